// Verification of drafted tokens against the target model's distributions (speculative decoding),
// gfx950.  The random numbers are inputs, so the answer is a function of them.
//
// Sequence i has rows cu[i] .. cu[i + 1] of logits, one per token of the chunk it was given; row r
// decides on the draft ids[r + 1], its last row on none.  With p_r = softmax(l_r / T_i) and
// q_r the distribution that the draft was taken from (the point at the draft, without one):
//   draft r is accepted while  u_r q_r(x) < p_r(x)  holds for it and all before it;
//   after the first rejected row r the next token has the distribution max(p_r - q_r, 0) / sum
//   (p_r where that is nowhere positive), after a last accepted draft p of the last row;
//   it is the first v with  sum_{w <= v} weight(w) > u sum weight,  u the sequence's last one,
// which is distributed as a token of the target.  T = 0, and a row whose maximum is not finite
// (a NaN, nothing left by a mask), stand for the point at the row's argmax in torch's order.
// The reference samples one row at a time on the host (needle/model/sampler.py:16-46).
//
// Bound: every logit read once, and what each launch waits for.  Three or four launches (us at 304
// rows of 64 sequences, 151,936 bfloat16 logits, draft distributions / 5 rows of one, without):
//   stats   row slices: maximum, its index, sum of exponentials, in one pass (fp32 terms); beside
//           them what decides on the drafts                        20.2 (4.6 TB/s) / 3.4
//   sums    per sequence: accepts (every workgroup by itself, from the slices), then the chosen
//           row's weights summed by slices                         12.6 / 5.2
//   left    with draft distributions: the sums of max(p - q, 0) by slices   8.7
//   pick    finds the slice, then the token                        5.6 / 4.6
// stats issues about 10 instructions an entry (12 of the 20 us), sums and left 15 of fp64 for the
// 64 chosen rows; the rest of the later three is trips to memory that wait for one another.
// The chosen row's weights and sums are in fp64: a token's border is found among up to 2^17
// others, where fp32 sums (2^-24 of the total each) would pick a neighbour now and then.
// Sums run in a fixed order without atomics: the same inputs give the same tokens.
//
// Trees (TREE): the rows are nodes, row j of a sequence follows the node parents[j] before it (node 0,
// the newest token, is where the path begins).  At a node with children c1 < c2 < .., tokens x1, x2,
// .., the path goes on to the first ck with  u < p(x1) + .. + p(xk)  (a token that siblings share
// counts once); where there is none the next token has the node's p without its children's tokens.
// That is a draw of p for every node, so the tokens are distributed as the target's; a chain gives
// what points give above.  Four launches: after stats a workgroup per sequence walks its tree (walk),
// then sums and pick as above, the children's tokens as bits over a slice.  us, stats / walk / sums /
// pick: 32 trees of 16 to 64 nodes of 128,256 logits 53.1 (6.1 TB/s) / 5.8 / 7.0 / 5.5, a tree of 60
// of 151,936 6.4 / 5.3 / 3.0 / 4.9.  The walk takes a node's children one by one, each after a look at its
// earlier siblings for its token: a root with 1,023 children, none of which is taken, 1.3 ms a call (a
// chain of as many rows 0.03; 59 children 0.03).
#include "ndl_common.hpp"

#include <type_traits>

namespace ndl {
namespace {

constexpr int kThreads = 256;
constexpr int kStatSlice = 4096;     // elements of a slice at least
constexpr int kStatWgs = 1536;       // workgroups wanted over all rows: what the GPU holds at once
constexpr int kSumSlice = 2048;      // a step of a workgroup; slices are whole steps
constexpr int kSumWgs = 2048;        // of sums and left: likewise
constexpr int kStatSlices = 32;      // 8 rows' slices are combined at a time, at half a wave each
constexpr int kMaxSlices = 64;       // a lane of a wave each
constexpr int kPickLen = 6144;       // elements of a chosen row's slice at most (see pick)
constexpr int kMaxVocab = 1 << 18;
static_assert(kMaxVocab <= kMaxSlices * kPickLen, "a row's slices cover it");
constexpr int kRun = kSumSlice / kThreads;      // entries of a thread's step, next to each other
constexpr int kPickThreads = kPickLen / kRun;   // of the last launch: one workgroup per sequence
static_assert(kRun == 8 && kPickThreads % 64 == 0);
constexpr int kAccept = 64;          // rows decided on at a time

struct Info {            // of a sequence, written by `sums`
  int accepted;
  int kind;              // see Kind
  int64_t row;           // chosen row
  int64_t draft_row;     // its row of draft_probs (TREE: the node)
  int token;             // the point's token, or the draft that was rejected
  float top;             // the row's maximum
};
enum Kind { kNothing = 0, kPoint = 1, kAll = 2, kBut = 3, kLeft = 4 };
// kPoint: all weight at `token`; kAll: exp; kBut: exp but for `token`; kLeft: max(p - q, 0)

struct Drafted {         // of a drafted token, written by `stats`
  int x;                 // the token, -1 outside the vocabulary and without a draft row
  float l, q;            // its logit and its draft probability (TREE: its parent's bits)
  float u;
};
constexpr int kTreeNodes = 1024;     // of a sequence: further rows are no part of its tree
constexpr int kWalkThreads = 1024;
constexpr int kNodeBytes = 40;       // of LDS that the walk needs for one

struct VerifyArgs {
  const void* logits;
  int64_t stride;
  const void* ids;
  int ids64;
  const int32_t* cu;
  const float* uniforms;
  const float* temperature;    // null: 1
  const float* probs;          // null: the drafts are points
  int64_t probs_stride, probs_rows;
  void* tokens;
  int32_t* accepted;
  int64_t rows;
  int num_seqs, vocab;
  int slices, slice_len;       // of stats
  int sum_slices, sum_len;     // of sums, left
  float* part_max;             // [rows][slices]
  int* part_arg;
  float* part_sum;
  Drafted* drafted;            // [rows]
  Info* info;                  // [num_seqs]
  double* sums;                // [num_seqs][sum_slices]
  double* left;                // likewise
  const int32_t* parents;      // a tree's
  int32_t* path;
};

template <int FMT>
__device__ __forceinline__ float elem(const void* row, int64_t i) {
  if constexpr (FMT == kFmtF32)
    return static_cast<const float*>(row)[i];
  else
    return Elt<FMT == kFmtF16>::lo(static_cast<const u16*>(row)[i]);
}
template <int FMT>
__device__ __forceinline__ const void* row_at(const VerifyArgs& a, int64_t r) {
  return static_cast<const char*>(a.logits) + r * a.stride * (FMT == kFmtF32 ? 4 : 2);
}

// (va, ia) comes before (vb, ib) in torch's argmax order.
__device__ __forceinline__ bool better(float va, int ia, float vb, int ib) {
  const bool na = va != va, nb = vb != vb;
  if (na || nb) return na && (!nb || ia < ib);
  return va > vb || (va == vb && ia < ib);
}
// The value of the lane that a DPP pattern names (all of a row's lanes are active).
template <int PATTERN>
__device__ __forceinline__ float dpp(float v) {
  return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(v), PATTERN, 0xf, 0xf, true));
}
template <int PATTERN>
__device__ __forceinline__ double dpp(double v) {
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)w, PATTERN, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(uint32_t)(w >> 32), PATTERN, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Lane l ^ 16 (ROWS 16) or l ^ 32: v_permlane*_swap returns the lower row's value in one result
// and the upper one's in the other, so both lanes combine the same two in the same order.
template <int ROWS>
__device__ __forceinline__ u32x2 pair_of(uint32_t v) {
  if constexpr (ROWS == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return u32x2{r[0], r[1]};
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return u32x2{r[0], r[1]};
  }
}
template <int ROWS, class OP>
__device__ __forceinline__ float across(float v, OP op) {
  const u32x2 r = pair_of<ROWS>(__float_as_uint(v));
  return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int ROWS, class OP>
__device__ __forceinline__ double across(double v, OP op) {
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  const u32x2 lo = pair_of<ROWS>((uint32_t)w), hi = pair_of<ROWS>((uint32_t)(w >> 32));
  return op(__builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]),
            __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]));
}
// v combined over the wave's 64 lanes, on the VALU (a butterfly through the LDS crossbar takes
// about 100 cycles a step): pairs, quads, mirrored halves of 8 and of 16, then rows.
template <class T, class OP>
__device__ __forceinline__ T wave_all(T v, OP op) {
  v = op(v, dpp<0xb1>(v));      // quad_perm [1, 0, 3, 2]
  v = op(v, dpp<0x4e>(v));      // quad_perm [2, 3, 0, 1]
  v = op(v, dpp<0x141>(v));     // row_half_mirror
  v = op(v, dpp<0x140>(v));     // row_mirror
  v = across<16>(v, op);
  return across<32>(v, op);
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
  return wave_all(v, [](T x, T y) { return x + y; });
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_all(v, [](float x, float y) { return fmaxf(x, y); });
}

__device__ __forceinline__ int64_t draft_at(const VerifyArgs& a, int64_t i) {
  return a.ids64 ? static_cast<const int64_t*>(a.ids)[i]
                 : (int64_t)static_cast<const int32_t*>(a.ids)[i];
}
__device__ __forceinline__ void put_token(const VerifyArgs& a, int64_t i, int64_t v) {
  if (a.ids64)
    static_cast<int64_t*>(a.tokens)[i] = v;
  else
    static_cast<int32_t*>(a.tokens)[i] = (int32_t)v;
}

// Rows of sequence i, none where cu is not within the logits.
__device__ __forceinline__ int seq_rows(const VerifyArgs& a, int i, int64_t* first) {
  const int64_t f = a.cu[i], e = a.cu[i + 1];
  *first = f;
  return f < 0 || e > a.rows || e < f ? 0 : (int)(e - f);
}
__device__ __forceinline__ float temperature_of(const VerifyArgs& a, int i) {
  const float t = a.temperature ? a.temperature[i] : 1.f;
  return t > 0.f ? t : 0.f;     // 0, negative, NaN: the argmax
}

// log2(e) / T, within what keeps 0 * k and -inf * k what they should be.
__device__ __forceinline__ float rate_of(float temp) {
  return fmaxf(fminf(kLog2e / temp, 3e38f), 1e-30f);
}

// The drafted tokens of sequence i: what decides on them beside the rows' statistics, in the shadow
// of the rows' workgroups (three trips to memory).
template <int FMT, bool TREE>
__device__ __forceinline__ void gather_drafts(const VerifyArgs& a, int i) {
  int64_t first;
  const int n = seq_rows(a, i, &first);
  if constexpr (TREE) {
    for (int j = threadIdx.x; j < n; j += kThreads) {
      const int p = a.parents[first + j];
      const int64_t x = draft_at(a, first + j);
      Drafted g{-1, kNegInf, __int_as_float(-1), 0.f};
      if (p >= 0 && p < j) {
        g.q = __int_as_float(p);
        if (x >= 0 && x < a.vocab) {
          g.x = (int)x;
          g.l = elem<FMT>(row_at<FMT>(a, first + p), x);
        }
      }
      a.drafted[first + j] = g;
    }
    return;
  }
  for (int j = threadIdx.x; j < n - 1; j += kThreads) {
    const int64_t r = first + j, x = draft_at(a, r + 1), d = r - i;
    Drafted g{-1, kNegInf, 1.f, a.uniforms[r]};
    // (a row that draft_probs has not, as after a sequence without rows: nothing to judge it by)
    if (x >= 0 && x < a.vocab && (!a.probs || (d >= 0 && d < a.probs_rows))) {
      g.x = (int)x;
      g.l = elem<FMT>(row_at<FMT>(a, r), x);
      if (a.probs) g.q = a.probs[d * a.probs_stride + x];
    }
    a.drafted[r] = g;
  }
}

// A workgroup per sequence for gather_drafts, then one per row and slice: maximum and sum of
// exp((l - maximum) / T) in one pass.  Where the row is a point (T = 0, or a slice that holds a NaN
// or an infinity: the sum is NaN then), the maximum and its first index instead.
template <int FMT, bool TREE>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyArgs a) {
  constexpr int EB = FMT == kFmtF32 ? 4 : 2, PER = 16 / EB;
  constexpr int kBatch = 4;            // 16-byte words of a thread's step, the next in flight
  if (blockIdx.x < (unsigned)a.num_seqs) {
    gather_drafts<FMT, TREE>(a, (int)blockIdx.x);
    return;
  }
  const unsigned unit = blockIdx.x - (unsigned)a.num_seqs;
  const int64_t r = unit / (unsigned)a.slices;
  const int s = (int)(unit - (unsigned)r * a.slices), t = threadIdx.x;
  const char* const row = static_cast<const char*>(row_at<FMT>(a, r));
  const int b0 = s * a.slice_len;
  const int b1 = b0 + a.slice_len < a.vocab ? b0 + a.slice_len : a.vocab;
  // up to the first 16-byte boundary of the slice entry by entry, whole 16-byte words from there
  const int lead = (int)((16 - ((uintptr_t)(row + (int64_t)b0 * EB) & 15)) & 15) / EB;
  const int h0 = b0 + lead < b1 ? b0 + lead : b1;
  const int words = b1 > h0 ? (b1 - h0) / PER : 0, tail = h0 + words * PER;
  const char* const body = row + (int64_t)h0 * EB;
  u32x4 next[kBatch];
  auto load = [&](int w0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int w = w0 + u * kThreads;
      next[u] = ldg16(body + (int64_t)(w < words ? w : t) * 16);   // t < words
    }
  };
  if (t < words) load(t);
  // the row's sequence: its temperature
  int lo = 0, hi = a.num_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)a.cu[mid] <= r) lo = mid; else hi = mid - 1;
  }
  const float temp = temperature_of(a, lo);
  const float k = rate_of(temp);
  float top = kNegInf, sum = 0.f;
  __shared__ float sv[kThreads / 64], ss[kThreads / 64];
  __shared__ int si[kThreads / 64];
  bool point = !(temp > 0.f);
  if (!point) {
    // entries past the slice and lanes without any: -inf, whose term is 0
    auto raise = [&](float best) {
      if (best > top) {
        sum *= fast_exp2((top - best) * k);      // exp2(-inf) = 0 the first time
        top = best;
      }
    };
    auto term = [&](float l) {
      return fast_exp2((l - (top == kNegInf ? 0.f : top)) * k);
    };
    auto one = [&](float l) {
      raise(l);
      sum += term(l);
    };
    // a step's entries; WHOLE: its words are all within the slice
    auto step = [&](int w0, auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      float v[kBatch * PER], best = kNegInf;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const bool in = WHOLE || w0 + u * kThreads < words;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if constexpr (FMT == kFmtF32) {
            v[4 * u + x] = in ? __uint_as_float(next[u][x]) : kNegInf;
          } else {
            using T = Elt<FMT == kFmtF16>;
            v[8 * u + 2 * x] = in ? T::lo(next[u][x]) : kNegInf;
            v[8 * u + 2 * x + 1] = in ? T::hi(next[u][x]) : kNegInf;
          }
        }
      }
      if (w0 + kBatch * kThreads < words) load(w0 + kBatch * kThreads);
#pragma unroll
      for (int e = 0; e < kBatch * PER; ++e) best = fmaxf(best, v[e]);
      raise(best);
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < kBatch * PER; ++e) part[e & 3] += term(v[e]);
      sum += (part[0] + part[1]) + (part[2] + part[3]);
    };
    int w0 = t;
    for (; w0 + (kBatch - 1) * kThreads < words; w0 += kBatch * kThreads)
      step(w0, std::true_type{});
    if (w0 < words) step(w0, std::false_type{});
    if (t < h0 - b0) one(elem<FMT>(row, b0 + t));
    for (int i = tail + t; i < b1; i += kThreads) one(elem<FMT>(row, i));
    float wtop = top;
    wtop = wave_max(wtop);
    // (a lane with nothing: -inf and 0, whose factor must not be NaN)
    sum = wave_sum(top == wtop || sum == 0.f ? sum : sum * fast_exp2((top - wtop) * k));
    if ((t & 63) == 0) {
      sv[t >> 6] = wtop;
      ss[t >> 6] = sum;
    }
    __syncthreads();
    top = fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]));
    sum = 0.f;
    for (int w = 0; w < kThreads / 64; ++w)
      sum += sv[w] == top || ss[w] == 0.f ? ss[w] : ss[w] * fast_exp2((sv[w] - top) * k);
    point = sum != sum;
    __syncthreads();
  }
  int arg = b0 < b1 ? b0 : 0x7fffffff;   // what a slice of nothing but -inf has
  if (point) {
    // The maximum, and of each thread the step it is in; then the first such entry there.
    auto entry = [&](int u, int x) {
      if constexpr (FMT == kFmtF32)
        return __uint_as_float(next[u][x]);
      else
        return x & 1 ? Elt<FMT == kFmtF16>::hi(next[u][x >> 1])
                     : Elt<FMT == kFmtF16>::lo(next[u][x >> 1]);
    };
    float edge = kNegInf;      // of the entries that are not in whole words
    int edge_at = 0x7fffffff, in = -1;
    bool nan = false;
    top = kNegInf;
    auto one = [&](int i) {
      const float v = elem<FMT>(row, i);
      nan |= v != v;
      if (v > edge) {
        edge = v;
        edge_at = i;
      }
    };
    if (t < h0 - b0) one(b0 + t);
    for (int i = tail + t; i < b1; i += kThreads) one(i);
    if (t < words) load(t);
    for (int w0 = t; w0 < words; w0 += kBatch * kThreads) {
      float best = kNegInf;       // words past the slice repeat the thread's first
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
#pragma unroll
        for (int x = 0; x < PER; ++x) {
          nan |= entry(u, x) != entry(u, x);
          best = fmaxf(best, entry(u, x));
        }
      if (w0 + kBatch * kThreads < words) load(w0 + kBatch * kThreads);
      if (best > top) {
        top = best;
        in = w0;
      }
    }
    const bool wnan = __builtin_amdgcn_ballot_w64(nan) != 0;
    float wtop = fmaxf(top, edge);
    wtop = wave_max(wtop);
    if ((t & 63) == 0) sv[t >> 6] = wnan ? __uint_as_float(0x7fc00000u) : wtop;
    __syncthreads();
    wtop = fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]));
    if (sv[0] != sv[0] || sv[1] != sv[1] || sv[2] != sv[2] || sv[3] != sv[3])
      wtop = __uint_as_float(0x7fc00000u);
    int at = 0x7fffffff;
    if (wtop != wtop) {           // the first NaN
      for (int i = b0 + t; i < b1 && at == 0x7fffffff; i += kThreads) {
        const float v = elem<FMT>(row, i);
        at = v != v ? i : at;
      }
    } else if (wtop > kNegInf) {
      if (edge == wtop) at = edge_at;
      if (in >= 0 && top == wtop) {
        load(in);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
          for (int x = 0; x < PER; ++x) {
            const int w = in + u * kThreads, i = h0 + w * PER + x;
            if (w < words && entry(u, x) == wtop && i < at) at = i;
          }
      }
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      const int o = __shfl_xor(at, m, 64);
      at = o < at ? o : at;
    }
    if ((t & 63) == 0) si[t >> 6] = at;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) at = si[w] < at ? si[w] : at;
    top = wtop;
    if (wtop != wtop || wtop > kNegInf) arg = at;
  }
  if (t == 0) {
    const int64_t o = r * a.slices + s;
    a.part_max[o] = top;
    a.part_arg[o] = arg;
    a.part_sum[o] = sum;
  }
}

// A row's statistics from its slices: a lane's slice, then combined over a group of `width` lanes
// (a power of two, at least the slices).
struct RowStats {
  float top = kNegInf;
  int arg = 0x7fffffff;
  double sum = 0.0;
};
struct RowPart {
  float top = kNegInf, sum = 0.f;
  int arg = 0x7fffffff;
};
__device__ __forceinline__ RowPart load_part(const VerifyArgs& a, int64_t r, int s) {
  RowPart p;
  const int64_t o = r * a.slices + (s < a.slices ? s : 0);
  p.top = a.part_max[o];
  p.arg = a.part_arg[o];
  p.sum = a.part_sum[o];
  if (s >= a.slices) p = RowPart{};
  return p;
}
// v combined over groups of `width` lanes (1 to 32), as wave_all does over the wave.
template <class OP>
__device__ __forceinline__ double group_sum(double v, int width, OP op) {
  if (width > 1) v = op(v, dpp<0xb1>(v));
  if (width > 2) v = op(v, dpp<0x4e>(v));
  if (width > 4) v = op(v, dpp<0x141>(v));
  if (width > 8) v = op(v, dpp<0x140>(v));
  if (width > 16) v = across<16>(v, op);
  return v;
}
__device__ __forceinline__ RowStats row_stats(const RowPart& p, int width, float k) {
  // (maximum, index) as one 64-bit word, moved like a double
  auto word = [](float top, int arg) {
    return __builtin_bit_cast(double, (uint64_t)__float_as_uint(top) << 32 | (uint32_t)arg);
  };
  auto top_of = [](double w) {
    return __uint_as_float((uint32_t)(__builtin_bit_cast(uint64_t, w) >> 32));
  };
  auto arg_of = [](double w) { return (int)(uint32_t)__builtin_bit_cast(uint64_t, w); };
  const double w = group_sum(word(p.top, p.arg), width, [&](double x, double y) {
    return better(top_of(y), arg_of(y), top_of(x), arg_of(x)) ? y : x;
  });
  RowStats f{top_of(w), arg_of(w), 0.0};
  f.sum = group_sum(p.sum == 0.f ? 0.0
                    : p.top == f.top ? (double)p.sum
                                     : (double)p.sum * fast_exp2((p.top - f.top) * k),
                    width, [](double x, double y) { return x + y; });
  return f;
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

// 2^(j / 64)
__device__ const double kPowers[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
};

// exp((l - top) / T) in fp64, to about 1e-13 of it, 0 for a masked entry: 2^(n / 64) from the
// table, and 2^(r / 64), |r| <= 1/2, by the exponential's series to the fourth power.  n is read
// from the low bits of a sum with 1.5 * 2^52 (fp64 conversions run at a quarter of the rate).
struct Exp {
  const double* table;     // kPowers in LDS
  double rate;             // 64 / (T ln 2)
  __device__ __forceinline__ double operator()(float l, float top) const {
    constexpr double c = 0.01083042469624914545;            // ln 2 / 64
    // at most 0; -inf and what underflows anyway to a power that does
    const double z = __builtin_fmax(((double)l - (double)top) * rate, -140000.0);
    const double shifted = z + 6755399441055744.0;
    const int n = (int)(uint32_t)__builtin_bit_cast(uint64_t, shifted);
    const double r = z - (shifted - 6755399441055744.0);
    const double t = table[n & 63];
    const double q = fma(fma(fma(r, c * c * c * c / 24, c * c * c / 6), r, c * c / 2), r, c) * r;
    return __builtin_amdgcn_ldexp(fma(q, t, t), n >> 6);
  }
};
// Every thread calls it; a barrier is due before the first use.
__device__ __forceinline__ Exp make_exp(double* table, float temp) {
  if (threadIdx.x < 64) table[threadIdx.x] = kPowers[threadIdx.x];
  return Exp{table, 92.33248261893164817 / (double)temp};
}
__device__ __forceinline__ double positive(double x) { return x > 0.0 ? x : 0.0; }   // NaN: 0

// Entries v0 .. v0 + 7 of a row, -inf past b1.  A row begins at any multiple of its entries' size:
// the loads are of unaligned words.
template <int FMT>
__device__ __forceinline__ void load_eight(const void* row, int v0, int b1, float (&l)[kRun]) {
  if (v0 + kRun <= b1) {
    if constexpr (FMT == kFmtF32) {
      __builtin_memcpy(l, static_cast<const float*>(row) + v0, sizeof(l));
    } else {
      using T = Elt<FMT == kFmtF16>;
      uint32_t w[4];
      __builtin_memcpy(w, static_cast<const u16*>(row) + v0, sizeof(w));
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        l[2 * x] = T::lo(w[x]);
        l[2 * x + 1] = T::hi(w[x]);
      }
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < kRun; ++u) l[u] = v0 + u < b1 ? elem<FMT>(row, v0 + u) : kNegInf;
}

// The tokens of a tree's children at node `at`, one bit each over entries b0 .. b1 - 1 of the
// vocabulary (all threads; `bits` holds them).
template <int THREADS>
__device__ __forceinline__ void child_bits(const VerifyArgs& a, int64_t first, int n, int64_t at,
                                           int b0, int b1, uint32_t* bits) {
  for (int w = threadIdx.x; w < (b1 - b0 + 31) / 32; w += THREADS) bits[w] = 0;
  __syncthreads();
  if (n > kTreeNodes) n = kTreeNodes;
  for (int j = threadIdx.x; j < n; j += THREADS) {
    const Drafted d = a.drafted[first + j];
    if (__float_as_int(d.q) == at && d.x >= b0 && d.x < b1)
      atomicOr(&bits[(d.x - b0) >> 5], 1u << ((d.x - b0) & 31));
  }
  __syncthreads();
}
// The bits of entries v0 .. v0 + 7, v0 a multiple of 8 from b0 on.
__device__ __forceinline__ uint32_t eight_bits(const uint32_t* bits, int v0, int b0) {
  return (bits[(v0 - b0) >> 5] >> ((v0 - b0) & 31)) & 0xffu;
}

// A workgroup per sequence: its tree walked from node 0.  Rows' statistics by groups of lanes, the
// nodes' probabilities by threads, then one wave goes from node to node.
template <int FMT>
__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(VerifyArgs a) {
  extern __shared__ double walk_lds[];
  const int i = blockIdx.x, t = threadIdx.x, lane = t & 63;
  int64_t first;
  const int rows = seq_rows(a, i, &first);
  if (rows <= 0) {
    if (t == 0) {
      a.accepted[i] = 0;
      a.info[i] = Info{0, kNothing, 0, 0, 0, 0.f};
    }
    return;
  }
  const int n = rows < kTreeNodes ? rows : kTreeNodes;
  double* const totals = walk_lds;                        // [n] each
  double* const chance = totals + n;                      // of a node where it hangs
  float* const tops = reinterpret_cast<float*>(chance + n);
  int* const args = reinterpret_cast<int*>(tops + n);
  int* const up = args + n;
  int* const token = up + n;
  float* const us = reinterpret_cast<float*>(token + n);
  int* const trail = reinterpret_cast<int*>(us + n);      // the path
  static_assert(2 * sizeof(double) + 6 * 4 == kNodeBytes, "per node");
  __shared__ double table[64];
  __shared__ int steps, last_kids;
  const float temp = temperature_of(a, i);
  const float k = rate_of(temp);
  const Exp ex = make_exp(table, temp);
  int width = 1;                       // lanes that a row's slices take
  while (width < a.slices) width <<= 1;
  const int gs = kWalkThreads / width, g = t / width;
  RowPart next = load_part(a, first + (g < n ? g : 0), t & (width - 1));
  for (int j = g; j < n; j += gs) {
    const RowPart part = next;
    next = load_part(a, first + (j + gs < n ? j + gs : j), t & (width - 1));
    const RowStats f = row_stats(part, width, k);
    if ((t & (width - 1)) == 0) {
      tops[j] = f.top;
      args[j] = f.arg;
      totals[j] = f.sum;
    }
  }
  for (int j = t; j < n; j += kWalkThreads) {
    const Drafted d = a.drafted[first + j];
    up[j] = __float_as_int(d.q);
    token[j] = d.x;
    us[j] = a.uniforms[first + j];
    trail[j] = -1;
    chance[j] = (double)d.l;           // its logit for now
  }
  __syncthreads();
  for (int j = t; j < n; j += kWalkThreads) {
    const int p = up[j], x = token[j];
    double c = 0.0;
    if (p >= 0 && x >= 0)
      c = temp > 0.f && finite(tops[p]) ? ex((float)chance[j], tops[p]) / totals[p]
                                        : (x == args[p] ? 1.0 : 0.0);
    chance[j] = c;
  }
  __syncthreads();
  if (t < 64) {
    int at = 0, acc = 0, kids = 0;
    for (;;) {
      if (lane == 0) trail[acc] = at;
      double upto = 0.0;
      const double u = (double)us[at];
      int to = -1;
      kids = 0;
      for (int base = at + 1; base < n && to < 0; base += 64) {
        const int j = base + lane;
        uint64_t mine = __builtin_amdgcn_ballot_w64(j < n && up[j < n ? j : 0] == at &&
                                                    token[j < n ? j : 0] >= 0);
        kids |= mine != 0;
        for (; mine && to < 0; mine &= mine - 1) {
          const int c = base + __builtin_ctzll(mine), x = token[c];
          bool again = false;          // an earlier sibling has the token
          for (int b = at + 1; b < c && !again; b += 64) {
            const int o = b + lane < c ? b + lane : c;
            again = __builtin_amdgcn_ballot_w64(o < c && up[o] == at && token[o] == x) != 0;
          }
          if (again) continue;
          upto += chance[c];
          if (u < upto) to = c;
        }
      }
      if (to < 0) break;
      at = to;
      ++acc;
    }
    if (lane == 0) {
      steps = acc;
      last_kids = kids;
    }
  }
  __syncthreads();
  const int acc = steps;
  for (int j = t; j < rows; j += kWalkThreads) {
    const int node = j < n ? trail[j] : -1;
    a.path[first + j] = node;
    if (j != acc) put_token(a, first + j, j < acc ? draft_at(a, first + trail[j + 1]) : -1);
  }
  if (t != 0) return;
  a.accepted[i] = acc;
  const int at = trail[acc];
  Info f;
  f.accepted = acc;
  f.row = first + at;
  f.draft_row = at;
  f.top = tops[at];
  f.token = args[at];
  f.kind = !(temp > 0.f) || !finite(f.top) ? kPoint : last_kids ? kBut : kAll;
  a.info[i] = f;
}

// Workgroup (slice, sequence): the sequence's accepted drafts and chosen row, then the sum of its
// slice of that row's weights.  Slice 0 writes what the later launches read.
template <int FMT, bool TREE>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs a) {
  const int i = blockIdx.y, s = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
  int64_t first;
  const int n = seq_rows(a, i, &first);
  const float temp = temperature_of(a, i);
  const float k = rate_of(temp);
  __shared__ double table[64];
  __shared__ uint32_t bits[TREE ? kPickLen / 32 : 1];
  __shared__ int reject;
  __shared__ double sums[kThreads / 64];
  __shared__ float tops[kAccept];
  __shared__ int args[kAccept], drafts[kAccept];
  __shared__ double totals[kAccept];
  const Exp ex = make_exp(table, temp);
  int width = 1;                       // lanes that a row's slices take
  while (width < a.slices) width <<= 1;
  Info f;
  if constexpr (TREE) {
    __syncthreads();
    f = a.info[i];
    if (n <= 0 || f.kind == kNothing) return;
  } else {
    __syncthreads();
    if (n <= 0) {
      if (s == 0 && t == 0) {
        a.accepted[i] = 0;
        a.info[i] = Info{0, kNothing, 0, 0, 0, 0.f};
      }
      return;
    }
    // kAccept rows at a time: their statistics by waves, the drafts' own entries by threads.  The
    // last row (or the first rejected) ends it, its statistics still there.
    int acc = 0, j0 = 0;
    for (;; j0 += kAccept) {
      const int m = n - j0 < kAccept ? n - j0 : kAccept;
      const bool draft = t < m && j0 + t < n - 1;
      const int g = t / width, gs = kThreads / width;
      const Drafted d = a.drafted[first + j0 + (t < m ? t : 0)];
      RowPart next = load_part(a, first + j0 + (g < m ? g : 0), t & (width - 1));
      for (int j = g; j < m; j += gs) {
        const RowPart part = next;
        next = load_part(a, first + j0 + (j + gs < m ? j + gs : j), t & (width - 1));
        const RowStats f = row_stats(part, width, k);
        if ((t & (width - 1)) == 0) {
          tops[j] = f.top;
          args[j] = f.arg;
          totals[j] = f.sum;
        }
      }
      __syncthreads();
      if (t < m) {
        drafts[t] = d.x;
        bool ok = false;
        if (draft && d.x >= 0) {
          const double uq = (double)d.u * (double)d.q;
          ok = temp > 0.f && finite(tops[t]) ? uq * totals[t] < ex(d.l, tops[t])
                                             : uq < (d.x == args[t] ? 1.0 : 0.0);
        }
        // the first row that is not accepted (the last has nothing to accept): t < m <= 64
        const uint64_t no = __builtin_amdgcn_ballot_w64(!ok);
        if (t == 0) reject = no ? j0 + __builtin_ctzll(no) : n;
      }
      __syncthreads();
      acc = reject;
      if (acc < n) break;
      __syncthreads();
    }
    const int64_t r = first + acc;
    f.accepted = acc;
    f.row = r;
    f.draft_row = r - i;
    f.top = tops[acc - j0];
    f.token = args[acc - j0];
    if (!(temp > 0.f) || !finite(f.top)) {
      f.kind = kPoint;
    } else if (acc == n - 1) {
      f.kind = kAll;
    } else if (a.probs) {
      f.kind = f.draft_row >= 0 && f.draft_row < a.probs_rows ? kLeft : kAll;
    } else {
      f.kind = kBut;
      f.token = drafts[acc - j0];
    }
    if (s == 0 && t == 0) a.info[i] = f;
  }
  if (f.kind == kPoint) return;
  const void* const row = row_at<FMT>(a, f.row);
  const int b0 = s * a.sum_len, b1 = b0 + a.sum_len < a.vocab ? b0 + a.sum_len : a.vocab;
  const int but = !TREE && f.kind == kBut ? f.token : -1;
  if (TREE && f.kind == kBut)
    child_bits<kThreads>(a, first, n, f.draft_row, b0, b1, bits);
  double z = 0.0;
  for (int v0 = b0 + t * kRun; v0 < b1; v0 += kSumSlice) {
    float l[kRun];
    load_eight<FMT>(row, v0, b1, l);
#pragma unroll
    for (int u = 0; u < kRun; ++u)
      if (v0 + u == but) l[u] = kNegInf;      // no weight
    if (TREE && f.kind == kBut) {
      const uint32_t kids = eight_bits(bits, v0, b0);
#pragma unroll
      for (int u = 0; u < kRun; ++u)
        if ((kids >> u) & 1u) l[u] = kNegInf;
    }
#pragma unroll
    for (int u = 0; u < kRun; ++u) z += ex(l[u], f.top);
  }
  z = wave_sum(z);
  if (lane == 0) sums[wv] = z;
  __syncthreads();
  if (t == 0) a.sums[(int64_t)i * a.sum_slices + s] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// The slices' sums added in every lane (at most 64).
__device__ __forceinline__ double slice_total(const double* p, int n, int lane) {
  return wave_sum(lane < n ? p[lane] : 0.0);
}

// Workgroup (slice, sequence): the sum of max(p - q, 0) over its slice of the chosen row.
template <int FMT>
__global__ __launch_bounds__(kThreads) void verify_left_kernel(VerifyArgs a) {
  const int i = blockIdx.y, s = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const Info f = a.info[i];
  if (f.kind != kLeft) return;
  __shared__ double table[64];
  __shared__ double part[kThreads / 64];
  const Exp ex = make_exp(table, temperature_of(a, i));
  const double scale =
      1.0 / slice_total(a.sums + (int64_t)i * a.sum_slices, a.sum_slices, lane);
  __syncthreads();
  const void* const row = row_at<FMT>(a, f.row);
  const float* const q = a.probs + f.draft_row * a.probs_stride;
  const int b0 = s * a.sum_len, b1 = b0 + a.sum_len < a.vocab ? b0 + a.sum_len : a.vocab;
  double z = 0.0;
  for (int v0 = b0 + t * kRun; v0 < b1; v0 += kSumSlice) {
    float l[kRun], d[kRun];
    load_eight<FMT>(row, v0, b1, l);
    load_eight<kFmtF32>(q, v0, b1, d);
#pragma unroll
    for (int u = 0; u < kRun; ++u)
      z += positive(ex(l[u], f.top) * scale - positive((double)d[u]));
  }
  z = wave_sum(z);
  if (lane == 0) part[t >> 6] = z;
  __syncthreads();
  if (t == 0) a.left[(int64_t)i * a.sum_slices + s] = (part[0] + part[1]) + (part[2] + part[3]);
}

// Inclusive prefix sum: over the 16 lanes of a row by shifts, then the rows before it.
__device__ __forceinline__ double wave_prefix(double v, int lane) {
  v += dpp<0x111>(v);           // row_shr:1, 0 from outside the row
  v += dpp<0x112>(v);
  v += dpp<0x114>(v);
  v += dpp<0x118>(v);
  double before = 0.0;
#pragma unroll
  for (int r = 0; r < 3; ++r) {
    const uint64_t w = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)w, 16 * r + 15);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(w >> 32), 16 * r + 15);
    before += lane > 16 * r + 15 ? __builtin_bit_cast(double, (uint64_t)hi << 32 | lo) : 0.0;
  }
  return v + before;
}

// Workgroup per sequence: its tokens.  The slice whose prefix passes the goal; then the thread
// (each takes a run of the slice), then the entry.
template <int FMT, bool TREE>
__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(VerifyArgs a) {
  const int i = blockIdx.x, t = threadIdx.x, lane = t & 63, wv = t >> 6;
  int64_t first;
  const int n = seq_rows(a, i, &first);
  const double plain = lane < a.sum_slices ? a.sums[(int64_t)i * a.sum_slices + lane] : 0.0;
  const double less =
      a.probs && lane < a.sum_slices ? a.left[(int64_t)i * a.sum_slices + lane] : 0.0;
  if (n <= 0) return;
  const Info f = a.info[i];
  if (f.accepted >= n) return;     // cu has changed since the launches before
  if constexpr (TREE) {
    if (f.kind == kNothing) return;
  } else {
    for (int j = t; j < n; j += kPickThreads)
      if (j != f.accepted)
        put_token(a, first + j, j < f.accepted ? draft_at(a, first + j + 1) : -1);
    if (t == 0) a.accepted[i] = f.accepted;
  }
  const int64_t to = first + f.accepted;
  if (f.kind == kPoint) {
    if (t == 0) put_token(a, to, f.token);
    return;
  }
  __shared__ double table[64];
  __shared__ uint32_t bits[TREE ? kPickLen / 32 : 1];
  __shared__ double wsum[kPickThreads / 64];
  __shared__ int cross[kPickThreads / 64], last[kPickThreads / 64];
  const Exp ex = make_exp(table, temperature_of(a, i));
  const double whole = wave_sum(plain);
  const double rest = f.kind == kLeft ? wave_sum(less) : 0.0;
  const bool left = rest > 0.0;        // else q covers p everywhere: p itself
  const double total = left ? rest : whole;
  if (!(total > 0.0)) {   // nothing but the rejected draft has weight
    if constexpr (TREE) {                // but its children: the likeliest, the row's argmax
      float l = kNegInf;
      int x = 0x7fffffff;
      for (int j = t; t < 64 && j < n && j < kTreeNodes; j += 64) {
        const Drafted d = a.drafted[first + j];
        if (__float_as_int(d.q) == f.draft_row && d.x >= 0 && better(d.l, d.x, l, x)) {
          l = d.l;
          x = d.x;
        }
      }
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) {
        const float ol = __shfl_xor(l, m, 64);
        const int ox = __shfl_xor(x, m, 64);
        if (better(ol, ox, l, x)) {
          l = ol;
          x = ox;
        }
      }
      if (t == 0) put_token(a, to, x == 0x7fffffff ? 0 : x);
    } else {
      if (t == 0) put_token(a, to, f.token < 0 ? 0 : f.token);
    }
    return;
  }
  const float u0 = a.uniforms[first + n - 1];
  const double u = u0 > 0.f ? (u0 < 1.f ? (double)u0 : 1.0) : 0.0;
  const double goal = u * total;
  // every wave finds the slice: the first whose prefix of the sums passes the goal, or, by the
  // roundings of the total, the last with weight
  const double x = left ? less : plain;
  const double upto = wave_prefix(x, lane);
  const uint64_t past = __builtin_amdgcn_ballot_w64(x > 0.0 && upto > goal);
  const uint64_t some = __builtin_amdgcn_ballot_w64(x > 0.0);
  const int pick = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
  const double before = __shfl(upto - x, pick, 64);
  const double scale = 1.0 / whole;
  const void* const row = row_at<FMT>(a, f.row);
  const float* const q = left ? a.probs + f.draft_row * a.probs_stride : nullptr;
  const int b0 = pick * a.sum_len, b1 = b0 + a.sum_len < a.vocab ? b0 + a.sum_len : a.vocab;
  const int v0 = b0 + t * kRun;
  float l[kRun], d[kRun];
  load_eight<FMT>(row, v0, b1, l);
  if (left) load_eight<kFmtF32>(q, v0, b1, d);
  double run[kRun], mine = 0.0;
  __syncthreads();
  uint32_t kids = 0;
  if (TREE && f.kind == kBut) {
    child_bits<kPickThreads>(a, first, n, f.draft_row, b0, b1, bits);
    kids = v0 < b1 ? eight_bits(bits, v0, b0) : 0u;
  }
#pragma unroll
  for (int e = 0; e < kRun; ++e) {
    run[e] = ex(l[e], f.top);
    if (left) run[e] = positive(run[e] * scale - positive((double)d[e]));
    if (TREE ? (kids >> e) & 1u : f.kind == kBut && v0 + e == f.token) run[e] = 0.0;
    mine += run[e];
  }
  // prefix over the threads
  const double incl = wave_prefix(mine, lane);
  if (lane == 63) wsum[wv] = incl;
  __syncthreads();
  double c = before + (incl - mine);
#pragma unroll
  for (int w = 0; w < kPickThreads / 64; ++w) c += w < wv ? wsum[w] : 0.0;
  // the first thread whose run passes the goal, and the last with weight: one of each wave's
  // lanes, then one of the waves (same-address LDS atomics take a cycle or more per lane)
  const uint64_t over = __builtin_amdgcn_ballot_w64(mine > 0.0 && c + mine > goal);
  const uint64_t any = __builtin_amdgcn_ballot_w64(mine > 0.0);
  if (lane == 0) {
    cross[wv] = over ? 64 * wv + __builtin_ctzll(over) : -1;
    last[wv] = any ? 64 * wv + 63 - __builtin_clzll(any) : -1;
  }
  __syncthreads();
  int who = -1, end = -1;
#pragma unroll
  for (int w = 0; w < kPickThreads / 64; ++w) {
    who = who < 0 ? cross[w] : who;
    end = last[w] >= 0 ? last[w] : end;
  }
  if (t != (who >= 0 ? who : end)) return;
  int token = v0;
  bool found = false;
#pragma unroll
  for (int e = 0; e < kRun; ++e) {
    c += run[e];
    if (run[e] > 0.0 && !found) {
      token = v0 + e;
      found = c > goal;
    }
  }
  put_token(a, to, token);
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }

struct Sizes {
  int slices, sum_len, sum_slices;
  size_t stat, drafted, info, sums, total;   // bytes of a part; three stats, two sums
};
Sizes sizes_of(int64_t rows, int num_seqs, int vocab) {
  Sizes z;
  const int64_t by_len = (vocab + kStatSlice - 1) / kStatSlice;
  const int64_t by_wgs = (kStatWgs + rows - 1) / rows;
  const int64_t few = by_len < by_wgs ? by_len : by_wgs;
  z.slices = (int)(few < kStatSlices ? few : kStatSlices);
  // one round of workgroups, as few slices as that takes: each decides on its drafts first (96 rows
  // of 50,257 float32: sums and left 8.8 + 7.0 us with 13 slices, 10.6 + 6.0 with 25)
  const int steps = (vocab + kSumSlice - 1) / kSumSlice;
  const int64_t wanted = ((int64_t)steps * num_seqs + kSumWgs - 1) / kSumWgs;
  const int most = kPickLen / kSumSlice, least = (steps + kMaxSlices - 1) / kMaxSlices;
  const int per = wanted < least ? least : wanted > most ? most : (int)wanted;
  z.sum_len = per * kSumSlice;
  z.sum_slices = (steps + per - 1) / per;
  z.stat = up((size_t)rows * z.slices * 4);
  z.drafted = up((size_t)rows * sizeof(Drafted));
  z.info = up((size_t)num_seqs * sizeof(Info));
  z.sums = up((size_t)num_seqs * z.sum_slices * 8);
  z.total = 3 * z.stat + z.drafted + z.info + 2 * z.sums;
  return z;
}

template <int FMT, bool TREE = false>
int launch_verify(const VerifyArgs& a, hipStream_t s) {
  const dim3 wg(kThreads);
  const unsigned seqs = (unsigned)a.num_seqs;
  hipLaunchKernelGGL((verify_stats_kernel<FMT, TREE>),
                     dim3((unsigned)(a.num_seqs + a.rows * a.slices)), wg, 0, s, a);
  int rc = check_launch();
  if (rc != NDL_OK) return rc;
  if constexpr (TREE) {
    const int lds = (int)(a.rows < kTreeNodes ? a.rows : kTreeNodes) * kNodeBytes;
    VerifyArgs args = a;
    void* params[] = {&args};
    if (hipLaunchKernel((const void*)verify_walk_kernel<FMT>, dim3(seqs), dim3(kWalkThreads), params,
                        lds, s) !=
        hipSuccess) {
      (void)hipGetLastError();
      return NDL_ERR_LAUNCH;
    }
    rc = check_launch();
    if (rc != NDL_OK) return rc;
  }
  hipLaunchKernelGGL((verify_sums_kernel<FMT, TREE>), dim3((unsigned)a.sum_slices, seqs), wg, 0, s,
                     a);
  rc = check_launch();
  if (rc != NDL_OK) return rc;
  if (a.probs != nullptr && a.probs_rows > 0) {
    hipLaunchKernelGGL((verify_left_kernel<FMT>), dim3((unsigned)a.sum_slices, seqs), wg, 0, s,
                       a);
    rc = check_launch();
    if (rc != NDL_OK) return rc;
  }
  hipLaunchKernelGGL((verify_pick_kernel<FMT, TREE>), dim3(seqs), dim3(kPickThreads), 0, s, a);
  return check_launch();
}

// The parts of the workspace and the slices of a call's rows.
void lay_out(VerifyArgs* a, const Sizes& z, void* workspace) {
  a->slices = z.slices;
  a->slice_len = (a->vocab + z.slices - 1) / z.slices;
  a->slice_len = (a->slice_len + 7) / 8 * 8;
  a->sum_slices = z.sum_slices;
  a->sum_len = z.sum_len;
  char* w = (char*)workspace;
  a->part_max = (float*)w;
  a->part_arg = (int*)(w + z.stat);
  a->part_sum = (float*)(w + 2 * z.stat);
  w += 3 * z.stat;
  a->drafted = (Drafted*)w;
  a->info = (Info*)(w + z.drafted);
  a->sums = (double*)(w + z.drafted + z.info);
  a->left = (double*)(w + z.drafted + z.info + z.sums);
}

}  // namespace
}  // namespace ndl

extern "C" size_t ndl_verify_drafts_workspace_bytes(int64_t num_rows, int num_seqs, int vocab) {
  if (num_rows <= 0 || num_seqs <= 0 || vocab <= 0) return 0;
  return ndl::sizes_of(num_rows, num_seqs, vocab).total;
}

extern "C" int ndl_verify_drafts(void* tokens, int32_t* accepted, const void* logits,
                                 int64_t row_stride, int dtype, const void* ids, int ids_are_int64,
                                 const int32_t* cu_seqlens, const float* uniforms,
                                 const float* temperature, const float* draft_probs,
                                 int64_t draft_stride, int64_t num_draft_rows, int64_t num_rows,
                                 int num_seqs, int vocab, void* workspace,
                                 size_t workspace_bytes, ndl_stream_t stream) {
  using namespace ndl;
  if (!dtype_known(dtype)) return NDL_ERR_UNSUPPORTED;
  if (num_rows < 0 || num_seqs < 0 || vocab <= 0) return NDL_ERR_INVALID_ARG;
  if (num_seqs == 0) return NDL_OK;
  if (num_rows == 0) return NDL_ERR_INVALID_ARG;   // every sequence has a row
  if (!tokens || !accepted || !logits || !ids || !cu_seqlens || !uniforms || row_stride < vocab)
    return NDL_ERR_INVALID_ARG;
  if (draft_probs != nullptr && (draft_stride < vocab || num_draft_rows < 0))
    return NDL_ERR_INVALID_ARG;
  const int eb = dtype_bytes(dtype);
  if ((uintptr_t)logits % eb || (uintptr_t)draft_probs & 3u || (uintptr_t)uniforms & 3u)
    return NDL_ERR_INVALID_ARG;
  if (num_rows > 65535 || num_seqs > 65535 || vocab > kMaxVocab)
    return NDL_ERR_UNSUPPORTED;
  const Sizes z = sizes_of(num_rows, num_seqs, vocab);
  if (!workspace || workspace_bytes < z.total || (uintptr_t)workspace & 255u)
    return NDL_ERR_WORKSPACE;
  VerifyArgs a{};
  a.logits = logits;
  a.stride = row_stride;
  a.ids = ids;
  a.ids64 = ids_are_int64 ? 1 : 0;
  a.cu = cu_seqlens;
  a.uniforms = uniforms;
  a.temperature = temperature;
  a.probs = draft_probs;
  a.probs_stride = draft_stride;
  a.probs_rows = num_draft_rows;
  a.tokens = tokens;
  a.accepted = accepted;
  a.rows = num_rows;
  a.num_seqs = num_seqs;
  a.vocab = vocab;
  lay_out(&a, z, workspace);
  const hipStream_t s = (hipStream_t)stream;
  if (dtype_is_f32(dtype)) return launch_verify<kFmtF32>(a, s);
  return dtype_is_f16(dtype) ? launch_verify<kFmtF16>(a, s) : launch_verify<kFmtBF16>(a, s);
}

extern "C" size_t ndl_verify_tree_workspace_bytes(int64_t num_rows, int num_seqs, int vocab) {
  return ndl_verify_drafts_workspace_bytes(num_rows, num_seqs, vocab);
}

extern "C" int ndl_verify_tree(void* tokens, int32_t* accepted, int32_t* path, const void* logits,
                               int64_t row_stride, int dtype, const void* ids, int ids_are_int64,
                               const int32_t* parents, const int32_t* cu_seqlens,
                               const float* uniforms, const float* temperature, int64_t num_rows,
                               int num_seqs, int vocab, void* workspace, size_t workspace_bytes,
                               ndl_stream_t stream) {
  using namespace ndl;
  if (!dtype_known(dtype)) return NDL_ERR_UNSUPPORTED;
  if (num_rows < 0 || num_seqs < 0 || vocab <= 0) return NDL_ERR_INVALID_ARG;
  if (num_seqs == 0) return NDL_OK;
  if (num_rows == 0) return NDL_ERR_INVALID_ARG;   // every sequence has a row
  if (!tokens || !accepted || !path || !logits || !ids || !parents || !cu_seqlens || !uniforms ||
      row_stride < vocab)
    return NDL_ERR_INVALID_ARG;
  if ((uintptr_t)logits % dtype_bytes(dtype) || (uintptr_t)uniforms & 3u)
    return NDL_ERR_INVALID_ARG;
  if (num_rows > 65535 || num_seqs > 65535 || vocab > kMaxVocab)
    return NDL_ERR_UNSUPPORTED;
  const Sizes z = sizes_of(num_rows, num_seqs, vocab);
  if (!workspace || workspace_bytes < z.total || (uintptr_t)workspace & 255u)
    return NDL_ERR_WORKSPACE;
  VerifyArgs a{};
  a.logits = logits;
  a.stride = row_stride;
  a.ids = ids;
  a.ids64 = ids_are_int64 ? 1 : 0;
  a.cu = cu_seqlens;
  a.uniforms = uniforms;
  a.temperature = temperature;
  a.tokens = tokens;
  a.accepted = accepted;
  a.rows = num_rows;
  a.num_seqs = num_seqs;
  a.vocab = vocab;
  a.parents = parents;
  a.path = path;
  lay_out(&a, z, workspace);
  const hipStream_t s = (hipStream_t)stream;
  if (dtype_is_f32(dtype)) return launch_verify<kFmtF32, true>(a, s);
  return dtype_is_f16(dtype) ? launch_verify<kFmtF16, true>(a, s)
                             : launch_verify<kFmtBF16, true>(a, s);
}
