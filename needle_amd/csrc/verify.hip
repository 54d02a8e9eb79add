// Verification of drafted tokens against the target model's distributions (speculative decoding),
// gfx950.  The random numbers are inputs, so the answer is a function of them.
//
// Sequence i has rows cu[i] .. cu[i + 1] of logits, one per token of the chunk it was given; row r
// judges the draft ids[r + 1], its last row has none to judge.  With p_r = softmax(l_r / T_i) and
// q_r the distribution that the draft was taken from (the point at the draft, without one):
//   draft r is accepted while  u_r q_r(x) < p_r(x)  holds for it and all before it;
//   after the first rejected row r the next token has the distribution max(p_r - q_r, 0) / sum
//   (p_r where that is nowhere positive), after a last accepted draft p of the last row;
//   it is the first v with  sum_{w <= v} weight(w) > u sum weight,  u the sequence's last one,
// which is distributed as a token of the target.  T = 0, and a row whose maximum is not finite
// (a NaN, nothing left by a mask), stand for the point at the row's argmax in torch's order.
// The reference samples one row at a time on the host (needle/model/sampler.py:16-46).
//
// Bound: every logit read once.  Three or four launches:
//   stats   row slices: maximum, its index, sum of exponentials, in one pass (fp32 terms)
//   sums    per sequence: accepts (every workgroup by itself, from the slices), then the chosen
//           row's weights summed by slices
//   left    with draft distributions: the sums of max(p - q, 0) by slices
//   pick    finds the slice, then the token
// The chosen row's weights and sums are in fp64: a token's border is found among up to 2^17
// others, where fp32 sums (2^-24 of the total each) would pick a neighbour now and then.
// Sums run in a fixed order without atomics: the same inputs give the same tokens.
#include "ndl_common.hpp"

namespace ndl {
namespace {

constexpr int kThreads = 256;
constexpr int kStatSlice = 4096;     // elements of a slice at least
constexpr int kStatWgs = 2048;       // workgroups wanted over all rows
constexpr int kSumSlice = 2048;
constexpr int kSumWgs = 1024;
constexpr int kMaxSlices = 64;       // a lane of a wave each

struct Info {            // of a sequence, written by `sums`
  int accepted;
  int kind;              // see Kind
  int64_t row;           // chosen row
  int64_t draft_row;     // its row of draft_probs
  int token;             // the point's token, or the draft that was rejected
  float top;             // the row's maximum
};
enum Kind { kNothing = 0, kPoint = 1, kAll = 2, kBut = 3, kLeft = 4 };
// kPoint: all weight at `token`; kAll: exp; kBut: exp but for `token`; kLeft: max(p - q, 0)

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
  Info* info;                  // [num_seqs]
  double* sums;                // [num_seqs][sum_slices]
  double* left;
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
__device__ __forceinline__ void wave_best(float& v, int& i) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const float ov = __shfl_xor(v, m, 64);
    const int oi = __shfl_xor(i, m, 64);
    if (better(ov, oi, v, i)) {
      v = ov;
      i = oi;
    }
  }
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
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
// exp((l - top) / T) as 2^((l - top) k); 0 for a masked entry (-inf * 0 is not asked).
__device__ __forceinline__ float term(float l, float top, float k) {
  const float x = (l - top) * k;
  return l == kNegInf ? 0.f : fast_exp2(x);
}

// Workgroup (slice s, row r): maximum, argmax and the sum of exp((l - maximum) / T).
template <int FMT>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyArgs a) {
  constexpr int EB = FMT == kFmtF32 ? 4 : 2, PER = 16 / EB;
  constexpr int kBatch = FMT == kFmtF32 ? 8 : 4;      // loads in flight (32 elements)
  const int s = blockIdx.x;
  const int64_t r = blockIdx.y;
  // the row's sequence: its temperature
  int lo = 0, hi = a.num_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)a.cu[mid] <= r) lo = mid; else hi = mid - 1;
  }
  const float temp = temperature_of(a, lo);
  const float k = rate_of(temp);
  const char* const row = static_cast<const char*>(row_at<FMT>(a, r));
  const int b0 = s * a.slice_len;
  const int b1 = b0 + a.slice_len < a.vocab ? b0 + a.slice_len : a.vocab;
  // the first 16-byte boundary of the slice, whole 16-byte words from there
  const int lead = (int)((16 - ((uintptr_t)(row + (int64_t)b0 * EB) & 15)) & 15) / EB;
  const int h0 = b0 + lead < b1 ? b0 + lead : b1;
  const int words = (b1 - h0) / PER, tail = h0 + words * PER;
  const char* const body = row + (int64_t)h0 * EB;
  float top = kNegInf, sum = 0.f;
  int arg = 0x7fffffff;
  auto one = [&](float v, int i) {
    if (better(v, i, top, arg)) {
      sum *= top == v ? 1.f : fast_exp2((top - v) * k);
      top = v;
      arg = i;
    }
    sum += term(v, top, k);
  };
  const int t = threadIdx.x;
  if (t < h0 - b0) one(elem<FMT>(row, b0 + t), b0 + t);
  for (int w0 = t; w0 < words; w0 += kBatch * kThreads) {
    u32x4 p[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int w = w0 + u * kThreads;
      p[u] = ldg16(body + (int64_t)(w < words ? w : w0) * 16);
    }
    float v[kBatch * PER];
    float best = kNegInf;
    int at = 0x7fffffff;
    bool nan = false;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int w = w0 + u * kThreads;
      const bool in = w < words;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if constexpr (FMT == kFmtF32) {
          v[4 * u + x] = in ? __uint_as_float(p[u][x]) : kNegInf;
        } else {
          using T = Elt<FMT == kFmtF16>;
          v[8 * u + 2 * x] = in ? T::lo(p[u][x]) : kNegInf;
          v[8 * u + 2 * x + 1] = in ? T::hi(p[u][x]) : kNegInf;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < kBatch * PER; ++e) {
      nan |= v[e] != v[e];
      best = fmaxf(best, v[e]);
    }
    if (nan || best > top || arg == 0x7fffffff) {     // a new maximum: where it is
      for (int u = kBatch - 1; u >= 0; --u)
#pragma unroll
        for (int x = PER - 1; x >= 0; --x) {
          float y = 0.f;
#pragma unroll
          for (int z = 0; z < kBatch; ++z) y = z == u ? v[z * PER + x] : y;
          const int i = h0 + (w0 + u * kThreads) * PER + x;
          if (w0 + u * kThreads < words && (nan ? y != y : y == best)) at = i;
        }
      const float nv = nan ? __uint_as_float(0x7fc00000u) : best;
      if (better(nv, at, top, arg)) {
        sum *= top == nv ? 1.f : fast_exp2((top - nv) * k);
        top = nv;
        arg = at;
      }
    }
    if (temp > 0.f) {
      float part = 0.f;
#pragma unroll
      for (int e = 0; e < kBatch * PER; ++e) part += term(v[e], top, k);
      sum += part;
    }
  }
  for (int i = tail + t; i < b1; i += kThreads) one(elem<FMT>(row, i), i);
  // the wave, then the workgroup
  float wtop = top;
  int warg = arg;
  wave_best(wtop, warg);
  // lanes with nothing hold top = -inf and sum = 0: their factor must not be NaN
  sum = wave_sum(top == wtop ? sum : sum == 0.f ? 0.f : sum * fast_exp2((top - wtop) * k));
  __shared__ float sv[kThreads / 64], ss[kThreads / 64];
  __shared__ int si[kThreads / 64];
  if ((t & 63) == 0) {
    sv[t >> 6] = wtop;
    si[t >> 6] = warg;
    ss[t >> 6] = sum;
  }
  __syncthreads();
  if (t == 0) {
    for (int w = 1; w < kThreads / 64; ++w)
      if (better(sv[w], si[w], wtop, warg)) {
        wtop = sv[w];
        warg = si[w];
      }
    float z = 0.f;
    for (int w = 0; w < kThreads / 64; ++w)
      if (ss[w] != 0.f) z += sv[w] == wtop ? ss[w] : ss[w] * fast_exp2((sv[w] - wtop) * k);
    const int64_t o = r * a.slices + s;
    a.part_max[o] = wtop;
    a.part_arg[o] = warg;
    a.part_sum[o] = z;
  }
}

// A row's statistics from its slices, in every lane of the wave.
__device__ __forceinline__ void row_stats(const VerifyArgs& a, int64_t r, int lane, float k,
                                          float* top, int* arg, double* sum) {
  float v = kNegInf, z = 0.f;
  int i = 0x7fffffff;
  if (lane < a.slices) {
    v = a.part_max[r * a.slices + lane];
    i = a.part_arg[r * a.slices + lane];
    z = a.part_sum[r * a.slices + lane];
  }
  *top = v;
  *arg = i;
  wave_best(*top, *arg);
  *sum = wave_sum(z == 0.f ? 0.0 : v == *top ? (double)z : (double)z * exp2((double)(v - *top) * k));
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

// weight of an entry: exp((l - top) / T) in fp64
__device__ __forceinline__ double weight(float l, float top, double inv_t) {
  return l == kNegInf ? 0.0 : exp(((double)l - (double)top) * inv_t);
}
__device__ __forceinline__ double positive(double x) { return x > 0.0 ? x : 0.0; }   // NaN: 0

// Workgroup (slice, sequence): the sequence's accepted drafts and chosen row, then the sum of its
// slice of that row's weights.  Slice 0 writes what the later launches read.
template <int FMT>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs a) {
  const int i = blockIdx.y, s = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
  int64_t first;
  const int n = seq_rows(a, i, &first);
  const float temp = temperature_of(a, i);
  const float k = rate_of(temp);
  const double inv_t = temp > 0.f ? 1.0 / (double)temp : 0.0;
  __shared__ int reject;
  __shared__ double part[kThreads / 64];
  if (t == 0) reject = n - 1;
  __syncthreads();
  for (int j = wv; j < n - 1; j += kThreads / 64) {
    const int64_t r = first + j;
    float top;
    int arg;
    double sum;
    row_stats(a, r, lane, k, &top, &arg, &sum);
    if (lane == 0) {
      const int64_t x = draft_at(a, r + 1);
      double p = 0.0, q = 1.0;
      if (x >= 0 && x < a.vocab) {
        if (temp > 0.f && finite(top))
          p = weight(elem<FMT>(row_at<FMT>(a, r), x), top, inv_t) / sum;
        else
          p = x == arg ? 1.0 : 0.0;
        const int64_t d = r - i;
        if (a.probs) q = d >= 0 && d < a.probs_rows ? a.probs[d * a.probs_stride + x] : 0.f;
      }
      if (!((double)a.uniforms[r] * q < p)) atomicMin(&reject, j);
    }
  }
  __syncthreads();
  if (n <= 0) {
    if (s == 0 && t == 0) {
      a.accepted[i] = 0;
      a.info[i] = Info{0, kNothing, 0, 0, 0, 0.f};
    }
    return;
  }
  const int acc = reject;
  const int64_t r = first + acc;
  float top;
  int arg;
  double fsum;
  row_stats(a, r, lane, k, &top, &arg, &fsum);
  Info f;
  f.accepted = acc;
  f.row = r;
  f.draft_row = r - i;
  f.top = top;
  if (!(temp > 0.f) || !finite(top)) {
    f.kind = kPoint;
    f.token = arg;
  } else if (acc == n - 1) {
    f.kind = kAll;
    f.token = arg;
  } else {
    const int64_t x = draft_at(a, r + 1);
    f.kind = a.probs ? (f.draft_row >= 0 && f.draft_row < a.probs_rows ? kLeft : kAll) : kBut;
    f.token = a.probs ? arg : x >= 0 && x < a.vocab ? (int)x : -1;
  }
  if (s == 0 && t == 0) a.info[i] = f;
  if (f.kind == kPoint) return;
  const void* const row = row_at<FMT>(a, r);
  const int b0 = s * a.sum_len, b1 = b0 + a.sum_len < a.vocab ? b0 + a.sum_len : a.vocab;
  double z = 0.0;
  for (int v0 = b0 + t; v0 < b1; v0 += 8 * kThreads) {
    float l[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int v = v0 + u * kThreads;
      l[u] = v < b1 ? elem<FMT>(row, v) : kNegInf;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const double w = weight(l[u], top, inv_t);
      z += f.kind == kBut && v0 + u * kThreads == f.token ? 0.0 : w;
    }
  }
  z = wave_sum(z);
  if (lane == 0) part[wv] = z;
  __syncthreads();
  if (t == 0) a.sums[(int64_t)i * a.sum_slices + s] = (part[0] + part[1]) + (part[2] + part[3]);
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
  const double inv_t = 1.0 / (double)temperature_of(a, i);
  const double total = slice_total(a.sums + (int64_t)i * a.sum_slices, a.sum_slices, lane);
  const void* const row = row_at<FMT>(a, f.row);
  const float* const q = a.probs + f.draft_row * a.probs_stride;
  const int b0 = s * a.sum_len, b1 = b0 + a.sum_len < a.vocab ? b0 + a.sum_len : a.vocab;
  double z = 0.0;
  for (int v0 = b0 + t; v0 < b1; v0 += 8 * kThreads) {
    float l[8], d[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int v = v0 + u * kThreads;
      l[u] = v < b1 ? elem<FMT>(row, v) : kNegInf;
      d[u] = v < b1 ? q[v] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      z += positive(weight(l[u], f.top, inv_t) / total - positive((double)d[u]));
  }
  z = wave_sum(z);
  __shared__ double part[kThreads / 64];
  if (lane == 0) part[t >> 6] = z;
  __syncthreads();
  if (t == 0) a.left[(int64_t)i * a.sum_slices + s] = (part[0] + part[1]) + (part[2] + part[3]);
}

__device__ __forceinline__ double wave_prefix(double v, int lane) {   // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  return v;
}

// Workgroup per sequence: its tokens.  The slice whose prefix passes the goal, then the thread
// (each takes a run of the slice), then the entry.
template <int FMT>
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyArgs a) {
  const int i = blockIdx.x, t = threadIdx.x, lane = t & 63, wv = t >> 6;
  int64_t first;
  const int n = seq_rows(a, i, &first);
  if (n <= 0) return;
  const Info f = a.info[i];
  for (int j = t; j < n; j += kThreads)
    if (j != f.accepted) put_token(a, first + j, j < f.accepted ? draft_at(a, first + j + 1) : -1);
  if (t == 0) a.accepted[i] = f.accepted;
  const int64_t to = first + f.accepted;
  if (f.kind == kPoint) {
    if (t == 0) put_token(a, to, f.token);
    return;
  }
  const int ns = a.sum_slices;
  const double* const plain = a.sums + (int64_t)i * ns;
  const double whole = slice_total(plain, ns, lane);
  bool left = f.kind == kLeft;
  const double* sums = plain;
  double total = whole;
  if (left) {
    const double rest = slice_total(a.left + (int64_t)i * ns, ns, lane);
    if (rest > 0.0) {
      sums = a.left + (int64_t)i * ns;
      total = rest;
    } else {
      left = false;     // q covers p everywhere: p itself
    }
  }
  if (!(total > 0.0)) {   // nothing but the rejected draft has weight
    if (t == 0) put_token(a, to, f.token < 0 ? 0 : f.token);
    return;
  }
  const float u0 = a.uniforms[first + n - 1];
  const double u = u0 > 0.f ? (u0 < 1.f ? (double)u0 : 1.0) : 0.0;
  const double goal = u * total;
  // every wave finds the slice: the first whose prefix of the sums passes the goal, or, by the
  // roundings of the total, the last with weight
  const double x = lane < ns ? sums[lane] : 0.0;
  const double upto = wave_prefix(x, lane);
  const uint64_t past = __builtin_amdgcn_ballot_w64(x > 0.0 && upto > goal);
  const uint64_t some = __builtin_amdgcn_ballot_w64(x > 0.0);
  const int pick = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
  const double before = __shfl(upto - x, pick, 64);
  const double inv_t = 1.0 / (double)temperature_of(a, i);
  const void* const row = row_at<FMT>(a, f.row);
  const float* const q = left ? a.probs + f.draft_row * a.probs_stride : nullptr;
  auto value = [&](int v) -> double {
    const double w = weight(elem<FMT>(row, v), f.top, inv_t);
    if (left) return positive(w / whole - positive((double)q[v]));
    return f.kind == kBut && v == f.token ? 0.0 : w;
  };
  const int b0 = pick * a.sum_len, b1 = b0 + a.sum_len < a.vocab ? b0 + a.sum_len : a.vocab;
  const int per = (b1 - b0 + kThreads - 1) / kThreads;
  const int v0 = b0 + t * per < b1 ? b0 + t * per : b1, v1 = v0 + per < b1 ? v0 + per : b1;
  double mine = 0.0;
  for (int v = v0; v < v1; ++v) mine += value(v);
  // prefix over the threads
  const double incl = wave_prefix(mine, lane);
  __shared__ double wsum[kThreads / 64];
  __shared__ int found, fallback;
  if (lane == 63) wsum[wv] = incl;
  if (t == 0) {
    found = 0x7fffffff;
    fallback = -1;
  }
  __syncthreads();
  double c = before + (incl - mine);
  for (int w = 0; w < wv; ++w) c += wsum[w];
  int hit = 0x7fffffff, seen = -1;
  if (mine > 0.0)
    for (int v = v0; v < v1; ++v) {
      const double x = value(v);
      c += x;
      if (x > 0.0) seen = v;
      if (x > 0.0 && c > goal) {
        hit = v;
        break;
      }
    }
  if (hit != 0x7fffffff) atomicMin(&found, hit);
  if (seen >= 0) atomicMax(&fallback, seen);
  __syncthreads();
  if (t == 0) put_token(a, to, found != 0x7fffffff ? found : fallback >= 0 ? fallback : 0);
}

int slices_for(int64_t rows, int vocab, int least, int wgs) {
  const int64_t by_len = (vocab + least - 1) / least;
  const int64_t by_wgs = (wgs + rows - 1) / rows;
  int64_t s = by_len < by_wgs ? by_len : by_wgs;
  return (int)(s < 1 ? 1 : s > kMaxSlices ? kMaxSlices : s);
}
size_t up(size_t n) { return (n + 255) / 256 * 256; }

struct Sizes {
  int slices, sum_slices;
  size_t stat, info, sums, total;    // bytes of a part; three stats, two sums
};
Sizes sizes_of(int64_t rows, int num_seqs, int vocab) {
  Sizes z;
  z.slices = slices_for(rows, vocab, kStatSlice, kStatWgs);
  z.sum_slices = slices_for(num_seqs, vocab, kSumSlice, kSumWgs);
  z.stat = up((size_t)rows * z.slices * 4);
  z.info = up((size_t)num_seqs * sizeof(Info));
  z.sums = up((size_t)num_seqs * z.sum_slices * 8);
  z.total = 3 * z.stat + z.info + 2 * z.sums;
  return z;
}

template <int FMT>
int launch_verify(const VerifyArgs& a, hipStream_t s) {
  const dim3 wg(kThreads), per_seq((unsigned)a.sum_slices, (unsigned)a.num_seqs);
  hipLaunchKernelGGL((verify_stats_kernel<FMT>), dim3((unsigned)a.slices, (unsigned)a.rows), wg,
                     0, s, a);
  int rc = check_launch();
  if (rc != NDL_OK) return rc;
  hipLaunchKernelGGL((verify_sums_kernel<FMT>), per_seq, wg, 0, s, a);
  rc = check_launch();
  if (rc != NDL_OK) return rc;
  if (a.probs != nullptr) {
    hipLaunchKernelGGL((verify_left_kernel<FMT>), per_seq, wg, 0, s, a);
    rc = check_launch();
    if (rc != NDL_OK) return rc;
  }
  hipLaunchKernelGGL((verify_pick_kernel<FMT>), dim3((unsigned)a.num_seqs), wg, 0, s, a);
  return check_launch();
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
  if (num_rows > 65535 || num_seqs > 65535 || vocab > (1 << 28)) return NDL_ERR_UNSUPPORTED;
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
  a.slices = z.slices;
  a.slice_len = (vocab + z.slices - 1) / z.slices;
  a.slice_len = (a.slice_len + 7) / 8 * 8;
  a.sum_slices = z.sum_slices;
  a.sum_len = (vocab + z.sum_slices - 1) / z.sum_slices;
  char* w = (char*)workspace;
  a.part_max = (float*)w;
  a.part_arg = (int*)(w + z.stat);
  a.part_sum = (float*)(w + 2 * z.stat);
  a.info = (Info*)(w + 3 * z.stat);
  a.sums = (double*)(w + 3 * z.stat + z.info);
  a.left = (double*)(w + 3 * z.stat + z.info + z.sums);
  const hipStream_t s = (hipStream_t)stream;
  if (dtype_is_f32(dtype)) return launch_verify<kFmtF32>(a, s);
  return dtype_is_f16(dtype) ? launch_verify<kFmtF16>(a, s) : launch_verify<kFmtBF16>(a, s);
}
