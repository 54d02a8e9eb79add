// The attention of chunks of new tokens over a paged pool (fp8_attention.hip, tree_attention.hip) cut
// into work: row blocks (the query columns that a workgroup holds at once), their tiles of keys laid
// end to end, and shares of those.
#pragma once

#include "ndl_common.hpp"

#include "chunk_shares.hpp"

namespace ndl {
namespace {

constexpr int kTile = 32;       // tokens per wave step

// What a launch's row blocks and shares are made of.
struct RowBlocks {
  const int32_t* block_table;
  int64_t bt_row_stride;
  int max_blocks;
  int tile_shift;               // log2(block_size / 16)
  const int32_t* cu_seqlens;    // null: one token per sequence
  const int32_t* context_lens;
  int num_seqs;
  int64_t num_tokens;
  int toks;                     // query tokens of a row block
  int blocks_per_seq;           // row blocks a sequence can have
  int items;                    // num_seqs * blocks_per_seq
  float scale_log2;
  // the split into equal shares (shares 0: a workgroup per row block)
  int shares;                   // per kv head
  int min_chunk;                // slots a share has at least
  int pad;                      // empty slots before each row block: what its start costs
  int nseg;                     // segment slots per kv head: shares + items
  float* ws_ml;                 // [kv head][segment][column][2]
  float* ws_acc;                // [kv head][segment][column][D]
};

// 32 bits of a mask row from bit `at` on (bits before the first count as set).
__device__ __forceinline__ uint32_t bits_at(const uint64_t* row, int words, int at) {
  if (at < 0) {
    const int s = -at;                       // below 32
    return (uint32_t)(row[0] << s) | ((1u << s) - 1u);
  }
  const int w = at >> 6, s = at & 63;
  uint64_t v = w < words ? row[w] >> s : 0u;
  if (s > 32 && w + 1 < words) v |= row[w + 1] << (64 - s);
  return (uint32_t)v;
}
// The low n bits (n of any size).
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
}

// A row block: tokens tok0 .. tok0 + n of the packed rows, the first at position pos.
struct Item {
  int64_t tok0;
  int n;
  int seq;
  int64_t pos;
  int64_t cap;                  // keys a table row holds
  int more;                     // tokens of the chunk past this row block that it may attend
  __device__ __forceinline__ int64_t keys() const {     // of its last token (and those)
    const int64_t k = pos + n + more;
    return n <= 0 || pos < 0 ? 0 : k < cap ? k : cap;
  }
  __device__ __forceinline__ int tiles() const { return (int)((keys() + kTile - 1) / kTile); }
};

// The sequence of row block e (32-bit: a 64-bit division takes a hundred instructions).
__device__ __forceinline__ int seq_of_item(const RowBlocks& a, int e) {
  return a.blocks_per_seq == 1 ? e : (int)((uint32_t)e / (uint32_t)a.blocks_per_seq);
}
// TREE: a token may attend any other of its chunk.
template <bool TREE = false>
__device__ __forceinline__ Item item_of(const RowBlocks& a, int e) {
  Item it;
  it.seq = seq_of_item(a, e);
  const int j0 = (e - it.seq * a.blocks_per_seq) * a.toks;
  int64_t first = it.seq, count = 1;
  if (a.cu_seqlens != nullptr) {
    first = a.cu_seqlens[it.seq];
    count = a.cu_seqlens[it.seq + 1] - first;
    if (first < 0 || first + count > a.num_tokens) count = 0;
  }
  it.tok0 = first + j0;
  it.n = (int)(count - j0 < a.toks ? count - j0 : a.toks);
  it.more = TREE && it.n > 0 ? (int)(count - j0) - it.n : 0;
  const int64_t ctx = a.context_lens[it.seq];
  it.pos = ctx < 0 ? -1 : ctx + j0;      // a negative context: nothing is attended
  it.cap = (int64_t)a.max_blocks << (4 + a.tile_shift);
  return it;
}

template <bool TREE>
__device__ __forceinline__ int slots_of(const RowBlocks& a, int e) {
  if (e >= a.items) return 0;
  const int n = item_of<TREE>(a, e).tiles();
  return n > 0 ? n + a.pad : 0;
}

// Inclusive prefix sum over the wave: by shifts within rows of 16 lanes, then the rows before.
template <int PATTERN>
__device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, PATTERN, 0xf, 0xf, true);
}
__device__ __forceinline__ int wave_scan(int v, int lane) {
  v = dpp_add<0x111>(v);         // row_shr:1, 0 from outside the row
  v = dpp_add<0x112>(v);
  v = dpp_add<0x114>(v);
  v = dpp_add<0x118>(v);
  const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31),
            r2 = __builtin_amdgcn_readlane(v, 47);
  return v + (lane >= 16 ? r0 : 0) + (lane >= 32 ? r1 : 0) + (lane >= 48 ? r2 : 0);
}

// The row blocks of a kv head laid end to end, in slots: their prefix sums, 64 to a step.  Up to
// kHeld row blocks stay in registers, loaded at once; more are read again where they are needed.
constexpr int kSteps = 4, kHeld = 64 * kSteps;
struct Place {
  int e, first, slots;          // a row block, its first slot, how many it has
};
template <bool TREE = false>
struct Stream {
  int total;
  Cut cut;
  int v[kSteps], incl[kSteps];

  __device__ __forceinline__ void read(const RowBlocks& a, int lane) {
    total = 0;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) v[k] = 64 * k < a.items ? slots_of<TREE>(a, 64 * k + lane) : 0;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      incl[k] = total;
      if (64 * k < a.items) {
        incl[k] = wave_scan(v[k], lane) + total;
        total = __builtin_amdgcn_readlane(incl[k], 63);
      }
    }
    for (int base = kHeld; base < a.items; base += 64)
      total += __builtin_amdgcn_readlane(wave_scan(slots_of<TREE>(a, base + lane), lane), 63);
    cut = cut_of(total, a.shares, a.min_chunk, a.pad);
  }
  // The row block that holds slot `at` (at < total), or row block `e` if that is not negative.
  __device__ __forceinline__ Place find(const RowBlocks& a, int lane, int at, int e) const {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const uint64_t hit = e >= 0 ? __builtin_amdgcn_ballot_w64(64 * k + lane == e)
                                  : __builtin_amdgcn_ballot_w64(v[k] > 0 && incl[k] > at);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        const int n = __builtin_amdgcn_readlane(v[k], l);
        return Place{64 * k + l, __builtin_amdgcn_readlane(incl[k], l) - n, n};
      }
    }
    int carry = __builtin_amdgcn_readlane(incl[kSteps - 1], 63);
    for (int base = kHeld; base < a.items; base += 64) {
      const int w = slots_of<TREE>(a, base + lane), in = wave_scan(w, lane) + carry;
      const uint64_t hit = e >= 0 ? __builtin_amdgcn_ballot_w64(base + lane == e)
                                  : __builtin_amdgcn_ballot_w64(w > 0 && in > at);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        const int n = __builtin_amdgcn_readlane(w, l);
        return Place{base + l, __builtin_amdgcn_readlane(in, l) - n, n};
      }
      carry = __builtin_amdgcn_readlane(in, 63);
    }
    return Place{a.items, carry, 0};
  }
  // Where share s begins.
  __device__ __forceinline__ int begin(const RowBlocks& a, int lane, int s) const {
    const int x = s * cut.chunk;   // fits 31 bits: make_plan
    if (x >= total) return total;
    const Place p = find(a, lane, x, -1);
    return share_begin(x, p.first, p.slots, cut.snap);
  }
};

// One workgroup per (row block, kv head, COLS columns): the parts that the shares hold,
// combined in their order; zeros for tokens with nothing to attend.  A row block inside one share
// was written by the attention.  MANY: whole steps of parts without a test for each, whose loads stay
// together (64 parts of one sequence: 12 us less), which takes registers (2 to 6 parts of 64 sequences:
// 2 us more).  put(row block, head, column, head_dim, outputs, maximum, sum).
constexpr int kMergeCols = 8;
constexpr int kMergeParts = 64;   // at a time

template <int D, bool TREE, int COLS = kMergeCols, bool MANY = false, class PUT>
__device__ __forceinline__ void merge_row_block(const RowBlocks& a, int group, PUT put) {
  constexpr int PER = COLS * D / 256;             // consecutive outputs of a thread
  constexpr int UNROLL = PER <= 4 ? 8 : 2;        // parts whose loads are under way
  __shared__ float2 part[kMergeParts][COLS];
  const int t = threadIdx.x, lane = t & 63;
  const int e = blockIdx.x, head = blockIdx.y, c0 = blockIdx.z * COLS;
  const Item it = item_of<TREE>(a, e);
  Stream<TREE> st;
  st.read(a, lane);
  const Place p = st.find(a, lane, 0, e);
  if (it.n <= 0 || c0 >= it.n * group) return;
  const int cols = it.n * group - c0 < COLS ? it.n * group - c0 : COLS;
  const int c = t * PER / D, d0 = t * PER - c * D;
  float o[PER];
#pragma unroll
  for (int x = 0; x < PER; ++x) o[x] = 0.f;
  float mx = kNegInf, l = 0.f;
  // its slots by the scan that gave its place and the cut: whatever the lengths are, or become while
  // this runs, share_parts names shares that there are, whose parts the workspace holds
  if (p.slots > 0) {
    int s0, s1;
    if (!share_parts(p.first, p.slots, st.cut, &s0, &s1)) return;   // written by the attention
    const int n = s1 - s0 + 1, per = a.toks * group;
    const int64_t seg = ((int64_t)head * a.nseg + s0 + e) * per + c0;
    const float2* const ml = reinterpret_cast<const float2*>(a.ws_ml) + seg;
    const float* const src = a.ws_acc + seg * D + (int64_t)(c < cols ? c : 0) * D + d0;
    // this thread's column's maximum over all parts, then 64 parts at a time
    const int64_t step = (int64_t)per * D;
    for (int pass = 0; pass < 2; ++pass) {
      for (int i0 = 0; i0 < n; i0 += kMergeParts) {
        const int m = n - i0 < kMergeParts ? n - i0 : kMergeParts;
        if (pass == 0 || n > kMergeParts) {
          __syncthreads();
          for (int i = t; i < m * COLS; i += 256)
            if (i % COLS < cols)
              part[i / COLS][i % COLS] =
                  ml[(int64_t)(i0 + i / COLS) * per + i % COLS];
          __syncthreads();
        }
        if (c >= cols) continue;
        if (pass == 0) {
          for (int i = 0; i < m; ++i) mx = fmaxf(mx, part[i][c].x);
          continue;
        }
        auto load = [&](int i, float* v) {
          const float* const q = src + (int64_t)(i0 + i) * step;
          if constexpr (PER >= 4) {
#pragma unroll
            for (int z = 0; z < PER; z += 4) {
              const f32x4 w = *reinterpret_cast<const f32x4*>(q + z);
#pragma unroll
              for (int x = 0; x < 4; ++x) v[z + x] = w[x];
            }
          } else {
            const f32x2 w = *reinterpret_cast<const f32x2*>(q);
            v[0] = w[0];
            v[1] = w[1];
          }
        };
        auto add = [&](int i, const float* v) {
          const float2 ms = part[i][c];
          const float f = ms.x == mx ? 1.f : fast_exp2(ms.x - mx);
          l += ms.y * f;
#pragma unroll
          for (int x = 0; x < PER; ++x) o[x] += v[x] * f;
        };
        int i = 0;
        for (; MANY && i + UNROLL <= m; i += UNROLL) {
          float v[UNROLL][PER];
#pragma unroll
          for (int y = 0; y < UNROLL; ++y) load(i + y, v[y]);
#pragma unroll
          for (int y = 0; y < UNROLL; ++y) add(i + y, v[y]);
        }
        for (; i < m; i += UNROLL) {
          float v[UNROLL][PER];
#pragma unroll
          for (int y = 0; y < UNROLL; ++y) load(i + y < m ? i + y : i, v[y]);
#pragma unroll
          for (int y = 0; y < UNROLL; ++y) {
            if (i + y >= m) break;
            add(i + y, v[y]);
          }
        }
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int x = 0; x < PER; ++x) o[x] *= inv;
  }
  if (c >= cols) return;
  put(it, head, c0 + c, d0, o, mx, l);
}

}  // namespace
}  // namespace ndl
