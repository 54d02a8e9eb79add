// Attention over the 16-bit paged pool whose weights are added up for every cached token and kv head,
// gfx950: what eviction from a bounded cache goes by.
//
//   out as paged_decode's and varlen_prefill's (tree_attention.hip's causal chunk), and
//   mass[x][kv] = decay * mass[x][kv] + sum_{t, h of kv's group} p[t][h][x]    (x < ctx),
//   mass[x][kv] = the sum alone                                                (the chunk's tokens),
//   p = softmax of the token's row, 0 where it does not attend x.
//
// The reference keeps no weights (needle/layers/attention.py:120-134, :291-310).
//
// The softmax's denominators are known only when a row is done, so the weights take a second look at
// the scores:
//   * Up to 32 columns (a decode step; tokens times heads of a group): the attention leaves its scores
//     behind (4 bytes each, where K and V are 512 bytes a token at head_dim 128) and a pass over
//     those takes the exponentials and sums (add_scores: 12 us where 64 sequences of 512 to 4,096
//     tokens have 32/8 heads; the call 125 us, 171 with the scores made again).
//   * More: the scores are made again, from K alone: the columns' Q in LDS in operand layout, a wave's
//     32 keys in registers for all columns, the sum over columns kept in the accumulator layout and
//     joined across lanes once, at the end.  (8 waves of 32 keys rather than 4 of 64: twice as many to a
//     SIMD, 26 us for 34 of 8 prompts of 2,000 to 16,000 tokens, 32 tokens each, 28/4 heads.)
// Scores kept are at most 1 GiB by the host's bounds (max_context_len, or all that the table holds).
// Bound (64 sequences' step): K and V read once, 4.3 TB/s over the call.  The 8 prompts' 84 us are the
// attention 42 (shares of 20 tiles), its merge 13 and the weights 26 (by instruction counts 5 of them
// products and 8 exponentials; the rest is trips to memory of workgroups that live for 256 keys).
// Sums run in a fixed order, without atomics; a key's number is written by one lane.
#include "fp8.hpp"
#include "tree_attention.hpp"

namespace ndl {
namespace {

constexpr int kKeys = 32;             // of a tile
constexpr int kMassWaves = 8;
constexpr int kMassKeys = kMassWaves * kKeys;      // of a workgroup: a tile for each wave
constexpr int kGroups = 4;            // 32-column groups in LDS at a time

struct MassArgs {
  float* mass;
  const u16* q;
  int64_t q_stride;
  const u16* kplane;
  int64_t num_blocks;
  int num_heads, num_kv_heads, group;
  const int32_t* block_table;
  int64_t bt_row_stride;
  int max_blocks;
  int block_shift;                    // log2(block_size)
  const int32_t* cu_seqlens;
  const int32_t* context_lens;
  int64_t num_tokens;
  int max_seqlen;
  int64_t max_keys;
  float scale_log2, decay;
  const float* lse;                   // [token][head]
  const float* scores;                // [kv head][sequence][column][score_keys]
  int64_t score_keys;
  int columns;                        // rows of scores per (kv head, sequence)
  int num_seqs;
};

struct Chunk {
  int64_t tok0;
  int n, ctx, keys;                   // tokens, cached ones before them, keys in all
};
__device__ __forceinline__ Chunk chunk_of(const MassArgs& a, int seq) {
  Chunk c{};
  int64_t first = seq, count = 1;
  if (a.cu_seqlens != nullptr) {
    first = a.cu_seqlens[seq];
    count = a.cu_seqlens[seq + 1] - first;
    if (first < 0 || count < 0 || first + count > a.num_tokens) count = 0;
  }
  if (count > a.max_seqlen) count = a.max_seqlen;
  c.tok0 = first;
  c.n = (int)count;
  c.ctx = a.context_lens[seq];
  const int64_t cap = (int64_t)a.max_blocks << a.block_shift;
  int64_t keys = c.ctx < 0 || c.n == 0 ? 0 : (int64_t)c.ctx + c.n;
  if (keys > cap) keys = cap;
  if (keys > a.max_keys) keys = a.max_keys;
  c.keys = (int)keys;
  return c;
}

// The number of position x of the sequence's kv head, null where its block id is invalid.
__device__ __forceinline__ float* number_of(const MassArgs& a, const int32_t* table, int x,
                                            int head) {
  const int b = table[x >> a.block_shift];
  if (b < 0 || b >= a.num_blocks) return nullptr;
  return a.mass + (((int64_t)b * a.num_kv_heads + head) << a.block_shift) +
         (x & ((1 << a.block_shift) - 1));
}
__device__ __forceinline__ void add_to(const MassArgs& a, float* at, int x, int ctx, float sum) {
  // (a decay of 0 forgets a NaN too)
  *at = x < ctx && a.decay != 0.f ? a.decay * *at + sum : sum;
}

// A thread per key, 256 of a (kv head, sequence): the exponentials of its columns' scores.
__global__ __launch_bounds__(256) void add_scores_kernel(MassArgs a) {
  const int head = blockIdx.x % a.num_kv_heads, seq = blockIdx.y;
  const int x = (int)(blockIdx.x / a.num_kv_heads) * 256 + threadIdx.x;
  const Chunk c = chunk_of(a, seq);
  if (x >= c.keys) return;
  float* const at = number_of(a, a.block_table + seq * a.bt_row_stride, x, head);
  if (at == nullptr) return;
  const float* s = a.scores + ((int64_t)head * a.num_seqs + seq) * a.columns * a.score_keys + x;
  const float* lse = a.lse + c.tok0 * a.num_heads + head * a.group;
  float sum = 0.f;
  for (int t = 0; t < c.n; ++t, lse += a.num_heads)
    for (int g = 0; g < a.group; ++g, s += a.score_keys) {
      // (a score past the token's last key is -inf, whatever its denominator is)
      const float v = *s;
      sum += v == kNegInf ? 0.f : fast_exp2(v - lse[g]);
    }
  add_to(a, at, x, c.ctx, sum);
}

template <int M>
__device__ __forceinline__ void halve(float* a, int lane) {
  const bool up = lane & M;
#pragma unroll
  for (int r = 0; r < M; ++r) {
    const float keep = up ? a[r + M] : a[r], give = up ? a[r] : a[r + M];
    a[r] = keep + __shfl_xor(give, M, 64);
  }
}
// v[r] summed over the lanes of its half (r: key 8 (r / 4) + 4 h + r % 4): the number of key
// `lane & 31` in lanes 0 to 31.  Halves of the registers change hands at each step, so that 16 sums
// take 16 exchanges.
__device__ __forceinline__ float sums_by_key(const f32x16& v, int lane) {
  float a[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) a[r] = v[r];
  // after the steps lane bits 3, 2, 1, 0 hold the bits of r that they took
  halve<8>(a, lane);
  halve<4>(a, lane);
  halve<2>(a, lane);
  halve<1>(a, lane);
  const float s = a[0] + __shfl_xor(a[0], 16, 64);       // of r = lane & 15, half lane >> 5
  // key k is r = 4 (k >> 3) + (k & 3) of half (k >> 2) & 1
  const int k = lane & 31;
  return __shfl(s, 4 * (k >> 3) + (k & 3) + 32 * ((k >> 2) & 1), 64);
}

// blockIdx.x: (block of kMassKeys keys, kv head), blockIdx.y: sequence.
template <int D, bool F16>
__global__ __launch_bounds__(64 * kMassWaves) void add_weights_kernel(MassArgs a) {
  using T = Elt<F16>;
  using X8 = typename T::x8;
  constexpr int KS = D / 16;
  __shared__ __attribute__((aligned(16))) u32x4 lq[kGroups][KS][64];
  __shared__ float llse[kGroups * 32];
  __shared__ int llim[kGroups * 32];
  const int lane = threadIdx.x & 63, c32 = lane & 31, h = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int head = blockIdx.x % a.num_kv_heads, seq = blockIdx.y;
  const int x0 = (int)(blockIdx.x / a.num_kv_heads) * kMassKeys + wv * kKeys;
  const Chunk c = chunk_of(a, seq);
  if ((int)(blockIdx.x / a.num_kv_heads) * kMassKeys >= c.keys) return;
  const int32_t* const table = a.block_table + seq * a.bt_row_stride;

  // This wave's keys, a row per lane: 16-byte pieces 2 s + h.  Keys past the last one and of invalid
  // blocks: the last block that there is (their sums are not written).
  X8 k[KS];
  {
    int x = x0 + c32;
    if (x >= c.keys) x = c.keys - 1;
    int b = table[x >> a.block_shift];
    if (b < 0 || b >= a.num_blocks) b = 0;
    const u16* const row = a.kplane + ((((int64_t)b * a.num_kv_heads + head) << a.block_shift) +
                                       (x & ((1 << a.block_shift) - 1))) * D + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s) k[s] = __builtin_bit_cast(X8, ld16(row + 16 * s));
  }
  f32x16 sum = {};
  const int cols = c.n * a.group;
  for (int col0 = 0; col0 < cols; col0 += 32 * kGroups) {
    const int here = cols - col0 < 32 * kGroups ? cols - col0 : 32 * kGroups;
    const int groups = (here + 31) / 32;
    if (col0 > 0) __syncthreads();
    for (int g = wv; g < groups; g += kMassWaves) {
      const int col = col0 + 32 * g + c32;
      const bool live = col < cols;
      const int tok = (live ? col : cols - 1) / a.group, sub = (live ? col : cols - 1) - tok * a.group;
      const int64_t at = (c.tok0 + tok) * a.num_heads + head * a.group + sub;
      const u16* const src =
          a.q + (c.tok0 + tok) * a.q_stride + (int64_t)(head * a.group + sub) * D + 8 * h;
#pragma unroll
      for (int s = 0; s < KS; ++s) lq[g][s][lane] = ld16(src + 16 * s);
      if (h == 0) {
        // (a sum of 0, where every score is -inf: no weight, as add_scores_kernel has it)
        const float lse = a.lse[at];
        llse[32 * g + c32] = lse == kNegInf ? -kNegInf : lse;
        llim[32 * g + c32] = live ? c.ctx + tok + 1 : 0;      // keys that the column attends
      }
    }
    __syncthreads();
    for (int g = 0; g < groups; ++g) {
      X8 q[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s) q[s] = __builtin_bit_cast(X8, lq[g][s][lane]);
      const float lse = llse[32 * g + c32];
      const int lim = llim[32 * g + c32];
      f32x16 sc = {};
#pragma unroll
      for (int s = 0; s < KS; ++s) sc = T::mfma32x32x16(k[s], q[s], sc);
      if (x0 + kKeys <= c.ctx && 32 * (g + 1) <= here) {     // every column attends every key
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[r] += fast_exp2(fmaf(sc[r], a.scale_log2, -lse));
      } else {
        const int left = lim - (x0 + 4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = fast_exp2(fmaf(sc[r], a.scale_log2, -lse));
          sum[r] += 8 * (r >> 2) + (r & 3) < left ? p : 0.f;
        }
      }
    }
  }
  const float s = sums_by_key(sum, lane);
  const int x = x0 + c32;
  if (h != 0 || x >= c.keys) return;
  float* const at = number_of(a, table, x, head);
  if (at != nullptr) add_to(a, at, x, c.ctx, s);
}

// What a call keeps of its scores, 0 where it makes them again: past kScoredColumns columns, or where
// the bounds that the host has would take more than kScoreBytes.
constexpr int64_t kScoreBytes = (int64_t)1 << 30;
struct MassSizes {
  int64_t score_keys;                 // 0: none kept
  size_t lse, scores, attention;
  size_t total() const { return lse + scores + attention; }
};
MassSizes sizes_of(const ChunkAttention& c) {
  MassSizes z{};
  z.lse = ((size_t)c.num_tokens * c.num_heads * 4 + 255) / 256 * 256;
  const int64_t cols = (int64_t)c.max_seqlen * (c.num_heads / c.num_kv_heads);
  if (cols <= kScoredColumns) {
    const int64_t keys = (c.max_keys + kKeys - 1) / kKeys * kKeys;
    const int64_t bytes = keys * 4 * cols * c.num_seqs * c.num_kv_heads;
    if (bytes <= kScoreBytes) {
      z.score_keys = keys;
      z.scores = ((size_t)bytes + 255) / 256 * 256;
    }
  }
  z.attention = chunk_attention_workspace(c);
  return z;
}

}  // namespace
}  // namespace ndl

extern "C" size_t ndl_attention_mass_workspace_bytes(int num_seqs, int64_t num_tokens,
                                                     int max_seqlen, int64_t max_keys,
                                                     int num_heads, int num_kv_heads, int head_dim,
                                                     int block_size) {
  using namespace ndl;
  if (num_seqs <= 0 || num_tokens <= 0 || max_seqlen <= 0 || max_keys <= 0 ||
      max_keys > 0x7fffff00 || (head_dim != 64 && head_dim != 128) ||
      block_tile_shift(block_size) < 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads != 0 || num_heads / num_kv_heads > 16)
    return 0;
  ChunkAttention c{};
  c.num_seqs = num_seqs;
  c.num_tokens = num_tokens;
  c.max_seqlen = max_seqlen;
  c.max_keys = max_keys;
  c.num_heads = num_heads;
  c.num_kv_heads = num_kv_heads;
  c.head_dim = head_dim;
  return sizes_of(c).total();
}

extern "C" int ndl_attention_mass(void* out, float* mass, const void* q, int64_t q_tok_stride,
                                  const void* kv_cache, int64_t num_blocks,
                                  const int32_t* block_table, int64_t bt_row_stride,
                                  int max_blocks_per_seq, const int32_t* cu_seqlens,
                                  const int32_t* context_lens, int num_seqs, int64_t num_tokens,
                                  int max_seqlen, int64_t max_keys, int num_heads,
                                  int num_kv_heads, int head_dim, int block_size, int dtype,
                                  float scale, float decay, void* workspace,
                                  size_t workspace_bytes, ndl_stream_t stream) {
  using namespace ndl;
  ChunkAttention c{};
  c.out = out;
  c.q = q;
  c.q_tok_stride = q_tok_stride;
  c.kv_cache = kv_cache;
  c.num_blocks = num_blocks;
  c.block_table = block_table;
  c.bt_row_stride = bt_row_stride;
  c.max_blocks_per_seq = max_blocks_per_seq;
  c.cu_seqlens = cu_seqlens;
  c.context_lens = context_lens;
  c.num_seqs = num_seqs;
  c.num_tokens = num_tokens;
  c.max_seqlen = max_seqlen;
  c.max_keys = max_keys;
  c.num_heads = num_heads;
  c.num_kv_heads = num_kv_heads;
  c.head_dim = head_dim;
  c.block_size = block_size;
  c.dtype = dtype;
  c.scale = scale;
  int rc = check_chunk_attention(c);
  if (rc != NDL_OK || num_seqs == 0 || num_tokens == 0) return rc;
  if (!mass || (uintptr_t)mass & 3u) return NDL_ERR_INVALID_ARG;
  const int64_t cap = (int64_t)max_blocks_per_seq * block_size;
  if (c.max_keys > cap) c.max_keys = cap;
  const MassSizes z = sizes_of(c);
  const int64_t blocks = (c.max_keys + 255) / 256 * num_kv_heads;
  static_assert(kMassKeys == 256, "keys of a workgroup, either way");
  const int threads = z.score_keys ? 256 : 64 * kMassWaves;      // of the weights' launch
  if (num_seqs > 65535 || !grid_fits(blocks, threads)) return NDL_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < z.total() || (uintptr_t)workspace & 255u)
    return NDL_ERR_WORKSPACE;
  c.lse = (float*)workspace;
  if (z.score_keys) {
    c.scores = (float*)((char*)workspace + z.lse);
    c.score_keys = z.score_keys;
  }
  const hipStream_t s = (hipStream_t)stream;
  rc = launch_chunk_attention(c, z.attention ? (char*)workspace + z.lse + z.scores : nullptr,
                              z.attention, s);
  if (rc != NDL_OK) return rc;
  MassArgs a{};
  a.mass = mass;
  a.q = (const u16*)q;
  a.q_stride = q_tok_stride;
  a.kplane = (const u16*)kv_cache;
  a.num_blocks = num_blocks;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.block_table = block_table;
  a.bt_row_stride = bt_row_stride;
  a.max_blocks = max_blocks_per_seq;
  a.block_shift = 4 + block_tile_shift(block_size);
  a.cu_seqlens = cu_seqlens;
  a.context_lens = context_lens;
  a.num_tokens = num_tokens;
  a.max_seqlen = max_seqlen;
  a.max_keys = c.max_keys;
  a.scale_log2 = scale * kLog2e;
  a.decay = decay;
  a.lse = c.lse;
  a.scores = c.scores;
  a.score_keys = c.score_keys;
  a.columns = max_seqlen * a.group;
  a.num_seqs = num_seqs;
  const dim3 grid((unsigned)blocks, (unsigned)num_seqs);
  if (z.score_keys) {
    hipLaunchKernelGGL(add_scores_kernel, grid, dim3(threads), 0, s, a);
    return check_launch();
  }
  const bool f16 = dtype_is_f16(dtype);
  if (head_dim == 128) {
    if (f16)
      hipLaunchKernelGGL((add_weights_kernel<128, true>), grid, dim3(threads), 0, s, a);
    else
      hipLaunchKernelGGL((add_weights_kernel<128, false>), grid, dim3(threads), 0, s, a);
  } else {
    if (f16)
      hipLaunchKernelGGL((add_weights_kernel<64, true>), grid, dim3(threads), 0, s, a);
    else
      hipLaunchKernelGGL((add_weights_kernel<64, false>), grid, dim3(threads), 0, s, a);
  }
  return check_launch();
}
