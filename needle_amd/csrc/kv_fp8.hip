// The 8-bit KV cache: rows of K and V quantised as they are written into the paged pool, and
// read back into the model's format.
//
// A row is one token's head_dim values of one head.  With a = max |x_d| over its finite values,
//   e = the smallest integer >= -126 with a <= 448 * 2^e,
//   code_d = e4m3(x_d * 2^-e)  (round to nearest even; NaN where x_d is not finite),
//   byte = e + 127,
// and the row's values are code_d * 2^e.  The scale is a power of two because e4m3 is a floating
// format: its step is relative (2^-4 of a value at most), so a finer scale gains nothing, the
// largest value lands in (224, 448] and everything down to 2^-14 of it keeps full precision; one
// byte per row then does, the multiplication is exact, and so is code * 2^e in bf16.  In fp16 it is
// between that format's ends: below 2^-14 it is rounded to a subnormal, and an fp16 row's values from
// 63,488 on have the code of 65,536, which reads back as infinity.
//
// The reference has no such pool; the slot rule is its append's (needle/layers/attention.py:
// 141-154, :224-237) and the rotation its _apply_rope (:277-288), as in rope_append.hip.
//
// Pools: codes [2][NB][Hkv][bs][D] bytes, scales [2][NB][Hkv][bs] bytes.
#include "fp8.hpp"

namespace ndl {
namespace {

struct QuantArgs {
  uint8_t* codes;
  uint8_t* scales;
  int64_t plane_rows;          // rows (token, head) of a plane
  int64_t num_blocks;
  int num_heads, num_kv_heads;
  int block_shift;             // log2(block_size)
  const u16* k;
  const u16* v;
  int64_t k_stride, v_stride;
  const u16* q;                // rotated into q_out (null: no q)
  u16* q_out;
  int64_t q_stride;
  const u16* cos;              // null: k (and q) as they are
  const u16* sin;
  int64_t cs_stride;
  const int32_t* block_table;
  int64_t bt_row_stride;
  int max_blocks;
  const int32_t* cu_seqlens;
  const int32_t* context_lens; // of a read: the first position of each sequence
  int num_seqs;
  int64_t num_tokens;
  u16* k_out;                  // of a read
  u16* v_out;
};

// Row index in a plane of (token t, kv head 0), or -1: t past the last sequence, a negative
// position, an invalid block id.  t is wave-uniform.
__device__ __forceinline__ int64_t slot_row(const QuantArgs& a, int64_t t) {
  int i;
  int64_t p;
  if (a.cu_seqlens == nullptr) {
    i = (int)t;
    p = a.context_lens[i];
  } else {
    if (t < (int64_t)a.cu_seqlens[0] || t >= (int64_t)a.cu_seqlens[a.num_seqs]) return -1;
    int lo = 0, hi = a.num_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((int64_t)a.cu_seqlens[mid] <= t) lo = mid; else hi = mid - 1;
    }
    i = lo;
    p = (int64_t)a.context_lens[i] + (t - a.cu_seqlens[i]);
  }
  if (p < 0) return -1;
  int64_t col = p >> a.block_shift;
  if (col > a.max_blocks - 1) col = a.max_blocks - 1;
  const int64_t b = a.block_table[(int64_t)i * a.bt_row_stride + col];
  if (b < 0 || b >= a.num_blocks) return -1;
  return ((b * a.num_kv_heads) << a.block_shift) + (p & ((1 << a.block_shift) - 1));
}

// One wave per (token, kRounds rounds of 64 items); an item is 8 elements of a row's first half and
// the 8 they rotate with, so D / 16 lanes hold a row and its maximum is a butterfly over them, and
// a lane's elements of cos and sin are the same in every round.  A token's items are the 2 Hkv
// rows of K and V, then the H rows of q.  All loads go out first, then the slot is looked up; what
// lies past the last item loads a valid one again and stores nothing.
//
// Bound by the bytes: 15,596 tokens of 28/4 heads of 128 with RoPE (279.6 MB, four fifths of them q
// in and out) take 50.3 us, 5.6 TB/s.  Two rounds a wave: one takes 54 us (cos, sin and the slot read
// twice as often), six 54.6 (fewer waves).  A step of a few tokens is its launch and two trips to
// memory: 4.2 us.
constexpr int kRounds = 2;

template <int D, bool F16>
__global__ __launch_bounds__(256) void kv_append_fp8_kernel(QuantArgs a) {
  constexpr int CPH = D / 16, HALF = D / 2, RPR = 64 / CPH;    // rows per round
  const int lane = threadIdx.x & 63;
  const int64_t w =
      (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int H = a.q ? a.num_heads : 0, Hkv = a.num_kv_heads;
  const int kv_rounds = (2 * Hkv + RPR - 1) / RPR, rounds = kv_rounds + (H + RPR - 1) / RPR;
  const int groups = (rounds + kRounds - 1) / kRounds;
  const int64_t t = w / groups;
  const int r0 = (int)(w - t * groups) * kRounds;
  if (t >= a.num_tokens) return;
  const int d0 = 8 * (lane % CPH);
  u32x4 lo[kRounds], hi[kRounds], clo, chi, slo, shi;
  const bool rope = a.cos != nullptr;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int r = r0 + i < rounds ? r0 + i : rounds - 1;
    const bool kv = r < kv_rounds;
    const int rows = kv ? 2 * Hkv : H;
    int row = (kv ? r : r - kv_rounds) * RPR + lane / CPH;
    if (row >= rows) row = rows - 1;
    const u16* src = kv ? (row >= Hkv ? a.v + t * a.v_stride - (int64_t)Hkv * D
                                      : a.k + t * a.k_stride)
                        : a.q + t * a.q_stride;
    src += (int64_t)row * D + d0;
    lo[i] = ld16(src);
    hi[i] = ld16(src + HALF);
  }
  if (rope) {
    const u16 *cs = a.cos + t * a.cs_stride + d0, *sn = a.sin + t * a.cs_stride + d0;
    clo = ld16(cs);
    chi = ld16(cs + HALF);
    slo = ld16(sn);
    shi = ld16(sn + HALF);
  }
  const int64_t slot = r0 < kv_rounds ? slot_row(a, t) : -1;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int r = r0 + i;
    if (r >= rounds) return;
    const bool kv = r < kv_rounds;
    const int row = (kv ? r : r - kv_rounds) * RPR + lane / CPH;
    const bool live = row < (kv ? 2 * Hkv : H), is_v = kv && row >= Hkv;
    if (rope) {
      u32x4 rlo, rhi;
      rope8<F16>(lo[i], hi[i], clo, chi, slo, shi, rlo, rhi);
      if (!is_v) {
        lo[i] = rlo;
        hi[i] = rhi;
      }
    }
    if (!kv) {
      if (live) {
        u16* const dst = a.q_out + (t * H + row) * D + d0;
        st16(dst, lo[i]);
        st16(dst + HALF, hi[i]);
      }
      continue;
    }
    const int byte = scale_byte<CPH, F16>(lo[i], hi[i]);
    const float mul = __uint_as_float((uint32_t)(254 - byte) << 23);
    if (live && slot >= 0) {
      const int h = is_v ? row - Hkv : row;
      const int64_t at = (is_v ? a.plane_rows : 0) + slot + ((int64_t)h << a.block_shift);
      uint8_t* const dst = a.codes + at * D + d0;
      *reinterpret_cast<u32x2*>(dst) = quant8<F16>(lo[i], mul);
      *reinterpret_cast<u32x2*>(dst + HALF) = quant8<F16>(hi[i], mul);
      if (d0 == 0) a.scales[at] = (uint8_t)byte;
    }
  }
}

constexpr int kReadItems = 512;   // 8-code items a wave has in flight: 4 KiB of codes, 8 KiB out

// The slot row of token t of a lane's own, as slot_row.  cu of up to 64 sequences is in the lanes
// of `starts` (lane i: cu[i + 1]): the sequence is found by exchanges, without loads that wait for
// one another.
__device__ __forceinline__ int64_t slot_row_of_lane(const QuantArgs& a, int64_t t, int starts) {
  const int n = a.num_seqs;
  int i = 0;                       // sequences that end at or before t
  if (n <= 64) {
#pragma unroll
    for (int step = 32; step >= 1; step >>= 1) {
      const int probe = i + step - 1;
      const int end = __shfl(starts, probe < 64 ? probe : 63, 64);
      if (probe < n && end <= t) i += step;
    }
    // (64 sequences that all end before t: step 32 .. 1 sum to 63)
    const int end = __shfl(starts, i < 64 ? i : 63, 64);
    if (i < n && end <= t) ++i;
  } else {
    int lo = 0, hi = n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.cu_seqlens[mid + 1] <= t) lo = mid + 1; else hi = mid;
    }
    i = lo;
  }
  if (i >= n) return -2;           // past the last sequence
  const int first = a.cu_seqlens[i];
  if (t < first) return -2;
  const int64_t p = (int64_t)a.context_lens[i] + (t - first);
  if (p < 0) return -1;
  int64_t col = p >> a.block_shift;
  if (col > a.max_blocks - 1) col = a.max_blocks - 1;
  const int64_t b = a.block_table[(int64_t)i * a.bt_row_stride + col];
  if (b < 0 || b >= a.num_blocks) return -1;
  return ((b * a.num_kv_heads) << a.block_shift) + (p & ((1 << a.block_shift) - 1));
}

// One wave per kReadItems items of the packed tokens; an item is 8 codes of one of a token's
// 2 Hkv rows, in the order of the tokens, so that a wave stores 1 KiB at once.  Lane k first finds
// the slot of the wave's k-th token.  Positions that have no slot read as zeros, tokens past the
// last sequence are not written.
//
// Bound by the bytes: 34,224 tokens of 8 heads of 128 (210.8 MB) take 37.2 us, 5.7 TB/s, with eight
// loads of a lane in flight; one load a wave, its slot looked up before it, takes 41.
template <int D, bool F16>
__global__ __launch_bounds__(256) void kv_read_fp8_kernel(QuantArgs a) {
  constexpr int CPR = D / 8, U = kReadItems / 64;
  const int lane = threadIdx.x & 63;
  const int64_t w =
      (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int Hkv = a.num_kv_heads, ipt = 2 * Hkv * CPR;     // items per token, at least 16
  const int64_t item0 = w * kReadItems, tok0 = item0 / ipt;
  if (tok0 >= a.num_tokens) return;
  const int starts = a.cu_seqlens[lane < a.num_seqs ? lane + 1 : a.num_seqs];
  const int64_t mine = slot_row_of_lane(a, tok0 + lane, starts);
  const int off = (int)(item0 - tok0 * ipt);
  const float inv = 1.f / (float)ipt;
  u32x2 c[U];
  float scale[U];
  u16* dst[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = off + 64 * u + lane;                    // under 2^20: the quotient is exact
    const int k = (int)(((float)at + 0.5f) * inv), item = at - k * ipt;
    const int row = item / CPR, d0 = 8 * (item - row * CPR);
    const bool is_v = row >= Hkv;
    const int h = is_v ? row - Hkv : row;
    const int64_t slot = __shfl(mine, k, 64);
    const bool in = slot >= 0;
    const int64_t src = in ? (is_v ? a.plane_rows : 0) + slot + ((int64_t)h << a.block_shift) : 0;
    c[u] = ld8(a.codes + src * D + (in ? d0 : 0));
    scale[u] = __uint_as_float((uint32_t)a.scales[src] << 23);
    if (!in) c[u] = u32x2{0u, 0u};
    dst[u] = slot == -2 || tok0 + k >= a.num_tokens
                 ? nullptr
                 : (is_v ? a.v_out : a.k_out) + ((tok0 + k) * Hkv + h) * D + d0;
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (dst[u] != nullptr)
      st16(dst[u],
           u32x4{value2<F16, false>(c[u][0], scale[u]), value2<F16, true>(c[u][0], scale[u]),
                 value2<F16, false>(c[u][1], scale[u]), value2<F16, true>(c[u][1], scale[u])});
}

int log2_of(int block_size) {
  const int s = block_tile_shift(block_size);
  return s < 0 ? -1 : s + 4;
}

}  // namespace
}  // namespace ndl

extern "C" int ndl_kv_append_fp8(void* codes, void* scales, int64_t num_blocks, int num_kv_heads,
                                 int block_size, int head_dim, int dtype, const void* k,
                                 int64_t k_tok_stride, const void* v, int64_t v_tok_stride,
                                 void* q_out, const void* q, int64_t q_tok_stride, int num_heads,
                                 const void* cos, const void* sin, int64_t cs_tok_stride,
                                 const int32_t* block_table, int64_t bt_row_stride,
                                 int max_blocks_per_seq, const int32_t* cu_seqlens,
                                 const int32_t* context_lens, int num_seqs, int64_t num_tokens,
                                 ndl_stream_t stream) {
  using namespace ndl;
  if (!dtype_supported(dtype) || (head_dim != 64 && head_dim != 128) || log2_of(block_size) < 0)
    return NDL_ERR_UNSUPPORTED;
  if (num_tokens < 0 || num_seqs < 0 || num_kv_heads <= 0 || num_blocks <= 0 ||
      max_blocks_per_seq <= 0 || bt_row_stride < max_blocks_per_seq)
    return NDL_ERR_INVALID_ARG;
  if (num_tokens == 0) return NDL_OK;
  if (!codes || !scales || !k || !v || !block_table || !context_lens || num_seqs == 0)
    return NDL_ERR_INVALID_ARG;
  if ((cos == nullptr) != (sin == nullptr) || (q == nullptr) != (q_out == nullptr) ||
      (q != nullptr && cos == nullptr))
    return NDL_ERR_INVALID_ARG;   // q is here to be rotated
  if (cu_seqlens == nullptr && num_tokens != num_seqs) return NDL_ERR_INVALID_ARG;
  const int64_t kv_row = (int64_t)num_kv_heads * head_dim;
  if (k_tok_stride < kv_row || v_tok_stride < kv_row ||
      (q != nullptr && (num_heads <= 0 || q_tok_stride < (int64_t)num_heads * head_dim)) ||
      (cos != nullptr && cs_tok_stride < head_dim))
    return NDL_ERR_INVALID_ARG;
  if (((uintptr_t)codes | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)q_out |
       (uintptr_t)cos | (uintptr_t)sin) & 15u)
    return NDL_ERR_INVALID_ARG;
  if ((k_tok_stride | v_tok_stride | (q ? q_tok_stride : 0) | (cos ? cs_tok_stride : 0)) & 7)
    return NDL_ERR_INVALID_ARG;
  QuantArgs a{};
  a.codes = (uint8_t*)codes;
  a.scales = (uint8_t*)scales;
  a.plane_rows = num_blocks * num_kv_heads * (int64_t)block_size;
  a.num_blocks = num_blocks;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.block_shift = log2_of(block_size);
  a.k = (const u16*)k;
  a.v = (const u16*)v;
  a.k_stride = k_tok_stride;
  a.v_stride = v_tok_stride;
  a.q = (const u16*)q;
  a.q_out = (u16*)q_out;
  a.q_stride = q_tok_stride;
  a.cos = (const u16*)cos;
  a.sin = (const u16*)sin;
  a.cs_stride = cs_tok_stride;
  a.block_table = block_table;
  a.bt_row_stride = bt_row_stride;
  a.max_blocks = max_blocks_per_seq;
  a.cu_seqlens = cu_seqlens;
  a.context_lens = context_lens;
  a.num_seqs = num_seqs;
  a.num_tokens = num_tokens;
  const int64_t rpr = 64 / (head_dim / 16);
  const int64_t rounds = (2 * num_kv_heads + rpr - 1) / rpr + (q ? (num_heads + rpr - 1) / rpr : 0);
  const int64_t groups = (rounds + kRounds - 1) / kRounds;
  const int64_t blocks = (num_tokens * groups + 3) / 4;
  if (!grid_fits(blocks, 256)) return NDL_ERR_INVALID_ARG;
  const dim3 grid((unsigned)blocks), wg(256);
  const hipStream_t s = (hipStream_t)stream;
  const bool f16 = dtype_is_f16(dtype);
  if (head_dim == 128) {
    if (f16)
      hipLaunchKernelGGL((kv_append_fp8_kernel<128, true>), grid, wg, 0, s, a);
    else
      hipLaunchKernelGGL((kv_append_fp8_kernel<128, false>), grid, wg, 0, s, a);
  } else {
    if (f16)
      hipLaunchKernelGGL((kv_append_fp8_kernel<64, true>), grid, wg, 0, s, a);
    else
      hipLaunchKernelGGL((kv_append_fp8_kernel<64, false>), grid, wg, 0, s, a);
  }
  return check_launch();
}

extern "C" int ndl_kv_read_fp8(void* k_out, void* v_out, const void* codes, const void* scales,
                               int64_t num_blocks, int num_kv_heads, int block_size,
                               int head_dim, int dtype, const int32_t* block_table,
                               int64_t bt_row_stride, int max_blocks_per_seq,
                               const int32_t* first, const int32_t* cu_seqlens, int num_seqs,
                               int64_t num_tokens, ndl_stream_t stream) {
  using namespace ndl;
  if (!dtype_supported(dtype) || (head_dim != 64 && head_dim != 128) || log2_of(block_size) < 0)
    return NDL_ERR_UNSUPPORTED;
  if (num_tokens < 0 || num_seqs < 0 || num_kv_heads <= 0 || num_blocks <= 0 ||
      max_blocks_per_seq <= 0 || bt_row_stride < max_blocks_per_seq)
    return NDL_ERR_INVALID_ARG;
  if (num_tokens == 0 || num_seqs == 0) return NDL_OK;
  if (!k_out || !v_out || !codes || !scales || !block_table || !first || !cu_seqlens)
    return NDL_ERR_INVALID_ARG;
  if (((uintptr_t)codes | (uintptr_t)k_out | (uintptr_t)v_out) & 15u) return NDL_ERR_INVALID_ARG;
  QuantArgs a{};
  a.codes = (uint8_t*)const_cast<void*>(codes);
  a.scales = (uint8_t*)const_cast<void*>(scales);
  a.plane_rows = num_blocks * num_kv_heads * (int64_t)block_size;
  a.num_blocks = num_blocks;
  a.num_kv_heads = num_kv_heads;
  a.block_shift = log2_of(block_size);
  a.block_table = block_table;
  a.bt_row_stride = bt_row_stride;
  a.max_blocks = max_blocks_per_seq;
  a.cu_seqlens = cu_seqlens;
  a.context_lens = first;
  a.num_seqs = num_seqs;
  a.num_tokens = num_tokens;
  a.k_out = (u16*)k_out;
  a.v_out = (u16*)v_out;
  const int64_t items = num_tokens * 2 * num_kv_heads * (head_dim / 8);
  const int64_t blocks = (items + 4 * kReadItems - 1) / (4 * kReadItems);
  if (num_kv_heads > 4096) return NDL_ERR_UNSUPPORTED;
  if (!grid_fits(blocks, 256)) return NDL_ERR_INVALID_ARG;
  const dim3 grid((unsigned)blocks), wg(256);
  const hipStream_t s = (hipStream_t)stream;
  const bool f16 = dtype_is_f16(dtype);
  if (head_dim == 128) {
    if (f16)
      hipLaunchKernelGGL((kv_read_fp8_kernel<128, true>), grid, wg, 0, s, a);
    else
      hipLaunchKernelGGL((kv_read_fp8_kernel<128, false>), grid, wg, 0, s, a);
  } else {
    if (f16)
      hipLaunchKernelGGL((kv_read_fp8_kernel<64, true>), grid, wg, 0, s, a);
    else
      hipLaunchKernelGGL((kv_read_fp8_kernel<64, false>), grid, wg, 0, s, a);
  }
  return check_launch();
}
