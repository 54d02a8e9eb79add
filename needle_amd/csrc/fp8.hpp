// What the kernels of the 8-bit pool (kv_fp8.hip, fp8_attention.hip) share, and what they ask of
// the 16-bit prefill (varlen_prefill.hip).
#pragma once

#include "ndl_common.hpp"

namespace ndl {

// Whether a launch's first grid dimension can be that many workgroups: HIP counts its threads in 32
// bits, and launches the rest of a larger one without an error.
inline bool grid_fits(int64_t workgroups, int threads) {
  return workgroups <= (int64_t)0xffffffffu / threads;
}

// Two e4m3 codes of w's low or high half times scale (a power of two), in the 16-bit format.
template <bool F16, bool HI>
__device__ __forceinline__ uint32_t value2(uint32_t w, float scale) {
  if constexpr (F16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}

// Largest finite magnitude of the two 16-bit elements of w, as 16 bits; `inf`: the format's
// infinity.
__device__ __forceinline__ uint32_t finite_max(uint32_t w, uint32_t inf) {
  const uint32_t a = w & 0x7fffu, b = (w >> 16) & 0x7fffu;
  const uint32_t x = a < inf ? a : 0u, y = b < inf ? b : 0u;
  return x > y ? x : y;
}

// Two 16-bit elements -> two codes in the low half (HI: the high half) of `old`.
template <bool F16, bool HI>
__device__ __forceinline__ int quant2(uint32_t w, float mul, int old) {
  using T = Elt<F16>;
  // what is not finite becomes NaN (a saturating conversion would hide an infinity)
  const float nan = __uint_as_float(0x7fc00000u);
  constexpr uint32_t inf = F16 ? 0x7c00u : 0x7f80u;
  const float x = (w & 0x7fffu) < inf ? T::lo(w) * mul : nan;
  const float y = ((w >> 16) & 0x7fffu) < inf ? T::hi(w) * mul : nan;
  return __builtin_amdgcn_cvt_pk_fp8_f32(x, y, old, HI);
}
template <bool F16>
__device__ __forceinline__ u32x2 quant8(const u32x4& w, float mul) {
  const int a = quant2<F16, true>(w[1], mul, quant2<F16, false>(w[0], mul, 0));
  const int b = quant2<F16, true>(w[3], mul, quant2<F16, false>(w[2], mul, 0));
  return u32x2{(uint32_t)a, (uint32_t)b};
}

// The scale byte of the row that LANES lanes hold, 8 elements of each half in lo and hi.
template <int LANES, bool F16>
__device__ __forceinline__ int scale_byte(const u32x4& lo, const u32x4& hi) {
  constexpr uint32_t inf = F16 ? 0x7c00u : 0x7f80u;
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t x = finite_max(lo[e], inf), y = finite_max(hi[e], inf);
    m = m > x ? m : x;
    m = m > y ? m : y;
  }
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) {
    const uint32_t x = (uint32_t)__shfl_xor((int)m, o, 64);
    m = m > x ? m : x;
  }
  // 448 = 1.75 * 2^8: the row's exponent less 8, one more where its mantissa is past 1.75
  const uint32_t bits = __float_as_uint(Elt<F16>::lo(m));
  const int e8 = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e8 < 1 ? 1 : e8;
}

// lds_dma16 with an address of each lane's own.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void lds_dma16_each(const void* src, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds_addr)), "v"(src)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// varlen_prefill.hip's attention for a caller with long, uneven prefixes: as
// ndl_varlen_prefill_split, but split too where whole tiles would leave much of their last round
// idle.  The sequences may be some of a batch's, from any on: num_tokens are the batch's rows,
// seqs_tokens bounds these sequences'.  Its workspace: prefill_rounds_workspace_bytes (of
// seqs_tokens).
size_t prefill_rounds_workspace_bytes(int num_seqs, int64_t num_tokens, int max_seqlen,
                                      int max_blocks_per_seq, int num_heads, int num_kv_heads,
                                      int head_dim, int block_size);
int launch_prefill_rounds(void* out, const void* q, int64_t q_tok_stride, const void* kv_cache,
                          int64_t num_blocks, const int32_t* block_table, int64_t bt_row_stride,
                          int max_blocks_per_seq, const int32_t* cu_seqlens,
                          const int32_t* context_lens, int num_seqs, int64_t num_tokens,
                          int64_t seqs_tokens, int max_seqlen, int max_context_len, int num_heads,
                          int num_kv_heads, int head_dim, int block_size, int dtype, float scale,
                          void* workspace, size_t workspace_bytes, ndl_stream_t stream);

}  // namespace ndl
