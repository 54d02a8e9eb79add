// What the kernels of the 8-bit pool (kv_fp8.hip, fp8_attention.hip) share, and what they ask of
// the 16-bit prefill (varlen_prefill.hip).
#pragma once

#include "ndl_common.hpp"

namespace ndl {

// Two e4m3 codes of w's low or high half times scale (a power of two), in the 16-bit format.
template <bool F16, bool HI>
__device__ __forceinline__ uint32_t value2(uint32_t w, float scale) {
  if constexpr (F16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}

// varlen_prefill.hip's attention for a caller with long, uneven prefixes: as
// ndl_varlen_prefill_split, but split too where whole tiles would leave much of their last round
// idle.  Its workspace: prefill_rounds_workspace_bytes.
size_t prefill_rounds_workspace_bytes(int num_seqs, int64_t num_tokens, int max_seqlen,
                                      int max_blocks_per_seq, int num_heads, int num_kv_heads,
                                      int head_dim, int block_size);
int launch_prefill_rounds(void* out, const void* q, int64_t q_tok_stride, const void* kv_cache,
                          int64_t num_blocks, const int32_t* block_table, int64_t bt_row_stride,
                          int max_blocks_per_seq, const int32_t* cu_seqlens,
                          const int32_t* context_lens, int num_seqs, int64_t num_tokens,
                          int max_seqlen, int max_context_len, int num_heads, int num_kv_heads,
                          int head_dim, int block_size, int dtype, float scale, void* workspace,
                          size_t workspace_bytes, ndl_stream_t stream);

}  // namespace ndl
