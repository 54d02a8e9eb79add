// What tree_attention.hip offers attention_mass.hip and fp8_attention.hip.
#pragma once

#include "ndl_common.hpp"

namespace ndl {

// Attention of a chunk of new tokens per sequence over a 16-bit paged pool, or, of trees, an 8-bit one.
struct ChunkAttention {
  void* out;
  const void* q;
  int64_t q_tok_stride;
  const void* kv_cache;            // an 8-bit pool's codes
  const void* scales;              // and its scales; null: a 16-bit pool
  int64_t num_blocks;
  const int32_t* block_table;
  int64_t bt_row_stride;
  int max_blocks_per_seq;
  const int32_t* cu_seqlens;       // null: one token per sequence
  const int32_t* context_lens;
  const uint64_t* mask;            // null: causal
  int64_t mask_stride;
  int mask_words;
  float* lse;                      // [token][head], log2 of the softmax's denominator; null: none
  // [kv head][sequence][max_seqlen * group][score_keys], of at most kScoredColumns columns: scores
  // times scale and log2 e, those that are not attended -inf, of whole 32-key tiles.  Null: none.
  float* scores;
  int64_t score_keys;
  int num_seqs;
  int64_t num_tokens;
  int max_seqlen;
  int64_t max_keys;
  int num_heads, num_kv_heads, head_dim, block_size, dtype;
  float scale;
};

constexpr int kScoredColumns = 32;     // tokens times heads of a group that scores are kept of

// Whether a launch can be made of these, NDL_OK or the error.
int check_chunk_attention(const ChunkAttention& c);
size_t chunk_attention_workspace(const ChunkAttention& c);
int launch_chunk_attention(const ChunkAttention& c, void* workspace, size_t workspace_bytes,
                           hipStream_t s);

}  // namespace ndl
