// The arithmetic by which fp8_attention.hip cuts the row blocks of a kv head into equal shares and
// finds the parts again: plain integers, nothing of the GPU.
//
// The row blocks lie end to end in slots, a slot per tile after `pad` empty ones.  Share s begins at
// slot s * chunk, or at a row block's end within `snap` slots of that: a sliver of a row block is
// not worth its part in the workspace.
#pragma once

#include <cstdint>

namespace ndl {

// A share's begin moves to a row block's end within an eighth of a share of it: us without / an
// eighth / a quarter / a third, 64 sequences of 512 to 4,096 tokens 50.9 / 48.8 / 48.9 / 51.9, with
// 1 to 8 new tokens each 56.2 / 56.0 / 60.0 / 60.4; 100 of up to 3,000, 28/4 heads 37.1 / 35.6 /
// 35.7 / 38.0.
constexpr int kSnap = 8;

struct Cut {
  int chunk, snap, shares;
};
__device__ __forceinline__ Cut cut_of(int total, int shares, int min_chunk, int pad) {
  const int c = (int)((uint32_t)(total + shares - 1) / (uint32_t)shares);
  const int chunk = c < min_chunk ? min_chunk : c;
  // (at least the empty slots: every part of a row block has a tile)
  return Cut{chunk, chunk / kSnap > pad ? chunk / kSnap : pad, shares};
}

// Where a share begins whose slot x is one of the row block's, first .. first + slots - 1.
__device__ __forceinline__ int share_begin(int x, int first, int slots, int snap) {
  if (x - first <= snap) return first;
  if (first + slots - x <= snap) return first + slots;
  return x;
}

// The tiles t0 .. t1 - 1 of a row block (its first slot, its tiles) within slots from .. to - 1.
__device__ __forceinline__ void share_tiles(int first, int pad, int ntiles, int from, int to,
                                            int* t0, int* t1) {
  const int base = first + pad;
  *t0 = from > base ? from - base : 0;
  *t1 = to < base + ntiles ? to - base : ntiles;
}

// Whether shares hold parts of a row block, and which: s0 .. s1, below the number of shares even
// where the row block is not of the lengths that the cut was made for.  Some begin inside it only
// where slots are left past those that share_begin moves to its ends; a shorter row block is one
// share's, wherever it lies (one that ends within `snap` slots of the stream's start has no last
// slot to divide).
__device__ __forceinline__ bool share_parts(int first, int slots, const Cut& cut, int* s0, int* s1) {
  if (slots < 2 * cut.snap + 2) return false;
  *s0 = (int)((uint32_t)(first + cut.snap) / (uint32_t)cut.chunk);
  *s1 = (int)((uint32_t)(first + slots - cut.snap - 1) / (uint32_t)cut.chunk);
  *s1 = *s1 < cut.shares ? *s1 : cut.shares - 1;
  return *s0 < *s1;
}

}  // namespace ndl
