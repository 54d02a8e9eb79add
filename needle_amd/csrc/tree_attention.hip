// Attention of drafted trees over the 16-bit paged pool, gfx950.  A sequence's chunk of new tokens
// are the nodes of a tree (the newest token its root); they are in the cache already, behind the
// context, at positions ctx + 0, ctx + 1, .. in the order of the chunk.
//
//   out[t][h] = sum_x softmax_x(scale * q[t][h] . k[x][h / g]) v[x][h / g],
//   x < ctx, and x = ctx + b for the set bits b of the token's mask row.
//
// Without a mask the chunk is causal (x <= ctx + t): what attention_mass.hip attends with.  The
// reference has no such attention; the arguments' meaning is its _prefill's and _decode's
// (needle/layers/attention.py:120-134, :291-310), with a cached prefix attended.
//
//   * Rows.  The g query heads of a kv head times the chunk's tokens are the columns, 32 to a wave
//     (S^T = K Q^T and O^T = V^T P^T on 32x32x16 MFMA, keys and head_dim as rows): of a workgroup's
//     eight waves CG (1, 2, 4, 8: what the row block's columns need) side by side hold up to 256
//     columns, so that a tree's keys are read once for all its nodes, and 8 / CG such groups take the
//     row block's 32-key tiles in turn.  (Four waves and 128 columns, trees of up to 256 columns: every
//     second row block reads all keys again, 170 us where this takes 155.)
//   * Keys.  A group's tile goes straight to its LDS ring in whole rows (1 KiB a load), K and V in
//     16-byte pieces swizzled by row so that the operand reads (K: ds_read_b128, V: transposing
//     ds_read_b64_tr_b16) spread over the banks.  Groups of several waves meet at a barrier for half
//     the ring's tiles (at each one: 165 us); the loads of single waves, which no other row
//     block repeats, pass the caches by (weights of 64 sequences' last tokens: 140 us for 125).
//   * An 8-bit pool's codes (trees of more than 64 columns, see fp8_attention.hip) go to a ring of each
//     wave's own; the wave unpacks what it has loaded, scale and all, into the group's 16-bit tiles.
//   * P^T needs no data movement: the accumulator layout of S^T is the operand's, with k order
//     8 h + e for key 16 t + 4 h + (e & 3) + 8 (e >> 2).
//   * Softmax in fp32 with exp2.  The maximum is raised (and the sums rescaled) only when a tile's
//     probabilities pass 256; P is rounded to the 16-bit format for the matrix cores (half a step of it,
//     what the output's own rounding costs too), its sum is taken before that.
//   * The mask costs nothing below the context: only tiles that reach into the chunk look at it, as
//     32 bits per column.
//   * Split: as fp8_attention.hip's (chunk_stream.hpp), a workgroup per (kv head, row block) or
//     equal shares of all of a kv head's tiles, merged by a second launch.
// Measured (us, a call): 64 trees of 16 to 64 nodes after 512 to 4,096 tokens, 32/8 heads of 128, bf16
// 155 to 162 (the keys at 2.8 to 2.95 TB/s, 470 to 490 TFLOP/s); 4 trees of 16 after 64 to 800, 14/2
// heads of 64, 8.7; 8 trees of 40 to 60 after 4,096 to 32,768 in an 8-bit pool, 28/4 heads of 128,
// float16, 165 (590 TFLOP/s).  What bounds the wide ones:
//   * Whole row blocks go to the XCDs in the order of the sequences, so uneven ones wait for the fullest
//     XCD: of those 64 trees its CUs have up to 137 steps of 32 keys where the mean is 94 (equal contexts
//     with as many keys, 111 for 97: 144 us).
//   * A step, 1.2 to 1.4 us on a full GPU, is neither bytes nor products: of a SIMD's cycles the matrix
//     cores take 27 %, the softmax 30 %, and LDS is busy for as many; two waves to a SIMD (222 of 256
//     registers) overlap them only in part.  Scores made a tile ahead took longer (195 us for 178, in
//     shares), a product put off past the barrier in half the waves too (172 for 165).
#include "chunk_stream.hpp"
#include "fp8.hpp"
#include "tree_attention.hpp"

#include <type_traits>

namespace ndl {
namespace {

constexpr float kRaiseSum = 256.f;   // a lane's sum of a tile's probabilities past which the
                                     // maximum is raised

// kScored: causal, and the scores stay behind in a.scores (row blocks of up to 32 columns).
enum Chunk { kCausal, kTree, kScored };

struct TreeOperands {
  u16* out;
  const u16* q;
  int64_t q_stride;
  const u16* kplane;
  const u16* vplane;
  int64_t num_blocks;
  int num_heads, num_kv_heads, group;
  const uint64_t* mask;         // null: causal
  int64_t mask_stride;
  int words;
  float* lse;
  float* scores;                // [kv head][sequence][column][score_keys], scaled, log2
  int64_t score_keys;
  int score_cols;
  const uint8_t* kscale;        // of an 8-bit pool, whose planes hold codes
  const uint8_t* vscale;
  uint32_t q_flip, q_keep;      // of two elements of q: signs flipped (scale < 0), kept (scale not 0)
};
struct TreeArgs : TreeOperands, RowBlocks {};

constexpr int kWaves = 8;

// With an 8-bit pool (FP8) a wave unpacks the codes that it has loaded itself, up to kCodeDepth steps
// ahead, into its group's 16-bit stages.
constexpr int kCodeDepth = 6;
template <int D>
struct TreeShape {
  static constexpr int kPlane = kTile * D * 2;             // bytes of a tile's K (or V)
  static constexpr int kStage = 2 * kPlane;
  static constexpr int kStages = (128 << 10) / kStage;     // of the ring, over all groups
  static constexpr int kPieces = kPlane / 1024;            // loads of a plane
  static constexpr int kRing = kStages * kStage;
  static constexpr int kSums = kWaves * 32 * D * 4;        // the waves' partial outputs
  static constexpr int kMl = 2 * kWaves * 32 * 4;
  static constexpr int kLds = (kRing > kSums ? kRing : kSums) + kMl;
};

// 16-byte piece of row r where its piece p lies.  K: 32 rows read at one piece, pairs of rows 8 apart
// and quads of neighbours at different banks.  V: four neighbouring rows read at 32 bytes.
template <int D>
__device__ __forceinline__ int k_swizzle(int r) {
  return D == 128 ? (((r & 3) << 2) | ((r >> 2) & 3)) : ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
}
__device__ __forceinline__ int v_swizzle(int r) { return (r & 3) << 1; }

// Waits until at most n (0 .. MAX) groups of I loads are in flight.
template <int I, int MAX>
__device__ __forceinline__ void wait_groups(int n) {
  if constexpr (MAX == 0) {
    vm_wait<0>();
  } else {
    if (n >= MAX)
      vm_wait<MAX * I>();
    else
      wait_groups<I, MAX - 1>(n);
  }
}

// Two outputs in the 16-bit format.  Of an 8-bit pool, in float16, those past it are its largest: they
// are sums of values of up to 65,504 and of what rounding the probabilities added.
template <bool F16, bool FP8>
__device__ __forceinline__ uint32_t pack_out(float x, float y) {
  if constexpr (F16 && FP8) {
    x = x > 65504.f ? 65504.f : x < -65504.f ? -65504.f : x;     // (a NaN stays)
    y = y > 65504.f ? 65504.f : y < -65504.f ? -65504.f : y;
  }
  return Elt<F16>::pack(x, y);
}

// 0xffff in each half of w that is an infinity or a NaN.
template <bool F16>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t inf = F16 ? 0x7c00u : 0x7f80u;
  return ((w & inf) == inf ? 0xffffu : 0u) | ((w >> 16 & inf) == inf ? 0xffff0000u : 0u);
}

// A workgroup's share of the row blocks of one kv head.  Its eight waves are as many groups of columns
// (CG) side by side as a row block has columns for, times as many groups of keys (KG) as are left.
template <int D, bool F16, Chunk KIND, bool FP8 = false>
__global__ __launch_bounds__(64 * kWaves, 2) void tree_attention_kernel(TreeArgs a) {
  constexpr bool TREE = KIND == kTree;
  using T = Elt<F16>;
  using X8 = typename T::x8;
  using S = TreeShape<D>;
  constexpr int NW = kWaves;
  constexpr int KS = D / 16;      // k steps of the QK product
  constexpr int DT = D / 32;      // 32-row tiles of O^T
  constexpr int CPR = D / 8;      // 16-byte pieces of a row
  constexpr int RPL = 512 / D;    // rows per load
  __shared__ __attribute__((aligned(16))) unsigned char smem[S::kLds];

  const int lane0 = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));

  // The kv heads of one share (or row block) run on one XCD at about the same time: workgroups
  // are dealt to the XCDs in turn, and heads share the tables, lengths and masks.
  const int Hkv = a.num_kv_heads;
  const unsigned per8 = 8u * Hkv, grp = blockIdx.x / per8, in8 = blockIdx.x - grp * per8;
  const int head = (int)(in8 >> 3);
  const int unit = (int)(grp * 8 + (in8 & 7));

  int e, first = 0, from = 0, to = 0;   // the row block, its first slot; the share's slots
  const bool whole = a.shares == 0;
  if (whole) {
    e = unit;
    if (e >= a.items) return;
  } else {
    if (unit >= a.shares) return;
    Stream<TREE> st;
    st.read(a, lane0);
    from = st.begin(a, lane0, unit);
    to = st.begin(a, lane0, unit + 1);
    if (from >= to) return;
    const Place p = st.find(a, lane0, from, -1);
    e = p.e;
    first = p.first;
  }

  for (; e < a.items; ++e) {
    const Item it = item_of<TREE>(a, e);
    const int ntiles = it.tiles();
    int t0 = 0, t1 = ntiles;
    if (!whole) {
      if (ntiles == 0) continue;
      if (first >= to) break;
      share_tiles(first, a.pad, ntiles, from, to, &t0, &t1);
      first += a.pad + ntiles;
      if (t0 >= t1) continue;     // only the empty slots are this share's
    } else if (it.n <= 0) {
      break;
    }
    const int cols = it.n * a.group;

    auto row_block = [&](auto groups) {
      constexpr int CG = decltype(groups)::value, KG = NW / CG;
      constexpr int NS = !FP8 ? S::kStages / KG : S::kStages / KG >= 8 ? 4 : 2;     // of a group
      constexpr int LOADS = 2 * S::kPieces / CG;       // of a wave, per stage
      // Steps between barriers: half of the ring is worked on while the other half is loaded.
      constexpr int BATCH = CG == 1 ? 1 : NS / 2, AHEAD = CG == 1 ? NS : BATCH;
      // (8-bit) loads of 1 KiB of a tile's codes, and how many of them are a wave's
      constexpr int CODE_LOADS = D / 16, MINE = CODE_LOADS > CG ? CODE_LOADS / CG : 1;
      constexpr int CODE_ROWS = 1024 / D;              // rows of a load
      constexpr int CODE_SLOT = MINE * 1280;           // a wave's codes of a stage, and their scales
      constexpr int ROOM = (S::kLds - S::kMl - NS * KG * S::kStage) / (NW * CODE_SLOT);
      constexpr int DEPTH = ROOM < kCodeDepth ? ROOM : kCodeDepth;      // stages of codes in flight
      static_assert(!FP8 || DEPTH >= 3, "room for the codes");
      static_assert(LOADS >= 1 && NS % BATCH == 0 && AHEAD * LOADS < 64, "loads of a wave");
      // (the lane through an empty asm: what is worked out from it stays within the row block)
      int lane = lane0;
      asm volatile("" : "+v"(lane));
      const int c = lane & 31, h = lane >> 5;
      const int kg = wv / CG, cg = wv % CG;
      const unsigned char* const ring = smem + kg * NS * S::kStage;
      const uint32_t ring_lds = lds_addr(ring);

      // This group's tiles: t0 + kg, t0 + kg + KG, ..  Lane 2 u + s of a window holds 16-token half s
      // of the window's tile u (32 of the group's tiles): its index in units of 16 rows of the plane
      // (block 0's where the id is invalid, with the lane's bit in win_bad).
      const int32_t* const table = a.block_table + (int64_t)it.seq * a.bt_row_stride;
      uint32_t window;
      uint64_t win_bad;
      auto load_window = [&](int u0) {
        const uint32_t tt = 2u * (uint32_t)(t0 + kg + KG * (u0 + (lane >> 1))) + (lane & 1);
        uint32_t col = tt >> a.tile_shift;
        if (col > (uint32_t)a.max_blocks - 1) col = (uint32_t)a.max_blocks - 1;
        const int b = table[col];
        const bool ok = b >= 0 && b < a.num_blocks;
        window = ((uint32_t)(ok ? b : 0) * (uint32_t)a.num_kv_heads + (uint32_t)head)
                     << a.tile_shift | (tt & ((1u << a.tile_shift) - 1u));
        win_bad = __builtin_amdgcn_ballot_w64(!ok);
      };
      load_window(0);

      // This lane's column: query token col / g, head head * g + col % g.
      const int col = 32 * cg + c;
      const bool live = col < cols;
      const int tok = (live ? col : cols - 1) / a.group;     // a column past the last repeats it
      const uint64_t* const mrow = TREE ? a.mask + (it.tok0 + tok) * a.mask_stride : nullptr;
      X8 q[KS];
      {
        const u16* const src =
            a.q + (it.tok0 + tok) * a.q_stride +
            (int64_t)(head * a.group + (live ? col : cols - 1) - tok * a.group) * D + 8 * h;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          u32x4 w = ld16(src + 16 * s);
          w = (w ^ a.q_flip) & a.q_keep;
          q[s] = __builtin_bit_cast(X8, w);
        }
      }
      const int all_keys = (int)it.keys();
      // position of the chunk's first token; below `open` every column attends
      const int pos = (int)it.pos, ctx = pos - (e - it.seq * a.blocks_per_seq) * a.toks;
      const int open = TREE ? ctx : pos + 1;

      f32x16 acc[DT];
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[t] = f32x16{};
      float m = kNegInf, l = 0.f;

      const int cnt = t1 - t0 > kg ? (t1 - t0 - kg + KG - 1) / KG : 0;   // this group's tiles
      const int steps = CG == 1 ? cnt : (t1 - t0 + KG - 1) / KG;         // barriers: every group's
      const int full = ((open < all_keys ? open : all_keys) / kTile) - t0 - kg;
      int plain = full > 0 ? (full + KG - 1) / KG : 0;                   // steps without a mask
      if (plain > cnt) plain = cnt;

      // A load's lane: row lane / CPR of its RPL rows, the piece that lands at lane % CPR.  Of K's
      // load p the swizzle has p in it too.
      const uint32_t src_row = (uint32_t)(lane / CPR) * (2 * D);
      const uint32_t src_k = src_row + 16u * ((lane % CPR) ^ k_swizzle<D>(lane / CPR));
      const uint32_t src_v = src_row + 16u * ((lane % CPR) ^ v_swizzle(lane / CPR));
      // What a wave loads of a stage: all (CG 1), K or V (2), half of K or of V (4), a quarter (8).
      const bool cg_v = 2 * cg / CG;
      const char* const my_plane = reinterpret_cast<const char*>(CG > 1 && cg_v ? a.vplane : a.kplane);
      const uint32_t my_src = cg_v ? src_v : src_k;
      uint32_t bad_bits = 0;        // two bits per stage: its halves with an invalid block id
      const uint32_t codes_lds =
          lds_addr(smem) + NS * KG * S::kStage + wv * DEPTH * CODE_SLOT;
      auto issue = [&](int u, int slot) {
        if (u > 0 && (u & 31) == 0) {
          load_window(u);
          asm volatile("" : "+v"(window));
        }
        if constexpr (FP8) {
#pragma unroll
          for (int i = 0; i < MINE; ++i) {
            // load x: of K below half of them, of V past them
            const int x = (cg + i * CG) % CODE_LOADS, row0 = x % (CODE_LOADS / 2) * CODE_ROWS;
            const bool v = x >= CODE_LOADS / 2;
            const uint32_t rows = (uint32_t)__builtin_amdgcn_readlane(
                                      (int)window, 2 * (u & 31) + row0 / 16) * 16u + row0 % 16;
            const uint32_t to = codes_lds + slot * CODE_SLOT + i * 1280;
            lds_dma16(reinterpret_cast<const char*>(v ? a.vplane : a.kplane) + (uint64_t)rows * D,
                      16u * lane, to);
            // the dword with the scale of the lane's row
            lds_dma4((v ? a.vscale : a.kscale) + rows, (uint32_t)(lane / (D / 16)) & ~3u, to + 1024);
          }
          bad_bits = (bad_bits & ~(3u << (2 * (u & 15)))) |
                     ((uint32_t)(win_bad >> (2 * (u & 31))) & 3u) << (2 * (u & 15));
          return;
        }
        const uint32_t st = ring_lds + slot * S::kStage;
        uint32_t off = my_src, off_v = src_v;
        asm volatile("" : "+v"(off), "+v"(off_v));   // (a load's own offset: no register over the loop)
#pragma unroll
        for (int s = 0; s < (CG >= 4 ? 1 : 2); ++s) {
          const int half = CG == 4 ? cg & 1 : CG == 8 ? (cg >> 1) & 1 : s;
          const uint64_t at =
              (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)window, 2 * (u & 31) + half) *
              (32 * D);
#pragma unroll
          for (int y = 0; y < (CG == 8 ? S::kPieces / 4 : S::kPieces / 2); ++y) {
            const int x = CG == 8 ? (cg & 1) * (S::kPieces / 4) + y : y;
            const uint32_t to = st + (uint32_t)(half * S::kPieces / 2 + x) * 1024;
            // (k_swizzle of a load's first row: the same in both halves)
            const uint32_t turn = 16u * k_swizzle<D>(x * RPL);
            if constexpr (CG == 1) {
              lds_dma16_nt(my_plane + at + 1024 * x, off ^ turn, to);
              lds_dma16_nt(reinterpret_cast<const char*>(a.vplane) + at + 1024 * x, off_v,
                           to + S::kPlane);
            } else {
              lds_dma16(my_plane + at + 1024 * x, cg_v ? off : off ^ turn,
                        cg_v ? to + S::kPlane : to);
            }
          }
        }
        if (win_bad || bad_bits)
          bad_bits = (bad_bits & ~(3u << (2 * slot))) |
                     ((uint32_t)(win_bad >> (2 * (u & 31))) & 3u) << (2 * slot);
      };
      // The wave's codes of a stage, into 16-bit stage u % NS.  In float16, which has no 65,536 (a row's
      // values from 63,488 on), keys are halved, for which the scores' scale makes up, and a value is
      // 65,504, the nearest there is.  A float16 row's values are multiples of 2^-24, so a halved key is
      // off by 2^-25 at most (odd multiples: 2^-24 of the key), every other is exact.
      auto unpack = [&](int u, int slot) {
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
          typedef const __attribute__((address_space(3))) u32x4* lds16;
          typedef __attribute__((address_space(3))) u32x4* lds16w;
          typedef const __attribute__((address_space(3))) uint32_t* lds4;
          const int x = (cg + i * CG) % CODE_LOADS, row0 = x % (CODE_LOADS / 2) * CODE_ROWS;
          const bool v = x >= CODE_LOADS / 2;
          const uint32_t from = codes_lds + slot * CODE_SLOT + i * 1280;
          const u32x4 w = *(lds16)(uintptr_t)(from + 16 * lane);
          const uint32_t four = *(lds4)(uintptr_t)(from + 1024 + 4 * lane);
          const int r = lane / (D / 16), row = row0 + r, p = 2 * (lane % (D / 16));
          float scale = __uint_as_float((four >> (8 * (r & 3)) & 0xffu) << 23);
          if (F16 && !v) scale *= 0.5f;
          uint32_t o[8];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            o[2 * y] = value2<F16, false>(w[y], scale);
            o[2 * y + 1] = value2<F16, true>(w[y], scale);
          }
          if (F16 && v && scale >= 256.f) {
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              if ((o[y] & 0x7fffu) == 0x7c00u) o[y] -= 1u;
              if ((o[y] & 0x7fff0000u) == 0x7c000000u) o[y] -= 0x10000u;
            }
          }
          const int swz = v ? v_swizzle(row) : k_swizzle<D>(row);
          const uint32_t to = ring_lds + (u % NS) * S::kStage + (v ? S::kPlane : 0) + row * (2 * D);
          *(lds16w)(uintptr_t)(to + 16 * (p ^ swz)) = u32x4{o[0], o[1], o[2], o[3]};
          *(lds16w)(uintptr_t)(to + 16 * ((p + 1) ^ swz)) = u32x4{o[4], o[5], o[6], o[7]};
        }
      };
      // What was loaded so far arrives here: the compiler's own waits in the loop would drain the
      // ring, whose loads it does not see, at every step.
      asm volatile("" : "+v"(window));
#pragma unroll 1
      for (int d = 0; d < (FP8 ? DEPTH : AHEAD) && d < cnt; ++d) issue(d, d);
#pragma unroll
      for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(q[s]));

      // Operand offsets in a stage, in bytes.
      uint32_t koff[KS], voff[DT];
#pragma unroll
      for (int s = 0; s < KS; ++s)
        koff[s] = ring_lds + 2 * (c * D + 8 * ((2 * s + h) ^ k_swizzle<D>(c)));
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const int r = (lane & 15) >> 2;              // of four rows, at 4 h
        const int piece = 4 * t + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        voff[t] = ring_lds + S::kPlane +
                  2 * ((4 * h + r) * D + 8 * (piece ^ v_swizzle(r)) + 4 * (lane & 1));
      }

      // One tile.  MASKED: some column may not attend some key.
      auto step = [&](int u, int slot, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        typedef const __attribute__((address_space(3))) u32x4* lds16;
        typedef __attribute__((address_space(3))) i16x4* lds4;
        const uint32_t st = slot * S::kStage;
        uint32_t mine = ~0u;                // the column's keys
        if constexpr (MASKED) {
          const uint32_t bad = (bad_bits >> (2 * (FP8 ? u & 15 : slot))) & 3u;
          const int kv0 = kTile * (t0 + kg + KG * u);
          // what any column attends, then this one
          uint32_t some = low_bits(all_keys - kv0);
          if (bad & 1) some &= 0xffff0000u;
          if (bad & 2) some &= 0x0000ffffu;
          mine = some;
          if (kv0 + kTile > open)
            mine &= TREE ? bits_at(mrow, a.words, kv0 - ctx) : low_bits(pos + tok + 1 - kv0);
          // values that no column attends may hold anything: 0 * NaN must not happen (each wave clears
          // them for itself)
          for (uint32_t none = ~some; none; none &= none - 1) {
            const uint32_t at = ring_lds + st + S::kPlane + __builtin_ctz(none) * (2 * D);
            if (lane < D / 2)
              *(__attribute__((address_space(3))) uint32_t*)(uintptr_t)(at + 4 * lane) = 0u;
          }
          asm volatile("" ::: "memory");
        }
        // S^T: lane (c, h) holds keys 8 (r / 4) + 4 h + r % 4 of column c
        f32x16 sc = {};
        {
          u32x4 ka[KS];
#pragma unroll
          for (int s = 0; s < KS; ++s) ka[s] = *(lds16)(uintptr_t)(koff[s] + st);
#pragma unroll
          for (int s = 0; s < KS; ++s)
            sc = T::mfma32x32x16(__builtin_bit_cast(X8, ka[s]), q[s], sc);
        }
        X8 va[2][DT];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const uint32_t at = voff[d] + st + 32 * t * D;
            const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)at);
            const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)(at + 16 * D));
            const u32x2 lo = __builtin_bit_cast(u32x2, x), hi = __builtin_bit_cast(u32x2, y);
            va[t][d] = __builtin_bit_cast(X8, u32x4{lo[0], lo[1], hi[0], hi[1]});
          }
        // Infinities and NaN in values that some columns attend and others do not (0 times one is NaN):
        // taken out of the product and put into the columns that attend them.
        bool odd = false;
        if constexpr (MASKED) {
          f32x16 probe = {};
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int d = 0; d < DT; ++d) probe = T::mfma32x32x16(va[t][d], X8{}, probe);
          float any = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) any += probe[r];
          odd = __builtin_amdgcn_ballot_w64(any != 0.f) != 0;
          if (odd) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int d = 0; d < DT; ++d) {
                u32x4 w = __builtin_bit_cast(u32x4, va[t][d]);
#pragma unroll
                for (int x = 0; x < 4; ++x) w[x] &= ~not_finite<F16>(w[x]);
                va[t][d] = __builtin_bit_cast(X8, w);
              }
          }
        }
        auto refill = [&] {     // what was read is in registers before the stage's next loads go out
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (u + NS < cnt) issue(u + NS, slot);
        };
        if constexpr (CG == 1 && !MASKED) refill();
        if constexpr (MASKED) {
          const uint32_t here = mine >> (4 * h);      // from the lane's first key on
#pragma unroll
          for (int r = 0; r < 16; ++r)
            sc[r] = (here >> (8 * (r >> 2) + (r & 3))) & 1u ? sc[r] : kNegInf;
        }

        if constexpr (KIND == kScored) {
          // four keys to a store; past the keys and where nothing is attended -inf (a context may be
          // longer than the call's bound, which the rows are of)
          if (live && col < a.score_cols && kTile * (int64_t)(t0 + kg + KG * u) < a.score_keys) {
            float* const at =
                a.scores +
                (((int64_t)head * a.num_seqs + it.seq) * a.score_cols + col) * a.score_keys +
                kTile * (t0 + kg + KG * u) + 4 * h;
#pragma unroll
            for (int x = 0; x < 4; ++x)
              *reinterpret_cast<f32x4*>(at + 8 * x) =
                  f32x4{sc[4 * x] * a.scale_log2, sc[4 * x + 1] * a.scale_log2,
                        sc[4 * x + 2] * a.scale_log2, sc[4 * x + 3] * a.scale_log2};
          }
        }

        // Probabilities against the running maximum as it stands.  Where a lane's sum of them exceeds
        // kRaiseSum, or while a column has no maximum yet, the maximum is raised, the sums are rescaled
        // and the probabilities taken again: no maximum is computed otherwise.
        uint32_t pw[8];
        float sum;
        auto probs = [&] {
          const float base = m == kNegInf ? 0.f : m;
          float p[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) p[r] = fast_exp2(fmaf(sc[r], a.scale_log2, -base));
#pragma unroll
          for (int r = 0; r < 8; ++r) pw[r] = T::pack(p[2 * r], p[2 * r + 1]);
#pragma unroll
          for (int w = 8; w >= 1; w >>= 1)
#pragma unroll
            for (int r = 0; r < w; ++r) p[r] += p[r + w];
          sum = p[0];
        };
        probs();
        if (__builtin_amdgcn_ballot_w64(!(sum <= kRaiseSum) || m == kNegInf)) {
          float mt = fmaxf(sc[0], sc[1]);
#pragma unroll
          for (int r = 2; r < 16; r += 2) mt = fmaxf(fmaxf(mt, sc[r]), sc[r + 1]);
          const float nm = fmaxf(m, max_xor32(mt) * a.scale_log2);
          const float f = m == nm ? 1.f : fast_exp2(m - nm);
          m = nm;
          l *= f;
#pragma unroll
          for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              // in place (a plain product may get other registers, and copies at every step); the
              // first one waits for f, which the compiler's hazard tracking does not see to in asm
              if (t == 0 && r == 0)
                asm volatile("s_nop 1\n\tv_mul_f32 %0, %0, %1" : "+v"(acc[t][r]) : "v"(f));
              else
                asm volatile("v_mul_f32 %0, %0, %1" : "+v"(acc[t][r]) : "v"(f));
            }
          probs();
        }
        l += sum;
        if constexpr (MASKED) {
          if (odd) {
#pragma unroll 1
            for (int key = 0; key < kTile; ++key) {
              const bool sees = (mine >> key) & 1u;
              const uint32_t at = ring_lds + st + S::kPlane + key * (2 * D);
#pragma unroll
              for (int x = 0; x < 4 * DT; ++x) {      // head_dim 8 x + 4 h ..
                typedef const __attribute__((address_space(3))) u32x2* lds8;
                u32x2 w = *(lds8)(uintptr_t)(at + 2 * (8 * (x ^ v_swizzle(key)) + 4 * h));
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  w[y] &= sees ? not_finite<F16>(w[y]) : 0u;
                  acc[x >> 2][4 * (x & 3) + 2 * y] += T::lo(w[y]);
                  acc[x >> 2][4 * (x & 3) + 2 * y + 1] += T::hi(w[y]);
                }
              }
            }
          }
          if constexpr (CG == 1) refill();
        }

        // O^T += V^T P^T
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const X8 pb = __builtin_bit_cast(X8, u32x4{pw[4 * t], pw[4 * t + 1], pw[4 * t + 2],
                                                     pw[4 * t + 3]});
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[d] = T::mfma32x32x16(va[t][d], pb, acc[d]);
        }
      };

      int u = 0, slot = 0, code = 0;     // code: FP8: the slot of the next tile's codes
      // The next tile's codes, which have arrived, become 16-bit ones; later codes take their place.
      auto next_codes = [&](int n) {     // n: the tile
        if constexpr (FP8) {
          if (n >= cnt) return;
          const int last = n + DEPTH - 1 < cnt - 1 ? n + DEPTH - 1 : cnt - 1;     // issued
          wait_groups<2 * MINE, DEPTH - 1>(last - n);
          asm volatile("" ::: "memory");
          unpack(n, code);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (n + DEPTH < cnt) issue(n + DEPTH, code);
          code = code + 1 == DEPTH ? 0 : code + 1;
        }
      };
      if constexpr (FP8)
        for (int n = 0; n < BATCH; ++n) next_codes(n);
      auto begin = [&] {
        if constexpr (FP8) {
          // every wave's part of these stages is there, every wave's reads of those before done
          if (u % BATCH == 0) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
          next_codes(u + BATCH);
          return;
        }
        if constexpr (CG > 1) {
          if (u % BATCH != 0) return;
          // every wave's loads of these stages are there, every wave's reads of those before done
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
          for (int x = BATCH; x < 2 * BATCH; ++x)
            if (u + x < cnt) issue(u + x, (u + x) % NS);
        } else {
          wait_groups<LOADS, AHEAD - 1>(cnt - 1 - u);
          asm volatile("" ::: "memory");
        }
      };
      auto end = [&] {
        slot = slot + 1 == NS ? 0 : slot + 1;
        ++u;
      };
      // (a wave without columns loads for the rest)
      const bool idle = CG > 1 && 32 * cg >= cols;
      // Two loops, the second from the first tile with a mask on: accumulators that both ways of one
      // loop write are copied at every step.
      bool begun = false;
      while (u < steps) {
        begin();
        begun = u >= plain || ((bad_bits >> (2 * (FP8 ? u & 15 : slot))) & 3u) != 0;
        if (begun) break;
        if (!idle) step(u, slot, std::false_type{});
        end();
      }
      while (u < steps) {
        if (!begun) begin();
        begun = false;
        // (a group may have a tile less than others)
        if (!idle && u < cnt) step(u, slot, std::true_type{});
        end();
      }

      // The groups' results joined; quad x of a wave's accumulators holds head_dim 32 (x / 4) +
      // 8 (x % 4) + 4 h .. + 3 of its lane's column.
      l = add_xor32(l);
      const bool part = !whole && (t0 > 0 || t1 < ntiles);
      int64_t row, seg;
      bool lead;                    // the lane that writes a column's statistics
      {
        // (worked out here, not kept over the loop)
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int col = 32 * cg + (ln & 31), tok = col / a.group;
        row = ((it.tok0 + tok) * a.num_heads + head * a.group + col - tok * a.group) * D +
              4 * (ln >> 5);
        seg = (((int64_t)head * a.nseg + unit + e) * a.toks * a.group + col) * D + 4 * (ln >> 5);
        lead = ln < 32;
      }
      auto put_stats = [&](float mm, float ll) {
        if (!lead) return;
        if (part)
          *reinterpret_cast<f32x2*>(a.ws_ml + seg / D * 2) = f32x2{mm, ll};
        else if (a.lse != nullptr)
          a.lse[row / D] = mm + __log2f(ll);
      };
      auto put = [&](int x, const f32x4& o, float inv) {
        if (part)
          *reinterpret_cast<f32x4*>(a.ws_acc + seg + 8 * x) = o;
        else
          *reinterpret_cast<u32x2*>(a.out + row + 8 * x) =
              u32x2{pack_out<F16, FP8>(o[0] * inv, o[1] * inv),
                    pack_out<F16, FP8>(o[2] * inv, o[3] * inv)};
      };
      auto quad = [&](int x) {
        return f32x4{acc[x >> 2][4 * (x & 3)], acc[x >> 2][4 * (x & 3) + 1],
                     acc[x >> 2][4 * (x & 3) + 2], acc[x >> 2][4 * (x & 3) + 3]};
      };
      if constexpr (KG == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;     // nothing attended: zeros
        if (live) {
          put_stats(m, l);
#pragma unroll
          for (int x = 0; x < 4 * DT; ++x) put(x, quad(x), inv);
        }
      } else {
        float* const ml = reinterpret_cast<float*>(smem + S::kLds - S::kMl);   // [2][wave][column]
        if (h == 0) {
          ml[32 * wv + c] = m;
          ml[32 * (NW + wv) + c] = l;
        }
        __syncthreads();
        float mm = kNegInf, ll = 0.f;
#pragma unroll
        for (int g = 0; g < KG; ++g) mm = fmaxf(mm, ml[32 * (g * CG + cg) + c]);
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          const float mw = ml[32 * (g * CG + cg) + c];
          ll += ml[32 * (NW + g * CG + cg) + c] * (mw == mm ? 1.f : fast_exp2(mw - mm));
        }
        const float f = m == mm ? 1.f : fast_exp2(m - mm);
        f32x4* const sums = reinterpret_cast<f32x4*>(smem);       // [wave][quad][lane]
#pragma unroll
        for (int x = 0; x < 4 * DT; ++x) sums[(wv * 4 * DT + x) * 64 + lane] = quad(x) * f;
        __syncthreads();
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        if (live) {
          if (kg == 0) put_stats(mm, ll);
#pragma unroll
          for (int y = 0; y < 4 * DT / KG; ++y) {
            const int x = y * KG + kg;
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int g = 0; g < KG; ++g) o += sums[((g * CG + cg) * 4 * DT + x) * 64 + lane];
            put(x, o, inv);
          }
        }
      }
    };
    if constexpr (KIND == kScored) {
      row_block(std::integral_constant<int, 1>{});
    } else if constexpr (FP8) {
      if (cols <= 128)
        row_block(std::integral_constant<int, 4>{});
      else
        row_block(std::integral_constant<int, 8>{});
    } else {
      if (cols <= 32)
        row_block(std::integral_constant<int, 1>{});
      else if (cols <= 64)
        row_block(std::integral_constant<int, 2>{});
      else if (cols <= 128)
        row_block(std::integral_constant<int, 4>{});
      else
        row_block(std::integral_constant<int, 8>{});
    }
    if (whole) return;
    __syncthreads();     // before the ring is written again
  }
}

// Columns of a workgroup of the merge: many where that makes workgroups enough, each of which finds its
// parts first (32 columns / 8, calls of us: 1 tree of 126 columns after 16,000, 28/4 heads, 51.7 / 44.1;
// 24 of 511 after 2,000 124 / 135).
constexpr int kJoinMany = 32, kJoinFew = 8, kJoinFrom = 512;
template <int D, bool F16, bool TREE, bool FP8, int COLS>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
  merge_row_block<D, TREE, COLS, true>(a, a.group, [&](const Item& it, int head, int col, int d0,
                                                 const float* o, float m, float l) {
    constexpr int PER = COLS * D / 256;
    const int tok = col / a.group;
    const int64_t row = (it.tok0 + tok) * a.num_heads + head * a.group + col - tok * a.group;
    uint32_t* const dst = reinterpret_cast<uint32_t*>(a.out + row * D + d0);
    uint32_t w[PER / 2];
#pragma unroll
    for (int x = 0; x < PER / 2; ++x) w[x] = pack_out<F16, FP8>(o[2 * x], o[2 * x + 1]);
    if constexpr (PER >= 8) {
#pragma unroll
      for (int x = 0; x < PER / 2; x += 4)
        st16(reinterpret_cast<u16*>(dst + x), u32x4{w[x], w[x + 1], w[x + 2], w[x + 3]});
    } else {
#pragma unroll
      for (int x = 0; x < PER / 2; ++x) dst[x] = w[x];
    }
    if (d0 == 0 && a.lse != nullptr) a.lse[row] = m + __log2f(l);
  });
}

// ---------------------------------------------------------------- launches

template <int D, bool F16>
const void* kernel_of(Chunk kind, bool fp8) {
  if (fp8) return (const void*)tree_attention_kernel<D, F16, kTree, true>;
  return kind == kTree     ? (const void*)tree_attention_kernel<D, F16, kTree>
         : kind == kScored ? (const void*)tree_attention_kernel<D, F16, kScored>
                           : (const void*)tree_attention_kernel<D, F16, kCausal>;
}
const void* kernel_for(int head_dim, bool f16, Chunk kind, bool fp8 = false) {
  if (head_dim == 128) return f16 ? kernel_of<128, true>(kind, fp8) : kernel_of<128, false>(kind, fp8);
  return f16 ? kernel_of<64, true>(kind, fp8) : kernel_of<64, false>(kind, fp8);
}
Chunk kind_of(const ChunkAttention& c) {
  return c.mask != nullptr ? kTree : c.scores != nullptr ? kScored : kCausal;
}

constexpr int kMinChunk = 8;      // slots a share has at least
constexpr int kWholeTiles = 48;   // tiles up to which a row block is one workgroup's
constexpr int kPad = 4;           // empty slots before a row block

struct Plan {
  int toks;
  int64_t blocks_per_seq, items;
  int shares;                 // 0: whole row blocks
  int64_t nseg;
  size_t ml_bytes, acc_bytes;
};

Plan plan_for(const ChunkAttention& c) {
  Plan p{};
  const int group = c.num_heads / c.num_kv_heads;
  // the formats' kernels use the same resources
  int64_t res = resident_workgroups(kernel_for(c.head_dim, false, kTree), 64 * kWaves);
  if (res <= 0) res = 256;
  const int64_t tiles = (c.max_keys + kTile - 1) / kTile;
  // Columns of a row block: all that the kernel takes, or, where row blocks are whole, as few as leave
  // no part of the GPU idle.
  int64_t units = 0;
  for (int cols = 32 * kWaves; cols >= 32; cols /= 2) {
    if (cols > 32 && (int64_t)c.max_seqlen * group <= cols / 2) continue;
    p.toks = cols / group;
    p.blocks_per_seq = ((int64_t)c.max_seqlen + p.toks - 1) / p.toks;
    p.items = c.num_seqs * p.blocks_per_seq;
    units = p.items * c.num_kv_heads;
    if (units * 2 > res || tiles > kWholeTiles) break;
  }
  // Whole row blocks where there are enough to even out: of wide ones two for each place (their parts
  // are large: 64 trees of 16 .. 64 nodes after up to 4,096 tokens, 32 heads on 8: 164 us whole, 178
  // in shares), of narrow ones four (those sequences' last tokens and their weights: 125 us in shares,
  // 139 whole).
  // (slots and segments are counted in 31 bits)
  const bool whole = tiles <= kWholeTiles || units >= (p.toks * group > 32 ? 2 : 4) * res ||
                     p.items * (tiles + kPad) + 2 * res * kMinChunk > 0x40000000;
  if (!whole) {
    int64_t s = res / c.num_kv_heads / 8 * 8;
    if (s < 8) s = 8;
    p.shares = (int)s;
    p.nseg = s + p.items;
    const size_t cols_of = (size_t)c.num_kv_heads * p.nseg * p.toks * group;
    p.ml_bytes = (cols_of * 8 + 255) / 256 * 256;
    p.acc_bytes = cols_of * c.head_dim * 4;
  }
  return p;
}

template <int D, bool F16, int COLS>
void launch_merge(const TreeArgs& a, bool tree, bool fp8, dim3 grid, hipStream_t s) {
  if (F16 && fp8)
    hipLaunchKernelGGL((tree_merge_kernel<D, F16, true, F16, COLS>), grid, dim3(256), 0, s, a);
  else if (tree)
    hipLaunchKernelGGL((tree_merge_kernel<D, F16, true, false, COLS>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((tree_merge_kernel<D, F16, false, false, COLS>), grid, dim3(256), 0, s, a);
}
template <int D, bool F16>
void launch_merge(const TreeArgs& a, bool tree, bool fp8, hipStream_t s) {
  const int cols = a.toks * a.group;
  const bool many = (int64_t)a.items * a.num_kv_heads * ((cols + kJoinMany - 1) / kJoinMany) >=
                    kJoinFrom;
  const int each = many ? kJoinMany : kJoinFew;
  const dim3 grid((unsigned)a.items, (unsigned)a.num_kv_heads, (unsigned)((cols + each - 1) / each));
  many ? launch_merge<D, F16, kJoinMany>(a, tree, fp8, grid, s)
       : launch_merge<D, F16, kJoinFew>(a, tree, fp8, grid, s);
}

// ---------------------------------------------------------------- masks from parents

// A workgroup per 256 tokens of sequence blockIdx.y: each walks up from its node, towards lower
// indices, and writes its row's words from the last to the first as it passes them.
constexpr int kHeldParents = 4096;   // of a sequence, in LDS
__global__ __launch_bounds__(256) void tree_mask_kernel(uint64_t* mask, int64_t stride, int words,
                                                        int32_t* depth, const int32_t* parents,
                                                        const int32_t* cu, int64_t num_tokens) {
  __shared__ int32_t up[kHeldParents];
  const int64_t first = cu[blockIdx.y], end = cu[blockIdx.y + 1];
  if (first < 0 || end > num_tokens || end <= first) return;
  const int64_t n = end - first, t0 = (int64_t)blockIdx.x * 256;
  if (t0 >= n) return;
  const int64_t need = t0 + 256 < n ? t0 + 256 : n;     // a walk leads to lower indices
  for (int64_t i = threadIdx.x; i < need && i < kHeldParents; i += 256) up[i] = parents[first + i];
  __syncthreads();
  const int64_t t = t0 + threadIdx.x;
  if (t >= n) return;
  uint64_t* const row = mask + (first + t) * stride;
  int64_t at = t;
  int w = words - 1, hops = 0;
  uint64_t word = 0;
  for (;;) {
    while ((int64_t)w > at >> 6) {
      row[w--] = word;
      word = 0;
    }
    if (at >> 6 == w) word |= (uint64_t)1 << (at & 63);     // (a node past the words has none)
    const int64_t p = at < kHeldParents ? up[at] : parents[first + at];
    if (p < 0 || p >= at) break;
    at = p;
    ++hops;
  }
  for (; w >= 0; --w) {
    row[w] = word;
    word = 0;
  }
  depth[first + t] = hops;
}

}  // namespace

int check_chunk_attention(const ChunkAttention& c) {
  if (!dtype_supported(c.dtype) || (c.head_dim != 64 && c.head_dim != 128) ||
      block_tile_shift(c.block_size) < 0 || c.num_heads <= 0 || c.num_kv_heads <= 0 ||
      c.num_heads % c.num_kv_heads != 0 || c.num_heads / c.num_kv_heads > 16)
    return NDL_ERR_UNSUPPORTED;
  if (c.num_seqs < 0 || c.num_tokens < 0 || c.num_blocks <= 0 || c.max_blocks_per_seq <= 0 ||
      c.bt_row_stride < c.max_blocks_per_seq || c.max_seqlen <= 0 || c.max_keys <= 0)
    return NDL_ERR_INVALID_ARG;
  if (c.num_seqs == 0 || c.num_tokens == 0) return NDL_OK;
  if (!c.out || !c.q || !c.kv_cache || !c.block_table || !c.context_lens)
    return NDL_ERR_INVALID_ARG;
  if (c.cu_seqlens == nullptr && (c.num_tokens != c.num_seqs || c.max_seqlen != 1))
    return NDL_ERR_INVALID_ARG;
  if (c.q_tok_stride < (int64_t)c.num_heads * c.head_dim || (c.q_tok_stride & 7))
    return NDL_ERR_INVALID_ARG;
  if (((uintptr_t)c.out | (uintptr_t)c.q | (uintptr_t)c.kv_cache) & 15u)
    return NDL_ERR_INVALID_ARG;
  if (c.mask != nullptr &&
      (c.mask_words <= 0 || c.mask_stride < c.mask_words || (uintptr_t)c.mask & 7u))
    return NDL_ERR_INVALID_ARG;
  if ((int64_t)c.max_blocks_per_seq * c.block_size > 0x7fffff00 || 
      c.num_blocks * c.num_kv_heads * (c.block_size / 16) > 0x7fffffff)
    return NDL_ERR_UNSUPPORTED;
  return NDL_OK;
}

static ChunkAttention within_table(ChunkAttention c) {
  const int64_t cap = (int64_t)c.max_blocks_per_seq * c.block_size;
  if (c.max_blocks_per_seq > 0 && c.max_keys > cap) c.max_keys = cap;
  return c;
}

size_t chunk_attention_workspace(const ChunkAttention& c) {
  const Plan p = plan_for(c);
  return p.ml_bytes + p.acc_bytes;
}

int launch_chunk_attention(const ChunkAttention& call, void* workspace, size_t workspace_bytes,
                           hipStream_t s) {
  const int rc0 = check_chunk_attention(call);
  if (rc0 != NDL_OK || call.num_seqs == 0 || call.num_tokens == 0) return rc0;
  const ChunkAttention c = within_table(call);
  const Plan p = plan_for(c);
  if (p.items > 0x7fffff00) return NDL_ERR_INVALID_ARG;
  TreeArgs a{};
  if (p.shares) {
    if (c.num_kv_heads > 65535) return NDL_ERR_UNSUPPORTED;     // a grid dimension of the merge
    if (!workspace || workspace_bytes < p.ml_bytes + p.acc_bytes || (uintptr_t)workspace & 255u)
      return NDL_ERR_WORKSPACE;
    a.ws_ml = (float*)workspace;
    a.ws_acc = (float*)((char*)workspace + p.ml_bytes);
  }
  a.out = (u16*)c.out;
  a.q = (const u16*)c.q;
  a.q_stride = c.q_tok_stride;
  a.kplane = (const u16*)c.kv_cache;
  const int64_t rows = c.num_blocks * c.num_kv_heads * (int64_t)c.block_size;     // of a plane
  a.vplane = a.kplane + rows * c.head_dim;
  if (c.scales != nullptr) {
    a.vplane = (const u16*)((const char*)c.kv_cache + rows * c.head_dim);
    a.kscale = (const uint8_t*)c.scales;
    a.vscale = a.kscale + rows;
  }
  a.num_blocks = c.num_blocks;
  a.num_heads = c.num_heads;
  a.num_kv_heads = c.num_kv_heads;
  a.group = c.num_heads / c.num_kv_heads;
  a.mask = c.mask;
  a.mask_stride = c.mask_stride;
  a.words = c.mask_words;
  a.lse = c.lse;
  a.scores = c.scores;
  a.score_keys = c.score_keys;
  a.score_cols = c.max_seqlen * a.group;
  a.block_table = c.block_table;
  a.bt_row_stride = c.bt_row_stride;
  a.max_blocks = c.max_blocks_per_seq;
  a.tile_shift = block_tile_shift(c.block_size);
  a.cu_seqlens = c.cu_seqlens;
  a.context_lens = c.context_lens;
  a.num_seqs = c.num_seqs;
  a.num_tokens = c.num_tokens;
  a.toks = p.toks;
  a.blocks_per_seq = (int)p.blocks_per_seq;
  a.items = (int)p.items;
  // the running maximum is of the scores before they are scaled: the scale's sign goes into q
  a.q_flip = c.scale < 0.f ? 0x80008000u : 0u;
  a.q_keep = c.scale == 0.f ? 0u : ~0u;
  a.scale_log2 = c.scale == 0.f ? 1.f : fabsf(c.scale) * kLog2e;
  if (c.scales != nullptr && dtype_is_f16(c.dtype)) a.scale_log2 *= 2.f;     // (keys are halved)
  a.shares = p.shares;
  a.min_chunk = kMinChunk;
  a.pad = kPad;
  a.nseg = (int)p.nseg;
  const int threads = 64 * kWaves;
  const int64_t units = a.shares ? a.shares : ((int64_t)a.items + 7) / 8 * 8;
  const int64_t wgs = units * a.num_kv_heads;
  if (!grid_fits(wgs, threads)) return NDL_ERR_INVALID_ARG;
  void* args[] = {&a};
  if (hipLaunchKernel(kernel_for(c.head_dim, dtype_is_f16(c.dtype), kind_of(c),
                                 c.scales != nullptr),
                      dim3((unsigned)wgs), dim3(threads), args, 0, s) != hipSuccess) {
    (void)hipGetLastError();  // clear the error so that the next call's check sees its own
    return NDL_ERR_LAUNCH;
  }
  const int rc = check_launch();
  if (rc != NDL_OK || a.shares == 0) return rc;
  const bool f16 = dtype_is_f16(c.dtype), tree = c.mask != nullptr, fp8 = c.scales != nullptr;
  if (c.head_dim == 128)
    f16 ? launch_merge<128, true>(a, tree, fp8, s) : launch_merge<128, false>(a, tree, fp8, s);
  else
    f16 ? launch_merge<64, true>(a, tree, fp8, s) : launch_merge<64, false>(a, tree, fp8, s);
  return check_launch();
}

}  // namespace ndl

extern "C" size_t ndl_tree_attention_workspace_bytes(int num_seqs, int max_seqlen, int64_t max_keys,
                                                     int num_heads, int num_kv_heads, int head_dim,
                                                     int block_size) {
  using namespace ndl;
  if (num_seqs <= 0 || max_seqlen <= 0 || max_keys <= 0 || max_keys > 0x7fffff00 ||
      (head_dim != 64 && head_dim != 128) || block_tile_shift(block_size) < 0 || num_heads <= 0 ||
      num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || num_heads / num_kv_heads > 16)
    return 0;
  ChunkAttention c{};
  c.num_seqs = num_seqs;
  c.max_seqlen = max_seqlen;
  c.max_keys = max_keys;
  c.num_heads = num_heads;
  c.num_kv_heads = num_kv_heads;
  c.head_dim = head_dim;
  return chunk_attention_workspace(c);
}

extern "C" int ndl_tree_attention(void* out, const void* q, int64_t q_tok_stride,
                                  const void* kv_cache, int64_t num_blocks,
                                  const int32_t* block_table, int64_t bt_row_stride,
                                  int max_blocks_per_seq, const int32_t* cu_seqlens,
                                  const int32_t* context_lens, const void* mask,
                                  int64_t mask_stride, int mask_words, int num_seqs,
                                  int64_t num_tokens, int max_seqlen, int64_t max_keys,
                                  int num_heads, int num_kv_heads, int head_dim, int block_size,
                                  int dtype, float scale, void* workspace, size_t workspace_bytes,
                                  ndl_stream_t stream) {
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
  c.mask = (const uint64_t*)mask;
  c.mask_stride = mask_stride;
  c.mask_words = mask_words;
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
  if (num_seqs > 0 && num_tokens > 0 && (!mask || !cu_seqlens)) return NDL_ERR_INVALID_ARG;
  return launch_chunk_attention(c, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int ndl_tree_mask(void* mask, int64_t mask_stride, int mask_words, int32_t* depth,
                             const int32_t* parents, const int32_t* cu_seqlens, int num_seqs,
                             int64_t num_tokens, int max_seqlen, ndl_stream_t stream) {
  using namespace ndl;
  if (num_seqs < 0 || num_tokens < 0 || max_seqlen < 0 || mask_words <= 0 ||
      mask_stride < mask_words)
    return NDL_ERR_INVALID_ARG;
  if (num_seqs == 0 || num_tokens == 0 || max_seqlen == 0) return NDL_OK;
  if (!mask || !depth || !parents || !cu_seqlens || (uintptr_t)mask & 7u)
    return NDL_ERR_INVALID_ARG;
  if (num_seqs > 65535) return NDL_ERR_UNSUPPORTED;
  const unsigned per = (unsigned)(((int64_t)max_seqlen + 255) / 256);
  if (!grid_fits(per, 256)) return NDL_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(tree_mask_kernel, dim3(per, (unsigned)num_seqs), dim3(256), 0,
                     (hipStream_t)stream, (uint64_t*)mask, mask_stride, mask_words, depth, parents,
                     cu_seqlens, num_tokens);
  return check_launch();
}
