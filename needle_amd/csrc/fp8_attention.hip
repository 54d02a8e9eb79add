// Attention of a chunk of new tokens per sequence over the 8-bit paged pool (kv_fp8.hip): one
// token (a decode step), a few (drafts to verify) or many (a prompt continued after a cached
// prefix), gfx950.
//
//   out[j][h] = sum_t softmax_t(scale * q[j][h] . k[t][h / g]) v[t][h / g],
//   t < min(ctx + j + 1, W * block_size),  k[t] = code * 2^(byte - 127), v likewise.
//
// The reference has no 8-bit pool; the meaning of the arguments is its _decode / _prefill's
// (needle/layers/attention.py:120-134, :291-310), with a cached prefix attended.
//
// Bound: the codes, each read once (2 (D + 1) bytes per token and kv head).
//   * Rows.  The g query heads of a kv head times the chunk's tokens are the N columns of
//     16x16x32 MFMA tiles whose M rows are tokens (S^T = K Q^T) or head_dim (O^T = V^T P^T):
//     up to 32 columns (NT tiles of 16) are a row block, longer chunks have several (64 columns
//     took more registers than there are).
//   * Codes to registers.  A wave takes 32 tokens at a time.  Their codes go straight to its own
//     LDS ring (1 KiB of contiguous bytes per load), two stages deep: a stage is refilled as soon
//     as its operands are in registers, so two tiles are in flight while a third computes, and
//     no barrier is needed before the waves' results are combined.
//   * Exact values.  e4m3 codes convert exactly to bf16 and fp16 (v_cvt_scalef32_pk_*_fp8), so
//     the products are the 16-bit kernels' (fp32 sums).  K's scale multiplies the scores, where
//     one factor is due anyway; V's is applied by the conversion, which is exact too but for fp16's
//     subnormals (its other end, 65,536, is worked round).
//   * P^T needs no data movement: with token slot 8 j + i of the PV product standing for token
//     4 j + i (i < 4) or 12 + 4 j + i, the accumulator layout of S^T is the operand's.
//   * Softmax in fp32 with exp2, scale * log2(e) folded.  The running maximum is raised (and the
//     sums rescaled) only when a tile exceeds it by 8, so probabilities stay below 256; a tile's
//     maximum is taken across lanes only then.
//     P is rounded to the 16-bit format for the matrix cores; its sum is taken before that.
//   * Long chunks (kUnpackRows columns, kUnpackScores scores) are bound by the products, not by the
//     codes: their keys are unpacked once into a 16-bit pool in the workspace and attended by
//     varlen_prefill.hip's kernels (see launch_unpacked).
//   * Split.  Either a workgroup per (kv head, row block), or, where those would leave the GPU
//     idle or unevenly loaded, all row blocks' tiles of a kv head laid end to end and cut into
//     equal shares, one per resident workgroup; what a share holds of a row block goes to a
//     workspace and is merged by a second launch.
// Measured (us, bytes read at): 64 sequences of 512 to 4,096 tokens, 32/8 heads of 128, one token
// each 47 + 4.8 of merge, 5.6 TB/s in the first launch; 24 sequences of 4,096 to 32,768, 28/4
// heads, float16, 72 + 6.9, 6.0 TB/s; 1 to 8 tokens each after 512 to 4,096 55 + 7.9, 4.9 TB/s.
// A few short sequences take 5 us, of which each step of a wave (a tile) is 1: about 270
// instructions, two waves to a SIMD; sixteen waves or deeper rings measured the same or slower.
#include "fp8.hpp"

#include "chunk_shares.hpp"

namespace ndl {
namespace {

constexpr int kTile = 32;       // tokens per wave step
constexpr float kRaise = 8.f;   // log2 of the largest probability before the maximum is raised

struct ChunkArgs {
  u16* out;
  const u16* q;
  int64_t q_stride;
  uint8_t* codes;               // written only with new rows
  uint8_t* scales;
  int64_t plane_rows;           // rows (token, head) of a plane
  int64_t num_blocks;
  int num_heads, num_kv_heads, group;
  const u16* new_k;             // rows to append, of one token per sequence (null: none)
  const u16* new_v;
  int64_t k_stride, v_stride;
  const u16* cos;               // with new rows: q and k are not rotated yet (null: they are)
  const u16* sin;
  int64_t cs_stride;
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

// A row block: tokens tok0 .. tok0 + n of the packed rows, the first at position pos.
struct Item {
  int64_t tok0;
  int n;
  int seq;
  int64_t pos;
  int64_t cap;                  // keys a table row holds
  __device__ __forceinline__ int64_t keys() const {     // of its last token
    const int64_t k = pos + n;
    return n <= 0 || pos < 0 ? 0 : k < cap ? k : cap;
  }
  __device__ __forceinline__ int tiles() const { return (int)((keys() + kTile - 1) / kTile); }
};

// The sequence of row block e (32-bit: a 64-bit division takes a hundred instructions).
__device__ __forceinline__ int seq_of_item(const ChunkArgs& a, int e) {
  return a.blocks_per_seq == 1 ? e : (int)((uint32_t)e / (uint32_t)a.blocks_per_seq);
}
__device__ __forceinline__ Item item_of(const ChunkArgs& a, int e) {
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
  const int64_t ctx = a.context_lens[it.seq];
  it.pos = ctx < 0 ? -1 : ctx + j0;      // a negative context: nothing is attended
  it.cap = (int64_t)a.max_blocks << (4 + a.tile_shift);
  return it;
}

__device__ __forceinline__ int slots_of(const ChunkArgs& a, int e) {
  if (e >= a.items) return 0;
  const int n = item_of(a, e).tiles();
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
struct Stream {
  int total;
  Cut cut;
  int v[kSteps], incl[kSteps];

  __device__ __forceinline__ void read(const ChunkArgs& a, int lane) {
    total = 0;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) v[k] = 64 * k < a.items ? slots_of(a, 64 * k + lane) : 0;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      incl[k] = total;
      if (64 * k < a.items) {
        incl[k] = wave_scan(v[k], lane) + total;
        total = __builtin_amdgcn_readlane(incl[k], 63);
      }
    }
    for (int base = kHeld; base < a.items; base += 64)
      total += __builtin_amdgcn_readlane(wave_scan(slots_of(a, base + lane), lane), 63);
    cut = cut_of(total, a.shares, a.min_chunk, a.pad);
  }
  // The row block that holds slot `at` (at < total), or row block `e` if that is not negative.
  __device__ __forceinline__ Place find(const ChunkArgs& a, int lane, int at, int e) const {
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
      const int w = slots_of(a, base + lane), in = wave_scan(w, lane) + carry;
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
  __device__ __forceinline__ int begin(const ChunkArgs& a, int lane, int s) const {
    const int x = s * cut.chunk;   // fits 31 bits: make_plan
    if (x >= total) return total;
    const Place p = find(a, lane, x, -1);
    return share_begin(x, p.first, p.slots, cut.snap);
  }
};

// Waits until at most n (0 .. MAX) groups of I loads are in flight.
template <int I, int MAX>
__device__ __forceinline__ void vm_wait_groups(int n) {
  if constexpr (MAX == 0) {
    vm_wait<0>();
  } else {
    if (n >= MAX)
      vm_wait<MAX * I>();
    else
      vm_wait_groups<I, MAX - 1>(n);
  }
}

// The power of two that byte r of w stands for: one instruction, where shifting and masking are
// two.
__device__ __forceinline__ float scale_of(uint32_t w, int r) {
  uint32_t x;
  if (r == 0)
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD "
        "src1_sel:BYTE_0" : "=v"(x) : "v"(23), "v"(w));
  else if (r == 1)
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD "
        "src1_sel:BYTE_1" : "=v"(x) : "v"(23), "v"(w));
  else if (r == 2)
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD "
        "src1_sel:BYTE_2" : "=v"(x) : "v"(23), "v"(w));
  else
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD "
        "src1_sel:BYTE_3" : "=v"(x) : "v"(23), "v"(w));
  return __uint_as_float(x);
}
// fmaxf of three without the compiler's quieting of each (no score is a signalling NaN).
__device__ __forceinline__ float max3(float x, float y, float z) {
  float m;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(x), "v"(y), "v"(z));
  return m;
}

// Two outputs in the 16-bit format.  In float16 those past it are its largest: they are sums of
// values of 65,536 that were 65,504 or less before they were codes.
template <bool F16>
__device__ __forceinline__ uint32_t pack_out(float x, float y) {
  if constexpr (F16) {
    x = x > 65504.f ? 65504.f : x < -65504.f ? -65504.f : x;     // (a NaN stays)
    y = y > 65504.f ? 65504.f : y < -65504.f ? -65504.f : y;
  }
  return Elt<F16>::pack(x, y);
}

// 0xff in every byte of w that is a NaN code (0x7f or 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t top = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  return (top >> 7) * 0xffu;
}

// NT: 16-column tiles of a row block; NW: waves of a workgroup, which take its tiles in turn.
template <int D, int NT, int NW>
struct Shape {
  static constexpr int kRowTile = kTile * D;                 // bytes of a tile's K (or V)
  static constexpr int kStage = 2 * kRowTile + 256;          // K, V, scales
  static constexpr int kDepth = 2;
  static constexpr int kRing = kDepth * kStage;
  static constexpr int kLoads = 2 * (kRowTile / 1024) + 1;   // per stage
  static constexpr int kSums = NW * NT * 16 * D * 4;         // bytes of the waves' partial outputs
  static constexpr int kMl = 2 * NW * NT * 16 * 4;
  static constexpr int kLds = (NW * kRing > kSums ? NW * kRing : kSums) + kMl;
};

// 8 elements of x rotated with the other half's, by rope8's roundings: x cos + turned sin.
template <bool F16>
__device__ __forceinline__ u32x4 rope_half(const u32x4& x, const u32x4& turned, const u32x4& c,
                                           const u32x4& s) {
#pragma clang fp contract(off)
  using T = Elt<F16>;
  u32x4 out;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t xc = T::pack(T::lo(x[w]) * T::lo(c[w]), T::hi(x[w]) * T::hi(c[w]));
    const uint32_t ts = T::pack(T::lo(turned[w]) * T::lo(s[w]), T::hi(turned[w]) * T::hi(s[w]));
    out[w] = T::pack(T::lo(xc) + T::lo(ts), T::hi(xc) + T::hi(ts));
  }
  return out;
}

// A decode step's new row as the projections left it, and its cos and sin: the four rows go
// straight to 1 KiB of LDS of the wave's own before the lengths arrive, and are used while the
// ring's first loads are under way, so that they take no registers in between.
template <int D, bool F16>
struct NewRow {
  static constexpr int kBytes = 1024, kRow = 2 * D;     // k, v, cos, sin
  static constexpr int CPH = D / 16;
  const unsigned char* at;
  __device__ __forceinline__ void load(const ChunkArgs& a, int64_t tok, int head, int lane,
                                       uint32_t lds) const {
    const int row = (lane / (D / 8)) & 3;      // (head_dim 64: all of it twice)
    const u16* src = (row == 1 ? a.new_v + tok * a.v_stride : a.new_k + tok * a.k_stride) +
                     (int64_t)head * D;
    if (row >= 2 && a.cos != nullptr) src = (row == 2 ? a.cos : a.sin) + tok * a.cs_stride;
    lds_dma16_each(src + 8 * (lane % (D / 8)), lds);
  }
  __device__ __forceinline__ u32x4 part(int row, int d) const {
    return *reinterpret_cast<const u32x4*>(at + row * kRow + 2 * d);
  }
  // q in the operand layout of chunk_attention_kernel: lane (j, c) holds head_dim 64 (i >> 1) +
  // 16 j + 8 (i & 1) .. + 7 in q[i].
  template <class X8>
  __device__ __forceinline__ void rotate(X8* q, int j) const {
    constexpr int KS = D / 32;
    u32x4 x[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) x[i] = __builtin_bit_cast(u32x4, q[i]);
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      // the other half is in q[i ^ 2], or, at head_dim 64, 32 lanes away; the first half takes it
      // negated
      const bool second = D == 128 ? i >= 2 : j >= 2;
      u32x4 turned;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t o =
            D == 128 ? x[i ^ (KS / 2)][w] : (uint32_t)__shfl_xor((int)x[i][w], 32, 64);
        turned[w] = second ? o : o ^ 0x80008000u;
      }
      const int d = 64 * (i >> 1) + 16 * j + 8 * (i & 1);
      q[i] = __builtin_bit_cast(X8, rope_half<F16>(x[i], turned, part(2, d), part(3, d)));
    }
  }
  // 8 codes of each half of k, or, in the odd groups of D / 16 lanes, of v; and the scale.
  __device__ __forceinline__ int quantise(bool rope, int lane, u32x2* codes_lo,
                                          u32x2* codes_hi) const {
    const int d0 = 8 * (lane % CPH), v = (lane / CPH) & 1;
    u32x4 lo = part(v, d0), hi = part(v, d0 + D / 2);
    if (rope) {
      u32x4 rlo, rhi;
      rope8<F16>(lo, hi, part(2, d0), part(2, d0 + D / 2), part(3, d0), part(3, d0 + D / 2), rlo,
                 rhi);
      lo = v ? lo : rlo;
      hi = v ? hi : rhi;
    }
    const int byte = scale_byte<CPH, F16>(lo, hi);
    const float mul = __uint_as_float((uint32_t)(254 - byte) << 23);
    *codes_lo = quant8<F16>(lo, mul);
    *codes_hi = quant8<F16>(hi, mul);
    return byte;
  }
};

// A workgroup's share of the row blocks of one kv head.  NEW: the sequence's new row is quantised
// by the wave whose tile holds its position, which puts it into the ring for itself and into the
// pool.  (head_dim 64: 128 registers, as without, so that as many workgroups are resident.)
template <int D, bool F16, int NT, int NW, bool NEW = false>
__global__ __launch_bounds__(64 * NW, NEW && D == 64 ? 4 : 8 / NW)
void chunk_attention_kernel(ChunkArgs a) {
  using T = Elt<F16>;
  using X8 = typename T::x8;
  using S = Shape<D, NT, NW>;
  constexpr int KS = D / 32;      // k steps of the QK product
  constexpr int DB = D / 16;      // 16-row tiles of O^T; head_dim index DB * m + b in tile b
  constexpr int VW = DB / 4;      // words of codes a lane holds of one V row
  using Row = NewRow<D, F16>;
  constexpr int kRows = NEW ? NW * Row::kBytes : 0;
  __shared__ __attribute__((aligned(16))) unsigned char smem[S::kLds + kRows];
  float* const ml = reinterpret_cast<float*>(smem + S::kLds - S::kMl);   // [2][wave][column]

  const int lane = threadIdx.x & 63, j = lane >> 4, c = lane & 15;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  unsigned char* const ring = smem + wv * S::kRing;
  const uint32_t ring_lds = lds_addr(ring);
  unsigned char* const fresh_lds = smem + S::kLds + wv * Row::kBytes;
  const Row fresh{fresh_lds};

  // The kv heads of one share (or row block) run on one XCD at about the same time: workgroups
  // are dealt to the XCDs in turn, and heads share the lines of scales, tables and lengths.
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
    Stream st;
    st.read(a, lane);
    from = st.begin(a, lane, unit);
    to = st.begin(a, lane, unit + 1);
    if (from >= to) return;
    const Place p = st.find(a, lane, from, -1);
    e = p.e;
    first = p.first;
  }

  const uint32_t swz = (uint32_t)((lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4));
  const int bshift = 4 + a.tile_shift;
  const uint32_t tmask = (1u << a.tile_shift) - 1;

  for (; e < a.items; ++e) {
    // This wave's tiles: t0 + wv, t0 + wv + NW, ..  Lane 2 u + s of a window holds the block id of
    // 16-token half s of the window's tile u (32 of the wave's tiles).
    const int32_t* const table = a.block_table + (int64_t)seq_of_item(a, e) * a.bt_row_stride;
    int t0 = 0, window;
    auto load_window = [&](int u0) {
      const int tt = 2 * (t0 + wv + NW * (u0 + (lane >> 1))) + (lane & 1);
      int col = tt >> a.tile_shift;
      if (col > a.max_blocks - 1) col = a.max_blocks - 1;
      window = table[col];
    };
    if constexpr (NEW) fresh.load(a, seq_of_item(a, e), head, lane, lds_addr(fresh_lds));
    if (whole) load_window(0);        // before the lengths arrive
    const Item it = item_of(a, e);
    const int ntiles = it.tiles();
    int t1 = ntiles;
    if (!whole) {
      if (ntiles == 0) continue;
      if (first >= to) break;
      share_tiles(first, a.pad, ntiles, from, to, &t0, &t1);
      first += a.pad + ntiles;
      if (t0 >= t1) continue;     // only the empty slot is this share's
      load_window(0);
    } else if (it.n <= 0) {
      break;
    }
    const int cols = it.n * a.group;

    // Columns: 16 nt + c is query token col / g, head head * g + col % g.
    X8 q[NT][KS];
    int lim[NT];                  // keys the column attends
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      int col = 16 * nt + c;
      if (col >= cols) col = cols - 1;      // computed like the last column, not stored
      const int tok = col / a.group;
      const u16* src = a.q + (it.tok0 + tok) * a.q_stride +
                       (int64_t)(head * a.group + col - tok * a.group) * D;
#pragma unroll
      for (int s = 0; s < KS; ++s)
        q[nt][s] = __builtin_bit_cast(X8, ld16(src + 64 * (s >> 1) + 16 * j + 8 * (s & 1)));
      const int64_t k = it.pos + tok + 1;
      lim[nt] = (int)(k < it.cap ? k : it.cap);
    }
    // the new row's position in the table (past the end the last column is written again, as an
    // append does) and the step of this wave that attends it
    int at_new = -1, u_new = -1;
    if constexpr (NEW) {
      if (it.pos >= 0)
        at_new = (int)(it.pos < it.cap ? it.pos
                                       : it.cap - (1 << bshift) + (it.pos & ((1 << bshift) - 1)));
      at_new = __builtin_amdgcn_readfirstlane(at_new);
      const int tile = at_new >> 5;
      if (at_new >= 0 && tile >= t0 && tile < t1 && (tile - t0) % NW == wv)
        u_new = (tile - t0) / NW;
    }
    const int64_t k_first = it.pos + 1 < it.cap ? it.pos + 1 : it.cap;
    const int all_keys = (int)it.keys();      // of the last token
    const int min_keys = k_first < 0 ? 0 : (int)k_first;   // of the first

    f32x4 acc[NT][DB];
    float m[NT], l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt] = kNegInf;
      l[nt] = 0.f;
#pragma unroll
      for (int b = 0; b < DB; ++b) acc[nt][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const int cnt = t1 - t0 > wv ? (t1 - t0 - wv + NW - 1) / NW : 0;
    uint32_t bad_bits = 0;        // two bits per stage: its halves with an invalid block id
    auto issue = [&](int u, int slot) {
      if (u > 0 && (u & 31) == 0) {
        load_window(u);
        asm volatile("" : "+v"(window));
      }
      const uint32_t st = ring_lds + slot * S::kStage;
      const int tile = t0 + wv + NW * u;
      uint32_t srow[2];
      uint32_t bad = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        int b = __builtin_amdgcn_readlane(window, 2 * (u & 31) + s);
        if (b < 0 || b >= a.num_blocks) {
          b = 0;
          bad |= 1u << s;
        }
        const int64_t row = (((int64_t)b * Hkv + head) << bshift) +
                            (((uint32_t)(2 * tile + s) & tmask) << 4);
        srow[s] = (uint32_t)row;
        const uint8_t* kb = a.codes + row * D;
        const uint8_t* vb = kb + a.plane_rows * D;
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
          lds_dma16_nt(kb + 1024 * x, swz, st + s * 16 * D + 1024 * x);
          lds_dma16_nt(vb + 1024 * x, (uint32_t)lane * 16,
                       st + S::kRowTile + s * 16 * D + 1024 * x);
        }
      }
      // scales: 4-byte word w of half s of plane p lands at word 8 p + 4 s + w
      const uint32_t off = (lane & 8 ? (uint32_t)a.plane_rows : 0u) +
                           (lane & 4 ? srow[1] : srow[0]) + 4u * (lane & 3);
      lds_dma4(a.scales, off, st + 2 * S::kRowTile);
      bad_bits = (bad_bits & ~(3u << (2 * slot))) | (bad << (2 * slot));
    };
    // What was loaded so far arrives here, q with the ring's first stages.  Left to the compiler its
    // waits would be where the values are used, in the loop, and drain the ring, whose loads it does
    // not see, at every step.
    auto arrive = [&]() {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < KS; ++x) asm volatile("" : "+v"(q[nt][x]));
    };
    asm volatile("" : "+v"(window));
    if constexpr (NEW) arrive();     // rotated while those are under way
#pragma unroll
    for (int d = 0; d < S::kDepth; ++d)
      if (d < cnt) issue(d, d);
    if constexpr (!NEW) arrive();

    constexpr int CPH = D / 16;
    u32x2 xlo, xhi;
    int xbyte = 0;
    if constexpr (NEW) {
      vm_wait_groups<S::kLoads, S::kDepth>(cnt);      // the rows are there, the ring need not be
      asm volatile("" ::: "memory");
      if (a.cos != nullptr) fresh.rotate(q[0], j);
      if (u_new >= 0) xbyte = fresh.quantise(a.cos != nullptr, lane, &xlo, &xhi);
    }

    int slot = 0;
    for (int u = 0; u < cnt; ++u) {
      vm_wait_groups<S::kLoads, S::kDepth - 1>(cnt - 1 - u);
      asm volatile("" ::: "memory");
      unsigned char* const st = ring + slot * S::kStage;
      if constexpr (NEW) {
        if (u == u_new) {       // (LDS accesses of a wave are in order: the reads below see it)
          int ln = lane;        // addresses worked out here: they would hold registers all along
          asm volatile("" : "+v"(ln));
          if (ln < 2 * CPH) {
            const int d0 = 8 * (ln % CPH), r = at_new & 15, half = (at_new >> 4) & 1;
            const bool v = ln >= CPH;
            auto place = [&](int d) {
              if (v) return S::kRowTile + (16 * half + r) * D + d;
              const int row = D == 128 ? r : r >> 1;
              const int chunk = D == 128 ? d >> 4 : (r & 1) * 4 + (d >> 4);
              return half * 16 * D + row * 128 + ((chunk ^ (row & 7)) << 4) + (d & 15);
            };
            *reinterpret_cast<u32x2*>(st + place(d0)) = xlo;
            *reinterpret_cast<u32x2*>(st + place(d0 + D / 2)) = xhi;
            if (d0 == 0) st[2 * S::kRowTile + (v ? 32 : 0) + 16 * half + r] = (uint8_t)xbyte;
            const int b = table[at_new >> bshift];
            if (b >= 0 && b < a.num_blocks) {
              const int64_t row = (v ? a.plane_rows : 0) + (((int64_t)b * Hkv + head) << bshift) +
                                  (at_new & ((1 << bshift) - 1));
              *reinterpret_cast<u32x2*>(a.codes + row * D + d0) = xlo;
              *reinterpret_cast<u32x2*>(a.codes + row * D + d0 + D / 2) = xhi;
              if (d0 == 0) a.scales[row] = (uint8_t)xbyte;
            }
          }
          asm volatile("" ::: "memory");
        }
      }
      // operands: K half s, 16 codes at head_dim 64 h + 16 j of row c; V rows of slots 8 j + i
      u32x4 kc[2][D / 64];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          const int o = D == 128 ? c * 128 + (((4 * h + j) ^ (c & 7)) << 4)
                                 : (c >> 1) * 128 + ((((c & 1) * 4 + j) ^ (c >> 1)) << 4);
          kc[s][h] = *reinterpret_cast<const u32x4*>(st + s * 16 * D + o);
        }
      uint32_t vc[8][VW];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = (i >> 2) * 16 + 4 * j + (i & 3);
        const unsigned char* p = st + S::kRowTile + row * D + DB * c;
        if constexpr (VW == 2) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(p);
          vc[i][0] = x[0];
          vc[i][1] = x[1];
        } else {
          vc[i][0] = *reinterpret_cast<const uint32_t*>(p);
        }
      }
      uint32_t sk[2], sv[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        sk[s] = *reinterpret_cast<const uint32_t*>(st + 2 * S::kRowTile + 16 * s + 4 * j);
        sv[s] = *reinterpret_cast<const uint32_t*>(st + 2 * S::kRowTile + 32 + 16 * s + 4 * j);
      }
      const uint32_t bad = (bad_bits >> (2 * slot)) & 3u;
      // in registers before the stage's next loads go out
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (u + S::kDepth < cnt) issue(u + S::kDepth, slot);
      slot = slot + 1 == S::kDepth ? 0 : slot + 1;

      // S^T: lane (j, c) holds tokens 16 s + 4 j + r of column c
      f32x4 sc[2][NT];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[s][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const u32x4 kw{value2<F16, false>(kc[s][h][2 * x], 1.f),
                           value2<F16, true>(kc[s][h][2 * x], 1.f),
                           value2<F16, false>(kc[s][h][2 * x + 1], 1.f),
                           value2<F16, true>(kc[s][h][2 * x + 1], 1.f)};
            const X8 k8 = __builtin_bit_cast(X8, kw);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              sc[s][nt] = T::mfma16x16x32(k8, q[nt][2 * h + x], sc[s][nt]);
          }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float ks = scale_of(sk[s], r) * a.scale_log2;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sc[s][nt][r] *= ks;
        }

      const int tile = t0 + wv + NW * u;
      const bool masked = bad != 0 || kTile * (tile + 1) > min_keys;
      uint32_t nan_any = 0;
      if (masked) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int at = kTile * tile + 16 * s + 4 * j;     // the lane's first token
          const bool off = (bad >> s) & 1;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int left = off ? 0 : lim[nt] - at;
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[s][nt][r] = r < left ? sc[s][nt][r] : kNegInf;
          }
          // what no column attends may hold anything, a NaN included: 0 * NaN must not happen,
          // nor 0 times the scale of 255, which is one too
          const int left = off ? 0 : all_keys - at;
          sv[s] &= left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int w = 0; w < VW; ++w) {
              vc[4 * s + r][w] = r < left ? vc[4 * s + r][w] : 0u;
              nan_any |= nan_bytes(vc[4 * s + r][w]);
            }
        }
      }

      X8 p[NT];
      bool raise = false;
      float mt[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mt[nt] = max3(max3(sc[0][nt][0], sc[0][nt][1], sc[0][nt][2]),
                      max3(sc[0][nt][3], sc[1][nt][0], sc[1][nt][1]),
                      max3(sc[1][nt][2], sc[1][nt][3], sc[1][nt][3]));
        raise |= mt[nt] > m[nt] + kRaise;
      }
      if (__builtin_amdgcn_ballot_w64(raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float nm = fmaxf(m[nt], max_xor32(max_xor16(mt[nt])));
          const float f = m[nt] == nm ? 1.f : fast_exp2(m[nt] - nm);
          m[nt] = nm;
          l[nt] *= f;
#pragma unroll
          for (int b = 0; b < DB; ++b) acc[nt][b] *= f;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float base = m[nt] == kNegInf ? 0.f : m[nt];    // nothing attended yet
        float e8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e8[i] = fast_exp2(sc[i >> 2][nt][i & 3] - base);
        l[nt] += ((e8[0] + e8[1]) + (e8[2] + e8[3])) + ((e8[4] + e8[5]) + (e8[6] + e8[7]));
        const u32x4 w{T::pack(e8[0], e8[1]), T::pack(e8[2], e8[3]), T::pack(e8[4], e8[5]),
                      T::pack(e8[6], e8[7])};
        p[nt] = __builtin_bit_cast(X8, w);
      }

      // A NaN in a value that some of the chunk's tokens attend and others do not: it is taken
      // out of the product and put into the columns that attend it.
      if (masked && a.toks > 1 && __builtin_amdgcn_ballot_w64(nan_any != 0)) {
        constexpr uint32_t one = F16 ? 0x3c00u : 0x3f80u;
        X8 seen[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int s = i >> 1, at = kTile * tile + 16 * s + 4 * j + 2 * (i & 1);
            const int left = (bad >> s) & 1 ? 0 : lim[nt] - at;
            w[i] = (left > 0 ? one : 0u) | (left > 1 ? one << 16 : 0u);
          }
          seen[nt] = __builtin_bit_cast(X8, w);
        }
#pragma unroll
        for (int b = 0; b < DB; ++b) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = (nan_bytes(vc[2 * i][b >> 2]) >> (8 * (b & 3))) & 0xffu;
            const uint32_t y = (nan_bytes(vc[2 * i + 1][b >> 2]) >> (8 * (b & 3))) & 0xffu;
            w[i] = (x ? one : 0u) | (y ? one << 16 : 0u);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const f32x4 hits = T::mfma16x16x32(__builtin_bit_cast(X8, w), seen[nt],
                                               f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (hits[r] > 0.f) acc[nt][b][r] = __uint_as_float(0x7fc00000u);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int w = 0; w < VW; ++w) vc[i][w] &= ~nan_bytes(vc[i][w]);
      }

      // A float16 row's values from 63,488 on are 256 * 2^8 as codes, 65,536, which float16 has not:
      // such a row is converted under 2^7 and its probabilities (256 at most) doubled, both exact.
      // Few rows reach 448 (a byte of 128): one test a step for all of them (us without / with, 24
      // sequences of 4,096 to 32,768, 28/4 heads 82.4 / 83.2; 64 of 2,048 to 4,096 with 5 drafts 85.1 /
      // 85.7).
      if constexpr (F16) {
        if (__builtin_amdgcn_ballot_w64(((sv[0] | sv[1]) & 0x80808080u) != 0)) {
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t big = ((sv[i >> 2] >> (8 * (i & 3))) & 0xffu) == 135u;
            sv[i >> 2] -= big << (8 * (i & 3));
            f[i] = big ? 2.f : 1.f;
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            u32x4 w = __builtin_bit_cast(u32x4, p[nt]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = T::pack(T::lo(w[i]) * f[2 * i], T::hi(w[i]) * f[2 * i + 1]);
            p[nt] = __builtin_bit_cast(X8, w);
          }
        }
      }

      // O^T += V^T P^T: a pair of head_dim tiles at a time, the rows' pairs of codes turned into
      // pairs of tokens
      asm volatile("" : "+v"(sv[0]), "+v"(sv[1]));     // the scales no sooner than they are used
      float vs[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) vs[i] = scale_of(sv[i >> 2], i & 3);
#pragma unroll
      for (int b2 = 0; b2 < DB / 2; ++b2) {
        uint32_t v2[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v2[i] = b2 & 1 ? value2<F16, true>(vc[i][b2 >> 1], vs[i])
                         : value2<F16, false>(vc[i][b2 >> 1], vs[i]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = pack_halves(v2[2 * i], v2[2 * i + 1], x == 1);
          const X8 v8 = __builtin_bit_cast(X8, w);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            acc[nt][2 * b2 + x] = T::mfma16x16x32(v8, p[nt], acc[nt][2 * b2 + x]);
        }
      }
    }

    // The waves' results: (m, l) first, then the outputs scaled to the common maximum, laid out
    // so that one wave's lanes hold head_dim DB (4 j + r) .. of column tile nt's columns.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      l[nt] = add_xor32(add_xor16(l[nt]));
      if (j == 0) {
        ml[wv * 16 * NT + 16 * nt + c] = m[nt];
        ml[(NW + wv) * 16 * NT + 16 * nt + c] = l[nt];
      }
    }
    __syncthreads();
    float* const sums = reinterpret_cast<float*>(smem);   // [wave][nt][r][lane][DB]
    float mm[NT], ll[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = 16 * nt + c;
      mm[nt] = ml[col];
#pragma unroll
      for (int w = 1; w < NW; ++w) mm[nt] = fmaxf(mm[nt], ml[w * 16 * NT + col]);
      ll[nt] = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float mw = ml[w * 16 * NT + col];
        ll[nt] += ml[(NW + w) * 16 * NT + col] * (mw == mm[nt] ? 1.f : fast_exp2(mw - mm[nt]));
      }
      const float f = m[nt] == mm[nt] ? 1.f : fast_exp2(m[nt] - mm[nt]);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int b = 0; b < DB; b += 4)
          *reinterpret_cast<f32x4*>(sums + (((wv * NT + nt) * 4 + r) * 64 + lane) * DB + b) =
              f32x4{acc[nt][b][r] * f, acc[nt][b + 1][r] * f, acc[nt][b + 2][r] * f,
                    acc[nt][b + 3][r] * f};
    }
    __syncthreads();
    const bool part = !whole && (t0 > 0 || t1 < ntiles);
    const int64_t seg = ((int64_t)head * a.nseg + unit + e) * (a.toks * a.group);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if ((nt * 4 + r) % NW != wv) continue;
        const int col = 16 * nt + c;
        float o[DB];
#pragma unroll
        for (int b = 0; b < DB; ++b) o[b] = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int b = 0; b < DB; ++b) o[b] += sums[(((w * NT + nt) * 4 + r) * 64 + lane) * DB + b];
        if (col >= cols) continue;
        const int d0 = DB * (4 * j + r);
        if (part) {
          float* const dst = a.ws_acc + (seg + col) * D + d0;
#pragma unroll
          for (int b = 0; b < DB; b += 4)
            *reinterpret_cast<f32x4*>(dst + b) = f32x4{o[b], o[b + 1], o[b + 2], o[b + 3]};
          if (d0 == 0) *reinterpret_cast<f32x2*>(a.ws_ml + (seg + col) * 2) = f32x2{mm[nt], ll[nt]};
        } else {
          const float inv = ll[nt] == 0.f ? 0.f : 1.f / ll[nt];   // nothing attended: zeros
          const int tok = col / a.group;
          u16* const dst = a.out + ((it.tok0 + tok) * a.num_heads + head * a.group + col -
                                    tok * a.group) * (int64_t)D + d0;
          uint32_t w[DB / 2];
#pragma unroll
          for (int b = 0; b < DB / 2; ++b) w[b] = pack_out<F16>(o[2 * b] * inv, o[2 * b + 1] * inv);
          if constexpr (DB == 8)
            st16(dst, u32x4{w[0], w[1], w[2], w[3]});
          else
            *reinterpret_cast<u32x2*>(dst) = u32x2{w[0], w[1]};
        }
      }
    }
    if (whole) return;
    __syncthreads();     // before the ring is written again
  }
  if constexpr (NEW) vm_wait<0>();     // rows of a row block that is not this share's
}

// One workgroup per (row block, kv head, kMergeCols columns): the parts that the shares hold,
// combined in their order; zeros for tokens with nothing to attend.  A row block inside one share
// was written by the attention.
constexpr int kMergeCols = 8;
constexpr int kMergeParts = 64;   // at a time

template <int D, bool F16>
__global__ __launch_bounds__(256) void chunk_merge_kernel(ChunkArgs a) {
  constexpr int PER = kMergeCols * D / 256;       // consecutive outputs of a thread: 4 or 2
  __shared__ float2 part[kMergeParts][kMergeCols];
  const int t = threadIdx.x, lane = t & 63;
  const int e = blockIdx.x, head = blockIdx.y, c0 = blockIdx.z * kMergeCols;
  const Item it = item_of(a, e);
  Stream st;
  st.read(a, lane);
  const Place p = st.find(a, lane, 0, e);
  if (it.n <= 0 || c0 >= it.n * a.group) return;
  const int cols = it.n * a.group - c0 < kMergeCols ? it.n * a.group - c0 : kMergeCols;
  const int c = t * PER / D, d0 = t * PER - c * D;
  float o[PER];
#pragma unroll
  for (int x = 0; x < PER; ++x) o[x] = 0.f;
  // its slots by the scan that gave its place and the cut: whatever the lengths are, or become while
  // this runs, share_parts names shares that there are, whose parts the workspace holds
  if (p.slots > 0) {
    int s0, s1;
    if (!share_parts(p.first, p.slots, st.cut, &s0, &s1)) return;   // written by the attention
    const int n = s1 - s0 + 1, per = a.toks * a.group;
    const int64_t seg = ((int64_t)head * a.nseg + s0 + e) * per + c0;
    const float2* const ml = reinterpret_cast<const float2*>(a.ws_ml) + seg;
    const float* const src = a.ws_acc + seg * D + (int64_t)(c < cols ? c : 0) * D + d0;
    // this thread's column's maximum over all parts, then 64 parts at a time
    const int64_t step = (int64_t)per * D;
    float mx = kNegInf, l = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      for (int i0 = 0; i0 < n; i0 += kMergeParts) {
        const int m = n - i0 < kMergeParts ? n - i0 : kMergeParts;
        if (pass == 0 || n > kMergeParts) {
          __syncthreads();
          for (int i = t; i < m * kMergeCols; i += 256)
            if (i % kMergeCols < cols)
              part[i / kMergeCols][i % kMergeCols] =
                  ml[(int64_t)(i0 + i / kMergeCols) * per + i % kMergeCols];
          __syncthreads();
        }
        if (c >= cols) continue;
        if (pass == 0) {
          for (int i = 0; i < m; ++i) mx = fmaxf(mx, part[i][c].x);
          continue;
        }
        for (int i = 0; i < m; i += 8) {
          float v[8][PER];
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const float* const q = src + (int64_t)(i0 + (i + y < m ? i + y : i)) * step;
            if constexpr (PER == 4) {
              const f32x4 w = *reinterpret_cast<const f32x4*>(q);
#pragma unroll
              for (int x = 0; x < PER; ++x) v[y][x] = w[x];
            } else {
              const f32x2 w = *reinterpret_cast<const f32x2*>(q);
              v[y][0] = w[0];
              v[y][1] = w[1];
            }
          }
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            if (i + y >= m) break;
            const float2 ms = part[i + y][c];
            const float f = ms.x == mx ? 1.f : fast_exp2(ms.x - mx);
            l += ms.y * f;
#pragma unroll
            for (int x = 0; x < PER; ++x) o[x] += v[y][x] * f;
          }
        }
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int x = 0; x < PER; ++x) o[x] *= inv;
  }
  if (c >= cols) return;
  const int col = c0 + c, tok = col / a.group;
  u16* const dst = a.out + ((it.tok0 + tok) * a.num_heads + head * a.group + col - tok * a.group) *
                               (int64_t)D + d0;
  if constexpr (PER == 4)
    *reinterpret_cast<u32x2*>(dst) = u32x2{pack_out<F16>(o[0], o[1]), pack_out<F16>(o[2], o[3])};
  else
    *reinterpret_cast<uint32_t*>(dst) = pack_out<F16>(o[0], o[1]);
}

// ---------------------------------------------------------------- long chunks

struct UnpackArgs {
  u16* pool;                    // [2][num_seqs * cols][Hkv][bs][D]
  int32_t* table;               // [num_seqs][cols + 1], the last one invalid: keys past the
                                // bound, which the prefill's column clamp leads there
  int32_t* lens;                // [num_seqs]: context_lens, 0 for a negative one
  int cols;
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t plane_rows, pool_rows;   // rows of a plane of the codes and of the 16-bit pool
  int64_t num_blocks;
  int num_kv_heads, num_heads, group;
  const int32_t* block_table;
  int64_t bt_row_stride;
  int tile_shift;
  const int32_t* cu_seqlens;
  const int32_t* context_lens;
  int64_t num_tokens;
  u16* out;
};
struct Chunk {
  int64_t tok0, pos, keys;
  int n;
};
__device__ __forceinline__ Chunk chunk_of_seq(const UnpackArgs& a, int seq) {
  Chunk c;
  c.tok0 = a.cu_seqlens[seq];
  const int64_t n = a.cu_seqlens[seq + 1] - c.tok0;
  c.n = c.tok0 < 0 || n <= 0 || c.tok0 + n > a.num_tokens ? 0 : (int)n;
  c.pos = a.context_lens[seq];
  const int64_t cap = (int64_t)a.cols << (4 + a.tile_shift), k = c.pos + c.n;
  c.keys = c.n == 0 || c.pos < 0 ? 0 : k < cap ? k : cap;
  return c;
}

// The attended 16-token tiles of sequence blockIdx.y into its blocks of the 16-bit pool, a wave
// per (tile, plane, kv head), heads next to each other as they lie in a block.  A NaN among the
// chunk's own values becomes 0 here and reaches the tokens that attend it in chunk_nan_kernel:
// the causal mask's 0 * NaN would bring it to those before it too.
// In float16, which has no 65,536 (a row's values from 63,488 on), keys are halved, for which the
// scores' scale makes up, and a value is 65,504, the nearest there is.
template <int D, bool F16>
__global__ __launch_bounds__(256) void chunk_unpack_kernel(UnpackArgs a) {
  constexpr int LPR = D / 8, RPL = 64 / LPR;     // lanes per row (8 codes each), rows per load
  const int lane = threadIdx.x & 63, seq = blockIdx.y, Hkv = a.num_kv_heads;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const Chunk ch = chunk_of_seq(a, seq);
  const int bshift = 4 + a.tile_shift;
  const uint32_t tmask = (1u << a.tile_shift) - 1;
  // a negative context attends nothing: its blocks are all invalid
  const int64_t keys = ch.pos < 0 ? ch.n : ch.keys;
  const int64_t tiles = (keys + 15) >> 4, items = tiles * 2 * Hkv;
  int32_t* const row = a.table + (int64_t)seq * (a.cols + 1);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.lens[seq] = ch.pos < 0 ? 0 : (int32_t)ch.pos;
    row[a.cols] = -1;
  }
  const int r = lane / LPR;
  for (int64_t item = (int64_t)blockIdx.x * 4 + wv; item < items; item += (int64_t)gridDim.x * 4) {
    const int64_t tile = item / (2 * Hkv);
    const int ph = (int)(item - tile * 2 * Hkv), plane = ph >= Hkv, head = ph - plane * Hkv;
    const int col = (int)(tile >> a.tile_shift);
    if (col >= a.cols) break;
    const int b = a.block_table[(int64_t)seq * a.bt_row_stride + col];
    const bool ok = b >= 0 && b < a.num_blocks && ch.pos >= 0;
    const int64_t in_block = (int64_t)((uint32_t)tile & tmask) << 4;
    const int64_t block = (int64_t)seq * a.cols + col;
    if (ph == 0 && in_block == 0 && lane == 0) row[col] = ok ? (int)block : -1;
    if (!ok) continue;
    const int64_t from =
        (plane ? a.plane_rows : 0) + (((int64_t)b * Hkv + head) << bshift) + in_block;
    u16* const dst = a.pool + ((plane ? a.pool_rows : 0) + ((block * Hkv + head) << bshift) +
                               in_block) * D + lane * 8;
    u32x2 c[16 / RPL];
    float scale[16 / RPL];
#pragma unroll
    for (int x = 0; x < 16 / RPL; ++x) {
      c[x] = ld8(a.codes + from * D + x * 512 + lane * 8);
      scale[x] = __uint_as_float((uint32_t)a.scales[from + x * RPL + r] << 23);
    }
#pragma unroll
    for (int x = 0; x < 16 / RPL; ++x) {
      if (plane && 16 * tile + x * RPL + r >= ch.pos) {
        c[x][0] &= ~nan_bytes(c[x][0]);
        c[x][1] &= ~nan_bytes(c[x][1]);
      }
      if (F16 && !plane) scale[x] *= 0.5f;
      u32x4 out{value2<F16, false>(c[x][0], scale[x]), value2<F16, true>(c[x][0], scale[x]),
                value2<F16, false>(c[x][1], scale[x]), value2<F16, true>(c[x][1], scale[x])};
      if (F16 && plane && scale[x] >= 256.f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((out[i] & 0x7fffu) == 0x7c00u) out[i] -= 1u;
          if ((out[i] & 0x7fff0000u) == 0x7c000000u) out[i] -= 0x10000u;
        }
      }
      st16(dst + x * 512, out);
    }
  }
}

// A wave per (16 tokens of a chunk, kv head) of sequence blockIdx.y: where one of their values is
// a NaN code, the output of that head_dim index becomes NaN from its token on.
template <int D>
__global__ __launch_bounds__(256) void chunk_nan_kernel(UnpackArgs a) {
  constexpr int PER = D / 64;
  const int lane = threadIdx.x & 63, seq = blockIdx.y, Hkv = a.num_kv_heads;
  const int64_t w =
      (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int head = (int)(w % Hkv);
  const int64_t j0 = w / Hkv * 16;
  const Chunk ch = chunk_of_seq(a, seq);
  if (j0 >= ch.n) return;
  const int bshift = 4 + a.tile_shift;
  // a lane per token for its slot, then a row of codes at a time, none behind a branch
  int64_t mine = -1;
  if (lane < 16) {
    const int64_t p = ch.pos + j0 + lane;
    if (j0 + lane < ch.n && ch.pos >= 0 && p < ch.keys) {
      const int b = a.block_table[(int64_t)seq * a.bt_row_stride + (p >> bshift)];
      if (b >= 0 && b < a.num_blocks)
        mine = (((int64_t)b * Hkv + head) << bshift) + (p & ((1 << bshift) - 1));
    }
  }
  uint32_t code[16];
  bool in[16];
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    const int row = __builtin_amdgcn_readlane((int)mine, x);    // plane_rows fits 31 bits
    in[x] = row >= 0;
    const uint8_t* const p = a.codes + (a.plane_rows + (in[x] ? row : 0)) * D + lane * PER;
    if constexpr (PER == 2)
      code[x] = *reinterpret_cast<const uint16_t*>(p);
    else
      code[x] = *p;
  }
  int first[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    first[e] = 16;
#pragma unroll
    for (int x = 15; x >= 0; --x)
      if (in[x] && ((code[x] >> (8 * e)) & 0x7f) == 0x7f) first[e] = x;
  }
  bool any = false;
#pragma unroll
  for (int e = 0; e < PER; ++e) any |= first[e] < 16;
  if (!__builtin_amdgcn_ballot_w64(any)) return;
  for (int64_t j = j0; j < ch.n; ++j)
    for (int g = 0; g < a.group; ++g)
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (first[e] < 16 && j0 + first[e] <= j)   // bf16 and fp16: all bits but the sign
          a.out[((ch.tok0 + j) * a.num_heads + head * a.group + g) * (int64_t)D + lane * PER + e] =
              0x7fffu;
}

// Where unpacking first is the faster way: enough columns for a row's codes to be used often, and
// enough scores in all to pay for its launches (unpacking, the prefill with its merge, the scan).
// us, here / unpacked, chunks of c tokens after t: 28/4 heads of 128, 1 sequence, t 4,000, c 128
// 36.6 / 46.6, 256 57.6 / 47.9; 4, t 1,000, 64 32.0 / 41.2, 128 48.9 / 43.9; 16, t 4,000, 16
// 55.2 / 88.4, 32 103 / 91.4, 64 206 / 129; 32/8 heads, 16, t 4,000, 32 98.6 / 149, 64 199 / 181,
// 128 367 / 216; 14/2 heads of 64, 4, t 12,000, 32 34.6 / 53.3, 128 93.2 / 68.7.
constexpr int64_t kUnpackRows = 224;
constexpr int64_t kUnpackScores = (int64_t)1 << 24;
// The 16-bit pool of a group of sequences, which are unpacked and attended together; one sequence is
// a group of its own up to kUnpackMost, past which its chunk stays row blocks.  (Tables are as wide
// as the longest sequence's, so the pool is the rectangle of all: one long prompt among many short
// ones would take all there is.)  A group's launches end before the next one's begin: us, 32
// sequences after 16,384, 32/8 heads of 128, in a pool of 2.1 GB / three of 0.7, 64 tokens each
// 1,094 / 1,150, 256 tokens 2,695 / 2,795; 64 of 128 after 8,192, 28/4 heads, one of 1.1 GB / two
// 1,347 / 1,356.
constexpr int64_t kUnpackBytes = NDL_FP8_UNPACK_BYTES;
constexpr int64_t kUnpackMost = (int64_t)16 << 30;

struct Unpacked {
  int cols, seqs;               // of the table; sequences of a group
  int64_t blocks;
  size_t table_bytes, lens_bytes, pool_bytes, prefill_bytes;
  size_t total() const { return table_bytes + lens_bytes + pool_bytes + prefill_bytes; }
};
// Tokens that a group of seqs sequences can have.
int64_t group_tokens(int64_t seqs, int64_t num_tokens, int max_seqlen) {
  const int64_t most = seqs * max_seqlen;
  return most < num_tokens ? most : num_tokens;
}
// Workgroups of chunk_nan_kernel per sequence.
int64_t nan_scan_workgroups(int max_seqlen, int num_kv_heads) {
  return (((int64_t)max_seqlen + 15) / 16 * num_kv_heads + 3) / 4;
}
// Whether a call takes this path, and its workspace.
bool unpacked_plan(int64_t num_seqs, int64_t num_tokens, int max_seqlen, int64_t max_keys,
                   int num_heads, int num_kv_heads, int head_dim, int block_size, Unpacked* u) {
  const int64_t rows = (int64_t)max_seqlen * (num_heads / num_kv_heads);
  if (rows < kUnpackRows ||
      (double)rows * (double)max_keys * (double)(num_seqs * num_kv_heads) < (double)kUnpackScores)
    return false;
  const int64_t cols = (max_keys + block_size - 1) / block_size;
  if (cols >= 0x7fffffff / block_size || !grid_fits(nan_scan_workgroups(max_seqlen, num_kv_heads), 256))
    return false;
  const int64_t each = cols * block_size * num_kv_heads * head_dim * 4;
  if (each > kUnpackMost) return false;
  int64_t most = kUnpackBytes / each;
  if (most > 65535) most = 65535;       // a grid dimension
  if (most < 1) most = 1;
  const int64_t groups = (num_seqs + most - 1) / most, seqs = (num_seqs + groups - 1) / groups;
  u->cols = (int)cols;
  u->seqs = (int)seqs;
  u->blocks = seqs * cols;
  u->table_bytes = ((size_t)(u->blocks + seqs) * 4 + 255) / 256 * 256;
  u->lens_bytes = ((size_t)seqs * 4 + 255) / 256 * 256;
  u->pool_bytes = ((size_t)(seqs * each) + 255) / 256 * 256;
  u->prefill_bytes = 0;
  for (const int64_t n : {seqs, num_seqs % seqs}) {     // even groups, the last one
    const size_t b = n == 0 ? 0
                            : prefill_rounds_workspace_bytes(
                                  (int)n, group_tokens(n, num_tokens, max_seqlen), max_seqlen,
                                  u->cols + 1, num_heads, num_kv_heads, head_dim, block_size);
    if (b > u->prefill_bytes) u->prefill_bytes = b;
  }
  return true;
}

template <int D, bool F16>
int launch_unpacked(const ChunkArgs& c, const Unpacked& u, int max_seqlen, int64_t max_keys,
                    int block_size, float scale, void* workspace, hipStream_t s) {
  UnpackArgs a{};
  a.table = (int32_t*)workspace;
  a.lens = (int32_t*)((char*)workspace + u.table_bytes);
  a.pool = (u16*)((char*)workspace + u.table_bytes + u.lens_bytes);
  a.cols = u.cols;
  a.codes = c.codes;
  a.scales = c.scales;
  a.plane_rows = c.plane_rows;
  a.pool_rows = u.blocks * c.num_kv_heads * (int64_t)block_size;
  a.num_blocks = c.num_blocks;
  a.num_kv_heads = c.num_kv_heads;
  a.num_heads = c.num_heads;
  a.group = c.group;
  a.bt_row_stride = c.bt_row_stride;
  a.tile_shift = c.tile_shift;
  a.num_tokens = c.num_tokens;
  a.out = c.out;
  // (the prefill sizes its split by the table, in the call as in the workspace query)
  const int64_t cached = (int64_t)(u.cols + 1) * block_size;
  const int64_t items = (max_keys + 15) / 16 * 2 * c.num_kv_heads;
  const int64_t scan = nan_scan_workgroups(max_seqlen, c.num_kv_heads);
  void* const ws = u.prefill_bytes ? (char*)workspace + u.total() - u.prefill_bytes : nullptr;
  if (F16) scale *= 2.f;     // of halved keys
  for (int64_t i0 = 0; i0 < c.num_seqs; i0 += u.seqs) {
    const int n = (int)(c.num_seqs - i0 < u.seqs ? c.num_seqs - i0 : u.seqs);
    a.block_table = c.block_table + i0 * c.bt_row_stride;
    a.cu_seqlens = c.cu_seqlens + i0;
    a.context_lens = c.context_lens + i0;
    // workgroups of a sequence: what the longest can use, 16,384 over all of the group
    int64_t wgs = (16384 + n - 1) / n;
    if (wgs > (items + 3) / 4) wgs = (items + 3) / 4;
    hipLaunchKernelGGL((chunk_unpack_kernel<D, F16>), dim3((unsigned)wgs, (unsigned)n), dim3(256),
                       0, s, a);
    int rc = check_launch();
    if (rc != NDL_OK) return rc;
    rc = launch_prefill_rounds(c.out, c.q, c.q_stride, a.pool, u.blocks, a.table, u.cols + 1,
                               u.cols + 1, a.cu_seqlens, a.lens, n, c.num_tokens,
                               group_tokens(n, c.num_tokens, max_seqlen), max_seqlen, (int)cached,
                               c.num_heads, c.num_kv_heads, D, block_size,
                               F16 ? NDL_DTYPE_F16 : NDL_DTYPE_BF16, scale, ws, u.prefill_bytes, s);
    if (rc != NDL_OK) return rc;
    hipLaunchKernelGGL((chunk_nan_kernel<D>), dim3((unsigned)scan, (unsigned)n), dim3(256), 0, s, a);
    rc = check_launch();
    if (rc != NDL_OK) return rc;
  }
  return NDL_OK;
}

// Column tiles of a row block: one where it holds max_seqlen tokens of a group's heads, else two.
int col_tiles(int64_t max_seqlen, int group) { return max_seqlen * group <= 16 ? 1 : 2; }

struct Plan {
  int nt, toks, waves, pad;
  int64_t blocks_per_seq, items;
  int shares;                 // 0: whole row blocks
  int64_t nseg;
  size_t ml_bytes, acc_bytes;
};

template <int D, bool F16>
const void* kernel_of(int nt, int waves, bool append = false) {
  if (append)       // one token per sequence: one column tile
    return waves == 4 ? (const void*)chunk_attention_kernel<D, F16, 1, 4, true>
                      : (const void*)chunk_attention_kernel<D, F16, 1, 8, true>;
  if (waves == 4)
    return nt == 1 ? (const void*)chunk_attention_kernel<D, F16, 1, 4>
                   : (const void*)chunk_attention_kernel<D, F16, 2, 4>;
  return nt == 1 ? (const void*)chunk_attention_kernel<D, F16, 1, 8>
                 : (const void*)chunk_attention_kernel<D, F16, 2, 8>;
}

// Slots a share has at least: two tiles for each of four waves.
constexpr int kMinChunk = 8;
// Tiles up to which a row block is one workgroup's, whatever else there is: the shares' scan, their
// parts and the merge launch cost more (us, shares / whole, decode of 8 sequences: 14/2 heads of
// 64, 1,000 tokens 12.2 / 8.2, 1,500 12.8 / 9.9, 3,000 14.6 / 15.8; 32/8 of 128 14.9 / 11.0,
// 16.1 / 14.2, 17.7 / 22.6; 500 tokens in tables of 1,500, all that the host knows of them, 16.6 /
// 7.7).  Chunks of 5 tokens and 64 sequences part at about 2,000 to 3,000 tokens, and at less where
// one sequence is much longer than the others.
constexpr int kWholeTiles = 48;
// Empty slots before a row block, one column tile or two (its start, its waves' sums): us at 0 and
// 0, 0 and 2, 1 and 4, 5 tokens each after up to 3,000: 32 sequences of 14/2 heads of 64 24.3 /
// 23.5 / 21.5, of 28/4 of 128 35.7 / 33.9 / 33.3, 100 of 32/8 70.3 / 69.2 / 66.7, one token each
// 52.5 / 52.8 / 51.2.
constexpr int kPad1 = 1, kPad2 = 4;

// resident: workgroups the GPU holds at once.
Plan make_plan(int64_t num_seqs, int64_t max_seqlen, int64_t max_keys, int group,
               int num_kv_heads, int head_dim, int64_t resident) {
  Plan p{};
  p.nt = col_tiles(max_seqlen, group);
  p.toks = 16 * p.nt / group;
  p.blocks_per_seq = (max_seqlen + p.toks - 1) / p.toks;
  p.items = num_seqs * p.blocks_per_seq;
  const int64_t tiles = (max_keys + kTile - 1) / kTile;
  const int64_t units = p.items * num_kv_heads;
  // (slots and segments are counted in 31 bits)
  const bool whole = tiles <= kWholeTiles || units >= 4 * resident ||
                     p.items * (tiles + kPad2) + 2 * resident * kMinChunk > 0x40000000;
  // Whole row blocks: eight waves where four would leave half the GPU without any (us, four /
  // eight, 16 sequences of 1,000 tokens: 14/2 heads of 64 9.5 / 8.3, 32/8 of 128 11.8 / 11.5; 128
  // of 32/8 28.4 / 34.8).  Shares: four (16 of 3,000, 32/8 heads, 1 and 8 tokens each 20.2 / 19.9
  // and 26.2 / 28.1, 14/2 of 64 14.5 / 15.3 and 18.4 / 24.3).
  p.waves = whole && units * 2 <= resident ? 8 : 4;
  p.pad = p.nt == 1 ? kPad1 : kPad2;
  if (!whole) {
    int64_t s = resident * 4 / p.waves / num_kv_heads / 8 * 8;
    if (s < 8) s = 8;
    p.shares = (int)s;
    p.nseg = s + p.items;
    const size_t cols = (size_t)num_kv_heads * p.nseg * p.toks * group;
    p.ml_bytes = (cols * 8 + 255) / 256 * 256;
    p.acc_bytes = cols * head_dim * 4;
  }
  return p;
}

bool shape_ok(int head_dim, int block_size, int num_heads, int num_kv_heads) {
  return (head_dim == 64 || head_dim == 128) && block_tile_shift(block_size) >= 0 &&
         num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0 &&
         num_heads / num_kv_heads <= 16;
}

Plan plan_for(int64_t num_seqs, int64_t max_seqlen, int64_t max_keys, int num_heads,
              int num_kv_heads, int head_dim) {
  const int group = num_heads / num_kv_heads, nt = col_tiles(max_seqlen, group);
  // the formats' kernels use the same resources
  int64_t res = resident_workgroups(
      head_dim == 128 ? kernel_of<128, false>(nt, 4) : kernel_of<64, false>(nt, 4), 256);
  if (res <= 0) res = 256;
  return make_plan(num_seqs, max_seqlen, max_keys, group, num_kv_heads, head_dim, res);
}

template <int D, bool F16>
int launch(ChunkArgs a, int nt, int waves, hipStream_t s) {
  const int64_t units = a.shares ? a.shares : ((int64_t)a.items + 7) / 8 * 8;
  const int64_t wgs = units * a.num_kv_heads;
  if (!grid_fits(wgs, 64 * waves)) return NDL_ERR_INVALID_ARG;
  void* args[] = {&a};
  if (hipLaunchKernel(kernel_of<D, F16>(nt, waves, a.new_k != nullptr), dim3((unsigned)wgs),
                      dim3(64 * waves), args, 0, s) != hipSuccess) {
    (void)hipGetLastError();  // clear the error so that the next call's check sees its own
    return NDL_ERR_LAUNCH;
  }
  const int rc = check_launch();
  if (rc != NDL_OK || a.shares == 0) return rc;
  const int groups = (a.toks * a.group + kMergeCols - 1) / kMergeCols;
  hipLaunchKernelGGL((chunk_merge_kernel<D, F16>),
                     dim3((unsigned)a.items, (unsigned)a.num_kv_heads, (unsigned)groups), dim3(256),
                     0, s, a);
  return check_launch();
}

}  // namespace
}  // namespace ndl

extern "C" size_t ndl_fp8_attention_workspace_bytes(int num_seqs, int64_t num_tokens,
                                                    int max_seqlen, int64_t max_keys,
                                                    int num_heads, int num_kv_heads, int head_dim,
                                                    int block_size) {
  using namespace ndl;
  if (num_seqs <= 0 || num_tokens <= 0 || max_seqlen <= 0 || max_keys <= 0 ||
      max_keys > 0x7fffff00 || !shape_ok(head_dim, block_size, num_heads, num_kv_heads))
    return 0;
  Unpacked u;
  if (unpacked_plan(num_seqs, num_tokens, max_seqlen, max_keys, num_heads, num_kv_heads, head_dim,
                    block_size, &u))
    return u.total();
  const Plan p = plan_for(num_seqs, max_seqlen, max_keys, num_heads, num_kv_heads, head_dim);
  return p.ml_bytes + p.acc_bytes;
}

// Both entry points; `a` holds the new rows and the rotation of the second one.
static int fp8_attention(ndl::ChunkArgs a, void* out, const void* q, int64_t q_tok_stride,
                         void* codes, void* scales, int64_t num_blocks,
                         const int32_t* block_table, int64_t bt_row_stride,
                         int max_blocks_per_seq, const int32_t* cu_seqlens,
                         const int32_t* context_lens, int num_seqs, int64_t num_tokens,
                         int max_seqlen, int64_t max_keys, int num_heads, int num_kv_heads,
                         int head_dim, int block_size, int dtype, float scale, void* workspace,
                         size_t workspace_bytes, ndl_stream_t stream) {
  using namespace ndl;
  if (!dtype_supported(dtype) || !shape_ok(head_dim, block_size, num_heads, num_kv_heads))
    return NDL_ERR_UNSUPPORTED;
  if (num_seqs < 0 || num_tokens < 0 || num_blocks <= 0 || max_blocks_per_seq <= 0 ||
      bt_row_stride < max_blocks_per_seq || max_seqlen <= 0 || max_keys <= 0)
    return NDL_ERR_INVALID_ARG;
  if (num_seqs == 0 || num_tokens == 0) return NDL_OK;
  if (!out || !q || !codes || !scales || !block_table || !context_lens)
    return NDL_ERR_INVALID_ARG;
  if (cu_seqlens == nullptr && (num_tokens != num_seqs || max_seqlen != 1))
    return NDL_ERR_INVALID_ARG;
  if (q_tok_stride < (int64_t)num_heads * head_dim || (q_tok_stride & 7))
    return NDL_ERR_INVALID_ARG;
  if (((uintptr_t)out | (uintptr_t)q | (uintptr_t)codes) & 15u || (uintptr_t)scales & 3u)
    return NDL_ERR_INVALID_ARG;
  a.plane_rows = num_blocks * num_kv_heads * (int64_t)block_size;
  // a scale's address is the pool's and a 32-bit offset; positions are 32-bit
  if (a.plane_rows > 0x7fffffff || (int64_t)max_blocks_per_seq * block_size > 0x7fffff00)
    return NDL_ERR_UNSUPPORTED;
  if (max_keys > (int64_t)max_blocks_per_seq * block_size)
    max_keys = (int64_t)max_blocks_per_seq * block_size;
  a.out = (u16*)out;
  a.q = (const u16*)q;
  a.q_stride = q_tok_stride;
  a.codes = (uint8_t*)codes;
  a.scales = (uint8_t*)scales;
  a.num_blocks = num_blocks;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.block_table = block_table;
  a.bt_row_stride = bt_row_stride;
  a.max_blocks = max_blocks_per_seq;
  a.tile_shift = block_tile_shift(block_size);
  a.cu_seqlens = cu_seqlens;
  a.context_lens = context_lens;
  a.num_seqs = num_seqs;
  a.num_tokens = num_tokens;
  const hipStream_t s = (hipStream_t)stream;
  const bool f16 = dtype_is_f16(dtype);
  Unpacked u;
  if (cu_seqlens != nullptr && unpacked_plan(num_seqs, num_tokens, max_seqlen, max_keys, num_heads,
                                             num_kv_heads, head_dim, block_size, &u)) {
    if (!workspace || workspace_bytes < u.total() || (uintptr_t)workspace & 255u)
      return NDL_ERR_WORKSPACE;
    if (head_dim == 128)
      return f16 ? launch_unpacked<128, true>(a, u, max_seqlen, max_keys, block_size, scale,
                                              workspace, s)
                 : launch_unpacked<128, false>(a, u, max_seqlen, max_keys, block_size, scale,
                                               workspace, s);
    return f16 ? launch_unpacked<64, true>(a, u, max_seqlen, max_keys, block_size, scale,
                                           workspace, s)
               : launch_unpacked<64, false>(a, u, max_seqlen, max_keys, block_size, scale,
                                            workspace, s);
  }
  const Plan p = plan_for(num_seqs, max_seqlen, max_keys, num_heads, num_kv_heads, head_dim);
  if (p.items > 0x7fffff00) return NDL_ERR_INVALID_ARG;
  if (p.shares) {
    if (num_kv_heads > 65535) return NDL_ERR_UNSUPPORTED;     // a grid dimension of the merge
    if (!workspace || workspace_bytes < p.ml_bytes + p.acc_bytes || (uintptr_t)workspace & 255u)
      return NDL_ERR_WORKSPACE;
    a.ws_ml = (float*)workspace;
    a.ws_acc = (float*)((char*)workspace + p.ml_bytes);
  }
  a.toks = p.toks;
  a.blocks_per_seq = (int)p.blocks_per_seq;
  a.items = (int)p.items;
  a.scale_log2 = scale * kLog2e;
  a.shares = p.shares;
  a.min_chunk = kMinChunk;
  a.pad = p.pad;
  a.nseg = (int)p.nseg;
  if (head_dim == 128)
    return f16 ? launch<128, true>(a, p.nt, p.waves, s) : launch<128, false>(a, p.nt, p.waves, s);
  return f16 ? launch<64, true>(a, p.nt, p.waves, s) : launch<64, false>(a, p.nt, p.waves, s);
}

extern "C" int ndl_fp8_attention(void* out, const void* q, int64_t q_tok_stride,
                                 const void* codes, const void* scales, int64_t num_blocks,
                                 const int32_t* block_table, int64_t bt_row_stride,
                                 int max_blocks_per_seq, const int32_t* cu_seqlens,
                                 const int32_t* context_lens, int num_seqs, int64_t num_tokens,
                                 int max_seqlen, int64_t max_keys, int num_heads,
                                 int num_kv_heads, int head_dim, int block_size, int dtype,
                                 float scale, void* workspace, size_t workspace_bytes,
                                 ndl_stream_t stream) {
  return fp8_attention({}, out, q, q_tok_stride, (void*)codes, (void*)scales, num_blocks,
                       block_table, bt_row_stride, max_blocks_per_seq, cu_seqlens, context_lens,
                       num_seqs, num_tokens, max_seqlen, max_keys, num_heads, num_kv_heads,
                       head_dim, block_size, dtype, scale, workspace, workspace_bytes, stream);
}

extern "C" int ndl_fp8_decode_append(void* out, const void* q, int64_t q_tok_stride, const void* k,
                                     int64_t k_tok_stride, const void* v, int64_t v_tok_stride,
                                     const void* cos, const void* sin, int64_t cs_stride,
                                     void* codes, void* scales, int64_t num_blocks,
                                     const int32_t* block_table, int64_t bt_row_stride,
                                     int max_blocks_per_seq, const int32_t* context_lens,
                                     int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                     int block_size, int dtype, float scale, void* workspace,
                                     size_t workspace_bytes, ndl_stream_t stream) {
  using namespace ndl;
  if (num_seqs > 0 && head_dim > 0 && num_kv_heads > 0) {
    const int64_t row = (int64_t)num_kv_heads * head_dim;
    if (!k || !v || k_tok_stride < row || v_tok_stride < row ||
        (k_tok_stride | v_tok_stride) & 7 || ((uintptr_t)k | (uintptr_t)v) & 15u)
      return NDL_ERR_INVALID_ARG;
    if ((cos == nullptr) != (sin == nullptr) ||
        (cos != nullptr && (cs_stride < head_dim || (cs_stride & 7) ||
                            ((uintptr_t)cos | (uintptr_t)sin) & 15u)))
      return NDL_ERR_INVALID_ARG;
  }
  ChunkArgs a{};
  a.new_k = (const u16*)k;
  a.new_v = (const u16*)v;
  a.k_stride = k_tok_stride;
  a.v_stride = v_tok_stride;
  a.cos = (const u16*)cos;
  a.sin = (const u16*)sin;
  a.cs_stride = cs_stride;
  const int64_t keys = (int64_t)max_blocks_per_seq * block_size;
  return fp8_attention(a, out, q, q_tok_stride, codes, scales, num_blocks, block_table,
                       bt_row_stride, max_blocks_per_seq, nullptr, context_lens, num_seqs,
                       num_seqs, 1, keys > 0 ? keys : 1, num_heads, num_kv_heads, head_dim,
                       block_size, dtype, scale, workspace, workspace_bytes, stream);
}
