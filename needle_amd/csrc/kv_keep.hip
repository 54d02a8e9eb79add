// Caches that keep some of their rows, gfx950: which tokens of a kv head stay when a cache is cut to a
// budget (kv_select), and the rows that stay moved together (kv_compact), after a selection or after
// the verification of a tree, whose accepted path lies scattered among its nodes.  The reference has
// neither; pool, table and positions are its attention's (needle/layers/attention.py:141-154).
#include "fp8.hpp"
#include "ndl_common.hpp"

namespace ndl {
namespace {

// ---------------------------------------------------------------- rows moved together
//
// Row first + j of a sequence <- row first + keep[j], j < count: of one kv head, or of all alike.
// Bound: the rows, read and written once, and the trips before them (length, index, block ids).
//   * A lane finds a row's source and place, for up to 64 rows of a wave's step and for several planes
//     (layers, K and V); then the wave's lanes take 16-byte pieces of those rows, 8 or 16 loads under
//     way, and the next step's rows are found meanwhile.  (A scale byte or a weight: a lane a row.)
//   * In place the indices ascend, so a row's source is never written before it is read: a later row
//     has a later source and a later place.  One wave (short lists) or the 16 of a workgroup (long
//     ones, a barrier between the reads of a step and its writes) take a list from front to back.
//   * Into other blocks nothing is ordered, and lists are cut into as many pieces as fill the GPU.
// us, in replayed graphs, rows out of the caches: the 2,048 rows that stay of 16 prompts of 4,096 to
// 16,384 tokens, 8 kv heads of 128, in place 74 (270 MB at 3.7 TB/s), into other blocks 65 (4.2); 512 of
// 8 caches of 530 to 640, 2 of 64, 6.2 either way; paths of 32 trees in 32 layers 11.9 (17 MB: a chain of
// trips, lengths and starts, list, tables, then a plane's rows and the next one's).
constexpr int kMaxPools = 128;
// Loads of a lane under way: us, 8 / 16, in place 32 layers of 32 trees' paths 12.2 / 14.9, into other
// blocks 16 x 2,048 rows of 8 heads 67 / 62 (fewer waves fit, but lists are longer).
constexpr int loads_of(bool in_place) { return in_place ? 8 : 16; }

struct MoveArgs {
  char* pool[kMaxPools];
  char* scales[kMaxPools];        // an 8-bit pool's
  int pools;
  float* mass;                    // or null
  int64_t num_blocks;
  int num_kv_heads, block_size, row_bytes;
  const int32_t* table;
  int64_t table_stride;
  int table_cols;
  const int32_t* to;
  int64_t to_stride;
  int to_cols;
  const int32_t* keep;            // [seq][kv head][width], or packed by cu, for every kv head alike
  const int32_t* cu;
  int width;
  int64_t keep_rows;              // with cu: entries of keep
  const int32_t* first;           // or null: 0
  const int32_t* counts;
  int num_seqs;
  int pieces, pieces_shift;       // of a row; their log2, or -1
  int planes_each;                // planes of the pools that a workgroup takes
};

// Source and place of row j of a list, as rows of a plane; kNone where there is nothing to do.
constexpr uint32_t kNone = ~0u;
struct Move {
  uint32_t from, to;
};

struct List {
  const int32_t* keep;
  const int32_t* table;
  const int32_t* to;
  int64_t base;
  int n;
};
__device__ __forceinline__ List list_of(const MoveArgs& a, int seq, int head) {
  List l;
  l.n = a.counts[seq];
  l.base = a.first ? a.first[seq] : 0;
  int64_t at = ((int64_t)seq * a.num_kv_heads + head) * a.width, most = a.width;
  if (a.cu) {
    at = a.cu[seq];
    const int64_t end = a.cu[seq + 1];
    most = at < 0 || end > a.keep_rows || end < at ? 0 : end - at;
  }
  l.keep = a.keep + at;
  if (l.n > most) l.n = (int)most;
  if (l.base < 0) l.n = 0;
  l.table = a.table + seq * a.table_stride;
  l.to = a.to + seq * a.to_stride;
  return l;
}
__device__ __forceinline__ Move move_of(const MoveArgs& a, const List& l, int j, int head) {
  const Move none{kNone, kNone};
  if (j >= l.n) return none;
  const int k = l.keep[j];
  const int64_t s = l.base + k, d = l.base + j;
  if (k < 0 || s >= (int64_t)a.table_cols * a.block_size ||
      d >= (int64_t)a.to_cols * a.block_size)
    return none;
  const uint32_t bs = (uint32_t)a.block_size, hkv = (uint32_t)a.num_kv_heads;
  const uint32_t sc = (uint32_t)s / bs, dc = (uint32_t)d / bs;
  const int sb = l.table[sc], db = l.to[dc];
  if (sb < 0 || sb >= a.num_blocks || db < 0 || db >= a.num_blocks) return none;
  const Move m{((uint32_t)sb * hkv + (uint32_t)head) * bs + ((uint32_t)s - sc * bs),
               ((uint32_t)db * hkv + (uint32_t)head) * bs + ((uint32_t)d - dc * bs)};
  return m.from == m.to ? none : m;
}

// A wave's rows j0, j0 + WAVES * per, .. of a list, `per` at a time.  A list in place is whole: every
// read of a step before its writes, within a wave by their order (a place written here is before the
// sources still on their way), across waves by a wait and a barrier.
template <int WAVES, bool IN_PLACE>
__device__ __forceinline__ void move_rows(const MoveArgs& a, const List& l, int head, int plane0,
                                          int plane1, int lane, int wave, int j0, int j1) {
  const int64_t plane_bytes = a.num_blocks * a.num_kv_heads * a.block_size * a.row_bytes;
  constexpr int kLoads = loads_of(IN_PLACE);
  const int per = a.pieces > kLoads ? kLoads * 64 / a.pieces : 64;
  auto find = [&](int base) {
    return lane < per && base + lane < j1 ? move_of(a, l, base + lane, head) : Move{kNone, kNone};
  };
  const int step = WAVES * per;
  Move next = find(j0 + wave * per);
  for (int base = j0; base < j1; base += step) {
    const Move m = next;
    const int mine = base + wave * per;
    if (mine + step < j1) next = find(mine + step);
    const int rows = j1 - mine < per ? j1 - mine : per, total = rows > 0 ? rows * a.pieces : 0;
    for (int y = plane0; y < plane1; ++y) {
      char* const plane = a.pool[y >> 1] + (y & 1) * plane_bytes;
      u32x4 v[kLoads];
#pragma unroll
      for (int x = 0; x < kLoads; ++x) {
        if (64 * x >= total) break;
        const int i = 64 * x + lane;
        const int r = a.pieces_shift >= 0 ? i >> a.pieces_shift : i / a.pieces;
        const uint32_t from = (uint32_t)__shfl((int)m.from, r & 63, 64);
        if (i < total && from != kNone)
          v[x] = *reinterpret_cast<const u32x4*>(plane + (int64_t)from * a.row_bytes +
                                                 16 * (i - r * a.pieces));
      }
      if constexpr (IN_PLACE && WAVES > 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
      }
#pragma unroll
      for (int x = 0; x < kLoads; ++x) {
        if (64 * x >= total) break;
        const int i = 64 * x + lane;
        const int r = a.pieces_shift >= 0 ? i >> a.pieces_shift : i / a.pieces;
        const uint32_t to = (uint32_t)__shfl((int)m.to, r & 63, 64);
        if (i < total && to != kNone)
          *reinterpret_cast<u32x4*>(plane + (int64_t)to * a.row_bytes + 16 * (i - r * a.pieces)) =
              v[x];
      }
    }
  }
}
// The same of numbers, one a row: scale bytes, weights.
template <int WAVES, bool IN_PLACE, class WORD>
__device__ __forceinline__ void move_words(const MoveArgs& a, const List& l, int head, WORD* plane,
                                           int lane, int wave, int j0, int j1) {
  const int step = WAVES * 64;
  Move next = j0 + 64 * wave + lane < j1 ? move_of(a, l, j0 + 64 * wave + lane, head)
                                         : Move{kNone, kNone};
  for (int base = j0; base < j1; base += step) {
    const Move m = next;
    const int j = base + step + 64 * wave + lane;
    WORD v{};
    if (m.from != kNone) v = plane[m.from];
    next = j < j1 ? move_of(a, l, j, head) : Move{kNone, kNone};
    if constexpr (IN_PLACE && WAVES > 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
    if (m.from != kNone) plane[m.to] = v;
  }
}

// blockIdx.x: lists (sequence, kv head), four to a workgroup where a wave takes one; blockIdx.y: groups
// of the pools' planes, then the planes of their scales, then the weights; blockIdx.z: a piece of the
// list.
template <int WAVES, bool IN_PLACE>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void kv_move_kernel(MoveArgs a) {
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int64_t unit = WAVES == 1 ? (int64_t)blockIdx.x * 4 + wv : blockIdx.x;
  const int wave = WAVES == 1 ? 0 : wv;
  if (unit >= (int64_t)a.num_seqs * a.num_kv_heads) return;
  const int seq = (int)(unit / a.num_kv_heads), head = (int)(unit - (int64_t)seq * a.num_kv_heads);
  const List l = list_of(a, seq, head);
  int j0 = 0, j1 = l.n;
  if (!IN_PLACE) {
    const int per = ((l.n + (int)gridDim.z - 1) / (int)gridDim.z + 63) / 64 * 64;
    if ((int64_t)per * blockIdx.z >= l.n) return;
    j0 = per * (int)blockIdx.z;
    j1 = l.n - j0 > per ? j0 + per : l.n;
  }
  if (j0 >= j1) return;
  const int main = 2 * a.pools, groups = (main + a.planes_each - 1) / a.planes_each;
  const int y = blockIdx.y;
  if (y < groups) {
    const int y0 = y * a.planes_each, y1 = y0 + a.planes_each < main ? y0 + a.planes_each : main;
    move_rows<WAVES, IN_PLACE>(a, l, head, y0, y1, lane, wave, j0, j1);
  } else if (y - groups < main && a.scales[0]) {
    const int s = y - groups;
    uint8_t* const plane = reinterpret_cast<uint8_t*>(a.scales[s >> 1]) +
                           (s & 1) * (a.num_blocks * a.num_kv_heads * a.block_size);
    move_words<WAVES, IN_PLACE>(a, l, head, plane, lane, wave, j0, j1);
  } else {
    move_words<WAVES, IN_PLACE>(a, l, head, a.mass, lane, wave, j0, j1);
  }
}

// ---------------------------------------------------------------- the rows that stay
//
// Of a kv head's L cached tokens the `budget` that stay: the first `sinks`, the last `recent`, and of
// those between the largest weights, of equal ones the first, in the order of their positions.
// A workgroup per (kv head, sequence): a radix select over the weights as ordered 32-bit keys, eight
// bits a pass from the top, then one pass that writes positions.  Bound: the passes' trips through
// LDS (keys are read from the pool once; those past kHeldMany again each pass) for few and short lists,
// which leave most of the GPU idle.  us: 8 caches of 530 to 640 tokens, 2 kv heads, 7.4; 16 of 4,096 to
// 16,384, 8 kv heads, 27 (all the weights at 0.15 TB/s).
constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
// Keys in LDS, by position: of a short table, or as many as a workgroup can have.
constexpr int kHeldFew = 8192, kHeldMany = 38912;

struct SelectArgs {
  int32_t* keep;                      // [seq][kv head][budget]
  int32_t* kept;                      // [seq]
  const float* mass;
  int64_t num_blocks;
  int num_kv_heads, block_size;
  const int32_t* table;
  int64_t table_stride;
  int table_cols;
  const int32_t* lens;
  int budget, sinks, recent;
};

// Keys in the order of the weights: -0 as 0, NaN the largest; 0 for a row without a block.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return ~0u;
  const uint32_t b = __float_as_uint(v + 0.f);           // (-0 + 0 = 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <int HELD>
__global__ __launch_bounds__(kSelThreads) void kv_select_kernel(SelectArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t keys[HELD];
  __shared__ uint32_t hist[256];
  __shared__ int above[kSelWaves], equal[kSelWaves];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  const int head = blockIdx.x, seq = blockIdx.y, t = threadIdx.x, lane = t & 63, wv = t >> 6;
  const int64_t cap = (int64_t)a.table_cols * a.block_size;
  int len = a.lens[seq];
  if (len < 0) len = 0;
  if (len > cap) len = (int)cap;
  int32_t* const out = a.keep + ((int64_t)seq * a.num_kv_heads + head) * a.budget;
  const int stay = len < a.budget ? len : a.budget;
  if (head == 0 && t == 0) a.kept[seq] = stay;
  for (int j = stay + t; j < a.budget; j += kSelThreads) out[j] = -1;
  if (len <= a.budget) {
    for (int j = t; j < stay; j += kSelThreads) out[j] = j;
    return;
  }
  // the ends (sinks + recent <= budget < len)
  for (int j = t; j < a.sinks; j += kSelThreads) out[j] = j;
  for (int j = t; j < a.recent; j += kSelThreads)
    out[a.budget - a.recent + j] = len - a.recent + j;
  const int want = a.budget - a.sinks - a.recent;        // of these:
  const int lo = a.sinks, hi = len - a.recent;           // candidates: more than want
  if (want == 0) return;
  const int32_t* const table = a.table + seq * a.table_stride;
  const uint32_t bs = (uint32_t)a.block_size;
  auto row_of = [&](uint32_t p, int b) {
    return ((int64_t)b * a.num_kv_heads + head) * bs + (p - p / bs * bs);
  };
  auto valid = [&](int b) { return b >= 0 && b < a.num_blocks; };
  auto load = [&](int p) {
    const int b = table[(uint32_t)p / bs];
    return valid(b) ? key_of(a.mass[row_of((uint32_t)p, b)]) : 0u;
  };
  auto key = [&](int p) { return p < HELD ? keys[p] : load(p); };
  if (bs % 4 == 0 && ((uintptr_t)a.mass & 15u) == 0) {
    // four positions a lane: all block ids, then all weights under way
    constexpr int kQuads = 4;
    const int end = hi < HELD ? hi : HELD;
    for (int p0 = 4 * t; p0 < end; p0 += 4 * kSelThreads * kQuads) {
      int b[kQuads];
#pragma unroll
      for (int x = 0; x < kQuads; ++x) {
        const int p = p0 + 4 * kSelThreads * x;
        b[x] = p < end ? table[(uint32_t)p / bs] : -1;
      }
      f32x4 v[kQuads];
#pragma unroll
      for (int x = 0; x < kQuads; ++x)
        if (valid(b[x]))
          v[x] = *reinterpret_cast<const f32x4*>(
              a.mass + row_of((uint32_t)(p0 + 4 * kSelThreads * x), b[x]));
#pragma unroll
      for (int x = 0; x < kQuads; ++x) {
        const int p = p0 + 4 * kSelThreads * x;
        if (p >= end) break;
        u32x4 k = {0u, 0u, 0u, 0u};
        if (valid(b[x])) k = u32x4{key_of(v[x][0]), key_of(v[x][1]), key_of(v[x][2]), key_of(v[x][3])};
        *reinterpret_cast<u32x4*>(&keys[p]) = k;
      }
    }
  } else {
    for (int p = t; p < hi && p < HELD; p += kSelThreads) keys[p] = load(p);
  }
  // The want-th largest key: its bits from the top, those above fixed as `prefix`.
  uint32_t prefix = 0;
  int left = want;                                       // of those that share the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (t < 256) hist[t] = 0;
    __syncthreads();
    const uint32_t fixed = shift == 24 ? 0u : ~0u << (shift + 8);
    for (int i = lo + t; i < hi; i += kSelThreads) {
      const uint32_t k = key(i);
      const bool in = (k & fixed) == prefix;
      // lanes with the first one's digit count at once (weights of 0 are many), the others each
      const uint32_t digit = (k >> shift) & 255u;
      const uint64_t active = __builtin_amdgcn_ballot_w64(in);
      if (!active) continue;
      const int leader = __builtin_ctzll(active);
      const uint32_t d0 = (uint32_t)__builtin_amdgcn_readlane((int)digit, leader);
      const uint64_t same = __builtin_amdgcn_ballot_w64(in && digit == d0);
      if (lane == leader) atomicAdd(&hist[d0], (uint32_t)__builtin_popcountll(same));
      if (in && digit != d0) atomicAdd(&hist[digit], 1u);
    }
    __syncthreads();
    if (wv == 0) {
      // digits from the top, four to a lane: the one where the count reaches `left`
      uint32_t c[4], sum = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        c[x] = hist[255 - 4 * lane - x];
        sum += c[x];
      }
      uint32_t incl = sum;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const uint32_t o = (uint32_t)__shfl_up((int)incl, m, 64);
        if (lane >= m) incl += o;
      }
      const uint64_t reach = __builtin_amdgcn_ballot_w64(incl >= (uint32_t)left);
      if (lane == __builtin_ctzll(reach)) {
        uint32_t before = incl - sum;
        int x = 0;
        for (; x < 3 && before + c[x] < (uint32_t)left; ++x) before += c[x];
        s_prefix = prefix | (uint32_t)(255 - 4 * lane - x) << shift;
        s_left = left - (int)before;
      }
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
  }
  // Each wave takes a run of positions: it counts, then writes behind those of the waves before.
  const int run = (hi - lo + kSelWaves - 1) / kSelWaves;
  const int i0 = lo + wv * run, i1 = i0 + run < hi ? i0 + run : hi;
  int more = 0, same = 0;
  for (int b = i0; b < i1; b += 64) {
    const uint32_t k = b + lane < i1 ? key(b + lane) : 0u;
    more += __builtin_popcountll(__builtin_amdgcn_ballot_w64(b + lane < i1 && k > prefix));
    same += __builtin_popcountll(__builtin_amdgcn_ballot_w64(b + lane < i1 && k == prefix));
  }
  if (lane == 0) {
    above[wv] = more;
    equal[wv] = same;
  }
  __syncthreads();
  int at = 0, ties = 0;                                  // written, equal ones seen before this run
  for (int w = 0; w < wv; ++w) {
    const int take = left - ties < equal[w] ? left - ties : equal[w];
    at += above[w] + (take > 0 ? take : 0);
    ties += equal[w];
  }
  const uint64_t below = lane ? ~0ull >> (64 - lane) : 0ull;
  for (int b = i0; b < i1; b += 64) {
    const bool in = b + lane < i1;
    const uint32_t k = in ? key(b + lane) : 0u;
    const uint64_t eq = __builtin_amdgcn_ballot_w64(in && k == prefix);
    const bool mine = in && (k > prefix || (k == prefix &&
                                            ties + __builtin_popcountll(eq & below) < left));
    const uint64_t take = __builtin_amdgcn_ballot_w64(mine);
    if (mine) out[a.sinks + at + __builtin_popcountll(take & below)] = b + lane;
    at += __builtin_popcountll(take);
    ties += __builtin_popcountll(eq);
  }
}

}  // namespace
}  // namespace ndl

extern "C" int ndl_kv_compact(void* const* pools, void* const* scales, int num_layers, float* mass,
                              int64_t num_blocks, int num_kv_heads, int block_size, int row_bytes,
                              const int32_t* block_table, int64_t bt_row_stride,
                              int max_blocks_per_seq, const int32_t* dst_table,
                              int64_t dst_row_stride, int dst_max_blocks, const int32_t* keep,
                              int keep_width, const int32_t* cu_seqlens, int64_t num_keep,
                              const int32_t* first, const int32_t* counts, int num_seqs,
                              ndl_stream_t stream) {
  using namespace ndl;
  if (num_layers < 0 || num_seqs < 0 || num_blocks <= 0 || num_kv_heads <= 0 || block_size <= 0 ||
      row_bytes <= 0 || row_bytes % 16 || max_blocks_per_seq <= 0 ||
      bt_row_stride < max_blocks_per_seq || keep_width < 0 || num_keep < 0)
    return NDL_ERR_INVALID_ARG;
  if (dst_table && (dst_max_blocks <= 0 || dst_row_stride < dst_max_blocks))
    return NDL_ERR_INVALID_ARG;
  const int64_t most = cu_seqlens ? num_keep : keep_width;       // rows of a list
  if (num_seqs == 0 || (num_layers == 0 && !mass) || most == 0) return NDL_OK;
  if ((num_layers && !pools) || !block_table || !keep || !counts) return NDL_ERR_INVALID_ARG;
  if (num_layers > kMaxPools || (int64_t)max_blocks_per_seq * block_size > 0x7fffff00 ||
      (int64_t)dst_max_blocks * block_size > 0x7fffff00 || most > 0x7fff0000 ||
      num_blocks > (int64_t)0xfffffff0 / num_kv_heads / block_size ||
      row_bytes > 16 * loads_of(true) * 64)
    return NDL_ERR_UNSUPPORTED;
  MoveArgs a{};
  for (int i = 0; i < num_layers; ++i) {
    a.pool[i] = (char*)pools[i];
    if (!pools[i] || (uintptr_t)pools[i] & 15u) return NDL_ERR_INVALID_ARG;
    for (int j = 0; j < i; ++j)      // (rows moved twice at once)
      if (pools[j] == pools[i]) return NDL_ERR_INVALID_ARG;
    if (!scales) continue;
    a.scales[i] = (char*)scales[i];
    if (!scales[i]) return NDL_ERR_INVALID_ARG;
  }
  if ((uintptr_t)mass & 3u) return NDL_ERR_INVALID_ARG;
  a.pools = num_layers;
  a.mass = mass;
  a.num_blocks = num_blocks;
  a.num_kv_heads = num_kv_heads;
  a.block_size = block_size;
  a.row_bytes = row_bytes;
  a.table = block_table;
  a.table_stride = bt_row_stride;
  a.table_cols = max_blocks_per_seq;
  a.to = dst_table ? dst_table : block_table;
  a.to_stride = dst_table ? dst_row_stride : bt_row_stride;
  a.to_cols = dst_table ? dst_max_blocks : max_blocks_per_seq;
  a.keep = keep;
  a.cu = cu_seqlens;
  a.width = keep_width;
  a.keep_rows = num_keep;
  a.first = first;
  a.counts = counts;
  a.num_seqs = num_seqs;
  a.pieces = row_bytes / 16;
  a.pieces_shift = -1;
  for (int x = 0; x < 16; ++x)
    if (a.pieces == 1 << x) a.pieces_shift = x;
  const int64_t units = (int64_t)num_seqs * num_kv_heads;
  const int main = 2 * num_layers, small = (scales ? main : 0) + (mass ? 1 : 0);
  const hipStream_t s = (hipStream_t)stream;
  if (!grid_fits(units, 1024)) return NDL_ERR_UNSUPPORTED;
  const bool waves = dst_table || most <= 64 || cu_seqlens;      // a wave a list, or a piece of one
  // Pieces of a list: 64 rows and more, up to two rounds of the waves that the GPU holds; planes to
  // a wave: more where there are lists enough.
  int64_t z = 1;
  a.planes_each = 1;
  if (waves) {
    const int64_t hold = 256 * 32;
    if (dst_table) {
      z = (most + 63) / 64;
      const int64_t fill = 2 * hold / (units * (main + small)) + 1;
      if (z > fill) z = fill;
      if (z > 65535) z = 65535;
    }
    const int64_t each = units * z * main / hold;
    a.planes_each = (int)(each < 1 ? 1 : each > 8 ? 8 : each);
  }
  const int groups = (main + a.planes_each - 1) / a.planes_each;
  const dim3 grid((unsigned)(waves ? (units + 3) / 4 : units), (unsigned)(groups + small),
                  (unsigned)z);
  if (dst_table)
    hipLaunchKernelGGL((kv_move_kernel<1, false>), grid, dim3(256), 0, s, a);
  else if (waves)
    hipLaunchKernelGGL((kv_move_kernel<1, true>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((kv_move_kernel<16, true>), grid, dim3(1024), 0, s, a);
  return check_launch();
}

extern "C" int ndl_kv_select(int32_t* keep, int32_t* kept, const float* mass, int64_t num_blocks,
                             int num_kv_heads, int block_size, const int32_t* block_table,
                             int64_t bt_row_stride, int max_blocks_per_seq, const int32_t* lens,
                             int num_seqs, int budget, int sinks, int recent, ndl_stream_t stream) {
  using namespace ndl;
  if (num_blocks <= 0 || num_kv_heads <= 0 || block_size <= 0 || max_blocks_per_seq <= 0 ||
      bt_row_stride < max_blocks_per_seq || num_seqs < 0 || budget <= 0 || sinks < 0 ||
      recent < 0 || (int64_t)sinks + recent > budget)
    return NDL_ERR_INVALID_ARG;
  if (num_seqs == 0) return NDL_OK;
  if (!keep || !kept || !mass || !block_table || !lens || (uintptr_t)mass & 3u)
    return NDL_ERR_INVALID_ARG;
  // (positions and entries of a list are counted on by a workgroup's threads in 31 bits)
  if (num_seqs > 65535 || budget > 0x7fff0000 || !grid_fits(num_kv_heads, kSelThreads) ||
      (int64_t)max_blocks_per_seq * block_size > 0x7fff0000)
    return NDL_ERR_UNSUPPORTED;
  SelectArgs a{keep, kept, mass, num_blocks, num_kv_heads, block_size, block_table, bt_row_stride,
               max_blocks_per_seq, lens, budget, sinks, recent};
  const dim3 grid((unsigned)num_kv_heads, (unsigned)num_seqs);
  if ((int64_t)max_blocks_per_seq * block_size <= kHeldFew)
    hipLaunchKernelGGL((kv_select_kernel<kHeldFew>), grid, dim3(kSelThreads), 0,
                       (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((kv_select_kernel<kHeldMany>), grid, dim3(kSelThreads), 0,
                       (hipStream_t)stream, a);
  return check_launch();
}
