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
// Bound: the rows, read and written once, and the trips before them (index, block id, row: three, the
// index and the block ids of the next rows under way while these move).
//   * A row is whole 16-byte pieces, a lane each (a scale byte or a weight: a lane a row).
//   * In place the indices ascend, so a row's source is never written before it is read: a later row
//     has a later source and a later place.  One wave (short lists) or one workgroup (long ones, a
//     barrier between the reads of a step and its writes) takes a list from front to back.
//   * Into other blocks nothing is ordered, and lists are cut into as many pieces as fill the GPU.
constexpr int kMaxPools = 128;
constexpr int kItems = 4;         // pieces of a lane under way

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
};

// Positions and blocks of row j of a list: byte offsets of its source and its place, -1 where there
// is none (nothing to do for row j).
struct Move {
  int64_t from, to;
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
__device__ __forceinline__ Move move_of(const MoveArgs& a, const List& l, int j, int head,
                                        int row_bytes) {
  Move m{-1, -1};
  if (j >= l.n) return m;
  const int k = l.keep[j];
  const int64_t s = l.base + k, d = l.base + j;
  if (k < 0 || s >= (int64_t)a.table_cols * a.block_size ||
      d >= (int64_t)a.to_cols * a.block_size)
    return m;
  const uint32_t bs = (uint32_t)a.block_size;
  const uint32_t sc = (uint32_t)s / bs, dc = (uint32_t)d / bs;
  const int sb = l.table[sc], db = l.to[dc];
  if (sb < 0 || sb >= a.num_blocks || db < 0 || db >= a.num_blocks) return m;
  const int64_t from =
      (((int64_t)sb * a.num_kv_heads + head) * bs + ((uint32_t)s - sc * bs)) * row_bytes;
  const int64_t to =
      (((int64_t)db * a.num_kv_heads + head) * bs + ((uint32_t)d - dc * bs)) * row_bytes;
  if (from == to) return m;
  return Move{from, to};
}

// THREADS threads take the rows j0 .. j1 - 1 of a list, WORD bytes a piece.
template <int THREADS, bool IN_PLACE, class WORD>
__device__ __forceinline__ void move_rows(const MoveArgs& a, const List& l, char* plane, int head,
                                          int row_bytes, int t, int j0, int j1) {
  const int pieces = row_bytes / (int)sizeof(WORD);      // of a row
  const int total = (j1 - j0) * pieces;                  // fits: the entry point checks
  auto slots = [&](int i0, Move* m) {
#pragma unroll
    for (int x = 0; x < kItems; ++x) {
      const int i = i0 + x * THREADS + t, j = (int)((uint32_t)i / (uint32_t)pieces);
      m[x] = i < total ? move_of(a, l, j0 + j, head, row_bytes) : Move{-1, -1};
      const int64_t in = (int64_t)(i - j * pieces) * (int)sizeof(WORD);
      if (m[x].from >= 0) {
        m[x].from += in;
        m[x].to += in;
      }
    }
  };
  Move next[kItems];
  slots(0, next);
  for (int i0 = 0; i0 < total; i0 += kItems * THREADS) {
    Move m[kItems];
    WORD v[kItems];
#pragma unroll
    for (int x = 0; x < kItems; ++x) {
      m[x] = next[x];
      if (m[x].from >= 0) v[x] = *reinterpret_cast<const WORD*>(plane + m[x].from);
    }
    if (i0 + kItems * THREADS < total) slots(i0 + kItems * THREADS, next);
    // every read of this step before its writes: within a wave by their order (a place written here
    // is before the sources still on their way), across waves by a wait and a barrier
    if constexpr (IN_PLACE && THREADS > 64) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < kItems; ++x)
      if (m[x].from >= 0) *reinterpret_cast<WORD*>(plane + m[x].to) = v[x];
  }
}

// blockIdx.x: lists (sequence, kv head), 256 / THREADS of them to a workgroup where a wave takes one;
// blockIdx.y: the planes of the pools, of their scales, the weights; blockIdx.z: a piece of the list.
template <int THREADS, bool IN_PLACE>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void kv_move_kernel(MoveArgs a) {
  constexpr int kBlock = THREADS < 256 ? 256 : THREADS;
  const int t = threadIdx.x % THREADS;
  const int64_t unit = (int64_t)blockIdx.x * (kBlock / THREADS) + threadIdx.x / THREADS;
  if (unit >= (int64_t)a.num_seqs * a.num_kv_heads) return;
  const int seq = (int)(unit / a.num_kv_heads), head = (int)(unit - (int64_t)seq * a.num_kv_heads);
  const List l = list_of(a, seq, head);
  int j0 = 0, j1 = l.n;
  if (!IN_PLACE) {
    const int per = (l.n + (int)gridDim.z - 1) / (int)gridDim.z;
    j0 = per * (int)blockIdx.z;
    j1 = j0 + per < l.n ? j0 + per : l.n;
  }
  if (j0 >= j1) return;
  const int64_t rows = a.num_blocks * a.num_kv_heads * a.block_size;    // of a plane
  const int y = blockIdx.y, main = 2 * a.pools;
  if (y < main) {
    move_rows<THREADS, IN_PLACE, u32x4>(a, l, a.pool[y >> 1] + (y & 1) * rows * a.row_bytes, head,
                                        a.row_bytes, t, j0, j1);
  } else if (y == main && a.mass) {
    move_rows<THREADS, IN_PLACE, uint32_t>(a, l, reinterpret_cast<char*>(a.mass), head, 4, t, j0,
                                           j1);
  } else {
    const int s = y - main - (a.mass ? 1 : 0);
    move_rows<THREADS, IN_PLACE, uint8_t>(a, l, a.scales[s >> 1] + (s & 1) * rows, head, 1, t, j0,
                                          j1);
  }
}

// ---------------------------------------------------------------- the rows that stay
//
// Of a kv head's L cached tokens the `budget` that stay: the first `sinks`, the last `recent`, and of
// those between the largest weights, of equal ones the first, in the order of their positions.
// A workgroup per (kv head, sequence): a radix select over the weights as ordered 32-bit keys, eight
// bits a pass from the top, then one pass that writes positions.  Bound: the passes' trips through
// LDS (keys are read from the pool once; those past kHeld again each pass) for few and short lists,
// which leave most of the GPU idle.
constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kHeld = 15360;          // keys in LDS (64 KiB in all: more a launch has to ask for)

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

__global__ __launch_bounds__(kSelThreads) void kv_select_kernel(SelectArgs a, int held) {
  extern __shared__ uint32_t keys[];                     // [held]
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
  const int n = len - a.sinks - a.recent;                // candidates, more than want
  if (want == 0) return;
  const int32_t* const table = a.table + seq * a.table_stride;
  const uint32_t bs = (uint32_t)a.block_size;
  auto load = [&](int i) {
    const uint32_t p = (uint32_t)(a.sinks + i), c = p / bs;
    const int b = table[c];
    if (b < 0 || b >= a.num_blocks) return 0u;
    return key_of(a.mass[((int64_t)b * a.num_kv_heads + head) * bs + (p - c * bs)]);
  };
  auto key = [&](int i) { return i < held ? keys[i] : load(i); };
#pragma unroll 4
  for (int i = t; i < n && i < held; i += kSelThreads) keys[i] = load(i);
  // The want-th largest key: its bits from the top, those above fixed as `prefix`.
  uint32_t prefix = 0;
  int left = want;                                       // of those that share the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (t < 256) hist[t] = 0;
    __syncthreads();
    const uint32_t fixed = shift == 24 ? 0u : ~0u << (shift + 8);
    for (int i = t; i < n; i += kSelThreads) {
      const uint32_t k = key(i);
      const bool in = (k & fixed) == prefix;
      // lanes with the digit of the first one count at once (weights of 0 are many)
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
  const int run = (n + kSelWaves - 1) / kSelWaves;
  const int i0 = wv * run, i1 = i0 + run < n ? i0 + run : n;
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
    if (mine) out[a.sinks + at + __builtin_popcountll(take & below)] = a.sinks + b + lane;
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
      (int64_t)dst_max_blocks * block_size > 0x7fffff00 || most * (row_bytes / 16) > 0x7fff0000)
    return NDL_ERR_UNSUPPORTED;
  MoveArgs a{};
  for (int i = 0; i < num_layers; ++i) {
    a.pool[i] = (char*)pools[i];
    if (!pools[i] || (uintptr_t)pools[i] & 15u) return NDL_ERR_INVALID_ARG;
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
  const int64_t units = (int64_t)num_seqs * num_kv_heads;
  const int planes = 2 * num_layers * (scales ? 2 : 1) + (mass ? 1 : 0);
  const hipStream_t s = (hipStream_t)stream;
  if (!grid_fits(units, 1024)) return NDL_ERR_UNSUPPORTED;
  if (dst_table) {
    // pieces of a list: what its longest needs, up to four rounds of the GPU's workgroups
    const int64_t step = (int64_t)256 * kItems * 16 / row_bytes;
    int64_t z = (most + step - 1) / step;
    const int64_t fill = (4 * 2048 + units * planes - 1) / (units * planes);
    if (z > fill) z = fill;
    if (z > 65535) z = 65535;
    hipLaunchKernelGGL((kv_move_kernel<256, false>),
                       dim3((unsigned)units, (unsigned)planes, (unsigned)z), dim3(256), 0, s, a);
  } else if (most <= 64 || cu_seqlens) {
    hipLaunchKernelGGL((kv_move_kernel<64, true>), dim3((unsigned)((units + 3) / 4), (unsigned)planes),
                       dim3(256), 0, s, a);
  } else {
    hipLaunchKernelGGL((kv_move_kernel<1024, true>), dim3((unsigned)units, (unsigned)planes),
                       dim3(1024), 0, s, a);
  }
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
  if (num_seqs > 65535 || (int64_t)max_blocks_per_seq * block_size > 0x7fffff00)
    return NDL_ERR_UNSUPPORTED;
  SelectArgs a{keep, kept, mass, num_blocks, num_kv_heads, block_size, block_table, bt_row_stride,
               max_blocks_per_seq, lens, budget, sinks, recent};
  const int64_t cap = (int64_t)max_blocks_per_seq * block_size;
  const int held = (int)(cap < kHeld ? cap : kHeld);
  hipLaunchKernelGGL(kv_select_kernel, dim3((unsigned)num_kv_heads, (unsigned)num_seqs),
                     dim3(kSelThreads), held * 4, (hipStream_t)stream, a, held);
  return check_launch();
}
