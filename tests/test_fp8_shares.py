"""The cut of row blocks into shares (needle_amd/csrc/chunk_shares.hpp), compiled for the host: the
parts that the attention's walk writes are the parts that its merge reads, all of them below
`shares + items`, and every tile is taken once (CPU)."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CXX = shutil.which("g++") or shutil.which("c++")

# The walk of chunk_attention_kernel over one kv head and the lookup of chunk_merge_kernel, with the
# header's arithmetic; Stream::find as a loop.
SOURCE = r"""
#define __device__
#define __forceinline__ inline
#include "chunk_shares.hpp"
#include <vector>
using namespace ndl;

// 0, or what is wrong; `worst` then holds (row block, its first slot, s0, s1).
extern "C" int check(const int* tiles, int items, int shares, int min_chunk, int pad, int* cuts,
                     int64_t* worst) {
  std::vector<int> first(items), slots(items);
  int total = 0;
  for (int e = 0; e < items; ++e) {
    first[e] = total;
    slots[e] = tiles[e] > 0 ? tiles[e] + pad : 0;
    total += slots[e];
  }
  const Cut cut = cut_of(total, shares, min_chunk, pad);
  cuts[0] = cut.chunk;
  cuts[1] = cut.snap;
  cuts[2] = 0;
  auto find = [&](int at) {
    int e = 0;
    while (!(slots[e] > 0 && first[e] + slots[e] > at)) ++e;
    return e;
  };
  auto begin = [&](int s) {
    const int x = s * cut.chunk;
    if (x >= total) return total;
    const int e = find(x);
    return share_begin(x, first[e], slots[e], cut.snap);
  };
  std::vector<std::vector<int>> written(items);   // shares with a part of the row block
  std::vector<int> done(items, 0), times(items, 0);
  for (int u = 0; u < shares; ++u) {
    const int from = begin(u), to = begin(u + 1);
    if (from >= to) continue;
    for (int e = find(from); e < items; ++e) {
      if (tiles[e] == 0) continue;
      if (first[e] >= to) break;
      int t0, t1;
      share_tiles(first[e], pad, tiles[e], from, to, &t0, &t1);
      if (t0 >= t1) return 1;                     // a share of empty slots only
      if (t0 != done[e]) return 2;                // a tile left out or taken twice
      done[e] = t1;
      if (t0 > 0 || t1 < tiles[e]) written[e].push_back(u);
      ++times[e];
    }
  }
  for (int e = 0; e < items; ++e) {
    if (done[e] != (tiles[e] > 0 ? tiles[e] : 0)) return 3;
    int s0 = 0, s1 = -1;
    const bool parts = slots[e] > 0 && share_parts(first[e], slots[e], cut, &s0, &s1);
    worst[0] = e;
    worst[1] = first[e];
    worst[2] = s0;
    worst[3] = s1;
    if (parts != !written[e].empty()) return 4;
    if (!parts) continue;
    ++cuts[2];
    if (s0 < 0 || s1 >= shares || (int)written[e].size() != s1 - s0 + 1) return 5;
    for (int s = s0; s <= s1; ++s)
      if (written[e][s - s0] != s || s + e >= shares + items) return 6;
  }
  return 0;
}

// Whether a row block at `first` of `slots`, whatever the cut was made for, has shares that there are.
extern "C" int within(int total, int shares, int min_chunk, int pad, int first, int slots) {
  int s0, s1;
  const Cut cut = cut_of(total, shares, min_chunk, pad);
  return !share_parts(first, slots, cut, &s0, &s1) || (s0 >= 0 && s0 < s1 && s1 < shares);
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if CXX is None:
        pytest.skip("no host C++ compiler")
    d = tmp_path_factory.mktemp("shares")
    (d / "shares.cpp").write_text(SOURCE)
    lib = d / "libshares.so"
    subprocess.check_call([CXX, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                           os.path.join(ROOT, "needle_amd", "csrc"), str(d / "shares.cpp"), "-o",
                           str(lib)])
    return ctypes.CDLL(str(lib))


@pytest.fixture
def check(lib):
    def run(tiles, shares, min_chunk, pad):
        cuts, worst = (ctypes.c_int * 3)(), (ctypes.c_int64 * 4)()
        rc = lib.check((ctypes.c_int * len(tiles))(*tiles), len(tiles), shares, min_chunk, pad, cuts, worst)
        assert rc == 0, (rc, tiles[:8], shares, min_chunk, pad, list(cuts), list(worst))
        return list(cuts)
    return run


def _tiles(tokens):
    return -(-tokens // 32)


@pytest.mark.parametrize("lens,shares,pad", [
    ([100] + [4000] * 63, 64, 1),            # 64 decodes of 32/8 heads of 128
    ([30] + [2048] * 31, 64, 1),
    ([200] + [16384] * 23, 128, 1),          # 28/4 heads of 128
    ([20] + [8000] * 63, 512, 1),            # 14/2 heads of 64
    ([100] + [2000] * 63, 64, 1),
    ([65] + [4005] * 63, 64, 4),             # chunks of five tokens
    ([1, 1, 1, 20, 0, 33] + [4000] * 60, 64, 1),
])
def test_short_row_blocks_before_long_ones(check, lens, shares, pad):
    chunk, snap, _ = check([_tiles(n) for n in lens], shares, 8, pad)
    assert snap > pad and _tiles(lens[0]) + pad <= snap


@pytest.mark.parametrize("pad", [1, 4])
def test_random_lengths(check, pad):
    rng = random.Random(7 + pad)
    snapped = 0
    for n in range(4000):
        items = rng.choice((1, 2, 3, 7, 24, 64, 65, 130, 300))
        shares = 8 * rng.choice((1, 2, 8, 16, 32, 64))
        chunk = rng.randint(8, 200)            # about what a share gets
        long = max(1, chunk * shares // items)
        kind = rng.random()
        tiles = [rng.randint(0, 2 * long) if kind < 0.4 else
                 int(long ** rng.random()) if kind < 0.7 else long for _ in range(items)]
        for e in range(rng.choice((0, 1, 1, 2, 5))):      # short ones in front, in between, last
            at = rng.choice((e % items, rng.randrange(items), items - 1))
            tiles[at] = rng.randint(0, 20)
        if not any(tiles):
            continue
        cuts = check(tiles, shares, 8, pad)
        snapped += cuts[1] > pad and cuts[2] > 0
    assert snapped > 500


def test_lengths_that_changed_since_the_cut(lib):
    """More than 256 row blocks are looked up by another read of the lengths than the cut's."""
    rng = random.Random(3)
    for _ in range(20000):
        total, slots = (int(2 ** rng.uniform(0, 24)) for _ in range(2))
        first = rng.choice((0, rng.randint(0, 2 * total)))
        assert lib.within(total, 8 * rng.randint(1, 128), 8, rng.choice((1, 4)), first, slots)
