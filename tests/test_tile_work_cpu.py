"""Who works on which chunk, and who arrives where, in the tile kernel of the 8-bit product: the kernel's own arithmetic
(csrc/tile_work.cuh) run on the host, with CTAs that give up at any of their units."""
import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "omnikv_b200" / "csrc"

SOURCE = r"""
#include <vector>
#include "tile_work.cuh"
using omnikv::TileWork;

// fail_at[cta]: the unit at which a CTA gives up (negative: never).  Returns 0, or which property does not hold.
extern "C" int run(int tiles, int shared, int sharers, int chunks, int ctas, const int* fail_at) {
  std::vector<int> counters(ctas, 0), seen((size_t)tiles * chunks, 0), finished(tiles, 0), first_of(ctas, -1);
  bool clean = true;
  int bad = 0;
  for (int cta = 0; cta < ctas; ++cta) {
    const TileWork work(tiles, shared, sharers, chunks, ctas, cta);
    const auto arrive = [&](const TileWork::Party& p, int tile) {
      if (p.first < 0 || p.first >= ctas || p.parts < 2) bad = 1;
      else if (first_of[p.first] >= 0 && first_of[p.first] != tile) bad = 2;  // one counter for two tiles
      else {
        first_of[p.first] = tile;
        if (++counters[p.first] == p.parts) counters[p.first] = 0, ++finished[tile];
      }
    };
    TileWork::Unit u;
    int n = 0;
    for (bool more = work.first(u); more; more = work.next(u), ++n) {
      if (u.tile < 0 || u.tile >= tiles || u.k0 < 0 || u.k0 >= u.k1 || u.k1 > chunks) return 3;
      if (fail_at[cta] == n) {
        clean = false;
        TileWork::Unit v = u;
        std::vector<int> left;
        for (bool m = true; m; m = work.next(v)) if (!work.whole(v)) left.push_back(v.tile);
        size_t i = 0;
        work.give_up(u, [&](const TileWork::Party& p) { arrive(p, left[i++]); });
        if (i != left.size()) return 4;
        break;
      }
      for (int k = u.k0; k < u.k1; ++k) ++seen[(size_t)u.tile * chunks + k];
      if (work.whole(u)) ++finished[u.tile];
      else arrive(work.party(u.tile), u.tile);
    }
  }
  if (bad) return bad;
  for (int c : counters) if (c) return 5;  // the next call would count from here
  if (clean)
    for (int s : seen) if (s != 1) return 6;
  for (int t = 0; t < tiles; ++t)
    if (finished[t] > 1 || (clean && finished[t] != 1)) return 7;
  return 0;
}
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    where = tmp_path_factory.mktemp("tile_work")
    (where / "t.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), str(where / "t.cpp"), "-o", str(where / "t.so")], check=True)
    lib = ctypes.CDLL(str(where / "t.so"))

    def call(tiles, shared, sharers, chunks, ctas, fail_at):
        return lib.run(tiles, shared, sharers, chunks, ctas, (ctypes.c_int * ctas)(*fail_at))

    return call


def layouts(rng):
    """(tiles, shared, sharers, chunks, ctas) as the plan makes them: whole tiles alone, m pieces per tile left over, or one
    piece per CTA."""
    ctas = 148
    chunks = rng.randint(2, 112)
    tiles = rng.randint(1, 5 * ctas)
    left = tiles % ctas
    if tiles <= ctas or not left:
        return tiles, 0, 0, chunks, min(ctas, tiles)
    pieces = [0] + [m * left for m in range(2, 7) if m * left <= ctas and m <= chunks] + ([ctas] if 2 * left > ctas else [])
    sharers = rng.choice(pieces)
    return tiles, left if sharers else 0, sharers, chunks, ctas


@pytest.mark.parametrize("seed", range(40))
def test_every_chunk_once_and_every_counter_back_at_zero(run, seed):
    rng = random.Random(seed)
    for _ in range(10):
        tiles, shared, sharers, chunks, ctas = layouts(rng)
        assert run(tiles, shared, sharers, chunks, ctas, [-1] * ctas) == 0, (tiles, shared, sharers, chunks)
        for share in (0.01, 0.3, 1.0):
            fail_at = [rng.randint(0, 3) if rng.random() < share else -1 for _ in range(ctas)]
            assert run(tiles, shared, sharers, chunks, ctas, fail_at) == 0, (tiles, shared, sharers, chunks, fail_at)
