// Which chunks of which tiles a CTA of the tile kernel (linear_w8a8.cu) works on, and who shares a tile with whom.  Plain
// arithmetic that the host can run too.
#pragma once

#ifdef __CUDACC__
#define OMNIKV_HD __host__ __device__ __forceinline__
#else
#include <algorithm>
#define OMNIKV_HD inline
#endif

namespace omnikv {
#ifndef __CUDACC__
using std::min;
#endif

// First the piece [lo, hi) of the list of all shared tiles' chunks (the last `shared` tiles, cut into `sharers` pieces of a
// chunk or more), then whole tiles: cta, cta + ctas, ...
struct TileWork {
  int chunks, whole_tiles, total, sharers, ctas, cta, lo, hi;

  struct Unit {
    int tile, k0, k1;
  };
  struct Party {  // the CTAs first, first + 1, ... that share a tile; `first` is that of no other tile
    int first, parts;
  };

  OMNIKV_HD TileWork(int tiles, int shared, int sharers_, int chunks_, int ctas_, int cta_)
      : chunks(chunks_), whole_tiles(tiles - shared), total(shared * chunks_), sharers(sharers_), ctas(ctas_), cta(cta_) {
    lo = piece_lo(cta);
    hi = piece_lo(cta + 1);
  }
  OMNIKV_HD int piece_lo(int i) const { return sharers ? (int)((long long)min(i, sharers) * total / sharers) : 0; }
  OMNIKV_HD bool first(Unit& u) const {  // false: no work
    if (lo < hi) u = Unit{whole_tiles + lo / chunks, lo % chunks, min(chunks, lo % chunks + hi - lo)};
    else u = Unit{cta, 0, chunks};
    return lo < hi || cta < whole_tiles;
  }
  OMNIKV_HD bool next(Unit& u) const {
    if (u.tile >= whole_tiles) {
      const int at = (u.tile - whole_tiles) * chunks + u.k1;
      if (at < hi) {
        u = Unit{u.tile + 1, 0, min(chunks, hi - at)};
        return true;
      }
      u = Unit{cta, 0, chunks};
    } else {
      u.tile += ctas;
    }
    return u.tile < whole_tiles;
  }
  OMNIKV_HD bool whole(const Unit& u) const { return u.k1 - u.k0 == chunks; }
  OMNIKV_HD int owner(int chunk) const {  // the CTA whose piece has this chunk
    int i = min(sharers - 1, (int)(((float)chunk + 0.5f) * (float)sharers / (float)total));
    while (piece_lo(i) > chunk) --i;
    while (piece_lo(i + 1) <= chunk) ++i;
    return i;
  }
  OMNIKV_HD Party party(int tile) const {
    const int at = (tile - whole_tiles) * chunks, first = owner(at);
    return Party{first, owner(at + chunks - 1) - first + 1};
  }
  // arrive(party) for every tile that this CTA shares, from unit u on: a CTA that gives up still arrives where others count it.
  template <typename Arrive>
  OMNIKV_HD void give_up(Unit u, const Arrive& arrive) const {
    for (bool more = true; more; more = next(u))
      if (!whole(u)) arrive(party(u.tile));
  }
};

}  // namespace omnikv
