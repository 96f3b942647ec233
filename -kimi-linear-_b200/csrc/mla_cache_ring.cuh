// mla_cache_ring.cuh -- places and barriers of the latent attention's ring of chunks.
// Plain C++, so that the order of waits, arms and copies can also be followed on a CPU
// (tests/test_latent_ring.py).
#pragma once

#ifdef __CUDACC__
#define KDA_RING_FN __host__ __device__ __forceinline__
#else
#define KDA_RING_FN inline
#endif

namespace kda {
namespace cache {

// A ring holds at most kRingTiles tiles of `tile_chunks` chunks.  A tile comes in two
// halves, chunks 0 .. half - 1 and the others (there may be none), that land and are freed
// apart: half h of tile k is half tile 2 k + h.  Barrier `full` of a half tile: it has
// landed; `freed`: the products have read it.
//
// `full` counts one arrival, the one that arms it with the bytes to come, and a second
// arrival in an unfinished phase is undefined.  The loading warp arms tile k before it
// waits for any of its places, when all it knows is that tile k - 1 had its own: that
// tile k - 5 has been read, but in a ring of more than three tiles not that tile k - 4 has
// landed.  So the barriers of tile k may be those of tile k - 8, not of tile k - 4.  (Armed
// behind the waits, four pairs would do; but the copies then go out later: 512 tokens
// against 8192 positions, KVL 512, 220 us for 212 us.)
constexpr int kRingTiles = 4, kStages = 8;
KDA_RING_FN constexpr int half_barrier(int half_tile) { return half_tile & (2 * kStages - 1); }
KDA_RING_FN constexpr unsigned half_parity(int half_tile) {
  return static_cast<unsigned>(half_tile) / (2 * kStages) & 1;
}

// Copies may be in flight for the half tiles from this one up to 2 tiles - 1, when `tiles`
// tiles have been armed: a ring's worth and the last one, which may have found no place;
// each has a barrier of its own.
KDA_RING_FN constexpr int first_in_flight(int tiles) {
  return tiles <= kRingTiles ? 0 : 2 * (tiles - kRingTiles - 1);
}

struct Ring {
  int tile_chunks, half;
  int ahead, spare;              // the ring in tiles, and the chunks over
  KDA_RING_FN Ring(int ring, int tile_chunks_, int half_)
      : tile_chunks(tile_chunks_), half(half_), ahead(ring / tile_chunks_), spare(ring % tile_chunks_) {}
  // The half tile that held the place of chunk c of tile k before (negative: none did).
  KDA_RING_FN int held_by(int k, int c) const {
    const int j = k - ahead - (c < spare), old = c - spare + (c < spare ? tile_chunks : 0);
    return 2 * j + (old >= half);
  }
  // A loader that gives up before chunk c of a tile has armed the whole tile: how many
  // chunks of half h it has not asked for.  With their bytes given back, what is armed
  // completes once the copies in flight have landed.
  KDA_RING_FN int missing(int c, int h) const {
    return h == 0 ? (c < half ? half - c : 0) : tile_chunks - (c < half ? half : c);
  }
};

}  // namespace cache
}  // namespace kda
