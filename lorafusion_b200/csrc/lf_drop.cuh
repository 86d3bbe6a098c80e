// Dropout whose mask is computed where it is used.
//
// Element (t, k) of the adapters' input is kept where a 16-bit random number is at least the row's threshold, 65536 times
// its adapter's rate.  The numbers come from Philox 4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", 2011): key = the seed's halves, counter = (k / 8, t, the offset's halves).  The 128
// bits serve elements k .. k + 7 of row t: word (k % 8) / 2, its low half for an even k.  A mask thus depends on seed,
// offset and position alone: forward and backward, every tiling and every path compute the same one.
#pragma once

#include <stdint.h>

#include "lf_internal.cuh"

namespace lf {

__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, uint64_t offset, uint64_t seed) {
  uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// All ones in each 16-bit half of `word` whose number keeps its element.  `threshold` is below 65536.
__device__ __forceinline__ uint32_t keep2(uint32_t word, uint32_t threshold) {
  return ((word & 0xffffu) >= threshold ? 0x0000ffffu : 0u) | ((word >> 16) >= threshold ? 0xffff0000u : 0u);
}

// Threshold of row `row` of tile `tile`: that of the segment that holds the row (several where the adapter has more than
// one virtual slot: theirs are the same).  0 where no segment does.
__device__ __forceinline__ uint32_t row_threshold(const Tables& tb, const DropArgs& d, int tile, int row) {
  const int e = tb.tile_st(tile + 1);
  for (int st = tb.tile_st(tile); st < e; ++st)
    if (row >= tb.st_lo(st) && row < tb.st_hi(st)) return d.threshold[tb.st_slot(st)];
  return 0;
}

}  // namespace lf
