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

// Numbers of N counters (c0[i], c1), round by round: 76 cycles of an SM quarter's issue a counter and warp, 97 where one
// counter's ten dependent rounds are all a warp has to do.
template <int N>
__device__ __forceinline__ void philox(const uint32_t (&c0)[N], uint32_t c1, const DropArgs& d, uint4 (&r)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j)
    r[j] = make_uint4(c0[j], c1, static_cast<uint32_t>(d.offset), static_cast<uint32_t>(d.offset >> 32));
#pragma unroll
  for (int i = 0; i < 10; ++i) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint64_t a = static_cast<uint64_t>(r[j].x) * 0xD2511F53u, b = static_cast<uint64_t>(r[j].z) * 0xCD9E8D57u;
      r[j] = make_uint4(static_cast<uint32_t>(b >> 32) ^ r[j].y ^ d.key[2 * i], static_cast<uint32_t>(b),
                        static_cast<uint32_t>(a >> 32) ^ r[j].w ^ d.key[2 * i + 1], static_cast<uint32_t>(a));
    }
  }
}
__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, const DropArgs& d) {
  const uint32_t c[1] = {c0};
  uint4 r[1];
  philox<1>(c, c1, d, r);
  return r[0];
}

// Two 16-bit elements, zeros where the word's halves drop them; `high` is the threshold (below 65536) shifted left by 16.
// The upper number is below the threshold where the whole word is below `high`.  (Built as a mask of compares and
// selects it took half as long as the generator itself.)
__device__ __forceinline__ uint32_t keep2(uint32_t v, uint32_t word, uint32_t high) {
  if (word < high) v &= 0x0000ffffu;
  if ((word << 16) < high) v &= 0xffff0000u;
  return v;
}

// Threshold of row `row` of tile `tile`: that of the segment that holds the row (several where the adapter has more than
// one virtual slot: theirs are the same).  0 where no segment does.
__device__ __forceinline__ uint32_t row_threshold(const Tables& tb, const DropArgs& d, int tile, int row) {
  const int e = tb.tile_st(tile + 1);
  for (int st = tb.tile_st(tile); st < e; ++st)
    if (row >= tb.st_lo(st) && row < tb.st_hi(st)) return d.threshold[tb.st_slot(st)];
  return 0;
}

// Masks tiles of 128 rows of 128 bytes (128-byte swizzle) in shared memory in place, a lane a row and four of its granules
// of eight elements at a time.  The numbers of the first four do not wait for the tile.
struct RowMask {
  uint32_t row, t, high;  // row of the tile, its number in the batch, `high` as in keep2
  __device__ __forceinline__ void numbers(int kb, int first, const DropArgs& d, uint4 (&r)[4]) const {
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = static_cast<uint32_t>(kb * 8 + first + j);  // kb: the block of K
    philox<4>(c, t, d, r);
  }
  __device__ __forceinline__ void keep(uint8_t* tile, int first, const uint4 (&r)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4* p = reinterpret_cast<uint4*>(tile + row * 128 + (((first + j) ^ (row & 7)) << 4));
      uint4 v = *p;
      v.x = keep2(v.x, r[j].x, high), v.y = keep2(v.y, r[j].y, high);
      v.z = keep2(v.z, r[j].z, high), v.w = keep2(v.w, r[j].w, high);
      *p = v;
    }
  }
};

}  // namespace lf
