// Microscaled 4-bit weights: layout and decoding.
//
// A value is q 2^E: q = (-1)^s {0, 0.5, 1, 1.5, 2, 3, 4, 6} in 4 bits (sign, two exponent bits, one of mantissa) and E
// shared by 32 neighbours along K, stored as the byte E + 127 (255: not a number), after the OCP microscaling formats.
//
// A weight [N, K] is cut into blocks of 128 rows x 64 columns, block (n / 128, k / 64) after block, K padded to 128 and
// N to 128 with zeros, so that whatever a tile of a product reads lies in the buffer.  A block is
//   codes   [2 halves of 32 columns][128 rows][16 bytes],
//   scales  [2 halves][128 rows], one byte each:
// a warp whose lanes are 32 rows reads 512 contiguous bytes, and the same bytes serve y = x V^T (64 columns of 128 rows)
// and grad_x = g V (64 rows of 128 columns).  Of eight codes in a 32-bit word, elements 0, 2, 4, 6 are in the low half
// and 1, 3, 5, 7 in the high half: elements 2p and 2p + 1 come out as one register of two 16-bit values.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace lf {

constexpr int kMx4Rows = 128, kMx4Cols = 64;
constexpr int kMx4HalfBytes = kMx4Rows * 16;                    // codes of 32 columns
constexpr int kMx4Codes = 2 * kMx4HalfBytes;                    // where the scales start
constexpr int kMx4Block = kMx4Codes + 2 * kMx4Rows;             // 4352 bytes
__host__ __device__ inline int mx4_row_tiles(int N) { return (N + kMx4Rows - 1) / kMx4Rows; }
__host__ __device__ inline int mx4_col_blocks(int K) { return (K + 127) / 128 * 2; }

// Four registers of two 16-bit values each from eight codes.  The code's exponent and mantissa bits, moved to the bottom
// of the type's exponent field, are the value times 2^-126 (bf16) or 2^-14 (f16), subnormal where the code's exponent is 0:
// a product with that power of two brings it back, a second one applies the scale.  Every step is exact (a power of two
// times two significant bits) while the value itself fits the type.  For f16 the first product stops 2^2 short and
// the scale makes up for it, so that scales down to 2^-26, those of float16's smallest weights, stay representable.
// 24 instructions for eight values; a table of byte permutes took as many.
template <typename T>
struct Mx4;
template <>
struct Mx4<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t scale(uint32_t s) {  // 2^(s - 127), twice
    const uint32_t v = s == 255u ? 0x7fc0u : s == 0u ? 0x0040u : s << 7;
    return v * 0x10001u;
  }
  static __device__ __forceinline__ uint32_t mul(uint32_t bits, uint32_t scale) {
    const uint32_t top = 0x7e807e80u;  // 2^126
    const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&bits),
                                     *reinterpret_cast<const __nv_bfloat162*>(&top));
    const __nv_bfloat162 r = __hmul2(v, *reinterpret_cast<const __nv_bfloat162*>(&scale));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint4 decode(uint32_t w, uint32_t scale) {
    constexpr uint32_t kMag = 0x01c001c0u, kSign = 0x80008000u;
    uint4 r;
    r.x = mul(((w << 6) & kMag) | ((w << 12) & kSign), scale);
    r.y = mul(((w << 2) & kMag) | ((w << 8) & kSign), scale);
    r.z = mul(((w >> 2) & kMag) | ((w << 4) & kSign), scale);
    r.w = mul(((w >> 6) & kMag) | (w & kSign), scale);
    return r;
  }
};
template <>
struct Mx4<__half> {
  static __device__ __forceinline__ uint32_t scale(uint32_t s) {  // 2^(s - 125), twice
    const int e = static_cast<int>(s) - 125;
    uint32_t v;
    if (s == 255u) v = 0x7e00u;
    else if (e >= -14) v = static_cast<uint32_t>((e < 15 ? e : 15) + 15) << 10;
    else v = e >= -24 ? 1u << (e + 24) : 0u;
    return v * 0x10001u;
  }
  static __device__ __forceinline__ uint32_t mul(uint32_t bits, uint32_t scale) {
    const uint32_t top = 0x6c006c00u;  // 2^12
    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&bits), *reinterpret_cast<const __half2*>(&top));
    const __half2 r = __hmul2(v, *reinterpret_cast<const __half2*>(&scale));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint4 decode(uint32_t w, uint32_t scale) {
    constexpr uint32_t kMag = 0x0e000e00u, kSign = 0x80008000u;
    uint4 r;
    r.x = mul(((w << 9) & kMag) | ((w << 12) & kSign), scale);
    r.y = mul(((w << 5) & kMag) | ((w << 8) & kSign), scale);
    r.z = mul(((w << 1) & kMag) | ((w << 4) & kSign), scale);
    r.w = mul(((w >> 3) & kMag) | (w & kSign), scale);
    return r;
  }
};

// 32 codes and their scale byte, in flight.  Weights are read once a tile: they do not displace what L1 holds.
struct Mx4Piece {
  uint4 codes;
  uint32_t scale;
};
__device__ __forceinline__ Mx4Piece mx4_load(const uint8_t* codes, const uint8_t* scale) {
  Mx4Piece p;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(p.codes.x), "=r"(p.codes.y), "=r"(p.codes.z), "=r"(p.codes.w)
               : "l"(codes));
  asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(p.scale) : "l"(scale));
  return p;
}
// The piece's 32 values as four 16-byte granules first .. first + 3 of a 128-byte row of shared memory with the 128-byte
// swizzle: granule g of row r lies at slot g ^ (r % 8).
template <typename T>
__device__ __forceinline__ void mx4_store(uint8_t* row, int r, int first, const Mx4Piece& p) {
  const uint32_t s = Mx4<T>::scale(p.scale);
  const uint32_t w[4] = {p.codes.x, p.codes.y, p.codes.z, p.codes.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(row + (((first + j) ^ (r & 7)) << 4)) = Mx4<T>::decode(w[j], s);
}

}  // namespace lf
