// Microscaled 4-bit weights: layout and decoding.
//
// A value is q 2^E: q = (-1)^s {0, 0.5, 1, 1.5, 2, 3, 4, 6} in 4 bits (sign, two exponent bits, one of mantissa) and E
// shared by 32 neighbours along K, stored as the byte E + 127 (255: not a number), after the OCP microscaling formats.
//
// A weight [N, K] is cut into pieces of 64 rows x 64 columns, two rows of pieces to a tile of 128 rows: piece
// ((n / 128, k / 64), n / 64 % 2) after piece, K padded to 128 and N to 128 with zeros, so that whatever a tile of a
// product reads lies in the buffer.  A piece is
//   codes   [2 halves of 32 columns][64 rows][16 bytes],
//   scales  [2 halves][64 rows], one byte each.
// Two pieces make a stage of either product, y = x V^T (128 rows of 64 columns: neighbours) or grad_x = g V (64
// rows of 128 columns: two copies), and a warp whose lanes are 32 rows reads 512 contiguous bytes.  Of eight codes in a 32-bit word, elements 0, 2, 4, 6 are in the low half
// and 1, 3, 5, 7 in the high half: elements 2p and 2p + 1 come out as one register of two 16-bit values.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace lf {

constexpr int kMx4Rows = 128, kMx4Cols = 64;
constexpr int kMx4HalfBytes = 64 * 16;                // codes of 64 rows x 32 columns
constexpr int kMx4Codes = 2 * kMx4HalfBytes;          // where a piece's scales start
constexpr int kMx4Piece = kMx4Codes + 2 * 64;         // 2176 bytes
constexpr int kMx4Block = 2 * kMx4Piece;              // 128 rows x 64 columns
// Byte offsets in a block (or a stage of two pieces) of row r's 16 bytes of codes and its scale in half c.
__host__ __device__ inline int mx4_code_at(int r, int c) { return (r >> 6) * kMx4Piece + c * kMx4HalfBytes + (r & 63) * 16; }
__host__ __device__ inline int mx4_scale_at(int r, int c) { return (r >> 6) * kMx4Piece + kMx4Codes + c * 64 + (r & 63); }
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

// 32 codes (half c of row r of a stage in shared memory) as granules 4c .. 4c + 3 of a 128-byte row with the 128-byte
// swizzle: granule g of row r lies at slot g ^ (r % 8).
__device__ __forceinline__ void mx4_fetch(const uint8_t* stage, int r, int c, uint4& codes, uint32_t& scale) {
  codes = *reinterpret_cast<const uint4*>(stage + mx4_code_at(r, c));
  scale = stage[mx4_scale_at(r, c)];
}
template <typename T>
__device__ __forceinline__ void mx4_store(uint8_t* row, int r, int c, const uint4& codes, uint32_t scale) {
  const uint32_t s = Mx4<T>::scale(scale);
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(row + (((4 * c + j) ^ (r & 7)) << 4)) = Mx4<T>::decode(w[j], s);
}

}  // namespace lf
