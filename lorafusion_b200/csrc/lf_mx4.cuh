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
// rows of 128 columns: two copies), and a warp whose lanes are 32 rows reads 512 contiguous bytes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace lf {

constexpr int kMx4Rows = 128;
constexpr int kMx4HalfBytes = 64 * 16;                // codes of 64 rows x 32 columns
constexpr int kMx4Codes = 2 * kMx4HalfBytes;          // where a piece's scales start
constexpr int kMx4Piece = kMx4Codes + 2 * 64;         // 2176 bytes
constexpr int kMx4Block = 2 * kMx4Piece;              // 128 rows x 64 columns
// Byte offsets in a block (or a stage of two pieces) of row r's 16 bytes of codes and its scale in half c.
__host__ __device__ inline int mx4_code_at(int r, int c) { return (r >> 6) * kMx4Piece + c * kMx4HalfBytes + (r & 63) * 16; }
__host__ __device__ inline int mx4_scale_at(int r, int c) { return (r >> 6) * kMx4Piece + kMx4Codes + c * 64 + (r & 63); }
__host__ __device__ inline int mx4_row_tiles(int N) { return (N + kMx4Rows - 1) / kMx4Rows; }
__host__ __device__ inline int mx4_col_blocks(int K) { return (K + 127) / 128 * 2; }

// Eight codes in a 32-bit word: elements 0, 2, 4, 6 in the low half, 1, 3, 5, 7 in the high half, so that elements 2p and
// 2p + 1 come out as one register of two 16-bit values.  A code's three bits of exponent and mantissa, moved to the bottom of
// the type's exponent field, are the value times 2^-126 (bf16) or 2^-14 (f16), subnormal where the code's exponent is 0; one
// product with that power and the scale brings it back, exactly while the value itself fits the type.  The bits of a
// half are placed so that most codes need one shift and one mask: 11 logic instructions and 4 products for eight
// values (codes in order took 15, and a byte table by permutes as many; the decoding warps of the CTA-pair GEMM are bound by
// what they issue).  Where the factor leaves the type's range, scales above 1 and NaN, the two powers are applied one
// after the other.
__device__ __forceinline__ void mx4_pairs(uint32_t codes, uint32_t& a, uint32_t& b) {
  const uint32_t even = codes & 0x0f0f0f0fu, odd = (codes >> 4) & 0x0f0f0f0fu;
  a = __byte_perm(even, odd, 0x5410);
  b = __byte_perm(even, odd, 0x7632);
}
template <typename T>
struct Mx4;
template <>
struct Mx4<__nv_bfloat16> {
  static constexpr uint32_t kMask = 0x81c081c0u, kSign = 0x80008000u;
  // the word of eight codes in order, four bits each
  static __device__ __forceinline__ uint32_t word(uint32_t codes) {
    uint32_t a, b;  // of each half: elements 0 and 2 (1 and 3), then 4 and 6 (5 and 7), a byte each
    mx4_pairs(codes, a, b);
    return (a & 0x00080008u) << 12 | (a & 0x00070007u) << 6 | (a & 0x08000800u) << 1 | (a & 0x07000700u) >> 5 |
           (b & 0x00080008u) << 6 | (b & 0x00070007u) | (b & 0x08000800u) << 3 | (b & 0x06000600u) << 1 |
           (b & 0x01000100u) << 5;
  }
  static __device__ __forceinline__ uint4 bits(uint32_t w) {
    uint4 r;
    r.x = w & kMask;
    r.y = (w << 3) & kMask;
    r.z = (w << 6) & kMask;
    r.w = ((w << 1) & kSign) | ((w >> 3) & 0x01800180u) | ((w >> 7) & 0x00400040u);
    return r;
  }
  static __device__ __forceinline__ uint32_t mul(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ bool one_factor(uint32_t s0, uint32_t s1) { return (s0 | s1) < 128u; }
  static __device__ __forceinline__ uint32_t factor(uint32_t s) { return s * 0x00800080u + 0x3f003f00u; }  // 2^(s - 1), twice
  static constexpr uint32_t kUp = 0x7e807e80u;                    // 2^126
  static __device__ __forceinline__ uint32_t scale(uint32_t s) {  // 2^(s - 127), twice
    return (s == 255u ? 0x7fc0u : s == 0u ? 0x0040u : s << 7) * 0x10001u;
  }
};
template <>
struct Mx4<__half> {
  static constexpr uint32_t kMask = 0x8e008e00u, kSign = 0x80008000u;
  static __device__ __forceinline__ uint32_t word(uint32_t codes) {
    uint32_t a, b;
    mx4_pairs(codes, a, b);
    return (a & 0x00080008u) << 12 | (a & 0x00070007u) << 9 | (a & 0x08000800u) << 1 | (a & 0x07000700u) >> 2 |
           (b & 0x00080008u) << 11 | (b & 0x00070007u) << 3 | (b & 0x08000800u) << 2 | (b & 0x07000700u) >> 8;
  }
  static __device__ __forceinline__ uint4 bits(uint32_t w) {
    constexpr uint32_t kMag = 0x0e000e00u;
    uint4 r;
    r.x = w & kMask;
    r.y = (w << 3) & kMask;
    r.z = ((w << 1) & kSign) | ((w << 6) & kMag);
    r.w = ((w << 2) & kSign) | ((w << 9) & kMag);
    return r;
  }
  static __device__ __forceinline__ uint32_t mul(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  // (a float16 weight's scales are 2^-26 at least)
  static __device__ __forceinline__ bool one_factor(uint32_t s0, uint32_t s1) { return (s0 | s1) < 128u && min(s0, s1) >= 99u; }
  static __device__ __forceinline__ uint32_t factor(uint32_t s) { return (s - 98u) * 0x04000400u; }  // 2^(s - 113), twice
  static constexpr uint32_t kUp = 0x6c006c00u;                    // 2^12: a fourth of the value, so that scales down to
  static __device__ __forceinline__ uint32_t scale(uint32_t s) {  // 2^(s - 125), twice: 2^-26 is still representable
    const int e = static_cast<int>(s) - 125;
    uint32_t v;
    if (s == 255u) v = 0x7e00u;
    else if (e >= -14) v = static_cast<uint32_t>((e < 15 ? e : 15) + 15) << 10;
    else v = e >= -24 ? 1u << (e + 24) : 0u;
    return v * 0x10001u;
  }
};

// 8 N values from N words that share a scale.
template <typename T, int N, bool kOne>
__device__ __forceinline__ void mx4_values(const uint32_t (&w)[N], uint32_t s, uint4* v) {
  const uint32_t f = kOne ? Mx4<T>::factor(s) : Mx4<T>::scale(s);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint4 b = Mx4<T>::bits(w[i]);
    if (!kOne) b.x = Mx4<T>::mul(b.x, Mx4<T>::kUp), b.y = Mx4<T>::mul(b.y, Mx4<T>::kUp), b.z = Mx4<T>::mul(b.z, Mx4<T>::kUp),
               b.w = Mx4<T>::mul(b.w, Mx4<T>::kUp);
    v[i].x = Mx4<T>::mul(b.x, f), v[i].y = Mx4<T>::mul(b.y, f), v[i].z = Mx4<T>::mul(b.z, f), v[i].w = Mx4<T>::mul(b.w, f);
  }
}

// 32 codes (half c of row r of a stage in shared memory) as granules 4c .. 4c + 3 of a 128-byte row with the 128-byte
// swizzle: granule g of row r lies at slot g ^ (r % 8).
__device__ __forceinline__ void mx4_fetch(const uint8_t* stage, int r, int c, uint4& codes, uint32_t& scale) {
  codes = *reinterpret_cast<const uint4*>(stage + mx4_code_at(r, c));
  scale = stage[mx4_scale_at(r, c)];
}
// Both halves of a row, 64 values.
template <typename T>
__device__ __forceinline__ void mx4_decode(const uint4 (&codes)[2], const uint32_t (&scale)[2], uint4 (&v)[8]) {
  const uint32_t w[2][4] = {{codes[0].x, codes[0].y, codes[0].z, codes[0].w}, {codes[1].x, codes[1].y, codes[1].z, codes[1].w}};
  if (Mx4<T>::one_factor(scale[0], scale[1])) {
    mx4_values<T, 4, true>(w[0], scale[0], v);
    mx4_values<T, 4, true>(w[1], scale[1], v + 4);
  } else {
    mx4_values<T, 4, false>(w[0], scale[0], v);
    mx4_values<T, 4, false>(w[1], scale[1], v + 4);
  }
}
}  // namespace lf
