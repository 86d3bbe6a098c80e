// A weight to microscaled 4-bit floating point and back (formats and layout: lf_mx4.cuh).
//
// Both are one pass: 2 bytes an element on the one side, 17/32 on the other.  Four lanes share a block of 32 along K, a
// warp takes 8 rows of 128 columns: 16-byte accesses on the dense side in runs of 64 bytes, runs of 128 bytes
// on the packed side, four loads of a lane in flight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "lf_internal.cuh"
#include "lf_mx4.cuh"

namespace lf {
namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ float to_f(uint32_t bits);
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(uint32_t bits) { return __uint_as_float(bits << 16); }
template <>
__device__ __forceinline__ float to_f<__half>(uint32_t bits) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

// Eight 16-bit elements k .. k + 7 of row n, zeros past the matrix.
__device__ __forceinline__ uint4 load8(const uint16_t* w, int n, int k, int N, int K, int64_t ld, bool vec) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (n >= N || k >= K) return v;
  const uint16_t* p = w + n * ld + k;
  if (vec) return *reinterpret_cast<const uint4*>(p);  // K and the row pitch are multiples of 8
  uint32_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = k + i < K ? p[i] : 0u;
  v.x = e[0] | e[1] << 16, v.y = e[2] | e[3] << 16, v.z = e[4] | e[5] << 16, v.w = e[6] | e[7] << 16;
  return v;
}

// Eight codes, the nearest of each value with ties to the even code and 6 for what is larger, value i in bits 4i .. 4i + 3.
__device__ __forceinline__ uint32_t encode8(const float (&f)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return r;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) mx4_quantize_kernel(const uint16_t* __restrict__ w, int N, int K, int64_t ld,
                                                                int vec, int64_t units, uint8_t* __restrict__ out) {
  const int lane = threadIdx.x & 31, j = lane & 3;
  const int spans = mx4_col_blocks(K) / 2;
  for (int64_t u = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 5; u < units;
       u += static_cast<int64_t>(gridDim.x) * (kThreads / 32)) {
    // a unit: 8 rows of one span of 128 columns; units of a span's 128 rows follow one another
    const int64_t at = u >> 4;
    const int span = static_cast<int>(at % spans), tile = static_cast<int>(at / spans);
    const int r = static_cast<int>(u & 15) * 8 + (lane >> 2), n = tile * kMx4Rows + r;
    uint4 v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = load8(w, n, span * 128 + c * 32 + j * 8, N, K, ld, vec != 0);
    uint8_t* blocks = out + (static_cast<int64_t>(tile) * spans + span) * (2 * kMx4Block);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t word[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
      // magnitudes compare as whole numbers; infinities and NaN are the largest
      uint32_t top = __vmaxu2(__vmaxu2(word[0] & 0x7fff7fffu, word[1] & 0x7fff7fffu),
                                   __vmaxu2(word[2] & 0x7fff7fffu, word[3] & 0x7fff7fffu));
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = max(top & 0xffffu, top >> 16);
      const uint32_t e = __float_as_uint(to_f<T>(top)) >> 23;  // floor(log2) + 127; 0 of a zero and of bf16's subnormals
      const bool bad = e == 255u;
      // E = floor(log2) - 2, at least -127; float16's blocks of zeros get the smallest scale that its other blocks have
      constexpr uint32_t kLeast = std::is_same_v<T, __half> ? 101u : 0u;
      const uint32_t s = bad ? 255u : e < kLeast + 2u ? kLeast : e - 2u;
      const float up = __uint_as_float((254u - (bad ? 127u : s)) << 23);  // 2^-E
      uint32_t code = 0;
      if (!bad) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[2 * i] = to_f<T>(word[i] & 0xffffu) * up, f[2 * i + 1] = to_f<T>(word[i] >> 16) * up;
        code = Mx4<T>::word(encode8(f));
      }
      uint8_t* b = blocks + (c >> 1) * kMx4Block;
      *reinterpret_cast<uint32_t*>(b + mx4_code_at(r, c & 1) + j * 4) = code;
      if (j == 0) b[mx4_scale_at(r, c & 1)] = static_cast<uint8_t>(s);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) mx4_dequantize_kernel(const uint8_t* __restrict__ in, int N, int K, int vec,
                                                                  int64_t units, uint16_t* __restrict__ w) {
  const int lane = threadIdx.x & 31, j = lane & 3;
  const int spans = mx4_col_blocks(K) / 2;
  for (int64_t u = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 5; u < units;
       u += static_cast<int64_t>(gridDim.x) * (kThreads / 32)) {
    const int64_t at = u >> 4;
    const int span = static_cast<int>(at % spans), tile = static_cast<int>(at / spans);
    const int r = static_cast<int>(u & 15) * 8 + (lane >> 2), n = tile * kMx4Rows + r;
    const uint8_t* blocks = in + (static_cast<int64_t>(tile) * spans + span) * (2 * kMx4Block);
    uint32_t code[4], scale[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint8_t* b = blocks + (c >> 1) * kMx4Block;
      code[c] = *reinterpret_cast<const uint32_t*>(b + mx4_code_at(r, c & 1) + j * 4);
      scale[c] = b[mx4_scale_at(r, c & 1)];
    }
    if (n >= N) continue;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int k = span * 128 + c * 32 + j * 8;
      if (k >= K) continue;
      const uint32_t one[1] = {code[c]};
      uint4 v;
      if (Mx4<T>::one_factor(scale[c], scale[c])) mx4_values<T, 1, true>(one, scale[c], &v);
      else mx4_values<T, 1, false>(one, scale[c], &v);
      uint16_t* p = w + static_cast<int64_t>(n) * K + k;
      if (vec) {
        *reinterpret_cast<uint4*>(p) = v;
        continue;
      }
      const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < K) p[i] = static_cast<uint16_t>(i & 1 ? word[i >> 1] >> 16 : word[i >> 1] & 0xffffu);
    }
  }
}

int64_t units_of(int N, int K) { return static_cast<int64_t>(mx4_row_tiles(N)) * (mx4_col_blocks(K) / 2) * 16; }
unsigned blocks_of(int64_t units, int num_sms) {
  const int64_t b = (units + kThreads / 32 - 1) / (kThreads / 32);
  return static_cast<unsigned>(b < 8 * num_sms ? b : 8 * num_sms);
}

}  // namespace

size_t mx4_bytes(int N, int K) {
  return static_cast<size_t>(mx4_row_tiles(N)) * static_cast<size_t>(mx4_col_blocks(K)) * kMx4Block;
}

cudaError_t mx4_quantize(int dtype, const void* w, int N, int K, int64_t ld, void* out, int num_sms, cudaStream_t st) {
  const int64_t units = units_of(N, K);
  if (units == 0) return cudaSuccess;
  const int vec = K % 8 == 0 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0;
  auto* k = dtype == LF_BF16 ? mx4_quantize_kernel<__nv_bfloat16> : mx4_quantize_kernel<__half>;
  k<<<blocks_of(units, num_sms), kThreads, 0, st>>>(static_cast<const uint16_t*>(w), N, K, ld, vec, units,
                                                    static_cast<uint8_t*>(out));
  return cudaGetLastError();
}

cudaError_t mx4_dequantize(int dtype, const void* in, int N, int K, void* w, int num_sms, cudaStream_t st) {
  const int64_t units = units_of(N, K);
  if (units == 0) return cudaSuccess;
  const int vec = K % 8 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0;
  auto* k = dtype == LF_BF16 ? mx4_dequantize_kernel<__nv_bfloat16> : mx4_dequantize_kernel<__half>;
  k<<<blocks_of(units, num_sms), kThreads, 0, st>>>(static_cast<const uint8_t*>(in), N, K, vec, units,
                                                    static_cast<uint16_t*>(w));
  return cudaGetLastError();
}

}  // namespace lf
