// Kernels of the adapters' dropout that stand apart from the products (numbers and mask: lf_drop.cuh).
//
//   drop_mask    xm = m x, bit for bit x or zero (1 / (1 - p) is in the adapters' factors: no rounding of its own).
//   drop_expand  delta[t] = m[t] (S_b[t] A_i), float32, which the grad_x GEMM adds to g W in its epilogue.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lf_drop.cuh"
#include "lf_internal.cuh"
#include "lf_launch.cuh"

namespace lf {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

// A warp a row: kB bytes an element.  Bound by HBM (2 kB bytes an element) and, about as much, by the generator's
// integer multiplies: 20 of them for 8 elements.
template <int kB>
__global__ void __launch_bounds__(kThreads) drop_mask_kernel(const uint8_t* __restrict__ x, int T, int K, int vec, Tables tb,
                                                             DropArgs d, uint8_t* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (t >= T) return;
  const uint32_t threshold =
      row_threshold(tb, d, static_cast<int>(t / LF_TILE_ROWS), static_cast<int>(t % LF_TILE_ROWS));
  const uint8_t* xr = x + t * K * kB;
  uint8_t* o = out + t * K * kB;
  for (int g = lane; g * 8 < K; g += 32) {
    const uint4 r = philox(static_cast<uint32_t>(g), static_cast<uint32_t>(t), d.offset, d.seed);
    const uint32_t word[4] = {r.x, r.y, r.z, r.w};
    if (vec) {  // rows of whole 16-byte pieces
      if (kB == 2) {
        uint4 v = reinterpret_cast<const uint4*>(xr)[g];
        const uint32_t high = threshold << 16;
        v.x = keep2(v.x, r.x, high), v.y = keep2(v.y, r.y, high), v.z = keep2(v.z, r.z, high), v.w = keep2(v.w, r.w, high);
        reinterpret_cast<uint4*>(o)[g] = v;
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 v = reinterpret_cast<const uint4*>(xr)[2 * g + h];
          const uint32_t a = word[2 * h], b = word[2 * h + 1];
          if ((a & 0xffffu) < threshold) v.x = 0;
          if ((a >> 16) < threshold) v.y = 0;
          if ((b & 0xffffu) < threshold) v.z = 0;
          if ((b >> 16) < threshold) v.w = 0;
          reinterpret_cast<uint4*>(o)[2 * g + h] = v;
        }
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = g * 8 + i;
      if (k >= K) break;
      const bool keep = (i & 1 ? word[i >> 1] >> 16 : word[i >> 1] & 0xffffu) >= threshold;
      if (kB == 2) reinterpret_cast<uint16_t*>(o)[k] = keep ? reinterpret_cast<const uint16_t*>(xr)[k] : uint16_t(0);
      else reinterpret_cast<uint32_t*>(o)[k] = keep ? reinterpret_cast<const uint32_t*>(xr)[k] : 0u;
    }
  }
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16*) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half*) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// delta [T, K] (float32): a CTA takes 128 rows x 128 columns, a warp 16 of the rows.  S comes as hi and lo halves (two
// products into one accumulator, so S enters to 2^-16), A_i^T [K, r_pad] per virtual slot.  The rank is short, so the
// products are few and the time goes into the 4 T K bytes written; warp-level MMAs read both operands where
// they lie.  Of a row's eight columns n .. n + 7, lane q of the four that hold them has 2q and 2q + 1, word q of one counter's
// numbers: each lane computes every fourth counter and the four exchange words.
constexpr int kExpandCols = 128;
template <typename T16>
__global__ void __launch_bounds__(kThreads) drop_expand_kernel(const uint16_t* __restrict__ s_hi, int64_t lo_off,
                                                               const uint16_t* __restrict__ at, int T, int K, Tables tb,
                                                               DropArgs d, float* __restrict__ delta) {
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int tile = blockIdx.x, k0 = blockIdx.y * kExpandCols;
  const int row0 = warp * 16;
  const int64_t t0 = static_cast<int64_t>(tile) * LF_TILE_ROWS + row0;
  if (t0 >= T) return;
  const int rp = tb.r_pad;
  float acc[kExpandCols / 8][4];
#pragma unroll
  for (int n = 0; n < kExpandCols / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  uint32_t threshold[2] = {0, 0};
  const int st1 = tb.tile_st(tile + 1);
  for (int st = tb.tile_st(tile); st < st1; ++st) {
    const int lo = tb.st_lo(st), hi = tb.st_hi(st);
    if (hi <= row0 || lo >= row0 + 16) continue;
    const int slot = tb.st_slot(st);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = row0 + g + 8 * h;
      if (row >= lo && row < hi) threshold[h] = d.threshold[slot];
    }
    const uint16_t* s = s_hi + (static_cast<int64_t>(st) * LF_TILE_ROWS + row0) * rp;
    for (int j = 0; j < rp; j += 16) {
      uint32_t a[2][4];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint16_t* sp = s + (p ? lo_off : 0) + j + 2 * q;
        a[p][0] = *reinterpret_cast<const uint32_t*>(sp + g * rp);
        a[p][1] = *reinterpret_cast<const uint32_t*>(sp + (g + 8) * rp);
        a[p][2] = *reinterpret_cast<const uint32_t*>(sp + g * rp + 8);
        a[p][3] = *reinterpret_cast<const uint32_t*>(sp + (g + 8) * rp + 8);
      }
      const uint16_t* b = at + (static_cast<int64_t>(slot) * K + k0) * rp + j + 2 * q;
#pragma unroll
      for (int n = 0; n < kExpandCols / 8; ++n) {
        if (k0 + n * 8 >= K) break;  // K is a multiple of 8
        const uint16_t* bn = b + static_cast<int64_t>(n * 8 + g) * rp;
        const uint32_t b0 = *reinterpret_cast<const uint32_t*>(bn), b1 = *reinterpret_cast<const uint32_t*>(bn + 8);
        mma16816(acc[n], a[0], b0, b1, static_cast<T16*>(nullptr));
        mma16816(acc[n], a[1], b0, b1, static_cast<T16*>(nullptr));
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t t = t0 + g + 8 * h;
#pragma unroll
    for (int n4 = 0; n4 < kExpandCols / 32; ++n4) {
      const uint4 r = philox(static_cast<uint32_t>(k0 / 8 + n4 * 4 + q), static_cast<uint32_t>(t), d.offset, d.seed);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // counter n4 * 4 + i is lane i's: this lane wants word q of it
        const uint32_t w0 = __shfl_sync(0xffffffffu, r.x, i, 4), w1 = __shfl_sync(0xffffffffu, r.y, i, 4);
        const uint32_t w2 = __shfl_sync(0xffffffffu, r.z, i, 4), w3 = __shfl_sync(0xffffffffu, r.w, i, 4);
        const uint32_t w = q == 0 ? w0 : q == 1 ? w1 : q == 2 ? w2 : w3;
        const int n = n4 * 4 + i, k = k0 + n * 8 + 2 * q;
        if (t < T && k < K) {
          float2 v;
          v.x = (w & 0xffffu) >= threshold[h] ? acc[n][2 * h] : 0.f;
          v.y = (w >> 16) >= threshold[h] ? acc[n][2 * h + 1] : 0.f;
          *reinterpret_cast<float2*>(delta + t * K + k) = v;
        }
      }
    }
  }
}

}  // namespace

cudaError_t drop_mask(int dtype, const void* x, int T, int K, const Tables& tb, const DropArgs& d, void* out,
                      cudaStream_t st) {
  if (T == 0 || K == 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(T) + kWarps - 1) / kWarps);
  const int vec = K % 8 == 0 && (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % 16 == 0;
  auto* k = dtype == LF_F32 ? drop_mask_kernel<4> : drop_mask_kernel<2>;
  k<<<grid, kThreads, 0, st>>>(static_cast<const uint8_t*>(x), T, K, vec, tb, d, static_cast<uint8_t*>(out));
  return cudaGetLastError();
}

cudaError_t drop_expand(int dtype, const void* s_ext, const void* at_pack, int T, int K, const Tables& tb, const DropArgs& d,
                        float* delta, cudaStream_t st) {
  if (T == 0 || K == 0) return cudaSuccess;
  const dim3 grid(static_cast<unsigned>(tb.n_tiles), static_cast<unsigned>((K + kExpandCols - 1) / kExpandCols));
  const int64_t lo = static_cast<int64_t>(tb.n_segtiles + 1) * LF_TILE_ROWS * tb.r_pad;  // plane of the low halves
  auto* k = dtype == LF_BF16 ? drop_expand_kernel<__nv_bfloat16> : drop_expand_kernel<__half>;
  k<<<grid, kThreads, 0, st>>>(static_cast<const uint16_t*>(s_ext), lo, static_cast<const uint16_t*>(at_pack), T, K, tb, d,
                               delta);
  return cudaGetLastError();
}

}  // namespace lf
