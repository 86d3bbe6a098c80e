// One shared projection with an adapter per row, the adapter's index read on the device:
//   y[t] = x[t] W^T + s_i (x[t] A_i^T) B_i^T,   i = row_slot[t]  (negative: no adapter).
//
// The adapters' part goes to a float32 buffer, and a GEMM whose last launch starts while that is still written adds it in
// its epilogue:
//   few rows     (decode) rows_lora: one launch.  A tile's rows are grouped by adapter, 8 at a time; a cluster takes
//                a few groups, its CTAs cut K for S = x A_i^T, exchange their sums through distributed
//                shared memory, then cut the output features for s_i S B_i^T, so that no grid-wide step lies
//                between A_i and B_i.  Few rows bring one adapter each: both products are streams of weights
//                through warp-level MMAs whose 8 columns are rows of one adapter, bound by bytes and latency.
//   many rows    (prompts) many_plan, many_shrink, many_expand: rows sorted by adapter, both products on tcgen05.
//   rows_gemm    y^T tiles of 128 output features x up to 256 rows with tcgen05 (the weight is the M operand, so a
//                decode step of a few rows wastes no tensor-memory lanes and streams W once), K split
//                over a cluster when the tiles alone would leave SMs idle.  Long batches go through
//                the CTA-pair GEMM of lf_tc.cu where its tiles fit better.
// Any order of rows works and no host plan is needed: the adapters are read on the device.
//
// S enters the second product as hi + lo halves of the input type after a per-row power-of-two scaling, so it is exact
// to about 2^-16 (bf16) or 2^-22 (f16) relative and a float16 S cannot overflow.  The row's largest magnitude becomes
// 1..2 (bf16) or 2^13..2^14 (f16, whose low halves of smaller values would leave its normal range otherwise: 2^-22
// then holds down to 2^-15 of the largest, 2^-37 of the largest below).  All sums are float32.
//
// Measured (replayed graph, weights from HBM; the shared projection alone by cuBLAS in brackets): 1 row 4096 -> 4096, rank 16
// 13.0 us (12.9); 64 rows of 56 adapters, ranks 8 to 64, 4096 -> 14336 43 us (23); 250 rows of 219 adapters
// of rank 16, 4096 -> 4096 37.5 us (11); 8192 rows of prompts, 64 adapters of ranks 8 to 64, 4096 -> 4096
// 254 us (178) in a burst, 300 after some seconds at the power cap (SM clock 1965 -> 1507 MHz).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>
#include <type_traits>

#include "lf_internal.cuh"
#include "lf_launch.cuh"
#include "lf_mx4.cuh"
#include "lf_ptx.cuh"

namespace lf {
namespace {

constexpr uint32_t kNoSlot = 0xffffffffu;
constexpr int kTileRows = 128;  // rows grouped by adapter together
constexpr int kShrinkThreads = 256;
constexpr int kShrinkWarps = kShrinkThreads / 32;
constexpr int kSteps = 8;  // rank steps of 16 that the groups of one batch have at most
// Lines of 128 bytes that a thread may ask of L2 ahead of its loads.  One row 4096 -> 4096: 15.0 -> 13.8 us, 250 rows of 219
// adapters 37.3 -> 35.2; with 14 (64 rows to 14336 features) or 24 lines a thread the requests hold up the
// loads behind them, 47 -> 50 and 94 -> 109 us.
constexpr int kPrefetchLines = 8;
constexpr int kSPitch = 24;  // elements from one row of a step of S to the next: no bank conflicts

// Slot and rank of row t as rank << 24 | slot, or kNoSlot.
__device__ __forceinline__ uint32_t row_adapter(const RowsArgs& p, int t, bool report) {
  const int64_t s = p.wide ? static_cast<const int64_t*>(p.row_slot)[t] : static_cast<const int32_t*>(p.row_slot)[t];
  if (s < 0) return kNoSlot;
  if (s >= p.n_slots) {
    if (report) record_error(p.err, kErrRowSlot);
    return kNoSlot;
  }
  const int r = min(p.slot_rank[s], p.r_pad);
  return r <= 0 ? kNoSlot : static_cast<uint32_t>(r) << 24 | static_cast<uint32_t>(s);
}
__device__ __forceinline__ int slot_of(uint32_t e) { return static_cast<int>(e & 0xffffffu); }
__device__ __forceinline__ int rank_of(uint32_t e) { return static_cast<int>(e >> 24); }
// Rank steps of 16 of the smallest kernel that covers the adapter.
__device__ __forceinline__ int width_of(uint32_t e) {
  const int n = (rank_of(e) + 15) >> 4;
  return n <= 2 ? n : n <= 4 ? 4 : 8;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// D (16 x 8, float32) = A (16 x 16) B (16 x 8) + D, one warp.  Lane 4g + q holds A rows g and g + 8, B
// column g, D rows g and g + 8 of columns 2q, 2q + 1.  The K order inside a step is free as long as A
// and B agree, so a lane takes consecutive elements of its rows with one wide load.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, __nv_bfloat16*) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, __half*) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// One warp's K steps k0 .. k1 - 1 (32 elements each) of a group's rows with A_i (rank up to 16 kMT), into its slot of
// `part`.  Few instructions a step count more here than anything else (with the bounds of K and of the rows
// tested on every load a step took 90): whole steps run without a test, and a row that the group does not
// have points at one that exists, for a column nobody reads.
template <typename T, int kMT, int kUnroll>
__device__ __forceinline__ void shrink_steps(float (&acc)[kMT][4], const T* xr, const T* ar, int K, int k, bool in) {
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 xv[kUnroll], lo[kUnroll][kMT], hi[kUnroll][kMT];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
#pragma unroll
    for (int m = 0; m < kMT; ++m) {
      lo[i][m] = in ? *reinterpret_cast<const uint4*>(ar + m * 16 * K + (k + i) * 32) : zero;
      hi[i][m] = in ? *reinterpret_cast<const uint4*>(ar + (m * 16 + 8) * K + (k + i) * 32) : zero;
    }
    xv[i] = in ? *reinterpret_cast<const uint4*>(xr + (k + i) * 32) : zero;
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i)
#pragma unroll
    for (int m = 0; m < kMT; ++m) {
      mma16816(acc[m], lo[i][m].x, hi[i][m].x, lo[i][m].y, hi[i][m].y, xv[i].x, xv[i].y, static_cast<T*>(nullptr));
      mma16816(acc[m], lo[i][m].z, hi[i][m].z, lo[i][m].w, hi[i][m].w, xv[i].z, xv[i].w, static_cast<T*>(nullptr));
    }
}
template <typename T, int kMT, int kUnroll>
__device__ __forceinline__ void shrink_groups(const T* xr, const T* ar, int K, int k0, int k1, float* dst) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  float acc[kMT][4];
#pragma unroll
  for (int m = 0; m < kMT; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
  const int whole = min(k1, K / 32);
  int k = k0;
#pragma unroll 1
  for (; k + kUnroll <= whole; k += kUnroll) shrink_steps<T, kMT, kUnroll>(acc, xr, ar, K, k, true);
  // a rest is a latency for each of its powers of two, not for each of its steps
  if constexpr (kUnroll >= 8)
    if (k + 4 <= whole) shrink_steps<T, kMT, 4>(acc, xr, ar, K, k, true), k += 4;
  if constexpr (kUnroll >= 4)
    if (k + 2 <= whole) shrink_steps<T, kMT, 2>(acc, xr, ar, K, k, true), k += 2;
#pragma unroll 1
  for (; k < k1; ++k) shrink_steps<T, kMT, 1>(acc, xr, ar, K, k, k * 32 + 8 * q < K);
#pragma unroll
  for (int m = 0; m < kMT; ++m) {
    float* at = dst + (m * 16 + g) * 8 + 2 * q;
    *reinterpret_cast<float2*>(at) = make_float2(acc[m][0], acc[m][1]);
    *reinterpret_cast<float2*>(at + 64) = make_float2(acc[m][2], acc[m][3]);
  }
}

// ============================================================================ adapters' part
// Rows of a tile grouped by adapter, at most 8 a group; groups of one adapter follow one another.
struct Groups {
  uint32_t eff[kTileRows];      // adapter of each row
  int16_t base[kTileRows];      // first group of the adapter whose first row this is
  int16_t start[kTileRows];     // first row of each group
  int16_t rows[kTileRows][8];   // rows of each group, -1: none
  int warp_groups[4];
  uint8_t order[kTileRows];     // the groups, widest adapters first
  uint32_t wide[4][4];          // groups 32 w .. + 31 of width 8, 4, 2, 1
};

// Number of groups of rows t0 .. t0 + rows - 1 (at most kTileRows).  All threads of the CTA call it; ends with a barrier.
__device__ __forceinline__ int group_rows(const RowsArgs& p, int t0, int rows, bool report, Groups& s) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t eff = kNoSlot;
  if (tid < kTileRows) {
    if (tid < rows) eff = row_adapter(p, t0 + tid, report);
    s.eff[tid] = eff;
    *reinterpret_cast<uint4*>(s.rows[tid]) = make_uint4(~0u, ~0u, ~0u, ~0u);
  }
  __syncthreads();
  // rows of the same adapter as a bit mask: the row's place among them, and its adapter's first row
  const bool on = tid < rows && eff != kNoSlot;
  int pos = 0, first_row = -1, groups = 0, before = 0;
  if (tid < kTileRows) {
    uint32_t m[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      m[w] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint4 u = *reinterpret_cast<const uint4*>(s.eff + w * 32 + i * 4);
        m[w] |= (static_cast<uint32_t>(u.x == eff) | static_cast<uint32_t>(u.y == eff) << 1 |
                 static_cast<uint32_t>(u.z == eff) << 2 | static_cast<uint32_t>(u.w == eff) << 3) << (4 * i);
      }
    }
    int total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < warp) pos += __popc(m[w]);
      if (w == warp) pos += __popc(m[w] & ((1u << lane) - 1));
      total += __popc(m[w]);
      if (first_row < 0 && m[w]) first_row = w * 32 + __ffs(m[w]) - 1;
    }
    groups = on && pos == 0 ? (total + 7) / 8 : 0;
    int sum = groups;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) s.warp_groups[warp] = sum;
    before = sum - groups;
  }
  __syncthreads();
  int n_groups = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < warp) before += s.warp_groups[w];
    n_groups += s.warp_groups[w];
  }
  if (groups > 0) s.base[tid] = static_cast<int16_t>(before);
  __syncthreads();
  if (on) {
    const int grp = s.base[first_row] + (pos >> 3);
    s.rows[grp][pos & 7] = static_cast<int16_t>(tid);
    if ((pos & 7) == 0) s.start[grp] = static_cast<int16_t>(tid);
  }
  __syncthreads();
  // Order by width: a cluster then takes every slices-th group, there and back, and all get about the same.
  const int width = tid < n_groups ? width_of(s.eff[s.start[tid]]) : 0;
  if (tid < kTileRows) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t m = __ballot_sync(0xffffffffu, width == 8 >> c);
      if (lane == 0) s.wide[c][warp] = m;
    }
  }
  __syncthreads();
  if (tid < n_groups) {
    int at = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t m = s.wide[c][w];
        if (width < 8 >> c || (width == 8 >> c && w < warp)) at += __popc(m);
        else if (width == 8 >> c && w == warp) at += __popc(m & ((1u << lane) - 1));
      }
    s.order[at] = static_cast<uint8_t>(tid);
  }
  __syncthreads();
  return n_groups;
}

// A row's values are divided by 2^ex, which brings the largest finite one to 2^kTop .. 2^(kTop + 1); 0 for a row that
// has none but zeros.  (Values that are not finite stay so, and must not take the others out of T's range.)
template <typename T>
constexpr int kTop = std::is_same<T, __half>::value ? 13 : 0;
template <typename T>
__device__ __forceinline__ int row_exponent(float top) {
  return top > 0.f ? max(-126, min(126, ilogbf(top) - kTop<T>)) : 0;
}
__device__ __forceinline__ float larger_finite(float top, float v) {
  return fabsf(v) <= 3.402823466e38f ? fmaxf(top, fabsf(v)) : top;
}
// w as high and low parts of one sign, of which neither is zero unless w is: both are multiplied by every entry of
// B_i, and with an infinite one the sum of both products has to be the infinity that w itself would give.  So the
// high part is rounded toward zero, and a w that it would hold alone becomes two equal parts (exact, and nothing
// below half of w's last bit, so sums that were exact stay so).  A part that would still be zero (w 2^-36 of the row's
// largest, 2^-126 for bf16) gets the smallest value.
__device__ __forceinline__ __nv_bfloat16 toward_zero(float w, __nv_bfloat16*) { return __float2bfloat16_rz(w); }
__device__ __forceinline__ __half toward_zero(float w, __half*) { return __float2half_rz(w); }
template <typename T>
__device__ __forceinline__ T at_least(T v, float w, float least) {
  return w != 0.f && to_f32(v) == 0.f ? from_f32<T>(copysignf(least, w)) : v;
}
template <typename T>
__device__ __forceinline__ void halves(float w, T& hi, T& lo) {
  T* const tag = nullptr;
  constexpr float least = std::is_same<T, __half>::value ? 0x1p-24f : 0x1p-126f;
  hi = toward_zero(w, tag);
  const float rest = w - to_f32(hi);
  const bool two = !(fabsf(rest) > 0.f);  // also infinities and NaN
  if (two) hi = toward_zero(0.5f * w, tag);
  lo = two ? hi : from_f32<T>(rest);
  hi = at_least(hi, w, least);
  lo = at_least(lo, w, least);
}

// One group of 8 rows as the second product sees it: S halves of row g (8 kSPitch from step to step), rows and
// factors of columns 2q, 2q + 1 (-1: the group has no such row).
template <typename T>
struct GroupRows {
  const T* hi;
  const T* lo;
  int row0, row1;
  float f0, f1;
};

// The second product of one group for output blocks b0 .. b1 - 1 (16 features each): kNM rank steps of 16, kPer blocks
// loaded together.  A block of a step is 512 contiguous bytes of B_i.  The order of K inside an MMA is free, so
// over two steps a lane takes 16 bytes: 8 ranks of one step, of which the first MMA multiplies 4 and the second the
// others.  The second half of a last, half block repeats the first, for results that land in the padding of
// `delta`.
template <typename T, int kNM, int kPer>
__device__ __forceinline__ void expand_blocks(const uint2* w, int N, int n, const uint2 (&sh)[kNM],
                                              const uint2 (&sl)[kNM], const GroupRows<T>& rows, float* o0, float* o1,
                                              bool second) {
  T* const tag = nullptr;
  uint2 u[kPer][kNM], v[kPer][kNM];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int half = n + i * 16 + 8 < N ? 32 : 0;
    if constexpr (kNM == 1) {
      u[i][0] = w[i * 64];
      v[i][0] = w[i * 64 + half];
    } else {
#pragma unroll
      for (int k = 0; k < kNM; k += 2) {
        const uint2* at = w + static_cast<size_t>(k) * N * 4 + i * 64;
        const uint4 a = *reinterpret_cast<const uint4*>(at), b = *reinterpret_cast<const uint4*>(at + half);
        u[i][k] = make_uint2(a.x, a.y), u[i][k + 1] = make_uint2(a.z, a.w);
        v[i][k] = make_uint2(b.x, b.y), v[i][k + 1] = make_uint2(b.z, b.w);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kNM; ++k) {
      mma16816(d, u[i][k].x, v[i][k].x, u[i][k].y, v[i][k].y, sh[k].x, sh[k].y, tag);
      mma16816(d, u[i][k].x, v[i][k].x, u[i][k].y, v[i][k].y, sl[k].x, sl[k].y, tag);
    }
    if (rows.row0 >= 0) o0[i * 16] = rows.f0 * d[0], o0[i * 16 + 8] = rows.f0 * d[2];
    if (second && rows.row1 >= 0) o1[i * 16] = rows.f1 * d[1], o1[i * 16 + 8] = rows.f1 * d[3];
  }
}
template <typename T, int kNM, int kPer>
__device__ __forceinline__ void expand_group(const RowsArgs& p, uint32_t e, int b0, int b1, const GroupRows<T>& rows) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int pitch = (p.N + 15) & ~15;
  uint2 sh[kNM], sl[kNM];
  const uint2 zero = make_uint2(0, 0);
  // the lane's step and first rank of a pair of steps (of the only step)
  const int step = kNM == 1 ? 0 : q >> 1, rank0 = kNM == 1 ? 4 * q : 8 * (q & 1);
#pragma unroll
  for (int k = 0; k < kNM; ++k) {
    const int at = (k & ~1) + step;  // beyond the rank nothing was written
    const bool on = 16 * at < rank_of(e);
    const int r = at * 8 * kSPitch + rank0 + 4 * (k & 1);
    sh[k] = on ? *reinterpret_cast<const uint2*>(rows.hi + r) : zero;
    sl[k] = on ? *reinterpret_cast<const uint2*>(rows.lo + r) : zero;
  }
  const bool second = __any_sync(0xffffffffu, rows.row1 >= 0);
  float* o0 = p.delta + static_cast<size_t>(max(rows.row0, 0)) * pitch + b0 * 16 + g;
  float* o1 = p.delta + static_cast<size_t>(max(rows.row1, 0)) * pitch + b0 * 16 + g;
  const uint2* w = static_cast<const uint2*>(p.b_bank) + rank0 / 4 +
                   ((static_cast<size_t>(slot_of(e)) * (p.r_pad >> 4) + step) * p.N + b0 * 16 + g) * 4;
  int n = b0 * 16;
  const int end = b1 * 16;
#pragma unroll 1
  for (; n + kPer * 16 <= end; n += kPer * 16, w += kPer * 64, o0 += kPer * 16, o1 += kPer * 16)
    expand_blocks<T, kNM, kPer>(w, p.N, n, sh, sl, rows, o0, o1, second);
  if constexpr (kPer >= 8)
    if (n + 64 <= end) {
      expand_blocks<T, kNM, 4>(w, p.N, n, sh, sl, rows, o0, o1, second);
      n += 64, w += 256, o0 += 64, o1 += 64;
    }
  if constexpr (kPer >= 4)
    if (n + 32 <= end) {
      expand_blocks<T, kNM, 2>(w, p.N, n, sh, sl, rows, o0, o1, second);
      n += 32, w += 128, o0 += 32, o1 += 32;
    }
#pragma unroll 1
  for (; n < end; n += 16, w += 64, o0 += 16, o1 += 16)
    expand_blocks<T, kNM, 1>(w, p.N, n, sh, sl, rows, o0, o1, second);
}

// Few rows.  Work items: (row tile, slice of its groups), each taken by a cluster of `kparts` CTAs that cut K for the first
// product and the output features for the second.  Partial products meet in shared memory, then across the
// cluster, in a fixed order.  The grid fits the GPU at once with one CTA an SM and leaves room for a CTA of the
// GEMM, which streams W meanwhile.
// Bound by latency: at 64 rows of 56 adapters, 4096 -> 14336, a CTA needs 4 us to sort its tile, 6 to 10 for its part of
// A_i, 8 for the exchange and S, and 8 to 19 for its part of B_i with 32 KB of loads in flight, while the
// GEMM is through after 28 us of the 42.  Tried without gain: 16 loads a lane instead of 8 for B_i (registers), bulk
// copies into a ring in the GEMM's epilogue, a third launch for the second product.
template <typename T, int kMT>
__global__ void __launch_bounds__(kShrinkThreads, 2) rows_lora_kernel(const RowsArgs p, int slices, int kparts) {
  constexpr int kRP = kMT * 16;  // padded rank
  __shared__ __align__(16) float part[kShrinkWarps][kSteps][16 * 8];
  __shared__ __align__(16) Groups s;
  __shared__ __align__(16) T s_hi[kSteps][8][kSPitch], s_lo[kSteps][8][kSPitch];
  __shared__ float s_fac[kSteps][8];
  __shared__ __align__(16) float s_sum[kSteps][16 * 8];
  __shared__ int s_more, s_go;  // whether this CTA, and so the cluster, has another batch
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, q = lane & 3;
  const int crank = blockIdx.x % kparts;
  const T* x = static_cast<const T*>(p.x);
  const T* bank = static_cast<const T*>(p.a_bank);
  const int K = p.K;
  const int n_blocks = (K + 31) / 32;  // 32 elements of K a step: 8 a lane
  const int out_blocks = (p.N + 15) >> 4;  // of 16 features; this CTA's: [nb0, nb1)
  const int nb0 = out_blocks * crank / kparts, nb1 = out_blocks * (crank + 1) / kparts;
  const int n_items = (p.T + kTileRows - 1) / kTileRows * slices;

  for (int item = blockIdx.x / kparts; item < n_items; item += gridDim.x / kparts) {
    const int slice = item % slices, t0 = item / slices * kTileRows;
    const int rows = min(kTileRows, p.T - t0);
    const int n_groups = group_rows(p, t0, rows, true, s);
    if (crank == 0 && slice == 0 && tid < rows) p.eff[t0 + tid] = s.eff[tid];
    // this cluster's groups: places slice, 2 slices - 1 - slice, 2 slices + slice, ... of the order
    auto group_at = [&](int j) { return static_cast<int>(s.order[j * slices + (j & 1 ? slices - 1 - slice : slice)]); };
    const int rest = n_groups % slices, rounds = n_groups / slices;
    const int mine = rounds + ((rounds & 1 ? slices - 1 - slice : slice) < rest);
    // Every CTA of a cluster sorts for itself, from slots that another stream must not change meanwhile.  If one does
    // all the same, the CTAs differ about the groups, and must not about the cluster's barriers: the first CTA says
    // whether a batch follows.
    for (int first = 0, batch; kparts > 1 || first < mine; first += batch) {
      int steps = 0, ranks = 0;  // as many groups as there is room for
      for (batch = 0; first + batch < mine; ++batch) {
        const uint32_t e = s.eff[s.start[group_at(first + batch)]];
        if (steps + width_of(e) > kSteps) break;
        steps += width_of(e);
        ranks += rank_of(e);
      }
      // This CTA's part of every A_i on its way to L2 at once: what the warps load at a time is too little to cover the
      // latency of HBM that the GEMM's stream of W keeps busy.
      const int k_lo = static_cast<int>(static_cast<int64_t>(crank) * n_blocks / kparts) * 32;
      const int k_hi = min(K, static_cast<int>(static_cast<int64_t>(crank + 1) * n_blocks / kparts) * 32);
      const int lines = (k_hi - k_lo + 63) >> 6;
      for (int u = 0; u < batch && ranks * lines <= kPrefetchLines * kShrinkThreads; ++u) {
        const uint32_t e = s.eff[s.start[group_at(first + u)]];
        const T* a = bank + static_cast<size_t>(slot_of(e)) * p.r_pad * K + k_lo;
        for (int l = tid; l < rank_of(e) * lines; l += kShrinkThreads)
          prefetch_l2(a + static_cast<size_t>(l / lines) * K + (l % lines) * 64);
      }
      // The warps divide the groups first, so that as many streams of A_i as there are warps are in flight, and K
      // where there are fewer groups than warps.
      const int lanes = batch >= 8 ? 8 : batch >= 4 ? 4 : batch >= 2 ? 2 : 1;  // groups at a time
      const int subs = kShrinkWarps / lanes, sub = warp / lanes;
      const int ranges = kparts * subs, me = crank * subs + sub;
      const int b0 = static_cast<int>(static_cast<int64_t>(me) * n_blocks / ranges);
      const int b1 = static_cast<int>(static_cast<int64_t>(me + 1) * n_blocks / ranges);
      for (int u = 0, at = 0; u < batch; ++u) {
        const int grp = group_at(first + u);
        const uint32_t e = s.eff[s.start[grp]];
        const int nm = width_of(e), slot_at = at;
        at += nm;
        if (u % lanes != warp % lanes) continue;
        const T* xr = x + static_cast<int64_t>(t0 + max(static_cast<int>(s.rows[grp][g]), 0)) * p.ldx + 8 * q;
        const T* ar = bank + (static_cast<size_t>(slot_of(e)) * p.r_pad + g) * K + 8 * q;
        float* dst = part[sub][slot_at];
        // the smallest kernel that covers the adapter's rank
        if (nm == 1) shrink_groups<T, 1, 8>(xr, ar, K, b0, b1, dst);
        else if (nm == 2) {
          if constexpr (kMT >= 2) shrink_groups<T, 2, 4>(xr, ar, K, b0, b1, dst);
        } else if (nm <= 4) {
          if constexpr (kMT >= 4) shrink_groups<T, 4, 2>(xr, ar, K, b0, b1, dst);
        } else if constexpr (kMT >= 8) {
          shrink_groups<T, 8, 1>(xr, ar, K, b0, b1, dst);
        }
      }
      // and its part of every B_i, which takes the time that the exchange below does
      const int b_lines = (nb1 - nb0) * 4;
      for (int u = 0; u < batch && steps * b_lines <= kPrefetchLines * kShrinkThreads; ++u) {
        const uint32_t e = s.eff[s.start[group_at(first + u)]];
        const char* b = static_cast<const char*>(p.b_bank) +
                        (static_cast<size_t>(slot_of(e)) * (p.r_pad >> 4) * p.N + nb0 * 16) * 32;
        const int bytes = (min(nb1 * 16, p.N) - nb0 * 16) * 32;
        for (int k = 0; 16 * k < rank_of(e); ++k)
          for (int l = tid * 128; l < bytes; l += kShrinkThreads * 128)
            prefetch_l2(b + static_cast<size_t>(k) * p.N * 32 + l);
      }
      __syncthreads();
      // The warps' sums, in the place of the first warp's; with a cluster every CTA reads the others' and adds them up
      // in the same order.  (Passing the sums on by remote stores, to the CTA that adds them and back, took two
      // cluster barriers and 5 us; this takes one.)
      for (int i = tid; i < steps * 128; i += kShrinkThreads) {
        float v = part[0][0][i];
        for (int w = 1; w < subs; ++w) v += part[w][0][i];
        if (kparts == 1) s_sum[0][i] = v;
        else part[0][0][i] = v;
      }
      if (kparts > 1) {
        if (tid == 0) s_more = first + batch < mine;
        __syncwarp();
        cluster_sync_all();
        float go = 0.f;  // the last warp has the least to add up
        if (tid == kShrinkThreads - 1) go = ld_cluster_f32(map_to_cta(smem_u32(&s_more), 0));
        for (int i = 4 * tid; i < steps * 128; i += 4 * kShrinkThreads) {
          const uint32_t at = smem_u32(&part[0][0][i]);
          float4 v[8];
#pragma unroll
          for (int c = 0; c < 8; ++c)
            if (c < kparts) v[c] = ld_cluster_f32x4(map_to_cta(at, c));
#pragma unroll
          for (int c = 1; c < 8; ++c)
            if (c < kparts) v[0].x += v[c].x, v[0].y += v[c].y, v[0].z += v[c].z, v[0].w += v[c].w;
          *reinterpret_cast<float4*>(&s_sum[0][i]) = v[0];
        }
        if (tid == kShrinkThreads - 1) s_go = __float_as_int(go);
        __syncwarp();
        cluster_arrive();  // the others may write their sums again once all have come here
      }
      __syncthreads();
      // S of each group, one warp a group; every CTA needs all of them for the second product
      for (int u = 0, at = 0; u < batch; ++u) {
        const int grp = group_at(first + u);
        const uint32_t e = s.eff[s.start[grp]];
        const int rank = rank_of(e), slot_at = at;
        at += width_of(e);
        if (u != warp) continue;
        float v[kRP / 4];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < kRP / 4; ++i) v[i] = (lane >> 3) + 4 * i < rank ? s_sum[slot_at][lane + 32 * i] : 0.f;
#pragma unroll
        for (int i = 0; i < kRP / 4; ++i) top = larger_finite(top, v[i]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const int ex = row_exponent<T>(top);
        const float down = scalbnf(1.f, -ex), fac = p.slot_scale[slot_of(e)] * scalbnf(1.f, ex);
        if (lane < 8) s_fac[u][lane] = fac;
#pragma unroll
        for (int i = 0; i < kRP / 4; ++i) {
          const int j = (lane >> 3) + 4 * i;
          if (j < ((rank + 15) & ~15))
            halves<T>(v[i] * down, s_hi[slot_at + (j >> 4)][lane & 7][j & 15], s_lo[slot_at + (j >> 4)][lane & 7][j & 15]);
        }
      }
      __syncthreads();
      // The warps divide the groups, then the features, here too; but the features alone where the groups' widths differ:
      // one warp would have four times another's work (64 rows of ranks 8 to 64 to 14336 features 46 -> 42 us; with equal
      // widths the other way was slower, 250 rows of rank 16 37.1 against 36.5).
      int lanes_b = lanes;
      if (batch > 1 && width_of(s.eff[s.start[group_at(first)]]) != width_of(s.eff[s.start[group_at(first + batch - 1)]]))
        for (lanes_b = 1; lanes_b < lanes && (nb1 - nb0) * lanes_b < 4 * kShrinkWarps;) lanes_b *= 2;
      const int subs_b = kShrinkWarps / lanes_b, sub_b = warp / lanes_b;
      const int f0 = nb0 + (nb1 - nb0) * sub_b / subs_b, f1 = nb0 + (nb1 - nb0) * (sub_b + 1) / subs_b;
      for (int u = 0, at = 0; u < batch; ++u) {
        const int grp = group_at(first + u);
        const uint32_t e = s.eff[s.start[grp]];
        const int nm = width_of(e), slot_at = at;
        at += nm;
        if (u % lanes_b != warp % lanes_b) continue;
        GroupRows<T> rows_of;
        const int r0 = s.rows[grp][2 * q], r1 = s.rows[grp][2 * q + 1];
        rows_of.hi = s_hi[slot_at][g];
        rows_of.lo = s_lo[slot_at][g];
        rows_of.row0 = r0 < 0 ? -1 : t0 + r0;
        rows_of.row1 = r1 < 0 ? -1 : t0 + r1;
        rows_of.f0 = s_fac[u][2 * q];
        rows_of.f1 = s_fac[u][2 * q + 1];
        if (nm == 1) expand_group<T, 1, 8>(p, e, f0, f1, rows_of);
        else if (nm == 2) {
          if constexpr (kMT >= 2) expand_group<T, 2, 4>(p, e, f0, f1, rows_of);
        } else if (nm <= 4) {
          if constexpr (kMT >= 4) expand_group<T, 4, 2>(p, e, f0, f1, rows_of);
        } else if constexpr (kMT >= 8) {
          expand_group<T, 8, 1>(p, e, f0, f1, rows_of);
        }
      }
      if (kparts > 1) {
        __syncwarp();
        cluster_wait();
        if (!s_go) break;
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

// ============================================================================ GEMM + expand
constexpr int kEpiWarps = 8;
constexpr int kGemmThreads = 64 + 32 * kEpiWarps;
constexpr int kWRows = 128;  // output features a tile: the M of the MMA
constexpr int kBK = 64;      // K elements of a stage: one 128-byte swizzle row
constexpr int kWBytes = kWRows * kBK * 2;
constexpr int kMaxStages = 28;

struct RowsGemm {
  RowsArgs a;
  int ksplit, stages;
  int sub;  // 64-element K blocks of a stage
  int slots;  // blocks of codes behind the stages (kMx4)
  uint32_t idesc;
};

// 32 tensor-memory lanes x kN columns, a lane's row in its registers.
template <int kN>
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, uint32_t (&v)[kN]) {
  static_assert(kN == 8 || kN == 32, "instruction shapes in use");
  if constexpr (kN == 32) {
    tmem_ld32(taddr, v);
  } else {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr));
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float a, float b) { return pack_f16x2(a, b); }

constexpr int kMaxSlots = 16;  // of codes (kMx4)

// kTN: rows (tokens) of a tile, the N of the MMA.  Warp 0 loads, warp 1 issues the MMAs, eight epilogue warps
// finish the tile.  kMx4: the weight is held in 4 bits (lf_mx4.cuh, map_w is not used).  One more warp copies its codes into
// a ring of their own, and the epilogue warps, idle until the tile is done, decode them into the stages.
template <typename T, int kTN, bool kMx4>
__global__ void __maxnreg__(80)
    rows_gemm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                     const __grid_constant__ RowsGemm prm) {
  constexpr int kXBytes = kTN * kBK * 2;
  constexpr int kCols = kTN < 32 ? 32 : kTN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_bar, drain_bar;
  __shared__ uint64_t code_full[kMx4 ? kMaxSlots : 1], code_empty[kMx4 ? kMaxSlots : 1];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  __shared__ uint8_t s_on[kTN];  // whether the row has an adapter
  const RowsArgs& p = prm.a;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  constexpr int w_bytes = kWBytes, block_bytes = w_bytes + kXBytes;
  // A stage holds `sub` blocks of 64 elements of K.  A block costs the loading warp two copies and the MMA warp four
  // MMAs, but each wait costs both about 0.1 us: with one block a stage, and with loops that only one lane ran, a
  // tile of few rows took 0.35 us a block however small its bytes; 1 row 4096 -> 4096 then took 12.1 us, now 11.0.
  const int sub = prm.sub, stage_bytes = sub * block_bytes;
  const int ks = prm.ksplit, stages = prm.stages;
  const int part = blockIdx.x % ks;  // rank in the cluster
  const int n0 = blockIdx.x / ks * kWRows;
  const int t0 = blockIdx.y * kTN;
  const int nkb = (p.K + kBK - 1) / kBK;
  const int kb0 = static_cast<int>(static_cast<int64_t>(part) * nkb / ks);
  const int kb1 = static_cast<int>(static_cast<int64_t>(part + 1) * nkb / ks);

  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], kMx4 ? 1 + kEpiWarps / 2 * sub : 1);
      mbar_init(&empty[s], 1);
    }
    if (kMx4)
      for (int i = 0; i < prm.slots; ++i) {
        mbar_init(&code_full[i], 1);
        mbar_init(&code_empty[i], kEpiWarps / 2);
      }
    mbar_init(&acc_bar, 1);
    mbar_init(&drain_bar, 1);
    abort_flag = 0;
    fence_mbar_init();
    if (!kMx4) tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0, issued = 0, parity = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; kb += sub) {
      if (!warp_wait_stage(&empty[stage], phase ^ 1, &abort_flag, p.err, kErrTimeoutEmpty)) {
        ok = false;
        break;
      }
      if (elect_one()) {
        uint8_t* w = ring + stage * stage_bytes;
        const int n = min(sub, kb1 - kb);
        mbar_arrive_expect_tx(&full[stage], n * (kMx4 ? kXBytes : block_bytes));
        for (int i = 0; i < n; ++i, w += block_bytes) {
          if (!kMx4) tma_load_2d(w, &map_w, &full[stage], (kb + i) * kBK, n0);
          tma_load_2d(w + w_bytes, &map_x, &full[stage], (kb + i) * kBK, t0);
        }
      }
      issued |= 1u << stage;
      parity = (parity & ~(1u << stage)) | (phase << stage);
      if (++stage == stages) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (!ok && lane == 0)  // let every copy that was started land before the memory is used again
      for (int s = 0; s < stages; ++s)
        if (issued & (1u << s)) drain_wait(&full[s], (parity >> s) & 1u, p.err);
    __syncwarp();
  } else if (warp == 1) {
    int stage = 0;
    uint32_t phase = 0, acc = 0;
    bool ok = true;
    // descriptors of the first block; addresses are in 16-byte units in their low bits
    const uint64_t w0 = umma_sdesc(smem_u32(ring), 16, 1024, 2);
    for (int kb = kb0; kb < kb1; kb += sub) {
      if (!warp_wait_stage(&full[stage], phase, &abort_flag, p.err, kErrTimeoutFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int n = min(sub, kb1 - kb);
      if (elect_one()) {
        uint64_t w = w0 + ((stage * stage_bytes) >> 4);
        for (int i = 0; i < n; ++i, w += block_bytes >> 4) {
          const uint64_t x = w + (w_bytes >> 4);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) umma_f16(tmem, w + 2 * k, x + 2 * k, prm.idesc, acc | i | k);
        }
        umma_commit(&empty[stage]);
      }
      __syncwarp();
      acc = 1;
      if (++stage == stages) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (elect_one()) {
      if (ok) {
        umma_commit(&acc_bar);
      } else if (acc) {
        umma_commit(&drain_bar);
        drain_wait(&drain_bar, 0, p.err);
      }
    }
    __syncwarp();
  } else if (kMx4 && warp == 2 + kEpiWarps) {
    const uint8_t* src = p.mx4.data + static_cast<int64_t>(n0 / kWRows) * p.mx4.col_blocks * kMx4Block;
    uint8_t* codes_at = ring + stages * stage_bytes;
    int slot = 0;
    uint32_t phase = 0, issued = 0, parity = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!warp_wait_stage(&code_empty[slot], phase ^ 1, &abort_flag, p.err, kErrTimeoutEmpty)) {
        ok = false;
        break;
      }
      if (elect_one()) {
        mbar_arrive_expect_tx(&code_full[slot], kMx4Block);
        bulk_load(codes_at + slot * kMx4Block, src + static_cast<int64_t>(kb) * kMx4Block, kMx4Block, &code_full[slot]);
      }
      __syncwarp();
      issued |= 1u << slot;
      parity = (parity & ~(1u << slot)) | (phase << slot);
      if (++slot == prm.slots) {
        slot = 0;
        phase ^= 1;
      }
    }
    if (!ok && lane == 0)
      for (int i = 0; i < prm.slots; ++i)
        if (issued & (1u << i)) drain_wait(&code_full[i], (parity >> i) & 1u, p.err);
    __syncwarp();
  } else {
    for (int i = tid - 64; i < kTN; i += kEpiWarps * 32)
      s_on[i] = p.row_slot != nullptr && t0 + i < p.T && row_adapter(p, t0 + i, false) != kNoSlot;
    named_barrier(1, kEpiWarps * 32);
    if constexpr (kMx4) {
      // Two groups of four warps take the blocks in turn, so that one decodes while the other waits or stores; where a
      // stage has two blocks each has one of them.
      const int w = warp - 2, row = (w & 3) * 32 + lane, group = w >> 2;
      const uint8_t* codes_at = ring + stages * stage_bytes;
      uint8_t* dst = ring + row * 128 + (sub == 2 ? group * block_bytes : 0);
      int stage = sub == 2 ? 0 : group, slot = group;
      uint32_t phase = 0, slot_phase = 0;
      bool fine = true;
      auto advance = [&]() {
        stage += sub == 2 ? 1 : 2;
        if (stage >= stages) {
          stage -= stages;
          phase ^= 1;
        }
      };
      // A wait on a slot must not come while the slot's use before is still on its way (the phases' parity would match the
      // one before that).  That use was another group's: it is over once this group's last stage, two blocks ago, was free
      // of what it held before, if there are enough slots, or once this block's stage is (rows_tc has the sizes).
      constexpr bool kStageFirst = kTN == 256;
      for (int kb = kb0 + group; kb < kb1; kb += 2) {
        if (kStageFirst) {
          fine = warp_wait_stage(&empty[stage], phase ^ 1, &abort_flag, p.err, kErrTimeoutEmpty);
          if (!fine) break;
        }
        fine = warp_wait_stage(&code_full[slot], slot_phase, &abort_flag, p.err, kErrTimeoutFull);
        if (!fine) break;
        uint4 codes[2], v[8];
        uint32_t scale[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) mx4_fetch(codes_at + slot * kMx4Block, row, c, codes[c], scale[c]);
        mx4_decode<T>(codes, scale, v);
        if (!kStageFirst) {
          fine = warp_wait_stage(&empty[stage], phase ^ 1, &abort_flag, p.err, kErrTimeoutEmpty);
          if (!fine) break;
        }
#pragma unroll
        for (int g = 0; g < 8; ++g) *reinterpret_cast<uint4*>(dst + stage * stage_bytes + ((g ^ (row & 7)) << 4)) = v[g];
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&full[stage]);
          mbar_arrive(&code_empty[slot]);
        }
        advance();
        slot += 2;
        if (slot >= prm.slots) {
          slot -= prm.slots;
          slot_phase ^= 1;
        }
      }
      // a last stage with one block
      if (fine && sub == 2 && group == 1 && ((kb1 - kb0) & 1) &&
          warp_wait_stage(&empty[stage], phase ^ 1, &abort_flag, p.err, kErrTimeoutEmpty) && lane == 0)
        mbar_arrive(&full[stage]);
      __syncwarp();
    }
  }
  const bool ok = warp_wait(&acc_bar, 0, &abort_flag, p.err, kErrTimeoutAcc);
  tc_fence_after();

  // The accumulator goes through the idle ring as [source CTA][row][feature], float32, so that a thread then
  // holds 8 features of a row.  Every CTA of the cluster finishes its own share of the features and gets
  // the others' partial sums of it.
  const int ew = warp - 2, quad = warp & 3;
  const int own = kWRows / ks, rows = min(kTN, p.T - t0);
  if (ks > 1) cluster_sync_all();  // every ring is idle
  if (ok && ew >= 0 && ew < kEpiWarps) {
    constexpr int kN = kTN >= 64 ? 32 : 8;  // rows a load
    constexpr int kHalf = kTN / 2;          // the two warps of a lane quarter take half the rows each
    const int f = quad * 32 + lane, first = (ew >> 2) * kHalf;
    uint32_t at = smem_u32(ring) + static_cast<uint32_t>((part * kTN * own + (f & (own - 1))) * 4);
    if (ks > 1) at = map_to_cta(at, f / own);
#pragma unroll 1
    for (int r = first; r < min(first + kHalf, rows); r += kN) {
      uint32_t v[kN];
      tmem_ld_rows<kN>(tmem + (static_cast<uint32_t>(quad * 32) << 16) + r, v);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < kN; ++i) st_cluster_f32(at + static_cast<uint32_t>((r + i) * own * 4), v[i]);
    }
  }
  if (ks > 1) cluster_sync_all();
  else __syncthreads();
  pdl_wait();  // the adapters' part
  if (ok) {
    const int nb = n0 + part * own;                       // this CTA's features
    const int shift = 4 - (31 - __clz(ks));               // log2 of 8-feature pieces a row
    const float* sums = reinterpret_cast<const float*>(ring);
    const int pitch = (p.N + 15) & ~15;
    for (int i = tid; i < rows << shift; i += kMx4 ? kGemmThreads + 32 : kGemmThreads) {
      const int r = i >> shift, f = (i & ((1 << shift) - 1)) * 8, n = nb + f;
      if (n >= p.N) continue;  // N is a multiple of 8
      float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
      if (s_on[r]) {
        const float4* d = reinterpret_cast<const float4*>(p.delta + static_cast<size_t>(t0 + r) * pitch + n);
        lo = d[0], hi = d[1];
      }
      float4 a0 = make_float4(0.f, 0.f, 0.f, 0.f), a1 = a0;
      for (int c = 0; c < ks; ++c) {  // fixed order
        const float4* w = reinterpret_cast<const float4*>(sums + (c * kTN + r) * own + f);
        a0.x += w[0].x, a0.y += w[0].y, a0.z += w[0].z, a0.w += w[0].w;
        a1.x += w[1].x, a1.y += w[1].y, a1.z += w[1].z, a1.w += w[1].w;
      }
      uint4 y;
      y.x = pack_pair<T>(a0.x + lo.x, a0.y + lo.y);
      y.y = pack_pair<T>(a0.z + lo.z, a0.w + lo.w);
      y.z = pack_pair<T>(a1.x + hi.x, a1.y + hi.y);
      y.w = pack_pair<T>(a1.z + hi.z, a1.w + hi.w);
      *reinterpret_cast<uint4*>(static_cast<T*>(p.y) + static_cast<size_t>(t0 + r) * p.N + n) = y;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, kCols);
}

// ============================================================================ many rows
// The adapters' part of long batches (prompts).  The rows are sorted by adapter on the device into tiles of up to 128
// rows of one adapter, and both products run on tcgen05 with the tile's rows as M: x is gathered row by row for the
// first, S kept in sorted order, and the second product's rows are written to their own places in `delta`.
// Which tile a row falls into, and where, depends on the order of atomics; a row's result does not, since
// no row of an MMA sees another.  (Other ways, 8192 x 4096 -> 4096, 64 adapters of rank up to 64, prompts / shuffled
// tokens, the part that is not hidden by the GEMM: groups of 8 rows with warp-level MMAs 154 / 373 us, every group
// fetching its A_i and B_i again; 128 rows as they come, multiplied by every adapter among them, 112 / 1110 us.)
struct ManyTile {
  uint32_t e;  // adapter
  int first;   // of the sorted rows
  int rows;
  int pad;
};

// Sorts at most kRowsChunk rows: a hash table of adapters in shared memory counts them, a scan places them.  One CTA,
// latency: 10 us for 8192 rows, 7 for 1000.
constexpr int kPlanThreads = 1024;
constexpr int kPlanSlots = 2 * kRowsChunk;  // of the table: never more than half full
constexpr int kPlanRows = kRowsChunk / kPlanThreads;
constexpr int kPlanSmem = kPlanSlots * 8 + kRowsChunk * 2;
__global__ void __launch_bounds__(kPlanThreads, 1) many_plan_kernel(const RowsArgs p, int log2_slots) {
  extern __shared__ uint32_t plan_smem[];
  uint32_t* key = plan_smem;
  const int slots = 1 << log2_slots;
  uint32_t* count = plan_smem + slots;  // then the first sorted row
  uint16_t* list = reinterpret_cast<uint16_t*>(count + slots);  // the table's slots in use
  __shared__ int warp_rows[32], warp_tiles[32], n_list;
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t e[kPlanRows];  // loads of one kind together: two latencies, not sixteen
  int64_t slot[kPlanRows];
#pragma unroll
  for (int i = 0; i < kPlanRows; ++i) {
    const int t = tid + i * kPlanThreads;
    slot[i] = t >= p.T ? -1 : p.wide ? static_cast<const int64_t*>(p.row_slot)[t] : static_cast<const int32_t*>(p.row_slot)[t];
  }
#pragma unroll
  for (int i = 0; i < kPlanRows; ++i) {
    const bool in = slot[i] >= 0 && slot[i] < p.n_slots;
    if (slot[i] >= p.n_slots) record_error(p.err, kErrRowSlot);
    const int r = in ? min(p.slot_rank[slot[i]], p.r_pad) : 0;
    e[i] = r <= 0 ? kNoSlot : static_cast<uint32_t>(r) << 24 | static_cast<uint32_t>(slot[i]);
    if (tid + i * kPlanThreads < p.T) p.eff[tid + i * kPlanThreads] = e[i];
  }
  for (int h = tid; h < slots; h += kPlanThreads) {
    key[h] = kNoSlot;
    count[h] = 0;
  }
  if (tid == 0) n_list = 0;
  __syncthreads();
  uint32_t at[kPlanRows], pos[kPlanRows];
#pragma unroll
  for (int i = 0; i < kPlanRows; ++i) {
    at[i] = pos[i] = 0;
    const uint32_t same = __match_any_sync(0xffffffffu, e[i]);
    const int lead = __ffs(same) - 1;
    if (e[i] != kNoSlot && lane == lead) {
      uint32_t h = (e[i] * 0x9e3779b1u) >> (32 - log2_slots);
      for (;;) {
        const uint32_t was = atomicCAS(&key[h], kNoSlot, e[i]);
        if (was == kNoSlot) list[atomicAdd(&n_list, 1)] = static_cast<uint16_t>(h);
        if (was == kNoSlot || was == e[i]) break;
        h = (h + 1) & (slots - 1);
      }
      at[i] = h;
      pos[i] = atomicAdd(&count[h], __popc(same));
    }
    at[i] = __shfl_sync(0xffffffffu, at[i], lead);
    pos[i] = __shfl_sync(0xffffffffu, pos[i], lead) + __popc(same & ((1u << lane) - 1));
  }
  __syncthreads();
  const int n = n_list;
  int row_base = 0, tile_base = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int h = i0 + tid < n ? list[i0 + tid] : 0, rows = i0 + tid < n ? static_cast<int>(count[h]) : 0;
    const int tiles = (rows + kTileRows - 1) / kTileRows;
    int row0 = rows, tile0 = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int r = __shfl_up_sync(0xffffffffu, row0, o), t = __shfl_up_sync(0xffffffffu, tile0, o);
      if (lane >= o) row0 += r, tile0 += t;
    }
    if (lane == 31) warp_rows[warp] = row0, warp_tiles[warp] = tile0;
    __syncthreads();
    row0 += row_base - rows, tile0 += tile_base - tiles;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      if (w < warp) row0 += warp_rows[w], tile0 += warp_tiles[w];
      row_base += warp_rows[w], tile_base += warp_tiles[w];
    }
    if (rows > 0) count[h] = row0;
    for (int r = 0; r < rows; r += kTileRows)
      static_cast<ManyTile*>(p.tiles)[tile0++] = ManyTile{key[h], row0 + r, min(kTileRows, rows - r), 0};
    __syncthreads();
  }
  if (tid == 0) *p.n_tiles = tile_base;
#pragma unroll
  for (int i = 0; i < kPlanRows; ++i)
    if (e[i] != kNoSlot) p.perm[count[at[i]] + pos[i]] = tid + i * kPlanThreads;
}

// S = x A_i^T of a tile, in sorted order.  K is cut over a cluster when there cannot be many tiles.  Four warps gather x
// with 16-byte copies, 8 lanes to the 128 bytes of a row and block of 64 elements, placed as the 128-byte swizzle
// would (a TMA gather of four rows takes about 50 ns however many are in flight: 99 us for 8192 rows); TMA
// loads A_i.  24 us for 8192 x 4096 and 64 adapters of ranks 8 to 64: a round of 87 tiles, half a microsecond for 128
// elements of K, where the MMA warp's eight small MMAs and their waits take what the copies do.
// All of a CTA's K goes into one accumulator.  The tensor core drops up to 2^-25 of the running sum a step of 16, so
// 14336 elements of one sign lose at most 2^-15 of S, as the shared projection beside it does: a hundredth of a bf16
// rounding of y, a sixteenth of a float16 one.  (The packed shrink rotates accumulators because its S also goes into
// gradients, which sum over all tokens.)
constexpr int kXBytes = kTileRows * kBK * 2;
constexpr int kShrinkMaxStages = 8;
constexpr int kLoadWarps = 4;
struct ManyShrink {
  RowsArgs a;
  int ksplit, pitch;  // floats from one row's S to the next in shared memory
  int stages;
  int ab_fmt;
};
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 1)
    many_shrink_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ ManyShrink prm) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kShrinkMaxStages], empty[kShrinkMaxStages], acc_full, drain_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  const RowsArgs& p = prm.a;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int ks = prm.ksplit, part = blockIdx.x % ks, stages = prm.stages;
  // two blocks of 64 elements a stage: a wait costs as much as a block's MMAs
  const int block_bytes = kXBytes + p.r_pad * kBK * 2, stage_bytes = 2 * block_bytes;
  float* s_part = reinterpret_cast<float*>(ring);  // [128][pitch], while the ring is idle
  const int nkb = (p.K + kBK - 1) / kBK;
  const int kb0 = static_cast<int>(static_cast<int64_t>(part) * nkb / ks);
  const int kb1 = static_cast<int>(static_cast<int64_t>(part + 1) * nkb / ks);
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1 + 32 * kLoadWarps);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full, 1);
    mbar_init(&drain_bar, 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, LF_BANK_MAX_RANK);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();  // not before this CTA has its tensor memory: the next kernel's could take it and wait for us
  pdl_wait();
  const uint32_t tmem = tmem_slot;
  const int n_tiles = *p.n_tiles;
  const uint64_t x0 = umma_sdesc(smem_u32(ring), 16, 1024, 2);
  int stage = 0;  // of every loading warp and of the MMA thread
  uint32_t phase = 0, issued = 0, parity = 0, done = 0, drained = 0;
  for (int i = blockIdx.x / ks; i < n_tiles; i += gridDim.x / ks, done ^= 1) {
    const ManyTile tile = static_cast<const ManyTile*>(p.tiles)[i];
    const int slot = slot_of(tile.e), rank = rank_of(tile.e), steps = (rank + 15) >> 4;
    if (warp == 0) {
      for (int kb = kb0; kb < kb1; kb += 2) {
        if (!warp_wait_stage(&empty[stage], phase ^ 1, &abort_flag, p.err, kErrTimeoutEmpty)) break;
        if (elect_one()) {
          const int n = min(2, kb1 - kb);
          mbar_arrive_expect_tx(&full[stage], n * steps * 16 * kBK * 2);
          uint8_t* d = ring + stage * stage_bytes + kXBytes;
          for (int b = 0; b < n; ++b, d += block_bytes)
            for (int k = 0; k < steps; ++k)
              tma_load_2d(d + k * 16 * kBK * 2, &map_a, &full[stage], (kb + b) * kBK, slot * p.r_pad + 16 * k);
        }
        issued |= 1u << stage;
        parity = (parity & ~(1u << stage)) | (phase << stage);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      const uint32_t idesc = umma_idesc_f16(kTileRows, steps * 16, prm.ab_fmt, 0, 0);
      uint32_t acc = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; kb += 2) {
        if (!warp_wait_stage(&full[stage], phase, &abort_flag, p.err, kErrTimeoutFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        fence_proxy_async_smem();  // x came by ordinary copies
        const int n = min(2, kb1 - kb);
        if (elect_one()) {
          uint64_t x = x0 + ((stage * stage_bytes) >> 4);
          for (int b = 0; b < n; ++b, x += block_bytes >> 4) {
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) umma_f16(tmem, x + 2 * k, x + (kXBytes >> 4) + 2 * k, idesc, acc | b | k);
          }
          umma_commit(&empty[stage]);
        }
        __syncwarp();
        acc = 1;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (elect_one()) {
        if (ok) umma_commit(&acc_full);
        else if (acc) {
          umma_commit(&drain_bar);
          drain_wait(&drain_bar, drained, p.err);
        }
      }
      __syncwarp();
      if (!ok && acc) drained ^= 1;
    } else {
      // rows (tid - 64) / 8 + kStep j, 16 bytes of each; a row that is not there reads nothing and becomes zeros
      constexpr int kStep = 4 * kLoadWarps, kPer = kTileRows / kStep;
      const int r0 = (tid - 64) >> 3, piece = tid & 7;
      const T* from[kPer];
      uint32_t bytes[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int row = r0 + kStep * j;
        from[j] = static_cast<const T*>(p.x) + piece * 8 + kb0 * kBK +
                  static_cast<int64_t>(p.perm[tile.first + min(row, tile.rows - 1)]) * p.ldx;
        bytes[j] = row < tile.rows ? 16 : 0;
      }
      const uint32_t to = smem_u32(ring) + static_cast<uint32_t>(r0 * 128 + ((piece ^ (r0 & 7)) << 4));
      for (int kb = warp < 2 + kLoadWarps ? kb0 : kb1; kb < kb1; kb += 2) {
        bool ok = true;
        if (lane == 0) ok = mbar_wait_stage(&empty[stage], phase ^ 1, &abort_flag, p.err, kErrTimeoutEmpty);
        if (!__shfl_sync(0xffffffffu, ok, 0)) break;
        const uint32_t d = to + stage * stage_bytes;
        if (kb + 2 <= kb1 && (kb + 2) * kBK <= p.K) {
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            cp_async16(d + j * kStep * 128, from[j], bytes[j]);
            cp_async16(d + block_bytes + j * kStep * 128, from[j] + kBK, bytes[j]);
            from[j] += 2 * kBK;
          }
        } else {
          for (int b = 0; b < min(2, kb1 - kb); ++b) {
            const bool in = (kb + b) * kBK + piece * 8 < p.K;  // zeros behind K
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
              cp_async16(d + b * block_bytes + j * kStep * 128, in ? from[j] : static_cast<const T*>(p.x), in ? bytes[j] : 0);
              from[j] += kBK;
            }
          }
        }
        cp_async_arrive(&full[stage]);  // once this thread's copies have landed
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      // the two warps of a lane quarter take alternate steps
      if (warp_wait_stage(&acc_full, done, &abort_flag, p.err, kErrTimeoutAcc)) {
        tc_fence_after();
        const int quad = warp & 3, row = quad * 32 + lane;
        if (quad * 32 < tile.rows) {
          for (int k = (warp - 2) >> 2; k < steps; k += 2) {
            uint32_t v[16];
            tmem_ld16(tmem + (static_cast<uint32_t>(quad * 32) << 16) + 16 * k, v);
            tmem_wait_ld();
            uint4* to_s = reinterpret_cast<uint4*>(s_part + row * prm.pitch + 16 * k);
#pragma unroll
            for (int j = 0; j < 4; ++j) to_s[j] = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
        }
        tc_fence_before();
      }
    }
    if (ks > 1) cluster_sync_all();
    else __syncthreads();
    tc_fence_after();
    // this CTA's rows of the tile: sum over the cluster in a fixed order, scale, split; 2 ks lanes a row, 8 values a time
    const int row = part + ks * (tid / (2 * ks)), sub = tid & (2 * ks - 1);
    if (tid < kEpiWarps * 32) {
      const size_t to = static_cast<size_t>(tile.first + row);
      float v[LF_BANK_MAX_RANK / 16][8];
      float top = 0.f;
#pragma unroll
      for (int c = 0; c < LF_BANK_MAX_RANK / 16; ++c) {
        const int j0 = 8 * (sub + 2 * ks * c);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] = 0.f;
        if (j0 < rank && row < tile.rows) {
          const uint32_t at = smem_u32(s_part + row * prm.pitch + j0);
          for (int peer = 0; peer < ks; ++peer) {
            const uint32_t from = ks == 1 ? at : map_to_cta(at, peer);
            const float4 lo = ld_cluster_f32x4(from), hi = ld_cluster_f32x4(from + 16);
            v[c][0] += lo.x, v[c][1] += lo.y, v[c][2] += lo.z, v[c][3] += lo.w;
            v[c][4] += hi.x, v[c][5] += hi.y, v[c][6] += hi.z, v[c][7] += hi.w;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j0 + j >= rank) v[c][j] = 0.f;  // columns past the rank: zero times x, which may not be finite
            top = larger_finite(top, v[c][j]);
          }
        }
      }
      for (int o = 1; o < 2 * ks; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int ex = row_exponent<T>(top);
      const float down = scalbnf(1.f, -ex);
      if (row < tile.rows) {
        if (sub == 0) p.factor[to] = p.slot_scale[slot] * scalbnf(1.f, ex);
#pragma unroll
        for (int c = 0; c < LF_BANK_MAX_RANK / 16; ++c) {
          const int j0 = 8 * (sub + 2 * ks * c);
          if (j0 < steps * 16) {
            __align__(16) T hi[8], lo[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) halves<T>(v[c][j] * down, hi[j], lo[j]);
            *reinterpret_cast<uint4*>(static_cast<T*>(p.s_hi) + to * p.r_pad + j0) = *reinterpret_cast<const uint4*>(hi);
            *reinterpret_cast<uint4*>(static_cast<T*>(p.s_lo) + to * p.r_pad + j0) = *reinterpret_cast<const uint4*>(lo);
          }
        }
      }
    }
    fence_proxy_async_smem();  // TMA writes here next
    if (ks > 1) cluster_sync_all();  // peers have read this CTA's sums
    else __syncthreads();
  }  // when a wait has run out the remaining tiles' waits end at once: the cluster's CTAs stay in step
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (warp == 0 && lane == 0 && abort_flag)  // let every copy that was started land before the memory is used again
    for (int s = 0; s < stages; ++s)
      if (issued & (1u << s)) drain_wait(&full[s], (parity >> s) & 1u, p.err);
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, LF_BANK_MAX_RANK);
}

// delta = s_i S B_i^T.  A unit is a tile x 256 features, and a CTA takes a run of them; the rank steps of S (high, then low
// halves) times those of B_i go into one of two accumulators.  38 us for 8192 x 4096 (117 MB written): bound by the
// epilogue's stores, 128 KB a unit at about 32 bytes a clock.  They go through shared memory so that a row's 128
// bytes leave together; sectors of 32 bytes straight from the registers took the operator from 248 to 252 us.
constexpr int kSStepBytes = kTileRows * 32;  // 16 ranks of 128 rows
constexpr int kBStepBytes = 256 * 32;        // 16 ranks of 256 features
constexpr int kExpandStages = 5, kExpandChunk = 2;  // rank steps of a stage, at most
constexpr int kExpandStepBytes = 2 * kSStepBytes + kBStepBytes;
constexpr int kExpandStageBytes = kExpandChunk * kExpandStepBytes;
constexpr int kDeltaStageBytes = 32 * 36 * 4;  // a warp's 32 rows x 32 columns, padded
struct ManyExpand {
  RowsArgs a;
  uint32_t idesc;
};
template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 1)
    many_expand_kernel(const __grid_constant__ CUtensorMap map_hi, const __grid_constant__ CUtensorMap map_lo,
                       const __grid_constant__ CUtensorMap map_b, const __grid_constant__ ManyExpand prm) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* out = ring + kExpandStages * kExpandStageBytes;
  __shared__ uint64_t full[kExpandStages], empty[kExpandStages], tfull[2], tempty[2], drain_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  const RowsArgs& p = prm.a;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < kExpandStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], kEpiWarps);
    }
    mbar_init(&drain_bar, 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();  // after the allocation, as above
  pdl_wait();
  const uint32_t tmem = tmem_slot;
  const ManyTile* tiles = static_cast<const ManyTile*>(p.tiles);
  const int blocks = (p.N + 255) / 256;
  const int64_t units = static_cast<int64_t>(*p.n_tiles) * blocks;
  const int u0 = static_cast<int>(units * blockIdx.x / gridDim.x), u1 = static_cast<int>(units * (blockIdx.x + 1) / gridDim.x);
  if (warp == 0) {
    fence_proxy_async_global();  // S was written by plain stores
    int stage = 0;
    uint32_t phase = 0, issued = 0, parity = 0;
    bool ok = true;
    for (int u = u0; u < u1 && ok; ++u) {
      const ManyTile tile = tiles[u / blocks];
      const int n0 = u % blocks * 256, steps = (rank_of(tile.e) + 15) >> 4;
      const int row_b = slot_of(tile.e) * (p.r_pad >> 4) * p.N + n0;
      for (int k0 = 0; k0 < steps; k0 += kExpandChunk) {
        if (!warp_wait_stage(&empty[stage], phase ^ 1, &abort_flag, p.err, kErrTimeoutEmpty)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          const int ns = min(kExpandChunk, steps - k0);
          mbar_arrive_expect_tx(&full[stage], ns * kExpandStepBytes);
          uint8_t* d = ring + stage * kExpandStageBytes;
          for (int k = k0; k < k0 + ns; ++k, d += kExpandStepBytes) {
            tma_load_2d(d, &map_hi, &full[stage], 16 * k, tile.first);
            tma_load_2d(d + kSStepBytes, &map_lo, &full[stage], 16 * k, tile.first);
            tma_load_2d(d + 2 * kSStepBytes, &map_b, &full[stage], 0, row_b + k * p.N);
          }
        }
        issued |= 1u << stage;
        parity = (parity & ~(1u << stage)) | (phase << stage);
        if (++stage == kExpandStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok && lane == 0)
      for (int s = 0; s < kExpandStages; ++s)
        if (issued & (1u << s)) drain_wait(&full[s], (parity >> s) & 1u, p.err);
    __syncwarp();
  } else if (warp == 1) {
    int stage = 0;
    uint32_t phase = 0;
    bool any = false, ok = true;
    const uint64_t s0 = umma_sdesc(smem_u32(ring), 16, 256, 6);
    for (int u = u0, i = 0; u < u1 && ok; ++u, ++i) {
      const int steps = (rank_of(tiles[u / blocks].e) + 15) >> 4, buf = i & 1;
      if (!warp_wait_stage(&tempty[buf], ((i >> 1) & 1) ^ 1, &abort_flag, p.err, kErrTimeoutAcc)) {
        ok = false;
        break;
      }
      const uint32_t d = tmem + buf * 256;
      for (int k0 = 0; k0 < steps; k0 += kExpandChunk) {
        if (!warp_wait_stage(&full[stage], phase, &abort_flag, p.err, kErrTimeoutFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          uint64_t s = s0 + ((stage * kExpandStageBytes) >> 4);
          for (int k = k0; k < min(steps, k0 + kExpandChunk); ++k, s += kExpandStepBytes >> 4) {
            const uint64_t w = s + ((2 * kSStepBytes) >> 4);
            umma_f16(d, s, w, prm.idesc, k > 0);
            umma_f16(d, s + (kSStepBytes >> 4), w, prm.idesc, 1);
          }
          umma_commit(&empty[stage]);
          if (k0 + kExpandChunk >= steps) umma_commit(&tfull[buf]);
        }
        __syncwarp();
        any = true;
        if (++stage == kExpandStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok && any && elect_one()) {
      umma_commit(&drain_bar);
      drain_wait(&drain_bar, 0, p.err);
    }
    __syncwarp();
  } else {
    // rows 32 quad .. + 31, columns 128 half .. + 127 of every unit
    const int ew = warp - 2, quad = warp & 3, half = ew >> 2;
    const int pitch = (p.N + 15) & ~15;
    float* stage_out = reinterpret_cast<float*>(out + ew * kDeltaStageBytes);
    int at = -1, rows = 0;
    float fac = 0.f;
    float* to[8];  // a lane writes 16 bytes of rows 4 i + lane / 8
    for (int u = u0, i = 0; u < u1; ++u, ++i) {
      if (u / blocks != at) {
        at = u / blocks;
        const ManyTile tile = tiles[at];
        rows = tile.rows - quad * 32;
        const int first = tile.first + quad * 32;
        if (rows > 0) {
          fac = p.factor[first + min(lane, rows - 1)];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            to[j] = p.delta + static_cast<size_t>(p.perm[first + min(4 * j + (lane >> 3), rows - 1)]) * pitch + 4 * (lane & 7);
        }
      }
      const int buf = i & 1, n0 = u % blocks * 256 + half * 128;
      if (!warp_wait_stage(&tfull[buf], (i >> 1) & 1, &abort_flag, p.err, kErrTimeoutAcc)) break;
      tc_fence_after();
      if (rows > 0) {
#pragma unroll 1
        for (int c0 = 0; c0 < 128 && n0 + c0 < p.N; c0 += 64) {
          uint32_t v[2][32];
          const uint32_t from = tmem + (static_cast<uint32_t>(quad * 32) << 16) + buf * 256 + half * 128 + c0;
          tmem_ld32(from, v[0]);
          tmem_ld32(from + 32, v[1]);
          tmem_wait_ld();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int n = n0 + c0 + 32 * h;
            float4* st = reinterpret_cast<float4*>(stage_out + lane * 36);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              st[i] = make_float4(fac * __uint_as_float(v[h][4 * i]), fac * __uint_as_float(v[h][4 * i + 1]),
                                  fac * __uint_as_float(v[h][4 * i + 2]), fac * __uint_as_float(v[h][4 * i + 3]));
            __syncwarp();
            // 128 contiguous bytes a row, four rows an access
            if (n + 4 * (lane & 7) < p.N) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                if (4 * j >= rows) break;
                const int r = 4 * j + (lane >> 3);
                if (r < rows)
                  *reinterpret_cast<float4*>(to[j] + n) = *reinterpret_cast<const float4*>(stage_out + r * 36 + 4 * (lane & 7));
              }
            }
            __syncwarp();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[buf]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ============================================================================ CUDA cores
// Float32 problems and shapes TMA cannot address.  One CTA a row for S; then 32 x 32 output tiles.  Sums are float32, cut
// so that their errors grow with K / 128 (S, one lane's share) or K / 32 (a step's sum first): 1.2e-7 of the
// result's norm at K = 256, where one float32 product with the library is off by 2.9e-7.  (The packed float32 path
// sums in 64 bits, for gradients and an oracle that it meets to the last bits; a served row needs no more than
// float32 products give.)
constexpr int kSimtShrink = 128;
template <typename T>
__global__ void __launch_bounds__(kSimtShrink) rows_shrink_simt_kernel(const RowsArgs p) {
  __shared__ float part[kSimtShrink / 32][8];
  pdl_launch_dependents();
  const int t = blockIdx.x, tid = threadIdx.x;
  const uint32_t e = row_adapter(p, t, true);
  if (tid == 0) p.eff[t] = e;
  if (e == kNoSlot) return;
  const int rank = rank_of(e), K = p.K;
  const T* x = static_cast<const T*>(p.x) + static_cast<int64_t>(t) * p.ldx;
  const T* a = static_cast<const T*>(p.a_bank) + static_cast<size_t>(slot_of(e)) * p.r_pad * K;
  float* s = static_cast<float*>(p.s_hi) + static_cast<size_t>(t) * p.r_pad;
  const float scale = p.slot_scale[slot_of(e)];
  for (int j0 = 0; j0 < rank; j0 += 8) {
    float acc[8] = {};
#pragma unroll 4
    for (int k = tid; k < K; k += kSimtShrink) {
      const float xv = to_f32(x[k]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j0 + j < rank) acc[j] = fmaf(xv, to_f32(a[static_cast<size_t>(j0 + j) * K + k]), acc[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
      if ((tid & 31) == 0) part[tid >> 5][j] = acc[j];
    }
    __syncthreads();
    if (tid < 8) {  // zeros behind the rank: the second product reads whole groups of four
      float v = part[0][tid];
#pragma unroll
      for (int w = 1; w < kSimtShrink / 32; ++w) v += part[w][tid];
      s[j0 + tid] = j0 + tid < rank ? scale * v : 0.f;
    }
    __syncthreads();
  }
}

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {  // 16-bit values at an address of any alignment they allow
  return make_float4(to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3]));
}

constexpr int kST = 32, kSK = 32;  // tile edge, K elements a step
template <typename T>
__global__ void __launch_bounds__(256) rows_gemm_simt_kernel(const RowsArgs p) {
  __shared__ float xs[kSK][kST + 1], wsm[kSK][kST + 1];
  const int n0 = blockIdx.x * kST, t0 = blockIdx.y * kST, tid = threadIdx.x;
  const int tr = tid / 16 * 2, tc = tid % 16 * 2;  // 2 rows x 2 features a thread
  const T* x = static_cast<const T*>(p.x);
  const T* w = static_cast<const T*>(p.w);
  float acc[2][2] = {};
  for (int k0 = 0; k0 < p.K; k0 += kSK) {
#pragma unroll
    for (int e = tid; e < kST * kSK; e += 256) {
      const int r = e / kSK, k = e % kSK;
      const bool in = k0 + k < p.K;
      xs[k][r] = in && t0 + r < p.T ? to_f32(x[static_cast<int64_t>(t0 + r) * p.ldx + k0 + k]) : 0.f;
      wsm[k][r] = in && n0 + r < p.N ? to_f32(w[static_cast<size_t>(n0 + r) * p.K + k0 + k]) : 0.f;
    }
    __syncthreads();
    float sum[2][2] = {};  // a step's sum first, then the running one: errors grow with K / 32, not K
#pragma unroll
    for (int k = 0; k < kSK; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) sum[i][j] = fmaf(xs[k][tr + i], wsm[k][tc + j], sum[i][j]);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] += sum[i][j];
    __syncthreads();
  }
  // The adapters' part of both rows and both features together, four ranks a load; which adapters they are does not
  // depend on the first launch.
  const T* b[2][2];
  int rank[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t e = t0 + tr + i < p.T ? row_adapter(p, t0 + tr + i, false) : kNoSlot;
    rank[i] = e == kNoSlot ? 0 : rank_of(e);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      b[i][j] = static_cast<const T*>(p.b_bank) +
                (rank[i] ? (static_cast<size_t>(slot_of(e)) * (p.r_pad >> 4) * p.N + min(n0 + tc + j, p.N - 1)) * 16 : 0);
  }
  pdl_wait();
  float add[2][2] = {};
#pragma unroll 2
  for (int r = 0; r < max(rank[0], rank[1]); r += 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (r >= rank[i]) continue;
      const float4 sv = *reinterpret_cast<const float4*>(static_cast<const float*>(p.s_hi) +
                                                         static_cast<size_t>(t0 + tr + i) * p.r_pad + r);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 bv = load4(b[i][j] + static_cast<size_t>(r >> 4) * p.N * 16 + (r & 15));
        add[i][j] = fmaf(sv.x, bv.x, fmaf(sv.y, bv.y, fmaf(sv.z, bv.z, fmaf(sv.w, bv.w, add[i][j]))));
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (t0 + tr + i < p.T && n0 + tc + j < p.N)
        static_cast<T*>(p.y)[static_cast<size_t>(t0 + tr + i) * p.N + n0 + tc + j] = from_f32<T>(acc[i][j] + add[i][j]);
}

// One adapter into its slot: A_i as it is, B_i in steps of 16 ranks, zeros past the rank.  One launch of a few
// microseconds whatever the rank (the same with tensor operations was seven, 43 us of host time).
template <typename T>
__global__ void __launch_bounds__(256) bank_load_kernel(const BankLoad p) {
  const T zero = from_f32<T>(0.f);
  const int64_t in_a = static_cast<int64_t>(p.r_pad) * p.K, all = in_a + static_cast<int64_t>(p.r_pad) * p.N;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < all; i += gridDim.x * 256ll) {
    if (i < in_a) {
      const int64_t r = i / p.K;
      static_cast<T*>(p.a_out)[i] = r < p.rank ? static_cast<const T*>(p.a)[r * p.lda + (i - r * p.K)] : zero;
    } else {
      const int64_t o = i - in_a, q = o >> 4, step = q / p.N;
      const int r = static_cast<int>(step) * 16 + static_cast<int>(o & 15);
      static_cast<T*>(p.b_out)[o] = r < p.rank ? static_cast<const T*>(p.b)[(q - step * p.N) * p.ldb + r] : zero;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *p.rank_out = p.rank;
    *p.scale_out = p.scale;
  }
}

// Opts a kernel into its dynamic shared memory once per device, and into the SM's largest shared-memory
// split (a kernel with a smaller one would keep the dependent GEMM's CTAs off its SMs).
cudaError_t allow_smem(const void* kernel, int bytes) {
  struct Done {
    const void* fn;
    int dev;
  };
  static std::mutex mu;
  static Done done[256];
  static int n = 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lk(mu);
  for (int i = 0; i < n; ++i)
    if (done[i].fn == kernel && done[i].dev == dev) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess && n < 256) done[n++] = Done{kernel, dev};
  return e;
}

// Shared memory of the stages.  Enough to keep HBM busy, little enough to leave room for a CTA of the
// adapters' kernel beside it, and more than a third of an SM, so that CTAs that share one always find
// tensor memory.  The epilogue passes kTN * 512 bytes of sums through it.
constexpr int ring_bytes(int tn) { return tn > 256 ? 0 : 160 * 1024; }
static_assert(ring_bytes(256) >= 256 * 512, "the sums fit the ring");

template <typename T, int kTN, bool kMx4>
cudaError_t launch_gemm(const RowsGemm& g, const CUtensorMap& w, const CUtensorMap& x, cudaStream_t st) {
  auto* k = rows_gemm_kernel<T, kTN, kMx4>;
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(k), ring_bytes(kTN) + 1024);
  if (e != cudaSuccess) return e;
  const dim3 grid(static_cast<unsigned>((g.a.N + kWRows - 1) / kWRows * g.ksplit),
                  static_cast<unsigned>((g.a.T + kTN - 1) / kTN));
  return launch_cluster(k, grid, g.ksplit, dim3(kMx4 ? kGemmThreads + 32 : kGemmThreads), ring_bytes(kTN) + 1024, st,
                        g.a.row_slot != nullptr, w, x, g);  // early beside the adapters' part only, which came after x
}

// The adapters' part of up to 256 rows: one CTA an SM, beside the GEMM's; few rows are cut over a larger cluster.
template <typename T>
cudaError_t lora_part(const RowsArgs& a, int num_sms, cudaStream_t st) {
  const int tiles = (a.T + kTileRows - 1) / kTileRows;
  int kparts = tiles == 1 ? 8 : 4;
  while (kparts > 1 && (a.K + 31) / 32 < kparts * kShrinkWarps) kparts /= 2;
  const int clusters = num_sms / kparts;
  int slices = clusters / tiles;
  slices = slices < 1 ? 1 : slices > kTileRows ? kTileRows : slices;
  if (slices > a.T) slices = a.T;
  const dim3 grid(static_cast<unsigned>((tiles * slices < clusters ? tiles * slices : clusters) * kparts));
  auto* k = a.r_pad == 16   ? rows_lora_kernel<T, 1>
            : a.r_pad == 32 ? rows_lora_kernel<T, 2>
            : a.r_pad == 64 ? rows_lora_kernel<T, 4>
                            : rows_lora_kernel<T, 8>;
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(k), 0);
  if (e != cudaSuccess) return e;
  return launch_cluster(k, grid, kparts, dim3(kShrinkThreads), 0, st, false, a, slices, kparts);
}

// The adapters' part of many rows, in three launches.
template <typename T>
cudaError_t many_part(const RowsArgs& a, int dtype, const ManyMaps& m, int num_sms, cudaStream_t st) {
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(many_plan_kernel), kPlanSmem);
  int log2_slots = 10;  // of the sort's table: at most half full
  while ((1 << log2_slots) < 2 * a.T) ++log2_slots;
  if (e == cudaSuccess) e = launch(many_plan_kernel, 1, kPlanThreads, (8u << log2_slots) + a.T * 2, st, false, a, log2_slots);
  if (e != cudaSuccess) return e;
  const int64_t most = static_cast<int64_t>(a.T / kTileRows) + a.n_slots;  // a slot has one tile that is not full
  const int tiles = static_cast<int>(most < a.T ? most : a.T);
  ManyShrink s{};
  s.a = a;
  s.ab_fmt = dtype == LF_BF16 ? 1 : 0;
  s.ksplit = 1;
  const int nkb = (a.K + kBK - 1) / kBK;
  while (s.ksplit < 8 && tiles * s.ksplit * 2 <= num_sms && nkb >= s.ksplit * 8) s.ksplit *= 2;
  s.pitch = a.r_pad + 4;
  constexpr int kMost = 224 * 1024;  // one limit for every rank: a kernel is opted into its shared memory once
  constexpr int kExpandSmem = kExpandStages * kExpandStageBytes + kEpiWarps * kDeltaStageBytes + 1024;
  static_assert(kExpandSmem <= kMost, "shared memory of an SM");
  static_assert(2 * 2 * (kXBytes + 16 * kBK * 2) >= kTileRows * (LF_BANK_MAX_RANK + 4) * 4, "the sums fit the ring");
  const int block = kXBytes + a.r_pad * kBK * 2;
  s.stages = (kMost - 1024) / (2 * block);
  if (s.stages > kShrinkMaxStages) s.stages = kShrinkMaxStages;
  auto* k = many_shrink_kernel<T>;
  int clusters = num_sms / s.ksplit;
  if (clusters > tiles) clusters = tiles;
  e = allow_smem(reinterpret_cast<const void*>(k), kMost);
  if (e == cudaSuccess)
    e = launch_cluster(k, dim3(static_cast<unsigned>(clusters * s.ksplit)), s.ksplit, dim3(kGemmThreads),
                       s.stages * 2 * block + 1024, st, true, m.a, s);
  if (e != cudaSuccess) return e;
  ManyExpand x{};
  x.a = a;
  x.idesc = umma_idesc_f16(kTileRows, 256, s.ab_fmt, 0, 0);
  const int64_t units = static_cast<int64_t>(tiles) * ((a.N + 255) / 256);
  auto* kx = many_expand_kernel<T>;
  e = allow_smem(reinterpret_cast<const void*>(kx), kExpandSmem);
  if (e != cudaSuccess) return e;
  return launch_cluster(kx, dim3(static_cast<unsigned>(units < num_sms ? units : num_sms)), 1, dim3(kGemmThreads),
                        kExpandSmem, st, true, m.s_hi, m.s_lo, m.b, x);
}

template <typename T>
cudaError_t adapters_part(const RowsArgs& a, int dtype, const ManyMaps* m, int num_sms, cudaStream_t st) {
  return m ? many_part<T>(a, dtype, *m, num_sms, st) : lora_part<T>(a, num_sms, st);
}

template <typename T, bool kMx4>
cudaError_t rows_tc(const RowsArgs& a, int dtype, const CUtensorMap& w, const CUtensorMap& x, const ManyMaps* m, int tn,
                    int ksplit, int num_sms, cudaStream_t st) {
  const cudaError_t e = a.row_slot ? adapters_part<T>(a, dtype, m, num_sms, st) : cudaSuccess;
  if (e != cudaSuccess) return e;
  RowsGemm g{};
  g.a = a;
  g.idesc = umma_idesc_f16(kWRows, tn, dtype == LF_BF16 ? 1 : 0, 0, 0);
  g.ksplit = ksplit;
  const int room = ring_bytes(tn), block = (kWRows + tn) * kBK * 2;
  g.sub = room / (2 * block) >= 3 ? 2 : 1;
  g.stages = room / (g.sub * block);
  if (kMx4) {  // three stages (two of 64 rows' pairs of blocks), the rest for codes: a CTA's K range of a few rows at once
    g.sub = tn <= 64 ? 2 : 1;
    g.stages = tn == 64 ? 2 : 3;
    g.slots = (room - g.stages * g.sub * block) / kMx4Block;
    if (g.slots > kMaxSlots) g.slots = kMaxSlots;
    if (g.slots < (tn == 256 ? g.stages : g.sub * g.stages + 2)) return cudaErrorInvalidValue;  // see the decoding loop
  }
  if (tn == 16) return launch_gemm<T, 16, kMx4>(g, w, x, st);
  if (tn == 32) return launch_gemm<T, 32, kMx4>(g, w, x, st);
  if (tn == 64) return launch_gemm<T, 64, kMx4>(g, w, x, st);
  if (tn == 128) return launch_gemm<T, 128, kMx4>(g, w, x, st);
  return launch_gemm<T, 256, kMx4>(g, w, x, st);
}

template <typename T>
cudaError_t rows_simt_t(const RowsArgs& a, cudaStream_t st) {
  cudaError_t e = launch(rows_shrink_simt_kernel<T>, a.T, kSimtShrink, 0, st, false, a);
  if (e != cudaSuccess) return e;
  const dim3 grid((a.N + kST - 1) / kST, (a.T + kST - 1) / kST);
  return launch_cluster(rows_gemm_simt_kernel<T>, grid, 1, dim3(256), 0, st, true, a);
}

}  // namespace

RowsTiles rows_tiles(int T, int K, int N, int num_sms) {
  RowsTiles t{};
  t.rows = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : T <= 128 ? 128 : 256;
  // K is split while the tiles leave more than half of the SMs without one and a part has 256 elements.
  // (Smaller tiles that cover every SM were slower: 32 features a tile and no split took 20 us where
  // 128 features and a split in four took 12.6, at 1 x 4096 -> 4096, and a GPU without free SMs cannot place the
  // adapters' CTAs beside the GEMM's.)
  const int64_t tiles = static_cast<int64_t>((N + kWRows - 1) / kWRows) * ((T + t.rows - 1) / t.rows);
  const int nkb = (K + kBK - 1) / kBK;
  t.ksplit = 1;
  while (t.ksplit < 8 && tiles * t.ksplit * 2 <= num_sms && nkb >= t.ksplit * 2 * 4) t.ksplit *= 2;
  return t;
}

cudaError_t rows_forward_tc(const RowsArgs& a, int dtype, const CUtensorMap& w, const CUtensorMap& x, const RowsTiles& t,
                            const ManyMaps* m, int num_sms, cudaStream_t st) {
  if (a.mx4.data)
    return dtype == LF_BF16 ? rows_tc<__nv_bfloat16, true>(a, dtype, w, x, m, t.rows, t.ksplit, num_sms, st)
                            : rows_tc<__half, true>(a, dtype, w, x, m, t.rows, t.ksplit, num_sms, st);
  return dtype == LF_BF16 ? rows_tc<__nv_bfloat16, false>(a, dtype, w, x, m, t.rows, t.ksplit, num_sms, st)
                          : rows_tc<__half, false>(a, dtype, w, x, m, t.rows, t.ksplit, num_sms, st);
}

cudaError_t rows_lora_part(const RowsArgs& a, int dtype, const ManyMaps* m, int num_sms, cudaStream_t st) {
  return dtype == LF_BF16 ? adapters_part<__nv_bfloat16>(a, dtype, m, num_sms, st)
                          : adapters_part<__half>(a, dtype, m, num_sms, st);
}

// Rounds of full tiles times the time of one (measured at K = 4096: 23 us for a 256 x 256 tile of a CTA pair, 32 us for
// a 128 x 256 tile of one CTA when every SM has one, a K part taking its share and the split about 5 us more).
bool rows_use_pairs(int T, int K, int N, int num_sms) {
  if (T <= 256) return false;
  const int64_t pair_tiles = static_cast<int64_t>((T + 255) / 256) * ((N + 255) / 256);
  const int64_t tiles = static_cast<int64_t>((T + 255) / 256) * ((N + kWRows - 1) / kWRows);
  const int ks = rows_tiles(T, K, N, num_sms).ksplit;
  const double pair = 23.0 * ((pair_tiles + num_sms / 2 - 1) / (num_sms / 2)) * K / 4096;
  const double one = 32.0 * ((tiles * ks + num_sms - 1) / num_sms) * K / 4096 / ks + 5.0;
  return pair < one;
}

// Over a weight in 4 bits both kernels are bound by the decoding, and a CTA pair's start, with its hand-over between the
// CTAs, costs more: the tiles of W as the M operand are faster or equal while every SM has at most one (333 rows
// 1000 -> 1048 16 us against 26, 512 rows 4096 -> 4096 28 against 36, 1024 rows 41 against 42), the pairs beyond that (700 rows
// 8192 -> 8192 96 against 121, 4096 rows 4096 -> 4096 119 against 141).
bool mx4_use_pairs(int T, int N, int num_sms) {
  return T > 256 && (static_cast<int64_t>(T) + 255) / 256 * ((N + kWRows - 1) / kWRows) > num_sms;
}

cudaError_t bank_load(const BankLoad& p, int dtype, int num_sms, cudaStream_t st) {
  const int64_t blocks = (static_cast<int64_t>(p.r_pad) * (static_cast<int64_t>(p.K) + p.N) + 255) / 256;
  const unsigned grid = static_cast<unsigned>(blocks < 16 * num_sms ? blocks : 16 * num_sms);
  auto* k = dtype == LF_F32    ? bank_load_kernel<float>
            : dtype == LF_BF16 ? bank_load_kernel<__nv_bfloat16>
                               : bank_load_kernel<__half>;
  return launch(k, grid, 256, 0, st, false, p);
}

cudaError_t rows_forward_simt(const RowsArgs& a, int dtype, cudaStream_t st) {
  if (dtype == LF_F32) return rows_simt_t<float>(a, st);
  return dtype == LF_BF16 ? rows_simt_t<__nv_bfloat16>(a, st) : rows_simt_t<__half>(a, st);
}

}  // namespace lf
