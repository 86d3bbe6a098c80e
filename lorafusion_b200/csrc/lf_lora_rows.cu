// One shared projection with an adapter per row, the adapter's index read on the device:
//   y[t] = x[t] W^T + s_i (x[t] A_i^T) B_i^T,   i = row_slot[t]  (negative: no adapter).
//
// Two launches, the second started while the first runs:
//   rows_lora    the adapters' part, float32: S = x[t] A_i^T, then s_i S B_i^T.  Rows are grouped by adapter on
//                the device, so any order of rows works and no host plan is needed.  A cluster takes a
//                few groups: its CTAs cut K for S, exchange their sums through distributed shared
//                memory, then cut the output features, so no grid-wide step lies between A_i and B_i.
//                Few rows bring one adapter each: both products are streams of weights through
//                warp-level MMAs whose 8 columns are rows of one adapter, bound by bytes.
//   rows_gemm    y^T tiles of 128 output features x up to 256 rows with tcgen05 (the weight is the
//                M operand, so a decode step of a few rows wastes no tensor-memory lanes and streams
//                W once), K split over a cluster when the tiles alone would leave SMs idle.  The
//                epilogue waits for the first launch, adds its part and writes y once.
//
// S enters the second product as hi + lo halves of the input type after a per-row power-of-two scaling (the
// row's largest magnitude becomes 1..2), so it is exact to about 2^-16 (bf16) or 2^-22 (f16)
// relative and a float16 S cannot overflow.  All sums are float32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

#include "lf_internal.cuh"
#include "lf_launch.cuh"
#include "lf_ptx.cuh"

namespace lf {
namespace {

constexpr uint32_t kNoSlot = 0xffffffffu;
constexpr int kTileRows = 128;  // rows grouped by adapter together
constexpr int kShrinkThreads = 256;
constexpr int kShrinkWarps = kShrinkThreads / 32;
constexpr int kPartBytes = 32 * 1024;  // per-warp partial products of one batch of groups

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

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// One warp's K steps k0 .. k1 - 1 (32 elements each) of up to kNB groups of one adapter (rank up to 16 kMT) into its
// slots of `part`.  Few instructions a step count more here than anything else (with the bounds of K and
// of the rows tested on every load a step took 90): whole steps run without a test, and a row that a group
// does not have points at one that exists, for columns nobody reads.
template <typename T, int kMT, int kNB, int kUnroll>
__device__ __forceinline__ void shrink_steps(float (&acc)[kMT][kNB][4], const T* const (&xr)[kNB], const T* ar, int K,
                                             int k, bool in) {
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 xv[kUnroll][kNB], lo[kUnroll][kMT], hi[kUnroll][kMT];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
#pragma unroll
    for (int m = 0; m < kMT; ++m) {
      lo[i][m] = in ? *reinterpret_cast<const uint4*>(ar + m * 16 * K + (k + i) * 32) : zero;
      hi[i][m] = in ? *reinterpret_cast<const uint4*>(ar + (m * 16 + 8) * K + (k + i) * 32) : zero;
    }
#pragma unroll
    for (int b = 0; b < kNB; ++b) xv[i][b] = in ? *reinterpret_cast<const uint4*>(xr[b] + (k + i) * 32) : zero;
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i)
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int b = 0; b < kNB; ++b) {
        mma16816(acc[m][b], lo[i][m].x, hi[i][m].x, lo[i][m].y, hi[i][m].y, xv[i][b].x, xv[i][b].y,
                 static_cast<T*>(nullptr));
        mma16816(acc[m][b], lo[i][m].z, hi[i][m].z, lo[i][m].w, hi[i][m].w, xv[i][b].z, xv[i][b].w,
                 static_cast<T*>(nullptr));
      }
}
template <typename T, int kMT, int kNB, int kUnroll, int kStride>
__device__ __forceinline__ void shrink_groups(const T* const (&xr)[kNB], const T* ar, int K, int k0, int k1, int nb,
                                              float* dst) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  float acc[kMT][kNB][4];
#pragma unroll
  for (int m = 0; m < kMT; ++m)
#pragma unroll
    for (int b = 0; b < kNB; ++b) acc[m][b][0] = acc[m][b][1] = acc[m][b][2] = acc[m][b][3] = 0.f;
  const int whole = min(k1, K / 32);
  int k = k0;
#pragma unroll 1
  for (; k + kUnroll <= whole; k += kUnroll) shrink_steps<T, kMT, kNB, kUnroll>(acc, xr, ar, K, k, true);
#pragma unroll 1
  for (; k < k1; ++k) shrink_steps<T, kMT, kNB, 1>(acc, xr, ar, K, k, k * 32 + 8 * q < K);
#pragma unroll
  for (int b = 0; b < kNB; ++b) {
    if (b < nb) {
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        float* at = dst + b * kStride + (m * 16 + g) * 8 + 2 * q;
        *reinterpret_cast<float2*>(at) = make_float2(acc[m][b][0], acc[m][b][1]);
        *reinterpret_cast<float2*>(at + 64) = make_float2(acc[m][b][2], acc[m][b][3]);
      }
    }
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
  int cost[kTileRows];          // what the groups up to each one (this one not) cost, and all of them
  int total;
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
  // a group's cost: its rank steps, and about one step for the rest
  if (warp == 0) {
    int sum = 0;
    for (int c = 0; c < n_groups; c += 32) {
      const int mine = c + lane < n_groups ? 1 + ((rank_of(s.eff[s.start[c + lane]]) + 15) >> 4) : 0;
      int up = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += v;
      }
      if (c + lane < n_groups) s.cost[c + lane] = sum + up - mine;
      sum += __shfl_sync(0xffffffffu, up, 31);
    }
    if (lane == 0) s.total = sum;
  }
  __syncthreads();
  return n_groups;
}

// First group of a slice: groups go to the slice that their cost's middle falls into.
__device__ __forceinline__ int slice_start(const Groups& s, int n_groups, int slice, int slices) {
  int lo = 0, hi = n_groups;  // the first group whose middle is at or past the slice's share
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    const int next = mid + 1 < n_groups ? s.cost[mid + 1] : s.total;
    if (static_cast<int64_t>(s.cost[mid] + next) * slices < 2ll * s.total * slice) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// 2^ex with the largest of a row's values over 1..2; 0 for a row that is all zero or not finite.
__device__ __forceinline__ int row_exponent(float top) {
  return top > 0.f && top <= 3.402823466e38f ? max(-126, min(126, ilogbf(top))) : 0;
}
// v scaled, as high and low halves; the high half of a value that is not finite says it all
template <typename T>
__device__ __forceinline__ void halves(float w, T& hi, T& lo) {
  hi = from_f32<T>(w);
  lo = from_f32<T>(fabsf(w) <= 4.f ? w - to_f32(hi) : 0.f);
}

// One group of 8 rows as the second product sees it: S halves of row g, rows and factors of columns 2q, 2q + 1 (-1:
// the group has no such row).
template <typename T>
struct GroupRows {
  const T* hi;
  const T* lo;
  int row0, row1;
  float f0, f1;
};

// The second product of up to kNB groups of one adapter for output blocks b0 .. b1 - 1 (16 features each): kNM rank
// steps of 16, kPer blocks loaded together.  B_i is stored in the order of the MMA's operand: one 16-byte load a
// lane and step.
template <typename T, int kNM, int kNB, int kPer>
__device__ __forceinline__ void expand_blocks(const uint4* w, int pitch, const uint2 (&sh)[kNB][kNM],
                                              const uint2 (&sl)[kNB][kNM], const GroupRows<T> (&rows)[kNB],
                                              float* const (&o0)[kNB], float* const (&o1)[kNB], int at, int nb,
                                              bool second) {
  T* const tag = nullptr;
  uint4 v[kPer][kNM];
#pragma unroll
  for (int i = 0; i < kPer; ++i)
#pragma unroll
    for (int k = 0; k < kNM; ++k) v[i][k] = w[k * pitch + (at + i) * 32];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
#pragma unroll
    for (int b = 0; b < kNB; ++b) {
      if (b < nb) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kNM; ++k) {
          mma16816(d, v[i][k].x, v[i][k].z, v[i][k].y, v[i][k].w, sh[b][k].x, sh[b][k].y, tag);
          mma16816(d, v[i][k].x, v[i][k].z, v[i][k].y, v[i][k].w, sl[b][k].x, sl[b][k].y, tag);
        }
        float* p0 = o0[b] + (at + i) * 16;
        float* p1 = o1[b] + (at + i) * 16;
        if (rows[b].row0 >= 0) p0[0] = rows[b].f0 * d[0], p0[8] = rows[b].f0 * d[2];
        if (second && rows[b].row1 >= 0) p1[0] = rows[b].f1 * d[1], p1[8] = rows[b].f1 * d[3];
      }
    }
  }
}
template <typename T, int kNM, int kNB, int kPer>
__device__ __forceinline__ void expand_group(const RowsArgs& p, uint32_t e, int b0, int b1,
                                             const GroupRows<T> (&rows)[kNB], int nb) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int blocks = (p.N + 15) >> 4, steps = p.r_pad >> 4;
  uint2 sh[kNB][kNM], sl[kNB][kNM];
  float *o0[kNB], *o1[kNB];
  bool odd = false;
#pragma unroll
  for (int b = 0; b < kNB; ++b) {
#pragma unroll
    for (int k = 0; k < kNM; ++k) {
      const bool on = 16 * k < rank_of(e);
      sh[b][k] = on ? *reinterpret_cast<const uint2*>(rows[b].hi + 16 * k + 4 * q) : make_uint2(0, 0);
      sl[b][k] = on ? *reinterpret_cast<const uint2*>(rows[b].lo + 16 * k + 4 * q) : make_uint2(0, 0);
    }
    o0[b] = p.delta + static_cast<size_t>(max(rows[b].row0, 0)) * blocks * 16 + g;
    o1[b] = p.delta + static_cast<size_t>(max(rows[b].row1, 0)) * blocks * 16 + g;
    odd = odd || rows[b].row1 >= 0;
  }
  const bool second = __any_sync(0xffffffffu, odd);
  const uint4* w = static_cast<const uint4*>(p.b_bank) + static_cast<size_t>(slot_of(e)) * steps * blocks * 32 + lane;
  int b = b0;
#pragma unroll 1
  for (; b + kPer <= b1; b += kPer)
    expand_blocks<T, kNM, kNB, kPer>(w, blocks * 32, sh, sl, rows, o0, o1, b, nb, second);
#pragma unroll 1
  for (; b < b1; ++b) expand_blocks<T, kNM, kNB, 1>(w, blocks * 32, sh, sl, rows, o0, o1, b, nb, second);
}

// Groups from `grp` on, at most kNB and `most`, that belong to one adapter.
template <int kNB>
__device__ __forceinline__ int unit_size(const Groups& s, int grp, int most) {
  int nb = 1;
  if (kNB > 1) {
    const uint32_t e = s.eff[s.start[grp]];
    while (nb < kNB && nb < most && s.eff[s.start[grp + nb]] == e) ++nb;
  }
  return nb;
}

// Work items: (row tile, slice of its groups), each taken by a cluster of `kparts` CTAs that cut K for the
// first product and the output features for the second.  Partial products
// meet in shared memory, then across the cluster, in a fixed order.  The grid fits the GPU at once, so
// the dependent GEMM streams its weight while this kernel runs.
// kNB = 1: a few rows, clusters.  kNB > 1: many rows (prompts), no cluster; up to kNB groups of one adapter share
// what is read of it.
template <typename T, int kMT, int kNB>
__global__ void __launch_bounds__(kShrinkThreads, 2) rows_lora_kernel(const RowsArgs p, int slices, int kparts_) {
  const int kparts = kNB > 1 ? 1 : kparts_;
  constexpr int kRP = kMT * 16;                                         // padded rank
  constexpr int kBatch = kPartBytes / (kShrinkWarps * kRP * 8 * 4);     // groups of 8 rows per batch
  constexpr int kPitch = kRP + 8;                                       // of S rows: no bank conflicts
  __shared__ float part[kShrinkWarps][kBatch][kRP * 8];
  __shared__ __align__(16) Groups s;
  __shared__ __align__(16) T s_hi[kBatch][8][kPitch], s_lo[kBatch][8][kPitch];
  __shared__ float s_fac[kBatch][8];
  __shared__ float s_in[kBatch * kRP * 8 + 8];  // the cluster's sums of this CTA's share (see below)
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
    const int g_lo = slice_start(s, n_groups, slice, slices);
    const int g_hi = slice + 1 < slices ? slice_start(s, n_groups, slice + 1, slices) : n_groups;
    for (int first = g_lo; first < g_hi; first += kBatch) {
      const int batch = min(kBatch, g_hi - first);
      // Up to kNB groups of one adapter are a unit.  The warps divide the units first, so that as many streams
      // of A_i as there are warps are in flight, and K where there are fewer units than warps.
      int n_units = 0;
      for (int u = 0; u < batch; u += unit_size<kNB>(s, first + u, batch - u)) ++n_units;
      const int lanes = n_units >= 8 ? 8 : n_units >= 4 ? 4 : n_units >= 2 ? 2 : 1;  // units at a time
      const int subs = kShrinkWarps / lanes, sub = warp / lanes;
      const int ranges = kparts * subs, me = crank * subs + sub;
      const int b0 = static_cast<int>(static_cast<int64_t>(me) * n_blocks / ranges);
      const int b1 = static_cast<int>(static_cast<int64_t>(me + 1) * n_blocks / ranges);
      for (int u = 0, index = 0, nb; u < batch; u += nb, ++index) {
        nb = unit_size<kNB>(s, first + u, batch - u);
        if (index % lanes != warp % lanes) continue;
        const uint32_t e = s.eff[s.start[first + u]];
        const int nm = (rank_of(e) + 15) >> 4;
        const T* xr[kNB];
#pragma unroll
        for (int b = 0; b < kNB; ++b) {
          const int row = b < nb ? s.rows[first + u + b][g] : 0;
          xr[b] = x + static_cast<int64_t>(t0 + max(row, 0)) * p.ldx + 8 * q;
        }
        const T* ar = bank + (static_cast<size_t>(slot_of(e)) * p.r_pad + g) * K + 8 * q;
        float* dst = part[sub][u];
        const T* const one_x[1] = {xr[0]};
        constexpr int kS = kRP * 8;
        // the smallest kernel that covers the adapter's rank and the groups at hand
        if (nm == 1) {
          if (kNB == 1 || nb == 1) shrink_groups<T, 1, 1, 8, kS>(one_x, ar, K, b0, b1, 1, dst);
          else shrink_groups<T, 1, kNB, 2, kS>(xr, ar, K, b0, b1, nb, dst);
        } else if (nm == 2) {
          if constexpr (kMT >= 2) {
            if (kNB == 1 || nb == 1) shrink_groups<T, 2, 1, 4, kS>(one_x, ar, K, b0, b1, 1, dst);
            else shrink_groups<T, 2, kNB, 2, kS>(xr, ar, K, b0, b1, nb, dst);
          }
        } else if (nm <= 4) {
          if constexpr (kMT >= 4) {
            if (kNB == 1 || nb == 1) shrink_groups<T, 4, 1, 2, kS>(one_x, ar, K, b0, b1, 1, dst);
            else shrink_groups<T, 4, kNB, 1, kS>(xr, ar, K, b0, b1, nb, dst);
          }
        } else if constexpr (kMT >= 8) {
          shrink_groups<T, 8, 1, 1, kS>(one_x, ar, K, b0, b1, 1, dst);
        }
      }
      __syncthreads();
      // The warps' sums, and with a cluster the CTAs': value i (of the batch's kRP x 8 a group) is summed by CTA
      // i / segment, which the others send theirs and which sends the sum to all.
      // The finished sums take the place of the first warp's.
      float* const s_sum = &part[0][0][0];
      const int values = batch * kRP * 8, segment = (values + kparts - 1) / kparts;
      for (int i = tid; i < values; i += kShrinkThreads) {
        float v = part[0][0][i];
        for (int w = 1; w < subs; ++w) v += part[w][0][i];
        if (kparts == 1) {
          s_sum[i] = v;
        } else {
          const int owner = i / segment;
          st_cluster_f32(map_to_cta(smem_u32(&s_in[crank * segment + i - owner * segment]), owner), __float_as_uint(v));
        }
      }
      if (kparts > 1) {
        cluster_sync_all();
        for (int i = tid; i < min(segment, values - crank * segment); i += kShrinkThreads) {
          float v = s_in[i];
          for (int c = 1; c < kparts; ++c) v += s_in[c * segment + i];
          const uint32_t at = smem_u32(&s_sum[crank * segment + i]);
          for (int c = 0; c < kparts; ++c) st_cluster_f32(map_to_cta(at, c), __float_as_uint(v));
        }
        cluster_sync_all();
      } else {
        __syncthreads();
      }
      // S of each group, one warp a group; every CTA needs all of them for the second product
      for (int u = warp; u < batch; u += kShrinkWarps) {
        const uint32_t e = s.eff[s.start[first + u]];
        const int rank = rank_of(e);
        float v[kRP / 4];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < kRP / 4; ++i) v[i] = (lane >> 3) + 4 * i < rank ? s_sum[u * kRP * 8 + lane + 32 * i] : 0.f;
#pragma unroll
        for (int i = 0; i < kRP / 4; ++i) {
          top = fmaxf(top, fabsf(v[i]));
          if (!(fabsf(v[i]) <= 3.402823466e38f)) top = __int_as_float(0x7f800000);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const int ex = row_exponent(top);
        const float down = scalbnf(1.f, -ex), fac = p.slot_scale[slot_of(e)] * scalbnf(1.f, ex);
        if (lane < 8) s_fac[u][lane] = fac;
#pragma unroll
        for (int i = 0; i < kRP / 4; ++i) {
          const int j = (lane >> 3) + 4 * i;
          if (j < ((rank + 15) & ~15)) halves<T>(v[i] * down, s_hi[u][lane & 7][j], s_lo[u][lane & 7][j]);
        }
      }
      __syncthreads();
      // the warps divide the units, then the features, here too
      const int f0 = nb0 + (nb1 - nb0) * sub / subs, f1 = nb0 + (nb1 - nb0) * (sub + 1) / subs;
      for (int u = 0, index = 0, nb; u < batch; u += nb, ++index) {
        nb = unit_size<kNB>(s, first + u, batch - u);
        if (index % lanes != warp % lanes) continue;
        const uint32_t e = s.eff[s.start[first + u]];
        const int nm = (rank_of(e) + 15) >> 4;
        GroupRows<T> rows_of[kNB];
#pragma unroll
        for (int b = 0; b < kNB; ++b) {
          const int v = u + min(b, nb - 1);
          rows_of[b].hi = s_hi[v][g];
          rows_of[b].lo = s_lo[v][g];
          const int r0 = b < nb ? s.rows[first + v][2 * q] : -1, r1 = b < nb ? s.rows[first + v][2 * q + 1] : -1;
          rows_of[b].row0 = r0 < 0 ? -1 : t0 + r0;
          rows_of[b].row1 = r1 < 0 ? -1 : t0 + r1;
          rows_of[b].f0 = s_fac[v][2 * q];
          rows_of[b].f1 = s_fac[v][2 * q + 1];
        }
        constexpr int kPer = kNB > 1 ? 4 : 8;  // 16-byte loads in flight a lane
        if (nm == 1) expand_group<T, 1, kNB, kPer>(p, e, f0, f1, rows_of, nb);
        else if (nm == 2) {
          if constexpr (kMT >= 2) expand_group<T, 2, kNB, kPer / 2>(p, e, f0, f1, rows_of, nb);
        } else if (nm <= 4) {
          if constexpr (kMT >= 4) expand_group<T, 4, kNB, kPer / 4>(p, e, f0, f1, rows_of, nb);
        } else if constexpr (kMT >= 8) {
          expand_group<T, 8, kNB, 1>(p, e, f0, f1, rows_of, nb);
        }
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

// kTN: rows (tokens) of a tile, the N of the MMA.  Warp 0 loads, warp 1 issues the MMAs, eight epilogue warps
// finish the tile.
template <typename T, int kTN>
__global__ void __maxnreg__(80)
    rows_gemm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                     const __grid_constant__ RowsGemm prm) {
  constexpr int kXBytes = kTN * kBK * 2;
  constexpr int kCols = kTN < 32 ? 32 : kTN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_bar, drain_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  __shared__ uint8_t s_on[kTN];  // whether the row has an adapter
  const RowsArgs& p = prm.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int w_bytes = kWBytes, block_bytes = w_bytes + kXBytes;
  // A stage holds `sub` blocks of 64 elements of K.  A block costs the loading thread two copies and the MMA
  // thread four MMAs, but each wait costs both about 0.1 us: with one block a stage, a tile of few rows took 0.35 us
  // a block however small its bytes.
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
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_bar, 1);
    mbar_init(&drain_bar, 1);
    abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_w);
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
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, parity = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; kb += sub) {
        if (!mbar_wait_stage(&empty[stage], phase ^ 1, &abort_flag, p.err, kErrTimeoutEmpty)) {
          ok = false;
          break;
        }
        uint8_t* w = ring + stage * stage_bytes;
        const int n = min(sub, kb1 - kb);
        mbar_arrive_expect_tx(&full[stage], n * block_bytes);
        for (int i = 0; i < n; ++i, w += block_bytes) {
          tma_load_2d(w, &map_w, &full[stage], (kb + i) * kBK, n0);
          tma_load_2d(w + w_bytes, &map_x, &full[stage], (kb + i) * kBK, t0);
        }
        issued |= 1u << stage;
        parity = (parity & ~(1u << stage)) | (phase << stage);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok)  // let every copy this thread started land before the memory is used again
        for (int s = 0; s < stages; ++s)
          if (issued & (1u << s)) drain_wait(&full[s], (parity >> s) & 1u, p.err);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, acc = 0;
      bool ok = true;
      // descriptors of the first block; addresses are in 16-byte units in their low bits
      const uint64_t w0 = umma_sdesc(smem_u32(ring), 16, 1024, 2);
      for (int kb = kb0; kb < kb1; kb += sub) {
        if (!mbar_wait_stage(&full[stage], phase, &abort_flag, p.err, kErrTimeoutFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int n = min(sub, kb1 - kb);
        uint64_t w = w0 + ((stage * stage_bytes) >> 4);
        for (int i = 0; i < n; ++i, w += block_bytes >> 4) {
          const uint64_t x = w + (w_bytes >> 4);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            umma_f16(tmem, w + 2 * k, x + 2 * k, prm.idesc, acc);
            acc = 1;
          }
        }
        umma_commit(&empty[stage]);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (ok) {
        umma_commit(&acc_bar);
      } else if (acc) {
        umma_commit(&drain_bar);
        drain_wait(&drain_bar, 0, p.err);
      }
    }
    __syncwarp();
  } else {
    for (int i = tid - 64; i < kTN; i += kEpiWarps * 32)
      s_on[i] = t0 + i < p.T && row_adapter(p, t0 + i, false) != kNoSlot;
    named_barrier(1, kEpiWarps * 32);
  }
  const bool ok = warp_wait(&acc_bar, 0, &abort_flag, p.err, kErrTimeoutAcc);
  tc_fence_after();

  // The accumulator goes through the idle ring as [source CTA][row][feature], float32, so that a thread then
  // holds 8 features of a row.  Every CTA of the cluster finishes its own share of the features and gets
  // the others' partial sums of it.
  const int ew = warp - 2, quad = warp & 3;
  const int own = kWRows / ks, rows = min(kTN, p.T - t0);
  if (ks > 1) cluster_sync_all();  // every ring is idle
  if (ok && ew >= 0) {
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
    for (int i = tid; i < rows << shift; i += kGemmThreads) {
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

// ============================================================================ CUDA cores
// Float32 problems and shapes TMA cannot address.  One CTA a row for S; then 32 x 32 output tiles.
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
    if (tid < 8 && j0 + tid < rank) {
      float v = part[0][tid];
#pragma unroll
      for (int w = 1; w < kSimtShrink / 32; ++w) v += part[w][tid];
      s[j0 + tid] = scale * v;
    }
    __syncthreads();
  }
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
  pdl_wait();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = t0 + tr + i;
    if (t >= p.T) continue;
    const uint32_t e = p.eff[t];
    const float* s = static_cast<const float*>(p.s_hi) + static_cast<size_t>(t) * p.r_pad;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = n0 + tc + j;
      if (n >= p.N) continue;
      float v = acc[i][j];
      if (e != kNoSlot) {
        // feature n of its block of 16, rank r of its step of 16: place 8 (4 (n % 8) + r / 4) + 4 (n / 8) + r % 4
        const int blocks = (p.N + 15) >> 4, f = n & 15;
        const T* b = static_cast<const T*>(p.b_bank) +
                     (static_cast<size_t>(slot_of(e)) * (p.r_pad >> 4) * blocks + (n >> 4)) * 256 + (f & 7) * 32 + (f >> 3) * 4;
        float add = 0.f;
        for (int r = 0; r < rank_of(e); ++r)
          add = fmaf(s[r], to_f32(b[static_cast<size_t>(r >> 4) * blocks * 256 + (r >> 2 & 3) * 8 + (r & 3)]), add);
        v += add;
      }
      static_cast<T*>(p.y)[static_cast<size_t>(t) * p.N + n] = from_f32<T>(v);
    }
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

template <typename T, int kTN>
cudaError_t launch_gemm(const RowsGemm& g, const CUtensorMap& w, const CUtensorMap& x, cudaStream_t st) {
  auto* k = rows_gemm_kernel<T, kTN>;
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(k), ring_bytes(kTN) + 1024);
  if (e != cudaSuccess) return e;
  const dim3 grid(static_cast<unsigned>((g.a.N + kWRows - 1) / kWRows * g.ksplit),
                  static_cast<unsigned>((g.a.T + kTN - 1) / kTN));
  return launch_cluster(k, grid, g.ksplit, dim3(kGemmThreads), ring_bytes(kTN) + 1024, st, true, w, x, g);
}

// The adapters' part of rows with `a`.  Up to 256 rows: one CTA an SM, beside the GEMM's; few rows are cut over a larger
// cluster.  More rows: two CTAs an SM and no cluster (the GEMM that follows needs whole SMs).
template <typename T>
cudaError_t lora_part(const RowsArgs& a, int num_sms, cudaStream_t st) {
  const int tiles = (a.T + kTileRows - 1) / kTileRows;
  const bool many = tiles > 2;
  int kparts = many ? 1 : tiles == 1 ? 8 : 4;
  while (kparts > 1 && (a.K + 31) / 32 < kparts * kShrinkWarps) kparts /= 2;
  const int clusters = (many ? 2 : 1) * num_sms / kparts;
  int slices = clusters / tiles;
  slices = slices < 1 ? 1 : slices > kTileRows ? kTileRows : slices;
  if (slices > a.T) slices = a.T;
  const dim3 grid(static_cast<unsigned>((tiles * slices < clusters ? tiles * slices : clusters) * kparts));
  cudaError_t e;
#define LF_LORA(MT, NB)                                                                                       \
  {                                                                                                           \
    auto* k = many ? rows_lora_kernel<T, MT, NB> : rows_lora_kernel<T, MT, 1>;                                \
    e = allow_smem(reinterpret_cast<const void*>(k), 0);                                                      \
    if (e == cudaSuccess) e = launch_cluster(k, grid, kparts, dim3(kShrinkThreads), 0, st, false, a, slices, kparts); \
  }
  if (a.r_pad == 16) LF_LORA(1, 4)
  else if (a.r_pad == 32) LF_LORA(2, 4)
  else if (a.r_pad == 64) LF_LORA(4, 2)
  else LF_LORA(8, 1)
#undef LF_LORA
  return e;
}

template <typename T>
cudaError_t rows_tc(const RowsArgs& a, int dtype, const CUtensorMap& w, const CUtensorMap& x, int tn, int ksplit,
                    int num_sms, cudaStream_t st) {
  const cudaError_t e = lora_part<T>(a, num_sms, st);
  if (e != cudaSuccess) return e;
  RowsGemm g{};
  g.a = a;
  g.idesc = umma_idesc_f16(kWRows, tn, dtype == LF_BF16 ? 1 : 0, 0, 0);
  g.ksplit = ksplit;
  const int room = ring_bytes(tn), block = (kWRows + tn) * kBK * 2;
  g.sub = room / (2 * block) >= 3 ? 2 : 1;
  g.stages = room / (g.sub * block);
  if (tn == 16) return launch_gemm<T, 16>(g, w, x, st);
  if (tn == 32) return launch_gemm<T, 32>(g, w, x, st);
  if (tn == 64) return launch_gemm<T, 64>(g, w, x, st);
  if (tn == 128) return launch_gemm<T, 128>(g, w, x, st);
  return launch_gemm<T, 256>(g, w, x, st);
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
  // 128 features and a split in four takes 12.6, at 1 x 4096 -> 4096, and a GPU without free SMs cannot place the
  // adapters' CTAs beside the GEMM's.)
  const int64_t tiles = static_cast<int64_t>((N + kWRows - 1) / kWRows) * ((T + t.rows - 1) / t.rows);
  const int nkb = (K + kBK - 1) / kBK;
  t.ksplit = 1;
  while (t.ksplit < 8 && tiles * t.ksplit * 2 <= num_sms && nkb >= t.ksplit * 2 * 4) t.ksplit *= 2;
  return t;
}

cudaError_t rows_forward_tc(const RowsArgs& a, int dtype, const CUtensorMap& w, const CUtensorMap& x, const RowsTiles& t,
                            int num_sms, cudaStream_t st) {
  return dtype == LF_BF16 ? rows_tc<__nv_bfloat16>(a, dtype, w, x, t.rows, t.ksplit, num_sms, st)
                          : rows_tc<__half>(a, dtype, w, x, t.rows, t.ksplit, num_sms, st);
}

cudaError_t rows_lora_part(const RowsArgs& a, int dtype, int num_sms, cudaStream_t st) {
  return dtype == LF_BF16 ? lora_part<__nv_bfloat16>(a, num_sms, st) : lora_part<__half>(a, num_sms, st);
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

cudaError_t rows_forward_simt(const RowsArgs& a, int dtype, cudaStream_t st) {
  if (dtype == LF_F32) return rows_simt_t<float>(a, st);
  return dtype == LF_BF16 ? rows_simt_t<__nv_bfloat16>(a, st) : rows_simt_t<__half>(a, st);
}

}  // namespace lf
