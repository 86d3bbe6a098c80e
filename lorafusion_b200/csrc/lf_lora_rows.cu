// One shared projection with an adapter per row, the adapter's index read on the device:
//   y[t] = x[t] W^T + s_i (x[t] A_i^T) B_i^T,   i = row_slot[t]  (negative: no adapter).
//
// Two launches, the second started while the first runs:
//   rows_shrink  S[t] = x[t] A_i^T.  Rows are grouped by adapter inside tiles of 128 rows, on the
//                device, so any order of rows works and no host plan is needed.  A group's A_i is
//                read once per tile.  Few rows bring one adapter each, so the product is a stream
//                of A_i through warp-level MMAs whose 8 columns are rows of one adapter: bound by the
//                bytes of A_i, and by x for long batches, never by the MMA rate.
//   rows_gemm    y^T tiles of 128 output features x up to 256 rows with tcgen05 (the weight is the
//                M operand, so a decode step of a few rows wastes no tensor-memory lanes and streams
//                W once), K split over a cluster when the tiles alone would leave SMs idle.  The
//                epilogue waits for the shrink, adds s_i S[t] B_i^T per 8 rows with warp-level MMAs on
//                the accumulator fragments, and writes y once.  B_i is prefetched into L2 while the
//                weight streams.
//
// S is kept as hi + lo halves of the input type after a per-row power-of-two scaling (the row's
// largest magnitude becomes 1..2), so it enters the expand to about 2^-16 (bf16) or 2^-22 (f16)
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
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, __half*) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ============================================================================ shrink
// Grid: (row tile, slice of its groups, K part); the K parts of one (tile, slice) form a cluster.
// Every warp takes its own K range of every group of 8 rows; partial products meet in shared memory,
// then across the cluster, in a fixed order.
template <typename T, int kMT>
__global__ void __launch_bounds__(kShrinkThreads) rows_shrink_kernel(const RowsArgs p, int slices, int kparts) {
  constexpr int kRP = kMT * 16;                                         // padded rank
  constexpr int kBatch = kPartBytes / (kShrinkWarps * kRP * 8 * 4);     // groups of 8 rows per batch
  __shared__ float part[kShrinkWarps][kBatch][kRP * 8];
  __shared__ uint32_t s_eff[kTileRows];
  __shared__ int16_t s_pos[kTileRows];
  __shared__ int16_t s_start[kTileRows];     // first row of each group
  __shared__ int16_t s_rows[kTileRows][8];   // rows of each group, -1: none
  __shared__ int s_warp_groups[4];
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int crank = blockIdx.x % kparts;
  const int slice = blockIdx.x / kparts % slices;
  const int t0 = blockIdx.x / (kparts * slices) * kTileRows;
  const int rows = min(kTileRows, p.T - t0);

  uint32_t eff = kNoSlot;
  if (tid < kTileRows) {
    if (tid < rows) {
      eff = row_adapter(p, t0 + tid, true);
      if (crank == 0 && slice == 0) p.eff[t0 + tid] = eff;
    }
    s_eff[tid] = eff;
#pragma unroll
    for (int i = 0; i < 8; ++i) s_rows[tid][i] = -1;
  }
  __syncthreads();
  // position of each row among its adapter's rows of the tile; every eighth starts a group
  int pos = 0;
  if (tid < rows && eff != kNoSlot)
    for (int j = 0; j < tid; ++j) pos += s_eff[j] == eff;
  const bool starts = tid < rows && eff != kNoSlot && (pos & 7) == 0;
  uint32_t vote = 0;
  if (tid < kTileRows) {
    s_pos[tid] = static_cast<int16_t>(pos);
    vote = __ballot_sync(0xffffffffu, starts);
    if (lane == 0) s_warp_groups[warp] = __popc(vote);
  }
  __syncthreads();
  int n_groups = 0, before = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < warp) before += s_warp_groups[w];
    n_groups += s_warp_groups[w];
  }
  if (starts) s_start[before + __popc(vote & ((1u << lane) - 1))] = static_cast<int16_t>(tid);
  __syncthreads();
  if (tid < rows && eff != kNoSlot) {
    const int want = pos & ~7;
    for (int u = 0; u < n_groups; ++u) {
      const int st = s_start[u];
      if (s_eff[st] == eff && s_pos[st] == want) {
        s_rows[u][pos & 7] = static_cast<int16_t>(tid);
        break;
      }
    }
  }
  __syncthreads();

  const int g = lane >> 2, q = lane & 3;
  const T* x = static_cast<const T*>(p.x);
  const T* bank = static_cast<const T*>(p.a_bank);
  const int K = p.K;
  const int n_blocks = (K + 31) / 32;  // 32 elements of K a step: 8 a lane
  const int ranges = kparts * kShrinkWarps, me = crank * kShrinkWarps + warp;
  const int b0 = static_cast<int>(static_cast<int64_t>(me) * n_blocks / ranges);
  const int b1 = static_cast<int>(static_cast<int64_t>(me + 1) * n_blocks / ranges);
  const uint4 zero = make_uint4(0, 0, 0, 0);

  const int mine = n_groups > slice ? (n_groups - slice + slices - 1) / slices : 0;  // groups slice, slice + slices, ..
  for (int first = 0; first < mine; first += kBatch) {
    const int batch = min(kBatch, mine - first);
    for (int u = 0; u < batch; ++u) {
      const int grp = slice + (first + u) * slices;
      const uint32_t e = s_eff[s_start[grp]];
      const int row = s_rows[grp][g];
      const int nm = (rank_of(e) + 15) >> 4;
      const T* xr = x + static_cast<int64_t>(t0 + max(row, 0)) * p.ldx + 8 * q;
      const T* ar = bank + (static_cast<size_t>(slot_of(e)) * p.r_pad + g) * K + 8 * q;
      float acc[kMT][4];
#pragma unroll
      for (int m = 0; m < kMT; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
#pragma unroll(kMT == 1 ? 4 : kMT == 2 ? 2 : 1)
      for (int b = b0; b < b1; ++b) {
        const bool in = b * 32 + 8 * q < K;
        const uint4 xv = in && row >= 0 ? *reinterpret_cast<const uint4*>(xr + b * 32) : zero;
        uint4 lo[kMT], hi[kMT];
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          const bool on = in && m < nm;
          lo[m] = on ? *reinterpret_cast<const uint4*>(ar + static_cast<size_t>(m * 16) * K + b * 32) : zero;
          hi[m] = on ? *reinterpret_cast<const uint4*>(ar + static_cast<size_t>(m * 16 + 8) * K + b * 32) : zero;
        }
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          if (m < nm) {
            mma16816(acc[m], lo[m].x, hi[m].x, lo[m].y, hi[m].y, xv.x, xv.y, static_cast<T*>(nullptr));
            mma16816(acc[m], lo[m].z, hi[m].z, lo[m].w, hi[m].w, xv.z, xv.w, static_cast<T*>(nullptr));
          }
        }
      }
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        float* dst = part[warp][u] + (m * 16 + g) * 8 + 2 * q;
        *reinterpret_cast<float2*>(dst) = make_float2(acc[m][0], acc[m][1]);
        *reinterpret_cast<float2*>(dst + 64) = make_float2(acc[m][2], acc[m][3]);
      }
    }
    __syncthreads();
    for (int i = tid; i < batch * kRP * 8; i += kShrinkThreads) {
      const int u = i / (kRP * 8), j = i % (kRP * 8);
      float v = part[0][u][j];
#pragma unroll
      for (int w = 1; w < kShrinkWarps; ++w) v += part[w][u][j];
      part[0][u][j] = v;
    }
    if (kparts > 1) cluster_sync_all();
    else __syncthreads();
    // group u of the batch is finished by CTA u % kparts of the cluster, one warp a group
    for (int u = warp * kparts + crank; u < batch; u += kShrinkWarps * kparts) {
      const int grp = slice + (first + u) * slices;
      const uint32_t e = s_eff[s_start[grp]];
      const int rank = rank_of(e), row = s_rows[grp][lane & 7];
      float v[kRP / 4];
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < kRP / 4; ++i) {
        const int j = (lane >> 3) + 4 * i;
        v[i] = 0.f;
        if (j < rank) {
          const uint32_t at = smem_u32(&part[0][u][j * 8 + (lane & 7)]);
          if (kparts > 1) {
            for (int c = 0; c < kparts; ++c) v[i] += ld_cluster_f32(map_to_cta(at, c));
          } else {
            v[i] = part[0][u][j * 8 + (lane & 7)];
          }
          top = fmaxf(top, fabsf(v[i]));
          if (!(fabsf(v[i]) <= 3.402823466e38f)) top = __int_as_float(0x7f800000);
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      // 2^exp: the largest magnitude over 1..2; a row that is all zero or not finite stays as it is
      int ex = 0;
      if (top > 0.f && top <= 3.402823466e38f) ex = max(-126, min(126, ilogbf(top)));
      const float down = scalbnf(1.f, -ex);
      if (row >= 0) {
        const size_t at = static_cast<size_t>(t0 + row) * p.r_pad;
        T* hi = static_cast<T*>(p.s_hi) + at;
        T* lo = static_cast<T*>(p.s_lo) + at;
        if (lane < 8) p.factor[t0 + row] = p.slot_scale[slot_of(e)] * scalbnf(1.f, ex);
#pragma unroll
        for (int i = 0; i < kRP / 4; ++i) {
          const int j = (lane >> 3) + 4 * i;
          if (j < ((rank + 15) & ~15)) {
            const float w = v[i] * down;
            const T h = from_f32<T>(w);
            const float rest = w - to_f32(h);
            hi[j] = h;
            lo[j] = from_f32<T>(fabsf(w) <= 4.f ? rest : 0.f);  // not finite: the high half says it all
          }
        }
      }
    }
    if (kparts > 1) cluster_sync_all();  // peers have read this CTA's sums
    else __syncthreads();
  }
}

// ============================================================================ GEMM + expand
constexpr int kGemmThreads = 256;
constexpr int kWRows = 128;  // output features a tile: the M of the MMA
constexpr int kBK = 64;      // K elements of a stage: one 128-byte swizzle row
constexpr int kWBytes = kWRows * kBK * 2;

struct RowsGemm {
  RowsArgs a;
  int ksplit, stages;
  uint32_t idesc;
};

__device__ __forceinline__ void tmem_ld_16x256(uint32_t taddr, float (&v)[4]) {
  uint32_t r[4];
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr));
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, const float (&v)[4]) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3])
               : "memory");
}

// c (16 output features x 8 rows, fragment layout) += s_i S B_i^T for the rows' adapters.  eff: adapter of
// row g of the 8; f0, f1: factors of rows 2q, 2q + 1.  Each distinct adapter of the 8 rows takes its
// own MMAs, and its result only reaches its own rows: values of another adapter that are not finite
// stay with their rows.
template <typename T>
__device__ __forceinline__ void expand8(const RowsArgs& p, float (&c)[4], int n_base, int tok0, uint32_t eff, float f0,
                                        float f1) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  if (__ballot_sync(0xffffffffu, eff != kNoSlot) == 0) return;
  uint32_t e[8];
  uint32_t lead = 0;
  int steps = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    e[i] = __shfl_sync(0xffffffffu, eff, 4 * i);
    bool first = e[i] != kNoSlot;
#pragma unroll
    for (int j = 0; j < i; ++j) first = first && e[j] != e[i];
    if (first) {
      lead |= 1u << i;
      steps = max(steps, (rank_of(e[i]) + 15) >> 4);
    }
  }
  const uint32_t col0 = __shfl_sync(0xffffffffu, eff, 8 * q), col1 = __shfl_sync(0xffffffffu, eff, 8 * q + 4);
  const T* bank = static_cast<const T*>(p.b_bank);
  const bool ok0 = n_base + g < p.N, ok1 = n_base + g + 8 < p.N;
  const size_t srow = static_cast<size_t>(eff != kNoSlot ? tok0 + g : 0) * p.r_pad + 4 * q;
  const T* hi = static_cast<const T*>(p.s_hi) + srow;
  const T* lo = static_cast<const T*>(p.s_lo) + srow;
  const uint2 zero = make_uint2(0, 0);
  float d[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < steps; ++k) {
    const bool live = eff != kNoSlot && 16 * k < rank_of(eff);
    const uint2 sh = live ? *reinterpret_cast<const uint2*>(hi + 16 * k) : zero;
    const uint2 sl = live ? *reinterpret_cast<const uint2*>(lo + 16 * k) : zero;
    uint2 u[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u[i] = v[i] = zero;
      if ((lead >> i & 1u) && 16 * k < rank_of(e[i])) {
        const T* b = bank + (static_cast<size_t>(slot_of(e[i])) * p.N + n_base + g) * p.r_pad + 16 * k + 4 * q;
        if (ok0) u[i] = *reinterpret_cast<const uint2*>(b);
        if (ok1) v[i] = *reinterpret_cast<const uint2*>(b + static_cast<size_t>(8) * p.r_pad);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if ((lead >> i & 1u) && 16 * k < rank_of(e[i])) {
        const bool m = eff == e[i];
        float t[4] = {0.f, 0.f, 0.f, 0.f};
        mma16816(t, u[i].x, v[i].x, u[i].y, v[i].y, m ? sh.x : 0u, m ? sh.y : 0u, static_cast<T*>(nullptr));
        mma16816(t, u[i].x, v[i].x, u[i].y, v[i].y, m ? sl.x : 0u, m ? sl.y : 0u, static_cast<T*>(nullptr));
        if (col0 == e[i]) d[0] += t[0], d[2] += t[2];
        if (col1 == e[i]) d[1] += t[1], d[3] += t[3];
      }
    }
  }
  if (col0 != kNoSlot) c[0] += f0 * d[0], c[2] += f0 * d[2];
  if (col1 != kNoSlot) c[1] += f1 * d[1], c[3] += f1 * d[3];
}

// Writes a fragment (16 features x 8 rows) to y through 256 bytes of the warp's shared memory, 16 bytes
// a store (N is a multiple of 8).
template <typename T>
__device__ __forceinline__ void store8rows(const RowsArgs& p, const float (&c)[4], int n_base, int tok0, T* stage) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  __syncwarp();
  stage[(2 * q) * 16 + g] = from_f32<T>(c[0]);
  stage[(2 * q + 1) * 16 + g] = from_f32<T>(c[1]);
  stage[(2 * q) * 16 + g + 8] = from_f32<T>(c[2]);
  stage[(2 * q + 1) * 16 + g + 8] = from_f32<T>(c[3]);
  __syncwarp();
  if (lane < 16) {
    const int t = tok0 + (lane >> 1), n = n_base + 8 * (lane & 1);
    if (t < p.T && n < p.N)
      *reinterpret_cast<uint4*>(static_cast<T*>(p.y) + static_cast<size_t>(t) * p.N + n) =
          *reinterpret_cast<const uint4*>(stage + (lane >> 1) * 16 + 8 * (lane & 1));
  }
}

// kTN: rows (tokens) of a tile, the N of the MMA.
template <typename T, int kTN>
__global__ void __launch_bounds__(kGemmThreads)
    rows_gemm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                     const __grid_constant__ RowsGemm prm) {
  constexpr int kXBytes = kTN * kBK * 2;
  constexpr int kStageBytes = kWBytes + kXBytes;
  constexpr int kCols = kTN < 32 ? 32 : kTN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[16], empty[16], acc_bar, drain_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  __shared__ uint32_t s_eff[kTN];
  __shared__ float s_fac[kTN];
  __shared__ __align__(16) T s_stage[8][128];
  const RowsArgs& p = prm.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, &abort_flag, p.err, kErrTimeoutEmpty)) {
          ok = false;
          break;
        }
        uint8_t* w = ring + stage * kStageBytes;
        mbar_arrive_expect_tx(&full[stage], kStageBytes);
        tma_load_2d(w, &map_w, &full[stage], kb * kBK, n0);
        tma_load_2d(w + kWBytes, &map_x, &full[stage], kb * kBK, t0);
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
      const uint32_t base = smem_u32(ring);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[stage], phase, &abort_flag, p.err, kErrTimeoutFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t w = base + stage * kStageBytes, x = w + kWBytes;
#pragma unroll
        for (int k = 0; k < kBK / 16; ++k) {
          umma_f16(tmem, umma_sdesc(w + k * 32, 16, 1024, 2), umma_sdesc(x + k * 32, 16, 1024, 2), prm.idesc, acc);
          acc = 1;
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
    // B_i of the rows this CTA will expand, into L2
    const int own = kWRows / ks;  // output features this CTA finishes
    const int nb = n0 + part * own;
    const int feats = min(own, p.N - nb);
    if (feats > 0) {
      const uint32_t bytes = static_cast<uint32_t>(feats) * p.r_pad * 2, lines = (bytes + 127) / 128;
      const int n_rows = min(kTN, p.T - t0);
      for (int r = warp - 2; r < n_rows; r += 6) {
        const uint32_t e = row_adapter(p, t0 + r, false);
        if (e == kNoSlot || (r > 0 && row_adapter(p, t0 + r - 1, false) == e)) continue;
        const char* b = static_cast<const char*>(p.b_bank) +
                        (static_cast<size_t>(slot_of(e)) * p.N + nb) * p.r_pad * 2;
        for (uint32_t l = lane; l < lines; l += 32)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(b + static_cast<size_t>(l) * 128));
      }
    }
  }
  bool ok = warp_wait(&acc_bar, 0, &abort_flag, p.err, kErrTimeoutAcc);
  tc_fence_after();
  pdl_wait();  // the shrink's results
  for (int i = tid; i < kTN; i += kGemmThreads) {
    const bool in = t0 + i < p.T;
    const uint32_t e = in ? p.eff[t0 + i] : kNoSlot;
    s_eff[i] = e;
    s_fac[i] = e != kNoSlot ? p.factor[t0 + i] : 0.f;
  }
  __syncthreads();

  const int g = lane >> 2, q = lane & 3;
  const int quad = warp & 3, half = warp >> 2;  // tensor-memory lanes of the warp; which row groups it takes
  constexpr int kGroups = kTN / 8;
  const int n_groups = min(kGroups, (p.T - t0 + 7) / 8);
  T* stage_out = s_stage[warp];
  if (ks == 1) {
    if (ok) {
      for (int c = half; c < n_groups; c += 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n_base = n0 + quad * 32 + h * 16;
          float v[4];
          tmem_ld_16x256(tmem + (static_cast<uint32_t>(quad * 32 + h * 16) << 16) + c * 8, v);
          if (n_base < p.N) {
            expand8<T>(p, v, n_base, t0 + c * 8, s_eff[c * 8 + g], s_fac[c * 8 + 2 * q], s_fac[c * 8 + 2 * q + 1]);
            store8rows<T>(p, v, n_base, t0 + c * 8, stage_out);
          }
        }
      }
    }
  } else {
    // every CTA of the cluster finishes kWRows / ks features: the others send it their partial sums
    const int per = 8 / ks;      // 16-feature blocks a CTA finishes
    cluster_sync_all();          // every ring is idle
    if (ok) {
      for (int c = half; c < n_groups; c += 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int mt = quad * 2 + h;
          float v[4];
          tmem_ld_16x256(tmem + (static_cast<uint32_t>(mt * 16) << 16) + c * 8, v);
          const uint32_t at = smem_u32(ring) + static_cast<uint32_t>(((part * per + mt % per) * kGroups + c) * 512 + lane * 16);
          st_cluster_v4(map_to_cta(at, mt / per), v);
        }
      }
    }
    cluster_sync_all();
    if (ok) {
      for (int u = warp; u < per * n_groups; u += 8) {
        const int m = u / n_groups, c = u % n_groups;
        const int n_base = n0 + (part * per + m) * 16;
        if (n_base >= p.N) continue;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < ks; ++s) {  // fixed order
          const float4 w = *reinterpret_cast<const float4*>(ring + ((s * per + m) * kGroups + c) * 512 + lane * 16);
          v[0] += w.x, v[1] += w.y, v[2] += w.z, v[3] += w.w;
        }
        expand8<T>(p, v, n_base, t0 + c * 8, s_eff[c * 8 + g], s_fac[c * 8 + 2 * q], s_fac[c * 8 + 2 * q + 1]);
        store8rows<T>(p, v, n_base, t0 + c * 8, stage_out);
      }
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
        const T* b = static_cast<const T*>(p.b_bank) + (static_cast<size_t>(slot_of(e)) * p.N + n) * p.r_pad;
        float add = 0.f;
        for (int r = 0; r < rank_of(e); ++r) add = fmaf(s[r], to_f32(b[r]), add);
        v += add;
      }
      static_cast<T*>(p.y)[static_cast<size_t>(t) * p.N + n] = from_f32<T>(v);
    }
  }
}

// Opts a kernel into its dynamic shared memory once per device.
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
  if (e == cudaSuccess && n < 256) done[n++] = Done{kernel, dev};
  return e;
}

constexpr int kRingBytes = 160 * 1024;  // largest ring: leaves room for a shrink CTA beside it

template <typename T, int kTN>
cudaError_t launch_gemm(const RowsGemm& g, const CUtensorMap& w, const CUtensorMap& x, cudaStream_t st) {
  const int stage = kWBytes + kTN * kBK * 2;
  const int smem = g.stages * stage + 1024;
  auto* k = rows_gemm_kernel<T, kTN>;
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(k), kRingBytes + 1024);
  if (e != cudaSuccess) return e;
  const dim3 grid(static_cast<unsigned>((g.a.N + kWRows - 1) / kWRows * g.ksplit),
                  static_cast<unsigned>((g.a.T + kTN - 1) / kTN));
  return launch_cluster(k, grid, g.ksplit, dim3(kGemmThreads), smem, st, true, w, x, g);
}

template <typename T>
cudaError_t rows_tc(const RowsArgs& a, int dtype, const CUtensorMap& w, const CUtensorMap& x, int tn, int num_sms,
                    cudaStream_t st) {
  // shrink: enough CTAs to fill the GPU once, K cut first (a cluster of up to 8), then the groups
  const int tiles = (a.T + kTileRows - 1) / kTileRows;
  int kparts = a.T <= 16 ? 8 : 4;
  while (kparts > 1 && (a.K + 31) / 32 < kparts * kShrinkWarps) kparts /= 2;
  int slices = 2 * num_sms / (tiles * kparts);
  slices = slices < 1 ? 1 : slices > kTileRows ? kTileRows : slices;
  if (slices > a.T) slices = a.T;
  const dim3 grid(static_cast<unsigned>(tiles) * slices * kparts);
  cudaError_t e;
#define LF_SHRINK(MT) \
  e = launch_cluster(rows_shrink_kernel<T, MT>, grid, kparts, dim3(kShrinkThreads), 0, st, false, a, slices, kparts)
  if (a.r_pad == 16) LF_SHRINK(1);
  else if (a.r_pad == 32) LF_SHRINK(2);
  else if (a.r_pad == 64) LF_SHRINK(4);
  else LF_SHRINK(8);
#undef LF_SHRINK
  if (e != cudaSuccess) return e;

  RowsGemm g{};
  g.a = a;
  g.idesc = umma_idesc_f16(kWRows, tn, dtype == LF_BF16 ? 1 : 0, 0, 0);
  const int64_t out_tiles = static_cast<int64_t>((a.N + kWRows - 1) / kWRows) * ((a.T + tn - 1) / tn);
  const int nkb = (a.K + kBK - 1) / kBK;
  g.ksplit = 1;
  while (g.ksplit < 8 && out_tiles * g.ksplit * 2 <= num_sms && nkb >= g.ksplit * 2 * 4) g.ksplit *= 2;
  const int stage = kWBytes + tn * kBK * 2;
  g.stages = kRingBytes / stage < 12 ? kRingBytes / stage : 12;
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

int rows_tile(int T) { return T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : T <= 128 ? 128 : 256; }

cudaError_t rows_forward_tc(const RowsArgs& a, int dtype, const CUtensorMap& w, const CUtensorMap& x, int num_sms,
                            cudaStream_t st) {
  const int tn = rows_tile(a.T);
  return dtype == LF_BF16 ? rows_tc<__nv_bfloat16>(a, dtype, w, x, tn, num_sms, st)
                          : rows_tc<__half>(a, dtype, w, x, tn, num_sms, st);
}

cudaError_t rows_forward_simt(const RowsArgs& a, int dtype, cudaStream_t st) {
  if (dtype == LF_F32) return rows_simt_t<float>(a, st);
  return dtype == LF_BF16 ? rows_simt_t<__nv_bfloat16>(a, st) : rows_simt_t<__half>(a, st);
}

}  // namespace lf
