// Kernels of the adapters' dropout that stand apart from the products (numbers and mask: lf_drop.cuh).
//
//   drop_mask    xm = m x, bit for bit x or zero (1 / (1 - p) is in the adapters' factors: no rounding of its own).
//   drop_expand  delta[t] = m[t] (S_b[t] A_i), float32, which the grad_x GEMM adds to g W in its epilogue.
#include "lf_drop.cuh"
#include "lf_internal.cuh"
#include "lf_launch.cuh"
#include "lf_ptx.cuh"

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
    const uint4 r = philox(static_cast<uint32_t>(g), static_cast<uint32_t>(t), d);
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

// delta [T, K] (float32) = m (S_b A_i), on tcgen05: units of 128 rows x 256 columns, persistent, one CTA an SM.  Warp 0 loads
// for every segment of the row tile its S_b (hi and lo halves: both products go to one accumulator, so S enters to 2^-16) and
// 256 rows of A_i^T [K, r_pad]; warp 1 issues the MMAs into one of two accumulators; eight warps mask 32 rows x 128
// columns each and store them through shared memory.  A lane has a row, so eight columns are one counter's numbers.
// The rank is short: what bounds it is the 4 T K bytes written, with the generator (1.3 us a unit of 2.9 us at the copy
// rate) behind them.  4096 x 4096 with rank 16 takes 23 us, 8192 rows with rank 64 36 (profiler, cold caches).  (With
// warp-level MMAs that read both operands where they lie: 61 and 220, bound by L1.)
constexpr int kExpandCols = 256;
constexpr int kExpandThreads = 320;
constexpr int kExpandRing = 128 * 1024;
constexpr int kExpandMaxStages = 8;
constexpr int kExpandStaging = 8 * 2 * 32 * 32 * 4;  // 8 warps x 2 buffers x (32 rows x 32 columns)
constexpr int kExpandSmem = 1024 + kExpandRing + kExpandStaging;
struct ExpandParams {
  int T, K, n_cols, units;  // n_cols: column blocks
  int stages, stage_bytes;
  int lo_row;               // where the plane of the low halves starts in the S map
  uint32_t idesc, layout, sbo;
  DropArgs drop;
  Tables tb;
};

__global__ void __launch_bounds__(kExpandThreads, 1)
    drop_expand_kernel(const __grid_constant__ CUtensorMap map_s, const __grid_constant__ CUtensorMap map_l,
                       const __grid_constant__ CUtensorMap map_d, const ExpandParams prm) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = ring + kExpandRing;
  __shared__ uint64_t full[kExpandMaxStages], empty[kExpandMaxStages], tfull[2], tempty[2], drain;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Tables& tb = prm.tb;
  const int rp = tb.r_pad, s_bytes = 128 * rp * 2;
  if (threadIdx.x == 0) {
    for (int i = 0; i < prm.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 8);
    }
    mbar_init(&drain, 1);
    abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_s);
    tma_prefetch_desc(&map_l);
    tma_prefetch_desc(&map_d);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();  // S_b

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0, issued = 0, parity = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < prm.units && ok; u += gridDim.x) {
      const int tile = u / prm.n_cols, c0 = (u - tile * prm.n_cols) * kExpandCols;
      const int st1 = tb.tile_st(tile + 1);
      for (int st = tb.tile_st(tile); st < st1; ++st) {
        ok = warp_wait_stage(&empty[stage], phase ^ 1, &abort_flag, tb.err, kErrTimeoutEmpty);
        if (!ok) break;
        const int slot = tb.st_slot(st);
        if (elect_one()) {
          uint8_t* p = ring + stage * prm.stage_bytes;
          mbar_arrive_expect_tx(&full[stage], 4 * s_bytes);
          tma_load_2d(p, &map_s, &full[stage], 0, st * 128);
          tma_load_2d(p + s_bytes, &map_s, &full[stage], 0, prm.lo_row + st * 128);
          tma_load_2d(p + 2 * s_bytes, &map_l, &full[stage], 0, slot * prm.K + c0);
          tma_load_2d(p + 3 * s_bytes, &map_l, &full[stage], 0, slot * prm.K + c0 + 128);
        }
        __syncwarp();
        issued |= 1u << stage;
        parity = (parity & ~(1u << stage)) | (phase << stage);
        if (++stage == prm.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok && lane == 0)  // let every copy that was started land
      for (int i = 0; i < prm.stages; ++i)
        if (issued & (1u << i)) drain_wait(&full[i], (parity >> i) & 1u, tb.err);
    __syncwarp();
  } else if (warp == 1) {
    int stage = 0, it = 0;
    uint32_t phase = 0;
    bool ok = true, any = false;
    for (int u = blockIdx.x; u < prm.units && ok; u += gridDim.x, ++it) {
      const int tile = u / prm.n_cols, buf = it & 1;
      ok = warp_wait_stage(&tempty[buf], ((it >> 1) & 1) ^ 1, &abort_flag, tb.err, kErrTimeoutAcc);
      if (!ok) break;
      tc_fence_after();
      uint32_t acc = 0;
      const int st1 = tb.tile_st(tile + 1);
      for (int st = tb.tile_st(tile); st < st1; ++st) {
        ok = warp_wait_stage(&full[stage], phase, &abort_flag, tb.err, kErrTimeoutFull);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t p = smem_u32(ring + stage * prm.stage_bytes);
          for (int half = 0; half < 2; ++half)
            for (int k = 0; k < rp / 16; ++k)
              umma_f16(tmem + buf * 256, umma_sdesc(p + half * s_bytes + k * 32, 16, prm.sbo, prm.layout),
                       umma_sdesc(p + 2 * s_bytes + k * 32, 16, prm.sbo, prm.layout), prm.idesc, acc | half | k);
          umma_commit(&empty[stage]);
        }
        __syncwarp();
        acc = 1;
        any = true;
        if (++stage == prm.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (ok && elect_one()) umma_commit(&tfull[buf]);
      __syncwarp();
    }
    if (!ok && any && elect_one()) {
      umma_commit(&drain);
      drain_wait(&drain, 0, tb.err);
    }
    __syncwarp();
  } else {
    const int w = warp - 2, q = warp & 3, half = w >> 2;
    uint8_t* mine = staging + w * (2 * 4096);
    int it = 0, buf_out = 0;
    for (int u = blockIdx.x; u < prm.units; u += gridDim.x, ++it) {
      const int tile = u / prm.n_cols, c0 = (u - tile * prm.n_cols) * kExpandCols + half * 128, buf = it & 1;
      const int row = q * 32 + lane;
      const uint32_t high = row_threshold(tb, prm.drop, tile, row) << 16;
      if (!warp_wait(&tfull[buf], (it >> 1) & 1, &abort_flag, tb.err, kErrTimeoutAcc)) break;
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < 128; c += 32) {
        uint32_t v[32];
        tmem_ld32(tmem + (static_cast<uint32_t>(q * 32) << 16) + buf * 256 + half * 128 + c, v);
        uint32_t ctr[4];
        uint4 r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) ctr[j] = static_cast<uint32_t>((c0 + c) / 8 + j);
        philox<4>(ctr, static_cast<uint32_t>(tile * LF_TILE_ROWS + row), prm.drop, r);
        tmem_wait_ld();
        if (c == 96) {  // accumulator fully read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tempty[buf]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t word[4] = {r[j].x, r[j].y, r[j].z, r[j].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if ((word[i] << 16) < high) v[8 * j + 2 * i] = 0u;
            if (word[i] < high) v[8 * j + 2 * i + 1] = 0u;
          }
        }
        if (c0 + c >= prm.K || tile * LF_TILE_ROWS + q * 32 >= prm.T) continue;
        uint8_t* out = mine + buf_out * 4096;
        if (lane == 0) bulk_wait_read<1>();  // the store that used this buffer has read it
        __syncwarp();
#pragma unroll
        for (int g = 0; g < 8; ++g)
          *reinterpret_cast<uint4*>(out + lane * 128 + ((g ^ (lane & 7)) << 4)) =
              make_uint4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&map_d, out, c0 + c, tile * LF_TILE_ROWS + q * 32);
          bulk_commit();
        }
        buf_out ^= 1;
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
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

cudaError_t drop_expand(int dtype, const CUtensorMap& s_map, const CUtensorMap& l_map, const CUtensorMap& delta_map, int T,
                        int K, const Tables& tb, const DropArgs& d, int num_sms, cudaStream_t st) {
  if (T == 0 || K == 0) return cudaSuccess;
  ExpandParams p{};
  p.T = T, p.K = K;
  p.n_cols = (K + kExpandCols - 1) / kExpandCols;
  const int64_t units = static_cast<int64_t>(tb.n_tiles) * p.n_cols;
  if (units > INT32_MAX) return cudaErrorInvalidValue;
  p.units = static_cast<int>(units);
  p.stage_bytes = 4 * 128 * tb.r_pad * 2;
  p.stages = kExpandRing / p.stage_bytes;
  if (p.stages > kExpandMaxStages) p.stages = kExpandMaxStages;
  p.lo_row = (tb.n_segtiles + 1) * LF_TILE_ROWS;
  p.idesc = umma_idesc_f16(128, kExpandCols, dtype == LF_BF16 ? 1 : 0, 0, 0);
  p.layout = umma_layout_for_span(tb.r_pad * 2);
  p.sbo = static_cast<uint32_t>(8 * tb.r_pad * 2);
  p.drop = d;
  p.tb = tb;
  const cudaError_t e =
      cudaFuncSetAttribute(drop_expand_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kExpandSmem);  // of this device
  if (e != cudaSuccess) return e;
  return launch(drop_expand_kernel, static_cast<unsigned>(p.units < num_sms ? p.units : num_sms), kExpandThreads, kExpandSmem,
                st, true, s_map, l_map, delta_map, p);
}

}  // namespace lf
