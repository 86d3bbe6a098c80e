// Per-adapter gradient norms, clipping and AdamW over many small tensors.
//
// A fine-tuning step of many adapters ends in hundreds of gradient blocks of a few thousand to a
// few million elements.  One launch covers all of them: every tensor is cut into chunks of kChunk
// elements, one CTA per chunk, so neither the count nor the sizes of the tensors shape the grid.
// The addresses of this step's gradients travel in the launch's parameter block (up to 32 KB),
// not through a copy to device memory: no copy precedes the kernels, and a captured launch holds
// its own table.
//
// All kernels stream: the norm pass reads every gradient once, the scale pass reads and writes the
// clipped ones, the update reads gradient, master, two moments and writes master, two moments and
// the rounded weight.  They are bound by HBM; passes that follow a norm pass walk the chunks
// backwards, so they start on what the norm pass left in the 126 MB L2.
//
// Measured, the seven projections of a Llama-3-8B block (896 tensors of 64 adapters, ranks 8 to 64), in brackets the time
// of the bytes at the rate of a copy: clipping 315 MB of bf16 gradients by adapter, of which 231 MB are
// beyond the limit and written, 144 us (83; the scale pass reads them from HBM again, 35); the AdamW step, 4.4 GB, 723 to
// 749 us (673); 256 adapters of rank 64 on 8192 x 28672, 16.9 GB, 2494 to 2594 us (2586).  Chunks of 8192 elements, all loads of a thread before the first use; small
// calls (11 us) are the launches and their host side.
//
// Sums of squares are held in float64 from the first product on: a float32 square overflows above
// 1.8e19 and vanishes below 1e-23, and the sums run over up to 10^9 elements.  Partial sums are
// added in a fixed order, so the norms are the same bits on every run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

#include "lf_internal.cuh"
#include "lf_launch.cuh"

namespace lf {
namespace {

constexpr int kChunk = 8192;      // elements a CTA handles: 4 to 8 16-byte loads a thread
constexpr int kThreads = 256;
constexpr int kFinalThreads = 512;
// CTAs that share a chunk's update (1 / 2 / 4, in turn on one GPU: 16 adapters of rank 16, 4096 -> 4096 22.4 / 20.8 / 20.5
// us, the 896 tensors named above 721 / 711 / 738).
constexpr int kUpdateParts = 2;
constexpr int kGroupsPerLaunch = 4096;  // groups whose presence bits fit one launch's parameters

// ------------------------------------------------------------------- element access
template <typename T>
struct Vec16 {  // 16 bytes of T as floats
  static constexpr int n = 16 / sizeof(T);
};
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[4], float*) {
  f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[8], __nv_bfloat16*) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[8], __half*) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = v.x, f[2 * i + 1] = v.y;
  }
}
__device__ __forceinline__ uint4 pack(const float (&f)[4], float*) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], __nv_bfloat16*) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    std::memcpy(&w[i], &v, 4);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], __half*) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    std::memcpy(&w[i], &v, 4);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load1(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store1(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ------------------------------------------------------------------- reductions
// kInf: the running value is the largest magnitude (a NaN stays a NaN), else a sum of squares.
template <bool kInf>
__device__ __forceinline__ double fold(double acc, float v) {
  if (kInf) {
    const double a = fabs(static_cast<double>(v));
    return (a > acc || a != a) ? a : acc;
  }
  const double d = v;
  return fma(d, d, acc);
}
template <bool kInf>
__device__ __forceinline__ double join(double a, double b) {
  if (kInf) return (b > a || b != b) ? b : a;
  return a + b;
}
// All threads' values joined in a fixed order; the result is valid in thread 0.
template <bool kInf, int kN>
__device__ double block_join(double v) {
  __shared__ double part[kN / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join<kInf>(v, __shfl_down_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = threadIdx.x < kN / 32 ? part[threadIdx.x] : 0.0;
#pragma unroll
    for (int o = kN / 64; o > 0; o >>= 1) v = join<kInf>(v, __shfl_down_sync(0xffffffffu, v, o));
  }
  return v;
}

template <bool kInf, typename T>
__device__ double chunk_fold(const T* p, int n) {
  constexpr int V = Vec16<T>::n;
  constexpr int kIters = kChunk / (kThreads * V);  // vectors a thread loads, all before the first use
  double acc[2] = {0.0, 0.0};
  if (aligned16(p)) {
    uint4 u[kIters];
    const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int at = (i * kThreads + threadIdx.x) * V;
      u[i] = at + V <= n ? *reinterpret_cast<const uint4*>(p + at) : zero;
    }
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      float f[V];
      unpack(u[i], f, static_cast<T*>(nullptr));
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j & 1] = fold<kInf>(acc[j & 1], f[j]);
    }
    const int tail = n / V * V + threadIdx.x;
    if (tail < n) acc[0] = fold<kInf>(acc[0], load1(p + tail));
  } else {
    for (int i = threadIdx.x; i < n; i += kThreads) acc[0] = fold<kInf>(acc[0], load1(p + i));
  }
  return join<kInf>(acc[0], acc[1]);
}

template <bool kInf>
__device__ double chunk_fold_any(uint64_t ptr, int dtype, uint32_t first, int n) {
  if (dtype == LF_F32) return chunk_fold<kInf>(reinterpret_cast<const float*>(ptr) + first, n);
  if (dtype == LF_BF16) return chunk_fold<kInf>(reinterpret_cast<const __nv_bfloat16*>(ptr) + first, n);
  return chunk_fold<kInf>(reinterpret_cast<const __half*>(ptr) + first, n);
}

// min(1, max_norm / (norm + 1e-6)); a NaN norm stays a NaN factor, an infinite limit clips nothing
__device__ __forceinline__ double clip_factor(double norm, double max_norm) {
  if (max_norm > 1.7976931348623157e308) return 1.0;
  const double c = max_norm / (norm + 1e-6);
  return c >= 1.0 ? 1.0 : c;
}

// ------------------------------------------------------------------- clipping
// One launch's tensors, by value: address, elements, first chunk (counted over all launches) and
// group << 2 | dtype.  Sizes in three classes, so a call with few tensors passes few bytes.
template <int kN>
struct GradPack {
  uint64_t ptr[kN];
  uint32_t numel[kN];
  uint32_t chunk0[kN];
  uint32_t group_dtype[kN];
  int n;
  int tensor0;  // index of ptr[0] over all launches
};

// Workspace of one clip call.
struct ClipWs {
  double* part;   // [n_chunks]
  int4* info;     // [n_tensors] first chunk, chunks, group
  float* factor;  // [n_groups]
};

template <int kN>
__device__ __forceinline__ int find_tensor(const GradPack<kN>& pk, uint32_t chunk) {
  int lo = 0, hi = pk.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pk.chunk0[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <bool kInf, int kN>
__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const __grid_constant__ GradPack<kN> pk, ClipWs ws) {
  pdl_launch_dependents();
  const uint32_t chunk = pk.chunk0[0] + blockIdx.x;
  const int t = find_tensor(pk, chunk);
  const uint32_t first = (chunk - pk.chunk0[t]) * kChunk;
  const uint32_t numel = pk.numel[t];
  const int n = min(static_cast<uint32_t>(kChunk), numel - first);
  const double v = block_join<kInf, kThreads>(
      chunk_fold_any<kInf>(pk.ptr[t], pk.group_dtype[t] & 3, first, n));
  if (threadIdx.x == 0) {
    ws.part[chunk] = v;
    if (first == 0)
      ws.info[pk.tensor0 + t] =
          make_int4(chunk, (numel + kChunk - 1) / kChunk, pk.group_dtype[t] >> 2, 0);
  }
}

// One CTA per group: joins the partial values of the group's chunks in a fixed order.
template <bool kInf>
__global__ void __launch_bounds__(kFinalThreads)
    clip_final_kernel(ClipWs ws, int n_tensors, int n_chunks, int n_groups, double max_norm, float* norms) {
  pdl_launch_dependents();
  pdl_wait();
  const int g = blockIdx.x;
  double acc = 0.0;
  if (n_groups == 1) {
    // one group: every chunk, without the tensor records
#pragma unroll 4
    for (int c = threadIdx.x; c < n_chunks; c += kFinalThreads) acc = join<kInf>(acc, ws.part[c]);
  } else {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int t0 = warp * 32; t0 < n_tensors; t0 += kFinalThreads) {
      int4 rec = make_int4(0, 0, -1, 0);
      if (t0 + lane < n_tensors) rec = ws.info[t0 + lane];
      uint32_t mine = __ballot_sync(0xffffffffu, rec.z == g);
      while (mine) {
        const int src = __ffs(mine) - 1;
        mine &= mine - 1;
        const int c0 = __shfl_sync(0xffffffffu, rec.x, src), nc = __shfl_sync(0xffffffffu, rec.y, src);
#pragma unroll 4
        for (int c = lane; c < nc; c += 32) acc = join<kInf>(acc, ws.part[c0 + c]);
      }
    }
  }
  acc = block_join<kInf, kFinalThreads>(acc);
  if (threadIdx.x == 0) {
    const double norm = kInf ? acc : sqrt(acc);
    norms[g] = static_cast<float>(norm);
    ws.factor[g] = static_cast<float>(clip_factor(norm, max_norm));
  }
}

template <typename T>
__device__ void chunk_scale(T* p, int n, float f) {
  constexpr int V = Vec16<T>::n;
  if (aligned16(p)) {
    constexpr int kIters = kChunk / (kThreads * V);
    uint4 u[kIters];
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int at = (i * kThreads + threadIdx.x) * V;
      if (at + V <= n) u[i] = *reinterpret_cast<const uint4*>(p + at);
    }
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int at = (i * kThreads + threadIdx.x) * V;
      if (at + V <= n) {
        float v[V];
        unpack(u[i], v, static_cast<T*>(nullptr));
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= f;
        *reinterpret_cast<uint4*>(p + at) = pack(v, static_cast<T*>(nullptr));
      }
    }
    const int tail = n / V * V + threadIdx.x;
    if (tail < n) store1(p + tail, load1(p + tail) * f);
  } else {
    for (int i = threadIdx.x; i < n; i += kThreads) store1(p + i, load1(p + i) * f);
  }
}

// Scales the chunks of clipped groups; a factor of 1 leaves a gradient as it is.
template <int kN>
__global__ void __launch_bounds__(kThreads) grad_scale_kernel(const __grid_constant__ GradPack<kN> pk, ClipWs ws) {
  pdl_wait();
  const uint32_t chunk = pk.chunk0[0] + (gridDim.x - 1 - blockIdx.x);
  const int t = find_tensor(pk, chunk);
  const float f = ws.factor[pk.group_dtype[t] >> 2];
  if (f == 1.0f) return;
  const uint32_t first = (chunk - pk.chunk0[t]) * kChunk;
  const int n = min(static_cast<uint32_t>(kChunk), pk.numel[t] - first);
  const int dtype = pk.group_dtype[t] & 3;
  if (dtype == LF_F32) chunk_scale(reinterpret_cast<float*>(pk.ptr[t]) + first, n, f);
  else if (dtype == LF_BF16) chunk_scale(reinterpret_cast<__nv_bfloat16*>(pk.ptr[t]) + first, n, f);
  else chunk_scale(reinterpret_cast<__half*>(pk.ptr[t]) + first, n, f);
}

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

uint64_t chunks_of(uint64_t numel) { return (numel + kChunk - 1) / kChunk; }

int elem_bytes(int dtype) { return dtype == LF_F32 ? 4 : 2; }

size_t clip_ws_bytes(uint64_t n_chunks, int n_tensors, int n_groups) {
  return align256(n_chunks * sizeof(double)) + align256(static_cast<size_t>(n_tensors) * sizeof(int4)) +
         align256(static_cast<size_t>(n_groups) * sizeof(float));
}

// Sum of the chunks of all tensors, or 0 with *ok = false when an argument is out of range.
uint64_t check_tensors(const lf_grad_tensor* t, int n, int n_groups, bool* ok) {
  uint64_t chunks = 0;
  *ok = true;
  for (int i = 0; i < n; ++i) {
    if (t[i].dtype < LF_F32 || t[i].dtype > LF_F16 || t[i].group < 0 || t[i].group >= n_groups ||
        t[i].numel >= (uint64_t(1) << 32) - kChunk || (t[i].numel > 0 && t[i].ptr == 0) ||
        t[i].ptr % elem_bytes(t[i].dtype) != 0) {
      *ok = false;
      return 0;
    }
    chunks += chunks_of(t[i].numel);
  }
  if (chunks > 0x7fffffffu) *ok = false;
  return chunks;
}

// No two tensors may share memory: both would be scaled by two launches' CTAs at once.
bool overlap(const lf_grad_tensor* t, int n) {
  std::vector<std::pair<uint64_t, uint64_t>> r;
  r.reserve(n);
  for (int i = 0; i < n; ++i)
    if (t[i].numel) r.emplace_back(t[i].ptr, t[i].ptr + t[i].numel * elem_bytes(t[i].dtype));
  if (!std::is_sorted(r.begin(), r.end())) std::sort(r.begin(), r.end());
  for (size_t i = 1; i < r.size(); ++i)
    if (r[i].first < r[i - 1].second) return true;
  return false;
}

template <int kN>
cudaError_t launch_norm(bool inf, const lf_grad_tensor* t, int n, int tensor0, uint32_t chunk0, uint32_t n_chunks,
                        const ClipWs& ws, int pass, bool pdl, cudaStream_t st) {
  GradPack<kN> pk;
  pk.n = n;
  pk.tensor0 = tensor0;
  uint32_t c = chunk0;
  for (int i = 0; i < n; ++i) {
    pk.ptr[i] = t[i].ptr;
    pk.numel[i] = static_cast<uint32_t>(t[i].numel);
    pk.chunk0[i] = c;
    pk.group_dtype[i] = static_cast<uint32_t>(t[i].group) << 2 | static_cast<uint32_t>(t[i].dtype);
    c += static_cast<uint32_t>(chunks_of(t[i].numel));
  }
  if (pass == 0)
    return inf ? launch(grad_norm_kernel<true, kN>, n_chunks, kThreads, 0, st, pdl, pk, ws)
               : launch(grad_norm_kernel<false, kN>, n_chunks, kThreads, 0, st, pdl, pk, ws);
  return launch(grad_scale_kernel<kN>, n_chunks, kThreads, 0, st, pdl, pk, ws);
}

constexpr int kPackMax = 1500;  // 20 bytes a tensor: a launch takes at most 32,764 parameter bytes

// One pass (0: norms, 1: scale) over all tensors, kPackMax of them a launch.
cudaError_t clip_pass(bool inf, const std::vector<lf_grad_tensor>& t, const ClipWs& ws, int pass, cudaStream_t st) {
  uint32_t chunk0 = 0;
  for (size_t at = 0; at < t.size(); at += kPackMax) {
    const int n = static_cast<int>(std::min<size_t>(kPackMax, t.size() - at));
    uint64_t c = 0;
    for (int i = 0; i < n; ++i) c += chunks_of(t[at + i].numel);
    const uint32_t nc = static_cast<uint32_t>(c);
    const lf_grad_tensor* p = t.data() + at;
    // only the launch right behind the final kernel may start early: it waits for that kernel alone
    const bool pdl = pass == 1 && at == 0;
    cudaError_t e;
    if (n <= 40) e = launch_norm<40>(inf, p, n, static_cast<int>(at), chunk0, nc, ws, pass, pdl, st);
    else if (n <= 200) e = launch_norm<200>(inf, p, n, static_cast<int>(at), chunk0, nc, ws, pass, pdl, st);
    else e = launch_norm<kPackMax>(inf, p, n, static_cast<int>(at), chunk0, nc, ws, pass, pdl, st);
    if (e != cudaSuccess) return e;
    chunk0 += nc;
  }
  return cudaSuccess;
}

// ------------------------------------------------------------------- AdamW
constexpr int kPtrMax = 3840;  // 8 bytes a tensor

template <int kN>
struct PtrPack {
  uint64_t ptr[kN];  // this step's gradients of tensors [tensor0, tensor0 + kN), 0: none
  int tensor0;
};
struct Presence {
  uint32_t bits[kGroupsPerLaunch / 32];
  int group0;
};

struct AdamTables {
  const lf_adamw_tensor* rec;
  const int32_t* chunk_tensor;
};

// What the update needs of a group: g' = factor g, p <- shrink p - size m / (sqrt(v) / root + eps).
struct AdamCoef {
  float factor, shrink, size, root;
};

template <int kN>
__global__ void __launch_bounds__(kThreads)
    adam_norm_kernel(const __grid_constant__ PtrPack<kN> pk, AdamTables tb, int grad_dtype, int chunk0, double* part) {
  pdl_launch_dependents();
  const int chunk = chunk0 + blockIdx.x;
  const int t = tb.chunk_tensor[chunk];
  const lf_adamw_tensor rec = tb.rec[t];
  const uint64_t ptr = pk.ptr[t - pk.tensor0];
  double v = 0.0;
  if (ptr != 0) {
    const uint32_t first = static_cast<uint32_t>(chunk - rec.chunk0) * kChunk;
    const int n = min(static_cast<uint32_t>(kChunk), rec.numel - first);
    v = chunk_fold_any<false>(ptr, grad_dtype, first, n);
  }
  v = block_join<false, kThreads>(v);
  if (threadIdx.x == 0) part[chunk] = v;
}

struct AdamFinal {
  const double* part;  // null: no norms wanted
  const double2* hyper;  // learning rate, weight decay per group
  int32_t* steps;
  AdamCoef* coef;
  float* norms;
  double beta1, beta2, max_norm;  // max_norm < 0: no clipping
  int n_tensors, skip_nonfinite;
};

// One CTA per group: its norm, clip factor, step count and bias corrections.  A group without
// gradients this step keeps its step count; its norm is 0.
__global__ void __launch_bounds__(kThreads)
    adam_final_kernel(const __grid_constant__ Presence pr, AdamTables tb, AdamFinal a) {
  pdl_launch_dependents();
  const int g = pr.group0 + blockIdx.x;
  const bool present = (pr.bits[blockIdx.x >> 5] >> (blockIdx.x & 31)) & 1u;
  AdamCoef c{1.0f, 1.0f, 0.0f, -1.0f};  // root < 0: leave the group as it is
  int t = 0;
  if (threadIdx.x == 0 && present) {  // all but the factor, while the norms are still summed
    t = a.steps[g] + 1;
    const double2 h = a.hyper[g];
    c.shrink = static_cast<float>(1.0 - h.x * h.y);
    c.size = static_cast<float>(h.x / (1.0 - pow(a.beta1, static_cast<double>(t))));
    c.root = static_cast<float>(sqrt(1.0 - pow(a.beta2, static_cast<double>(t))));
  }
  pdl_wait();
  double acc = 0.0;
  if (a.part != nullptr) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int t0 = warp * 32; t0 < a.n_tensors; t0 += kThreads) {
      int group = -1, c0 = 0, nc = 0;
      if (t0 + lane < a.n_tensors) {
        const lf_adamw_tensor& r = tb.rec[t0 + lane];
        group = r.group, c0 = r.chunk0, nc = r.n_chunks;
      }
      uint32_t mine = __ballot_sync(0xffffffffu, group == g);
      while (mine) {
        const int src = __ffs(mine) - 1;
        mine &= mine - 1;
        const int s0 = __shfl_sync(0xffffffffu, c0, src), sn = __shfl_sync(0xffffffffu, nc, src);
#pragma unroll 4
        for (int c = lane; c < sn; c += 32) acc += a.part[s0 + c];
      }
    }
    acc = block_join<false, kThreads>(acc);
  }
  if (threadIdx.x != 0) return;
  const double norm = sqrt(acc);
  if (a.part != nullptr) a.norms[g] = static_cast<float>(norm);
  const bool bad = a.skip_nonfinite && !(norm <= 1.7976931348623157e308);
  if (present && !bad) {
    a.steps[g] = t;
    if (a.max_norm >= 0.0) c.factor = static_cast<float>(clip_factor(norm, a.max_norm));
  } else {
    c.root = -1.0f;
  }
  a.coef[g] = c;
}

struct AdamState {
  float* exp_avg;
  float* exp_avg_sq;
  float* master;  // null for float32 weights
  const AdamCoef* coef;
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps;
};

// The update in float32; the weight is rounded once, from its float32 master.
__device__ __forceinline__ void adam_one(float g, float& p, float& m, float& v, const AdamCoef& c, const AdamState& s) {
  g *= c.factor;
  m = s.beta1 * m + s.one_minus_beta1 * g;
  v = s.beta2 * v + s.one_minus_beta2 * g * g;
  p = c.shrink * p - c.size * m / (sqrtf(v) / c.root + s.eps);
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    float a[4], b[4];
    unpack(*reinterpret_cast<const uint4*>(p), a, static_cast<float*>(nullptr));
    unpack(*reinterpret_cast<const uint4*>(p + 4), b, static_cast<float*>(nullptr));
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = a[i], f[4 + i] = b[i];
  } else {
    unpack(*reinterpret_cast<const uint4*>(p), f, static_cast<T*>(nullptr));
  }
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}

template <typename P, typename G, int kN>
__global__ void __launch_bounds__(kThreads)
    adam_update_kernel(const __grid_constant__ PtrPack<kN> pk, AdamTables tb, AdamState s, int chunk0) {
  constexpr bool kMaster = sizeof(P) == 2;
  const int part = blockIdx.x % kUpdateParts;  // of the chunk
  const int chunk = chunk0 + (gridDim.x - 1 - blockIdx.x) / kUpdateParts;
  const int t = tb.chunk_tensor[chunk];
  const lf_adamw_tensor rec = tb.rec[t];
  const G* grad = reinterpret_cast<const G*>(pk.ptr[t - pk.tensor0]);
  const uint32_t first = static_cast<uint32_t>(chunk - rec.chunk0) * kChunk;
  const int n = min(static_cast<uint32_t>(kChunk), rec.numel - first);
  P* w = reinterpret_cast<P*>(rec.param) + first;
  float* m = s.exp_avg + rec.state_off + first;
  float* v = s.exp_avg_sq + rec.state_off + first;
  float* q = kMaster ? s.master + rec.state_off + first : reinterpret_cast<float*>(w);
  pdl_wait();
  if (grad == nullptr) return;
  const AdamCoef c = s.coef[rec.group];
  if (c.root < 0.0f) return;
  grad += first;
  int done = 0;
  if (aligned16(grad) && aligned16(w)) {  // states start at multiples of 8 elements
    for (int at = (part * kThreads + threadIdx.x) * 8; at + 8 <= n; at += kUpdateParts * kThreads * 8) {
      float fg[8], fq[8], fm[8], fv[8];
      load8(grad + at, fg);
      load8(q + at, fq);
      load8(m + at, fm);
      load8(v + at, fv);
#pragma unroll
      for (int i = 0; i < 8; ++i) adam_one(fg[i], fq[i], fm[i], fv[i], c, s);
      store8(q + at, fq);
      store8(m + at, fm);
      store8(v + at, fv);
      if constexpr (kMaster) *reinterpret_cast<uint4*>(w + at) = pack(fq, static_cast<P*>(nullptr));
    }
    done = n / 8 * 8;
  }
  for (int at = done + part * kThreads + threadIdx.x; at < n; at += kUpdateParts * kThreads) {
    float fq = q[at], fm = m[at], fv = v[at];
    adam_one(load1(grad + at), fq, fm, fv, c, s);
    q[at] = fq, m[at] = fm, v[at] = fv;
    if constexpr (kMaster) store1(w + at, fq);
  }
}

template <int kN>
cudaError_t adam_pass_n(const lf_adamw_args* a, int t0, int t1, int pass, const AdamTables& tb, const AdamState& s,
                        double* part, cudaStream_t st) {
  PtrPack<kN> pk;
  pk.tensor0 = t0;
  for (int i = t0; i < t1; ++i) pk.ptr[i - t0] = a->grads[i];
  const int c0 = a->tensors[t0].chunk0;
  const int nc = a->tensors[t1 - 1].chunk0 + a->tensors[t1 - 1].n_chunks - c0;
  if (nc == 0) return cudaSuccess;
  if (pass == 0) return launch(adam_norm_kernel<kN>, nc, kThreads, 0, st, false, pk, tb, a->grad_dtype, c0, part);
  const bool pdl = t0 == 0;
  const int ctas = nc * kUpdateParts;
  const int pd = a->param_dtype, gd = a->grad_dtype;
  if (pd == LF_F32) return launch(adam_update_kernel<float, float, kN>, ctas, kThreads, 0, st, pdl, pk, tb, s, c0);
  if (pd == LF_BF16) {
    if (gd == LF_F32)
      return launch(adam_update_kernel<__nv_bfloat16, float, kN>, ctas, kThreads, 0, st, pdl, pk, tb, s, c0);
    return launch(adam_update_kernel<__nv_bfloat16, __nv_bfloat16, kN>, ctas, kThreads, 0, st, pdl, pk, tb, s, c0);
  }
  if (gd == LF_F32) return launch(adam_update_kernel<__half, float, kN>, ctas, kThreads, 0, st, pdl, pk, tb, s, c0);
  return launch(adam_update_kernel<__half, __half, kN>, ctas, kThreads, 0, st, pdl, pk, tb, s, c0);
}

cudaError_t adam_pass(const lf_adamw_args* a, int pass, const AdamTables& tb, const AdamState& s, double* part,
                      cudaStream_t st) {
  for (int t0 = 0; t0 < a->n_tensors; t0 += kPtrMax) {
    const int t1 = std::min(a->n_tensors, t0 + kPtrMax);
    cudaError_t e;
    if (t1 - t0 <= 100) e = adam_pass_n<100>(a, t0, t1, pass, tb, s, part, st);
    else if (t1 - t0 <= 500) e = adam_pass_n<500>(a, t0, t1, pass, tb, s, part, st);
    else e = adam_pass_n<kPtrMax>(a, t0, t1, pass, tb, s, part, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

size_t adam_ws_bytes(int64_t n_chunks, int n_groups) {
  return align256(static_cast<size_t>(n_chunks) * sizeof(double)) +
         align256(static_cast<size_t>(n_groups) * sizeof(AdamCoef));
}

}  // namespace
}  // namespace lf

using namespace lf;

extern "C" size_t lf_grad_clip_workspace_bytes(const lf_grad_tensor* tensors, int32_t n_tensors, int32_t n_groups) {
  if (n_tensors < 0 || n_groups < 0 || (n_tensors > 0 && !tensors)) return 0;
  bool ok = true;
  const uint64_t chunks = check_tensors(tensors, n_tensors, n_groups, &ok);
  return ok ? clip_ws_bytes(chunks, n_tensors, n_groups) : 0;
}

extern "C" int lf_grad_clip(const lf_grad_tensor* tensors, int32_t n_tensors, int32_t n_groups, int32_t inf_norm,
                            int32_t scale, double max_norm, float* norms_dev, void* workspace_dev,
                            size_t workspace_bytes, lf_stream_t stream) {
  if (n_tensors < 0 || n_groups < 0 || (n_tensors > 0 && !tensors)) return LF_ERR_INVALID_ARG;
  if (scale && !(max_norm >= 0.0)) return LF_ERR_INVALID_ARG;
  if (n_groups == 0) return n_tensors == 0 ? LF_OK : LF_ERR_INVALID_ARG;
  if (!norms_dev) return LF_ERR_INVALID_ARG;
  bool ok = true;
  const uint64_t chunks = check_tensors(tensors, n_tensors, n_groups, &ok);
  if (!ok) return LF_ERR_INVALID_ARG;
  if (!workspace_dev || workspace_bytes < clip_ws_bytes(chunks, n_tensors, n_groups)) return LF_ERR_CAPACITY;
  if (reinterpret_cast<uintptr_t>(workspace_dev) % 16 != 0) return LF_ERR_INVALID_ARG;
  try {
    if (scale && overlap(tensors, n_tensors)) return LF_ERR_INVALID_ARG;
    std::vector<lf_grad_tensor> t;
    t.reserve(n_tensors);
    for (int i = 0; i < n_tensors; ++i)
      if (tensors[i].numel) t.push_back(tensors[i]);
    char* w = static_cast<char*>(workspace_dev);
    ClipWs ws;
    ws.part = reinterpret_cast<double*>(w);
    w += align256(chunks * sizeof(double));
    ws.info = reinterpret_cast<int4*>(w);
    w += align256(static_cast<size_t>(n_tensors) * sizeof(int4));
    ws.factor = reinterpret_cast<float*>(w);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = clip_pass(inf_norm != 0, t, ws, 0, st);
    const bool pdl = !t.empty();
    const int nt = static_cast<int>(t.size()), nc = static_cast<int>(chunks);
    const double limit = scale ? max_norm : HUGE_VAL;
    if (e == cudaSuccess)
      e = inf_norm ? launch(clip_final_kernel<true>, n_groups, kFinalThreads, 0, st, pdl, ws, nt, nc, n_groups, limit,
                            norms_dev)
                   : launch(clip_final_kernel<false>, n_groups, kFinalThreads, 0, st, pdl, ws, nt, nc, n_groups,
                            limit, norms_dev);
    if (e == cudaSuccess && scale) e = clip_pass(inf_norm != 0, t, ws, 1, st);
    return e == cudaSuccess ? LF_OK : LF_ERR_CUDA;
  } catch (...) {
    return LF_ERR_CAPACITY;
  }
}

extern "C" int lf_adamw_plan(lf_adamw_tensor* tensors, int32_t n_tensors, int32_t n_groups, int32_t* chunk_tensor,
                             int64_t max_chunks, int64_t* n_chunks, int64_t* state_elems) {
  if (n_tensors < 0 || n_groups < 0 || (n_tensors > 0 && !tensors) || !n_chunks || !state_elems)
    return LF_ERR_INVALID_ARG;
  int64_t chunks = 0, off = 0;
  for (int i = 0; i < n_tensors; ++i) {
    lf_adamw_tensor& t = tensors[i];
    if (t.group < 0 || t.group >= n_groups || t.numel > 0xffffffffu - kChunk || (t.numel > 0 && t.param == 0))
      return LF_ERR_INVALID_ARG;
    const int64_t c = static_cast<int64_t>(chunks_of(t.numel));
    if (chunks + c > 0x7fffffff / kUpdateParts) return LF_ERR_INVALID_ARG;  // CTAs of a launch
    t.state_off = off;
    t.chunk0 = static_cast<int32_t>(chunks);
    t.n_chunks = static_cast<int32_t>(c);
    off += (static_cast<int64_t>(t.numel) + 7) / 8 * 8;
    if (chunk_tensor)
      for (int64_t k = chunks; k < chunks + c && k < max_chunks; ++k) chunk_tensor[k] = i;
    chunks += c;
  }
  *n_chunks = chunks;
  *state_elems = off;
  return chunk_tensor && max_chunks < chunks ? LF_ERR_CAPACITY : LF_OK;
}

extern "C" size_t lf_adamw_workspace_bytes(int64_t n_chunks, int32_t n_groups) {
  return n_chunks < 0 || n_groups < 0 ? 0 : adam_ws_bytes(n_chunks, n_groups);
}

extern "C" int lf_adamw_step(const lf_adamw_args* a, lf_stream_t stream) {
  if (!a || a->n_tensors < 0 || a->n_groups < 0 || a->n_chunks < 0) return LF_ERR_INVALID_ARG;
  if (a->n_tensors == 0 || a->n_groups == 0) return LF_OK;
  if (!a->tensors || !a->tensors_dev || !a->grads || !a->hyper_dev || !a->steps_dev) return LF_ERR_INVALID_ARG;
  const int pd = a->param_dtype, gd = a->grad_dtype;
  if (pd < LF_F32 || pd > LF_F16 || (gd != LF_F32 && gd != pd)) return LF_ERR_UNSUPPORTED;
  if (!(a->beta1 >= 0.0 && a->beta1 < 1.0) || !(a->beta2 >= 0.0 && a->beta2 < 1.0) || !(a->eps >= 0.0))
    return LF_ERR_INVALID_ARG;
  const bool norms = a->norms_dev != nullptr;
  if (!norms && (a->max_norm >= 0.0 || a->skip_nonfinite)) return LF_ERR_INVALID_ARG;
  if (a->max_norm != a->max_norm) return LF_ERR_INVALID_ARG;
  if (a->n_chunks > 0 && (!a->chunk_tensor_dev || !a->exp_avg_dev || !a->exp_avg_sq_dev ||
                          (pd != LF_F32 && !a->master_dev)))
    return LF_ERR_INVALID_ARG;
  for (const void* p : {static_cast<const void*>(a->exp_avg_dev), static_cast<const void*>(a->exp_avg_sq_dev),
                        static_cast<const void*>(a->master_dev), static_cast<const void*>(a->workspace_dev),
                        static_cast<const void*>(a->hyper_dev), static_cast<const void*>(a->tensors_dev)})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return LF_ERR_INVALID_ARG;
  if (!a->workspace_dev || a->workspace_bytes < adam_ws_bytes(a->n_chunks, a->n_groups)) return LF_ERR_CAPACITY;
  try {
    std::vector<uint8_t> present(a->n_groups, 0);
    for (int i = 0; i < a->n_tensors; ++i) {
      if (a->tensors[i].group < 0 || a->tensors[i].group >= a->n_groups) return LF_ERR_INVALID_ARG;
      if (a->grads[i] % elem_bytes(gd) != 0) return LF_ERR_INVALID_ARG;
      if (a->grads[i]) present[a->tensors[i].group] = 1;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    char* w = static_cast<char*>(a->workspace_dev);
    double* part = reinterpret_cast<double*>(w);
    AdamCoef* coef = reinterpret_cast<AdamCoef*>(w + align256(static_cast<size_t>(a->n_chunks) * sizeof(double)));
    const AdamTables tb{a->tensors_dev, a->chunk_tensor_dev};
    const AdamState s{a->exp_avg_dev,
                      a->exp_avg_sq_dev,
                      a->master_dev,
                      coef,
                      static_cast<float>(a->beta1),
                      static_cast<float>(1.0 - a->beta1),
                      static_cast<float>(a->beta2),
                      static_cast<float>(1.0 - a->beta2),
                      static_cast<float>(a->eps)};
    cudaError_t e = cudaSuccess;
    if (norms) e = adam_pass(a, 0, tb, s, part, st);
    const AdamFinal f{norms ? part : nullptr,
                      reinterpret_cast<const double2*>(a->hyper_dev),
                      a->steps_dev,
                      coef,
                      a->norms_dev,
                      a->beta1,
                      a->beta2,
                      a->max_norm,
                      a->n_tensors,
                      a->skip_nonfinite};
    for (int g0 = 0; g0 < a->n_groups && e == cudaSuccess; g0 += kGroupsPerLaunch) {
      const int n = std::min(kGroupsPerLaunch, a->n_groups - g0);
      Presence pr;
      std::memset(&pr, 0, sizeof(pr));
      pr.group0 = g0;
      for (int g = 0; g < n; ++g)
        if (present[g0 + g]) pr.bits[g >> 5] |= 1u << (g & 31);
      e = launch(adam_final_kernel, n, kThreads, 0, st, norms && g0 == 0 && a->n_chunks > 0, pr, tb, f);
    }
    if (e == cudaSuccess) e = adam_pass(a, 1, tb, s, part, st);
    return e == cudaSuccess ? LF_OK : LF_ERR_CUDA;
  } catch (...) {
    return LF_ERR_CAPACITY;
  }
}
