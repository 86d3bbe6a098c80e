// C ABI of the fused multi-adapter LoRA operator: argument checks, TMA descriptors,
// kernel dispatch.  No torch types cross this boundary; see include/lorafusion_b200.h.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <vector>

#include "lf_internal.cuh"
#include "lf_mx4.cuh"
#include "lf_ptx.cuh"

namespace lf {

// Device control word (one per device context): the status bounded waits inside the kernels
// record, and the wait limit they read.
__device__ DeviceCtl g_device_ctl = {0, 0, kWaitLimitNs};

namespace {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

struct DeviceState {
  bool ready = false;
  int num_sms = 0;
  int* status = nullptr;      // address of g_device_ctl.status on this device
  std::atomic<bool> no_cosched{false};  // the co-scheduled (cooperative) launch was refused here once
  std::atomic<int> refusal{0};          // the cudaError_t that refused launch returned
  std::vector<cudaEvent_t> events;  // lf_forward_host's stream-ordering events (grown on demand)
  std::mutex ev_mu;
};

std::mutex g_mu;
DeviceState g_dev[64];

// A profiling or checking tool injected into the process replays or serializes kernels, and a
// co-scheduled launch (whose CTAs wait on each other) then fails, so the default is "no
// co-scheduled launches" when one is present.  Signs of one: the variables CUDA tools set for
// their injection (CUDA_INJECTION64_PATH; Nsight Compute's NV_NSIGHT_INJECTION_* and
// NV_COMPUTE_PROFILER_PERFWORKS_DIR; NVIDIA_PROCESS_INJECTION_*), or an injection library mapped
// into the process.
bool tool_injected() {
  for (const char* v : {"CUDA_INJECTION64_PATH", "NV_NSIGHT_INJECTION_TRANSPORT_TYPE", "NV_COMPUTE_PROFILER_PERFWORKS_DIR",
                        "NVIDIA_PROCESS_INJECTION_CRASH_REPORTING"}) {
    const char* x = std::getenv(v);
    if (x != nullptr && x[0] != '\0') return true;
  }
  if (FILE* f = std::fopen("/proc/self/maps", "r")) {
    char line[1024];
    bool found = false;
    while (!found && std::fgets(line, sizeof(line), f))
      found = std::strstr(line, "libcuda-injection") != nullptr || std::strstr(line, "InjectionTarget") != nullptr;
    std::fclose(f);
    if (found) return true;
  }
  return false;
}
int default_cosched_mode() { return tool_injected() ? 0 : 1; }
// process-wide switch (lf_set_co_scheduling): 0 off, 1 dedicated, 2 prologue
std::atomic<int> g_cosched_mode{default_cosched_mode()};

// Test hook (lf_inject_stale_ready): co-scheduled launches that still make their GEMM CTAs wait
// for a ready value no shrink item publishes.
std::atomic<int> g_stale_ready{0};
uint64_t wait_generation(uint64_t gen) {
  int n = g_stale_ready.load();
  while (n > 0 && !g_stale_ready.compare_exchange_weak(n, n - 1)) {
  }
  return n > 0 ? gen + 2 : gen;
}

bool cosched_allowed(const DeviceState* ds) { return !ds->no_cosched.load() && g_cosched_mode.load() != 0; }

// A cooperative launch that returned `e` ran nothing: clear the (non-sticky) launch error, keep
// the code for lf_get_co_scheduling and use ordinary launches on this device from now on.
void refuse_cosched(DeviceState* ds, cudaError_t e) {
  (void)cudaGetLastError();
  int expect = 0;
  ds->refusal.compare_exchange_strong(expect, static_cast<int>(e));
  ds->no_cosched.store(true);
}
// Shrink inside the GEMM launch: on CTA pairs the GEMM's round count leaves idle (default, when
// there are at least four), or as every CTA's prologue (mode 2).
bool cosched_prologue() { return g_cosched_mode.load() == 2; }
EncodeTiledFn g_encode = nullptr;

int elem_bytes(int dtype) { return dtype == LF_F32 ? 4 : 2; }

cudaError_t device_state(DeviceState** out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lk(g_mu);
  DeviceState& d = g_dev[dev];
  if (!d.ready) {
    e = cudaDeviceGetAttribute(&d.num_sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    e = cudaGetSymbolAddress(reinterpret_cast<void**>(&d.status), g_device_ctl);
    if (e != cudaSuccess) return e;
    d.ready = true;
  }
  if (!g_encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
    if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !fn) return e != cudaSuccess ? e : cudaErrorUnknown;
    g_encode = reinterpret_cast<EncodeTiledFn>(fn);
  }
  *out = &d;
  return cudaSuccess;
}

// 2-D tile map over a row-major [outer, inner] matrix with row pitch `pitch_bytes`.
bool make_map(CUtensorMap* m, int dtype, const void* base, uint64_t inner, uint64_t outer, uint64_t pitch_bytes,
              uint32_t box_inner, uint32_t box_outer) {
  const uint32_t span = box_inner * static_cast<uint32_t>(elem_bytes(dtype));
  CUtensorMapSwizzle sw = span == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                          : span == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                       : CU_TENSOR_MAP_SWIZZLE_32B;
  if (span != 128 && span != 64 && span != 32) return false;
  const cuuint64_t dims[2] = {inner, outer};
  const cuuint64_t strides[1] = {pitch_bytes};
  const cuuint32_t box[2] = {box_inner, box_outer};
  const cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType dt = dtype == LF_BF16   ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                 : dtype == LF_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  std::memset(m, 0, sizeof(*m));
  CUresult r = g_encode(m, dt, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int to_status(cudaError_t e) { return e == cudaSuccess ? LF_OK : LF_ERR_CUDA; }

// segment tiles plus one all-zero block (index n_segtiles) the pair GEMM pads with
size_t segtile_elems(const lf_plan_info* info) {
  return static_cast<size_t>(info->n_segtiles + 1) * LF_TILE_ROWS * static_cast<size_t>(info->r_pad);
}

// One S_ext buffer, 256-byte multiple: f64 for the CUDA-core path, or four bf16/f16 planes for
// the tensor-core path.  A tensor-core shrink writes each value v as hi = round(v) in plane h and
// lo = round(v - hi) in plane kh + h, where kh (1 or 2) counts its K-half partial products (two
// when it runs inside the GEMM launch): planes [hi of each K half..., lo of each K half...].  The
// expand of a forward without dropout reads the hi planes, S rounded once as an activation is; the dA/dB grams and the
// expand of a forward with dropout read all 2*kh planes, so S enters their sums with about 16 significant bits
// instead of 8.
size_t sext_bytes(const lf_plan_info* info) { return (segtile_elems(info) * 8 + 255) & ~size_t(255); }

constexpr int kSextPlanes = 4;  // planes one tensor-core S_ext buffer holds

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

// ready flags of the (job, unit, K half) items when shrinks run inside the GEMM launch
// (one job in the forward, two in the backward)
size_t flag_bytes(const lf_plan_info* info, int jobs = 1) {
  return (static_cast<size_t>(info->n_shrink_units) * 2 * 8 * jobs + 255) & ~size_t(255);
}

// Per-launch flag value: unique within the process, so flags left in a reused workspace by an
// earlier launch never read as ready; a stray equal 64-bit value in fresh memory is the only
// (negligible) collision.
uint64_t next_generation() {
  static std::atomic<uint64_t> gen{
      (static_cast<uint64_t>(std::chrono::steady_clock::now().time_since_epoch().count()) << 1) | 1u};
  return gen.fetch_add(2, std::memory_order_relaxed) + 2;
}

int check_problem(const lf_problem* p, const lf_plan_info* info, const int32_t* table_dev) {
  if (!p || !info || (!table_dev && info->table_words > 0)) return LF_ERR_INVALID_ARG;
  if (p->dtype != LF_F32 && p->dtype != LF_BF16 && p->dtype != LF_F16) return LF_ERR_INVALID_ARG;
  if (p->T < 0 || p->K < 0 || p->N < 0) return LF_ERR_INVALID_ARG;
  if (p->T != info->total_rows) return LF_ERR_ROUTING;
  if (info->r_pad != 16 && info->r_pad != 32 && info->r_pad != 64) return LF_ERR_INVALID_ARG;
  return LF_OK;
}

// Tensor-core path: bf16/f16 with every row pitch and base 16-byte aligned (TMA).
bool tc_eligible(const lf_problem* p, std::initializer_list<const void*> ptrs) {
  if (p->dtype == LF_F32) return false;
  if (p->K == 0 || p->N == 0 || p->K % 8 != 0 || p->N % 8 != 0) return false;
  for (const void* q : ptrs)
    if (q && !aligned16(q)) return false;
  return true;
}

}  // namespace

Tables make_tables(const lf_plan_info* info, const int32_t* table_dev) {
  Tables t{};
  t.base = table_dev;
  t.off_tile_st = info->off_tile_st;
  t.off_st_tile = info->off_st_tile;
  t.off_st_lo = info->off_st_lo;
  t.off_st_hi = info->off_st_hi;
  t.off_st_slot = info->off_st_slot;
  t.off_st_scale = info->off_st_scale;
  t.off_slot_st = info->off_slot_st;
  t.off_slot_list = info->off_slot_list;
  t.off_slot_rank = info->off_slot_rank;
  t.off_rank_prefix = info->off_rank_prefix;
  t.off_slot_order = info->off_slot_order;
  t.off_unit_tile = info->off_unit_tile;
  t.off_unit_st0 = info->off_unit_st0;
  t.off_unit_nst = info->off_unit_nst;
  t.off_pair_lora = info->off_pair_lora;
  t.off_pl_a = info->off_pl_a;
  t.off_pl_b = info->off_pl_b;
  t.off_pl_slot = info->off_pl_slot;
  t.off_tile_unit = info->off_tile_unit;
  t.n_tiles = info->n_tiles;
  t.n_segtiles = info->n_segtiles;
  t.n_slots = info->n_slots;
  t.n_units = info->n_shrink_units;
  t.r_pad = info->r_pad;
  t.err = nullptr;
  return t;
}

}  // namespace lf

using namespace lf;

namespace lf {
size_t forward_min_workspace_bytes(const lf_plan_info* info) {
  return info ? align256(sext_bytes(info) + flag_bytes(info)) : 0;
}
}  // namespace lf

namespace {
size_t backward_min_workspace_bytes(const lf_plan_info* info) {
  return info ? align256(2 * sext_bytes(info) + flag_bytes(info, 2) +
                         gram_scratch_bytes(info->r_pad > 0 ? info->r_pad : 16))
              : 0;
}

// The K-split tail's scratch at byte `off` of a workspace of `bytes`: as many partial tiles as
// fit there (none: no split).
PairTail tail_scratch(void* ws, size_t bytes, size_t off) {
  PairTail t{};
  if (ws == nullptr || bytes < off + kTailFlagBytes + kTailPartialBytes) return t;
  char* base = static_cast<char*>(ws) + off;
  if (!aligned16(base)) return t;  // partial tiles are moved by bulk copies: no split tail
  t.flags = reinterpret_cast<uint64_t*>(base);
  t.partial = reinterpret_cast<float*>(base + kTailFlagBytes);
  const size_t fit = (bytes - off - kTailFlagBytes) / kTailPartialBytes;
  t.slots = static_cast<int>(fit < static_cast<size_t>(kTailSlots) ? fit : kTailSlots);
  t.gen = next_generation();
  return t;
}
}  // namespace

extern "C" size_t lf_forward_workspace_bytes(const lf_plan_info* info, int32_t dtype) {
  (void)dtype;
  return info ? forward_min_workspace_bytes(info) + tail_scratch_bytes() : 0;
}

extern "C" size_t lf_backward_workspace_bytes(const lf_plan_info* info, int32_t dtype) {
  (void)dtype;
  return info ? backward_min_workspace_bytes(info) + tail_scratch_bytes() : 0;
}

extern "C" int lf_pack_adapters(int32_t src_dtype, int32_t dst_dtype, const uint64_t* src_ptrs_dev,
                                const int32_t* slot_rank_dev, int32_t n_slots, int32_t rank_dim, int32_t other_dim,
                                int32_t transpose, int32_t d0, int32_t d1, void* dst_dev, lf_stream_t stream) {
  if (src_dtype < 0 || src_dtype > 2 || dst_dtype < 0 || dst_dtype > 2) return LF_ERR_INVALID_ARG;
  if (n_slots < 0 || d0 < 0 || d1 < 0 || other_dim < 0 || (rank_dim != 0 && rank_dim != 1)) return LF_ERR_INVALID_ARG;
  if (n_slots == 0 || d0 == 0 || d1 == 0) return LF_OK;
  if (!src_ptrs_dev || !slot_rank_dev || !dst_dev) return LF_ERR_INVALID_ARG;
  return to_status(pack_adapters(src_dtype, dst_dtype, src_ptrs_dev, slot_rank_dev, n_slots, rank_dim, other_dim,
                                 transpose, d0, d1, dst_dev, static_cast<cudaStream_t>(stream)));
}

namespace {
// What lf_options asks for, checked.
struct Options {
  bool mx4 = false;
  DropArgs drop{};
  char* scratch = nullptr;  // dropout's, and its size
  size_t scratch_bytes = 0;
};
size_t drop_scratch_mask(const lf_problem* p) {
  return align256(static_cast<size_t>(p->T) * static_cast<size_t>(p->K) * static_cast<size_t>(elem_bytes(p->dtype)));
}
int read_options(const lf_options* opt, const lf_problem* prob, const lf_plan_info* info, Options* out) {
  if (!opt) return LF_OK;
  if (opt->weight_format != LF_WEIGHT_DENSE && opt->weight_format != LF_WEIGHT_MX4) return LF_ERR_INVALID_ARG;
  out->mx4 = opt->weight_format == LF_WEIGHT_MX4;
  if (out->mx4 && prob->dtype == LF_F32) return LF_ERR_UNSUPPORTED;
  const lf_dropout* d = opt->dropout;
  if (!d || info->n_slots == 0 || info->n_segtiles == 0) return LF_OK;
  if (!d->slot_threshold_dev) return LF_ERR_INVALID_ARG;
  if (!aligned16(d->scratch_dev)) return LF_ERR_INVALID_ARG;
  out->drop.offset = d->offset;
  out->drop.threshold = d->slot_threshold_dev;
  for (uint32_t i = 0; i < 10; ++i) {
    out->drop.key[2 * i] = static_cast<uint32_t>(d->seed) + i * 0x9E3779B9u;
    out->drop.key[2 * i + 1] = static_cast<uint32_t>(d->seed >> 32) + i * 0xBB67AE85u;
  }
  out->scratch = static_cast<char*>(d->scratch_dev);
  out->scratch_bytes = d->scratch_dev ? d->scratch_bytes : 0;
  return LF_OK;
}
// Launches hand results to one another inside a grid through flags that hold a number no earlier launch used.  A launch
// captured into a graph repeats its number in every replay, so there the flags are cleared first, in the graph.
cudaError_t fresh_flags(bool captured, void* flags, size_t bytes, cudaStream_t st) {
  return captured && flags ? cudaMemsetAsync(flags, 0, bytes, st) : cudaSuccess;
}
bool is_captured(cudaStream_t st) {
  cudaStreamCaptureStatus s = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &s) != cudaSuccess) {
    (void)cudaGetLastError();  // the legacy stream beside another one's capture: not captured itself
    return false;
  }
  return s == cudaStreamCaptureStatusActive;
}
PairMx4 mx4_view(const void* data, int N, int K) {
  return PairMx4{static_cast<const uint8_t*>(data), mx4_row_tiles(N), mx4_col_blocks(K)};
}

// The forward stages; *sf_planes (if given) receives the K-half planes of S_f the shrink left in
// the workspace (2 when it ran inside the GEMM launch, 1 as a launch of its own, 0 without a
// tensor-core shrink), the value lf_backward_sf needs.
int forward_impl(const lf_problem* prob, const lf_plan_info* info, const int32_t* table_dev, void* y_dev,
                 void* workspace_dev, size_t workspace_bytes, void* tail_dev, size_t tail_bytes, int32_t stages,
                 lf_stream_t stream, int32_t* sf_planes, const lf_options* options = nullptr) {
  if (sf_planes) *sf_planes = 0;
  int rc = check_problem(prob, info, table_dev);
  if (rc != LF_OK) return rc;
  Options opt;
  rc = read_options(options, prob, info, &opt);
  if (rc != LF_OK) return rc;
  if (stages <= 0 || stages > 31 || ((stages & LF_STAGE_EXPAND) && (stages & LF_STAGE_BASE))) return LF_ERR_INVALID_ARG;
  const int T = prob->T, K = prob->K, N = prob->N;
  if (T == 0 || N == 0) return LF_OK;
  if (!prob->x_dev || !prob->w_dev || !prob->a_pack_dev || !prob->b_pack_dev || !y_dev) return LF_ERR_INVALID_ARG;
  if (workspace_bytes < forward_min_workspace_bytes(info) || !workspace_dev) return LF_ERR_CAPACITY;
  DeviceState* ds = nullptr;
  cudaError_t e = device_state(&ds);
  if (e != cudaSuccess) return LF_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Tables tb = make_tables(info, table_dev);
  tb.err = ds->status;
  const int dt = prob->dtype;
  const int rp = info->r_pad;
  const bool do_shrink = (stages & LF_STAGE_SHRINK) != 0;
  const bool do_gemm = (stages & (LF_STAGE_EXPAND | LF_STAGE_BASE)) != 0;
  const bool lora = (stages & LF_STAGE_EXPAND) != 0 && info->n_segtiles > 0;
  const PairMx4 mx4 = opt.mx4 ? mx4_view(prob->w_dev, N, K) : PairMx4{};
  const PairMx4* mx4p = opt.mx4 ? &mx4 : nullptr;
  const bool drop = opt.drop.threshold != nullptr;

  if (tc_eligible(prob, {prob->x_dev, prob->w_dev, prob->a_pack_dev, prob->b_pack_dev, y_dev, workspace_dev})) {
    const bool single = (stages & LF_STAGE_SINGLE_CTA) != 0;
    if (single && opt.mx4) return LF_ERR_UNSUPPORTED;
    const uint32_t nbox = single ? 256 : 128;  // rows of W / B_i per CTA and tile
    TcMaps maps;
    CUtensorMap a_map;
    const size_t es = 2;
    const uint64_t s_rows = kSextPlanes * static_cast<uint64_t>(info->n_segtiles + 1) * LF_TILE_ROWS;
    bool ok = make_map(&maps.p, dt, prob->x_dev, K, T, K * es, 64, 128) &&
              (opt.mx4 || make_map(&maps.q, dt, prob->w_dev, K, N, K * es, 64, nbox)) &&
              make_map(&a_map, dt, prob->a_pack_dev, K, static_cast<uint64_t>(info->n_slots) * rp, K * es, 64, rp);
    if (info->n_segtiles > 0)
      ok = ok && make_map(&maps.s, dt, workspace_dev, rp, s_rows, rp * es, rp, 128) &&
           make_map(&maps.l, dt, prob->b_pack_dev, rp, static_cast<uint64_t>(info->n_slots) * N, rp * es, rp, nbox);
    else
      maps.s = maps.l = maps.p;
    ok = ok && make_map(&maps.o, dt, y_dev, N, T, N * es, 64, 32);
    if (!ok) return LF_ERR_UNSUPPORTED;
    if (opt.mx4) maps.q = maps.p;  // not used
    // Shrink and expand requested together: run the shrink on CTA pairs the GEMM's round count
    // leaves idle, inside the same launch, when there are enough of them.
    const bool separate = (stages & LF_STAGE_SEPARATE) != 0;
    const bool fuse = !single && !separate && do_shrink && lora && cosched_allowed(ds) && !(drop && cosched_prologue());
    const int spare = fuse && !cosched_prologue() ? pair_spare_pairs(T, N, ds->num_sms, info->n_shrink_units) : 0;
    // the K-split tail needs a cooperative launch too
    const PairTail tail = tail_dev ? tail_scratch(tail_dev, tail_bytes, 0)
                                   : tail_scratch(workspace_dev, workspace_bytes, forward_min_workspace_bytes(info));
    const bool captured = is_captured(st);
    if (do_gemm) e = fresh_flags(captured, tail.flags, kTailFlagBytes, st);
    if (fuse && e == cudaSuccess)
      e = fresh_flags(captured, static_cast<char*>(workspace_dev) + sext_bytes(info), flag_bytes(info), st);
    if (e != cudaSuccess) return LF_ERR_CUDA;
    if (fuse && (spare > 0 || cosched_prologue())) {
      PairShrink sh{};
      sh.a_map = a_map;
      sh.s_ext = workspace_dev;
      sh.unit_ready = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace_dev) + sext_bytes(info));
      sh.gen = next_generation();
      sh.wait_gen = wait_generation(sh.gen);
      sh.n_pairs = spare;
      sh.prologue = cosched_prologue();
      sh.drop = opt.drop;
      e = tc_gemm_pair(dt, false, maps, T, N, K, lora, tb, y_dev, N, ds->num_sms, st, &sh, &tail, nullptr, mx4p, false, drop);
      if (e == cudaSuccess) {
        if (sf_planes) *sf_planes = 2;
        return LF_OK;
      }
      // The cooperative launch was refused (e.g. other work holds SMs, or a profiler
      // serializes launches): nothing ran; use the two-launch path from now on.
      refuse_cosched(ds, e);
    }
    if (do_shrink) {
      e = tc_shrink(dt, maps.p, a_map, K, tb, workspace_dev, ds->num_sms, st, &opt.drop);
      if (e != cudaSuccess) return LF_ERR_CUDA;
      if (sf_planes) *sf_planes = 1;
    }
    if (do_gemm) {
      if (single) {
        e = tc_gemm(dt, false, maps, T, N, K, lora, tb, y_dev, N, ds->num_sms, st);
      } else {
        const bool behind = do_shrink && lora;
        e = tc_gemm_pair(dt, false, maps, T, N, K, lora, tb, y_dev, N, ds->num_sms, st, nullptr,
                         cosched_allowed(ds) ? &tail : nullptr, nullptr, mx4p, behind, drop);
        if (e != cudaSuccess && cosched_allowed(ds)) {  // cooperative launch refused: nothing ran
          refuse_cosched(ds, e);
          e = tc_gemm_pair(dt, false, maps, T, N, K, lora, tb, y_dev, N, ds->num_sms, st, nullptr, nullptr, nullptr, mx4p,
                           behind, drop);
        }
      }
    }
    return to_status(e);
  }

  if (opt.mx4) return LF_ERR_UNSUPPORTED;
  if (drop && do_shrink && opt.scratch_bytes < drop_scratch_mask(prob)) return LF_ERR_CAPACITY;
  double* s_ext = static_cast<double*>(workspace_dev);
  if (do_shrink) {
    const void* xa = prob->x_dev;  // the adapters' input
    if (drop) {
      e = drop_mask(dt, prob->x_dev, T, K, tb, opt.drop, opt.scratch, st);
      if (e != cudaSuccess) return LF_ERR_CUDA;
      xa = opt.scratch;
    }
    e = simt_shrink(dt, xa, K, K, prob->a_pack_dev, tb, s_ext, st);
    if (e != cudaSuccess) return LF_ERR_CUDA;
  }
  if (do_gemm)
    e = simt_gemm(dt, prob->x_dev, K, prob->w_dev, K, 1, T, N, K, s_ext, lora ? prob->b_pack_dev : nullptr, tb, y_dev,
                  N, DropArgs{}, st);
  return to_status(e);
}
}  // namespace

extern "C" int lf_forward_stages(const lf_problem* prob, const lf_plan_info* info, const int32_t* table_dev,
                                 void* y_dev, void* workspace_dev, size_t workspace_bytes, int32_t stages,
                                 lf_stream_t stream) {
  return forward_impl(prob, info, table_dev, y_dev, workspace_dev, workspace_bytes, nullptr, 0, stages, stream,
                      nullptr);
}

extern "C" int lf_forward_sf(const lf_problem* prob, const lf_plan_info* info, const int32_t* table_dev, void* y_dev,
                             void* workspace_dev, size_t workspace_bytes, void* tail_dev, size_t tail_bytes,
                             int32_t* s_f_planes, lf_stream_t stream) {
  if (!s_f_planes) return LF_ERR_INVALID_ARG;
  return forward_impl(prob, info, table_dev, y_dev, workspace_dev, workspace_bytes, tail_dev, tail_bytes,
                      LF_STAGE_SHRINK | LF_STAGE_EXPAND, stream, s_f_planes);
}

extern "C" size_t lf_dropout_scratch_bytes(const lf_problem* p, int32_t backward) {
  if (!p || p->T < 0 || p->K < 0) return 0;
  const bool tc = tc_eligible(p, {p->x_dev, p->w_dev});
  if (!backward) return tc ? 0 : drop_scratch_mask(p);
  return drop_scratch_mask(p) + (tc ? align256(static_cast<size_t>(p->T) * static_cast<size_t>(p->K) * 4) : 0);
}

extern "C" int lf_forward_opt(const lf_problem* prob, const lf_plan_info* info, const int32_t* table_dev,
                              const lf_options* options, void* y_dev, void* workspace_dev, size_t workspace_bytes,
                              void* tail_dev, size_t tail_bytes, int32_t* s_f_planes, lf_stream_t stream) {
  int32_t planes = 0;
  const int rc = forward_impl(prob, info, table_dev, y_dev, workspace_dev, workspace_bytes, tail_dev, tail_bytes,
                              LF_STAGE_SHRINK | LF_STAGE_EXPAND, stream, &planes, options);
  if (s_f_planes) *s_f_planes = planes;
  return rc;
}

extern "C" size_t lf_forward_fixed_workspace_bytes(const lf_plan_info* info, int32_t dtype) {
  (void)dtype;
  return forward_min_workspace_bytes(info);
}

extern "C" int lf_forward_launch_count(const lf_problem* prob, const lf_plan_info* info) {
  if (!prob || !info) return -LF_ERR_INVALID_ARG;
  if (prob->T == 0 || prob->N == 0) return 0;
  DeviceState* ds = nullptr;
  if (device_state(&ds) != cudaSuccess) return -LF_ERR_CUDA;
  const bool tc = prob->dtype != LF_F32 && prob->K > 0 && prob->K % 8 == 0 && prob->N % 8 == 0;
  if (tc && info->n_segtiles > 0 && cosched_allowed(ds) &&
      (cosched_prologue() || pair_spare_pairs(prob->T, prob->N, ds->num_sms, info->n_shrink_units) > 0))
    return 1;
  return 2;
}

extern "C" int lf_backward_launch_count(const lf_problem* prob, const lf_plan_info* info) {
  if (!prob || !info) return -LF_ERR_INVALID_ARG;
  if (prob->T == 0) return 0;
  DeviceState* ds = nullptr;
  if (device_state(&ds) != cudaSuccess) return -LF_ERR_CUDA;
  const bool tc = prob->dtype != LF_F32 && prob->K > 0 && prob->K % 8 == 0 && prob->N % 8 == 0;
  const bool lora = info->n_segtiles > 0 && info->n_slots > 0;
  if (!tc) return 5;
  if (!lora) return 1;
  return (cosched_allowed(ds) &&
          (cosched_prologue() || pair_spare_pairs(prob->T, prob->K, ds->num_sms, info->n_shrink_units) > 0))
             ? 2
             : 4;
}

extern "C" int lf_set_co_scheduling(int32_t enable) {
  if (enable < 0 || enable > 2) return LF_ERR_INVALID_ARG;
  g_cosched_mode.store(enable);
  return LF_OK;
}

extern "C" int lf_set_wait_limit(uint64_t limit_ns) {
  if (limit_ns != 0 && (limit_ns < 1000000ull || limit_ns > 60000000000ull)) return LF_ERR_INVALID_ARG;
  const unsigned long long v = limit_ns == 0 ? kWaitLimitNs : limit_ns;
  DeviceState* ds = nullptr;
  if (device_state(&ds) != cudaSuccess) return LF_ERR_CUDA;
  if (cudaMemcpyToSymbol(g_device_ctl, &v, sizeof(v), offsetof(DeviceCtl, wait_limit_ns)) != cudaSuccess)
    return LF_ERR_CUDA;
  return LF_OK;
}

extern "C" int lf_inject_stale_ready(int32_t launches) {
  if (launches < 0) return LF_ERR_INVALID_ARG;
  g_stale_ready.store(launches);
  return LF_OK;
}

extern "C" int lf_get_co_scheduling(int32_t* mode, int32_t* refused_error) {
  if (!mode || !refused_error) return LF_ERR_INVALID_ARG;
  DeviceState* ds = nullptr;
  if (device_state(&ds) != cudaSuccess) return LF_ERR_CUDA;
  *mode = g_cosched_mode.load();
  *refused_error = ds->no_cosched.load() ? ds->refusal.load() : 0;
  return LF_OK;
}

extern "C" int lf_release(void) {
  for (DeviceState& d : g_dev) {
    std::lock_guard<std::mutex> lk(d.ev_mu);
    for (cudaEvent_t ev : d.events) (void)cudaEventDestroy(ev);
    d.events.clear();
  }
  return LF_OK;
}

extern "C" int lf_forward_host(const lf_problem* prob, const lf_host_chunk* chunks, int32_t n_chunks,
                               const void* x_host, void* y_host, void* x_dev, void* y_dev, void* workspace_dev,
                               size_t workspace_bytes, lf_stream_t stream, lf_stream_t h2d_stream,
                               lf_stream_t d2h_stream) {
  if (!prob || n_chunks < 0 || (n_chunks > 0 && (!chunks || !x_host || !y_host || !x_dev || !y_dev)))
    return LF_ERR_INVALID_ARG;
  if (prob->dtype != LF_F32 && prob->dtype != LF_BF16 && prob->dtype != LF_F16) return LF_ERR_INVALID_ARG;
  const size_t es = static_cast<size_t>(elem_bytes(prob->dtype));
  // Every chunk is checked before anything is enqueued, with the checks lf_forward makes, so a
  // bad chunk list fails with nothing in flight.
  int end = 0;
  for (int32_t c = 0; c < n_chunks; ++c) {
    const lf_host_chunk& ch = chunks[c];
    if (ch.row0 != end || ch.rows < 0 || !ch.info || ch.info->total_rows != ch.rows) return LF_ERR_INVALID_ARG;
    lf_problem pc = *prob;
    pc.T = ch.rows;
    const int rc = check_problem(&pc, ch.info, ch.table_dev);
    if (rc != LF_OK) return rc;
    if (ch.rows > 0 && prob->N > 0 && (workspace_bytes < forward_min_workspace_bytes(ch.info) || !workspace_dev))
      return LF_ERR_CAPACITY;
    end += ch.rows;
  }
  if (end != prob->T) return LF_ERR_INVALID_ARG;
  if (n_chunks == 0) return LF_OK;
  if (prob->N > 0 && (!prob->w_dev || !prob->a_pack_dev || !prob->b_pack_dev)) return LF_ERR_INVALID_ARG;
  DeviceState* ds = nullptr;
  if (device_state(&ds) != cudaSuccess) return LF_ERR_CUDA;
  const size_t n_ev = 2 * static_cast<size_t>(n_chunks) + 3;
  std::lock_guard<std::mutex> lk(ds->ev_mu);  // one enqueue at a time per device shares the events
  while (ds->events.size() < n_ev) {
    cudaEvent_t ev;
    if (cudaEventCreateWithFlags(&ev, cudaEventDisableTiming) != cudaSuccess) return LF_ERR_CUDA;
    ds->events.push_back(ev);
  }
  cudaEvent_t* ev = ds->events.data();
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  cudaStream_t si = static_cast<cudaStream_t>(h2d_stream);
  cudaStream_t so = static_cast<cudaStream_t>(d2h_stream);
  // the copies come after the work already on `stream` (earlier readers of x_dev / y_dev)
  if (cudaEventRecord(ev[0], cs) != cudaSuccess || cudaStreamWaitEvent(si, ev[0], 0) != cudaSuccess ||
      cudaStreamWaitEvent(so, ev[0], 0) != cudaSuccess)
    return LF_ERR_CUDA;
  const char* xh = static_cast<const char*>(x_host);
  char* yh = static_cast<char*>(y_host);
  char* xd = static_cast<char*>(x_dev);
  char* yd = static_cast<char*>(y_dev);
  const size_t row_in = static_cast<size_t>(prob->K) * es, row_out = static_cast<size_t>(prob->N) * es;
  int rc = LF_OK;
  for (int32_t c = 0; c < n_chunks && rc == LF_OK; ++c) {
    const lf_host_chunk& ch = chunks[c];
    const size_t r0 = static_cast<size_t>(ch.row0), nr = static_cast<size_t>(ch.rows);
    cudaEvent_t ev_in = ev[3 + 2 * c], ev_out = ev[4 + 2 * c];
    if (cudaMemcpyAsync(xd + r0 * row_in, xh + r0 * row_in, nr * row_in, cudaMemcpyHostToDevice, si) != cudaSuccess ||
        cudaEventRecord(ev_in, si) != cudaSuccess || cudaStreamWaitEvent(cs, ev_in, 0) != cudaSuccess) {
      rc = LF_ERR_CUDA;
      break;
    }
    lf_problem pc = *prob;
    pc.T = ch.rows;
    pc.x_dev = xd + r0 * row_in;
    rc = lf_forward(&pc, ch.info, ch.table_dev, yd + r0 * row_out, workspace_dev, workspace_bytes, stream);
    if (rc != LF_OK) break;
    if (cudaEventRecord(ev_out, cs) != cudaSuccess || cudaStreamWaitEvent(so, ev_out, 0) != cudaSuccess ||
        cudaMemcpyAsync(yh + r0 * row_out, yd + r0 * row_out, nr * row_out, cudaMemcpyDeviceToHost, so) != cudaSuccess)
      rc = LF_ERR_CUDA;
  }
  // `stream` waits for both copy streams, also after a failure part-way: the caller may release
  // x_dev / y_dev / the host buffers once `stream` has passed this point.
  const bool joined = cudaEventRecord(ev[1], so) == cudaSuccess && cudaStreamWaitEvent(cs, ev[1], 0) == cudaSuccess &&
                      cudaEventRecord(ev[2], si) == cudaSuccess && cudaStreamWaitEvent(cs, ev[2], 0) == cudaSuccess;
  if (rc == LF_OK && !joined) rc = LF_ERR_CUDA;
  return rc;
}

extern "C" int lf_forward(const lf_problem* prob, const lf_plan_info* info, const int32_t* table_dev, void* y_dev,
                          void* workspace_dev, size_t workspace_bytes, lf_stream_t stream) {
  return lf_forward_stages(prob, info, table_dev, y_dev, workspace_dev, workspace_bytes,
                           LF_STAGE_SHRINK | LF_STAGE_EXPAND, stream);
}

namespace {
// The backward; `sf_given` (planes `sf_planes`) is S_f = s x A_i^T as a forward left it in its
// workspace (tensor-core path only), or null to compute it here.
// `stages` 0: the whole backward (routed shrinks inside the grad_x launch when co-scheduling
// allows); otherwise the LF_BSTAGE_* bits, each a launch of its own (shrinks never co-scheduled).
int backward_impl(const lf_problem* prob, const lf_plan_info* info, const int32_t* table_dev, const void* grad_out_dev,
                  const void* sf_given, int sf_planes, int grad_f32, void* grad_x_dev, void* grad_a_dev,
                  void* grad_b_dev, void* workspace_dev, size_t workspace_bytes, lf_stream_t stream,
                  int stages = 0, const lf_peer_reduce* peer = nullptr, const lf_options* options = nullptr) {
  int rc = check_problem(prob, info, table_dev);
  if (rc != LF_OK) return rc;
  Options opt;
  rc = read_options(options, prob, info, &opt);
  if (rc != LF_OK) return rc;
  GramPeer gp{};
  if (peer != nullptr) {  // spanning adapters' blocks exchanged by the gram: tensor-core path only
    if (peer->world < 2 || peer->world > LF_MAX_PEERS || peer->rank < 0 || peer->rank >= peer->world ||
        peer->n_span <= 0 || !peer->slot_span_dev || !peer->span_info_dev || static_cast<uint32_t>(peer->gen) == 0 ||
        (peer->r_pad_x != 16 && peer->r_pad_x != 32 && peer->r_pad_x != 64))
      return LF_ERR_INVALID_ARG;
    for (int r = 0; r < peer->world; ++r)
      if (!peer->exchange[r] || !aligned16(peer->exchange[r])) return LF_ERR_INVALID_ARG;
    if (prob->dtype == LF_F32 || prob->T == 0 || info->n_segtiles == 0 || info->n_slots == 0)
      return LF_ERR_UNSUPPORTED;
    gp.world = peer->world;
    gp.rank = peer->rank;
    for (int r = 0; r < peer->world; ++r) gp.xbuf[r] = static_cast<uint8_t*>(peer->exchange[r]);
    gp.slot_span = peer->slot_span_dev;
    gp.span_info = peer->span_info_dev;
    gp.n_span = peer->n_span;
    gp.cblk_b = (prob->N + 127) / 128;
    gp.blocks_per_span = gp.cblk_b + (prob->K + 127) / 128;
    gp.n_blocks = gp.n_span * gp.blocks_per_span;
    gp.xr = peer->r_pad_x;
    gp.gen = peer->gen;
  }
  const GramPeer* gpp = peer != nullptr ? &gp : nullptr;
  const bool staged = stages != 0;
  const bool do_shrink = !staged || (stages & LF_BSTAGE_SHRINK) != 0;
  const bool do_gx = !staged || (stages & LF_BSTAGE_GRAD_X) != 0;
  const bool do_gab = !staged || (stages & LF_BSTAGE_GRAD_AB) != 0;
  const int T = prob->T, K = prob->K, N = prob->N;
  const size_t sb = sext_bytes(info);
  if (workspace_bytes < backward_min_workspace_bytes(info) || !workspace_dev) return LF_ERR_CAPACITY;
  DeviceState* ds = nullptr;
  cudaError_t e = device_state(&ds);
  if (e != cudaSuccess) return LF_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int dt = prob->dtype;
  const size_t es = static_cast<size_t>(elem_bytes(dt));
  if (do_gab && info->n_slots > 0 && (!grad_a_dev || !grad_b_dev)) return LF_ERR_INVALID_ARG;
  if (do_gab && (T == 0 || info->n_segtiles == 0)) {  // adapters whose routes are all empty: zero gradients
    const size_t ra = static_cast<size_t>(info->rank_total);
    const size_t gs = grad_f32 ? 4 : es;
    if (ra > 0 && K > 0 && cudaMemsetAsync(grad_a_dev, 0, ra * K * gs, st) != cudaSuccess) return LF_ERR_CUDA;
    if (ra > 0 && N > 0 && cudaMemsetAsync(grad_b_dev, 0, ra * N * gs, st) != cudaSuccess) return LF_ERR_CUDA;
  }
  if (T == 0) return LF_OK;
  if (!prob->x_dev || !prob->w_dev || !grad_out_dev || (do_gx && !grad_x_dev)) return LF_ERR_INVALID_ARG;
  if (info->n_slots > 0 && (!prob->a_pack_dev || !prob->bt_pack_dev || !prob->at_pack_dev))
    return LF_ERR_INVALID_ARG;
  Tables tb = make_tables(info, table_dev);
  tb.err = ds->status;
  const int rp = info->r_pad;
  char* ws = static_cast<char*>(workspace_dev);
  void* s_f = ws;
  void* s_b = ws + sb;
  const bool reuse_sf = sf_given != nullptr && prob->dtype != LF_F32 && (sf_planes == 1 || sf_planes == 2);
  if (reuse_sf) s_f = const_cast<void*>(sf_given);

  const bool tc_path = tc_eligible(prob, {prob->x_dev, prob->w_dev, prob->a_pack_dev, prob->bt_pack_dev,
                                          prob->at_pack_dev, grad_out_dev, grad_x_dev, workspace_dev});
  if ((peer != nullptr || opt.mx4) && !tc_path) return LF_ERR_UNSUPPORTED;
  const PairMx4 mx4 = opt.mx4 ? mx4_view(prob->w_dev, N, K) : PairMx4{};
  const PairMx4* mx4p = opt.mx4 ? &mx4 : nullptr;
  const bool drop = opt.drop.threshold != nullptr;
  if (drop && opt.scratch_bytes < lf_dropout_scratch_bytes(prob, 1)) return LF_ERR_CAPACITY;
  if (drop && (staged || reuse_sf)) return LF_ERR_UNSUPPORTED;
  const void* xa = drop ? opt.scratch : prob->x_dev;  // the adapters' input: m x is written on the way
  if (tc_path) {
    CUtensorMap p_x, p_g, a_map, bt_map, sf_map, sb_map;
    TcMaps dx;
    const PairTail tail = tail_scratch(workspace_dev, workspace_bytes, backward_min_workspace_bytes(info));
    const bool captured = is_captured(st);
    void* gram_scratch = ws + 2 * sb + flag_bytes(info, 2);
    if (do_gx) e = fresh_flags(captured, tail.flags, kTailFlagBytes, st);
    if (do_gx && e == cudaSuccess) e = fresh_flags(captured, ws + 2 * sb, flag_bytes(info, 2), st);
    if (do_gab && e == cudaSuccess)
      e = fresh_flags(captured, static_cast<char*>(gram_scratch) + gram_counters_offset(rp), kGramMaxCounters * 4 * 8, st);
    if (e != cudaSuccess) return LF_ERR_CUDA;
    const uint64_t s_rows = kSextPlanes * static_cast<uint64_t>(info->n_segtiles + 1) * LF_TILE_ROWS;
    bool ok = make_map(&p_x, dt, xa, K, T, K * es, 64, 128) &&
              make_map(&p_g, dt, grad_out_dev, N, T, N * es, 64, 128) &&
              (opt.mx4 || make_map(&dx.q, dt, prob->w_dev, K, N, K * es, 64, 64));
    const bool lora = info->n_segtiles > 0 && info->n_slots > 0;
    if (lora)
      ok = ok &&
           make_map(&a_map, dt, prob->a_pack_dev, K, static_cast<uint64_t>(info->n_slots) * rp, K * es, 64, rp) &&
           make_map(&bt_map, dt, prob->bt_pack_dev, N, static_cast<uint64_t>(info->n_slots) * rp, N * es, 64, rp) &&
           make_map(&sf_map, dt, s_f, rp, s_rows, rp * es, rp, 128) &&
           make_map(&sb_map, dt, s_b, rp, s_rows, rp * es, rp, 128) &&
           make_map(&dx.l, dt, prob->at_pack_dev, rp, static_cast<uint64_t>(info->n_slots) * K, rp * es, rp, 128);
    if (do_gx) ok = ok && make_map(&dx.o, dt, grad_x_dev, K, T, K * es, 64, 32);
    if (!ok) return LF_ERR_UNSUPPORTED;
    dx.p = p_g;
    if (opt.mx4) dx.q = p_g;  // not used
    int planes = 1;  // S_b's K-half planes (S_f's: sf_planes when reused, else the same as S_b's)
    bool gemm_done = !do_gx;
    if (lora && staged) {
      dx.s = sb_map;
      if (do_shrink) {
        if (!reuse_sf) {
          e = tc_shrink(dt, p_x, a_map, K, tb, s_f, ds->num_sms, st);
          if (e != cudaSuccess) return LF_ERR_CUDA;
        }
        e = tc_shrink(dt, p_g, bt_map, N, tb, s_b, ds->num_sms, st);
        if (e != cudaSuccess) return LF_ERR_CUDA;
      }
    } else if (lora) {
      dx.s = sb_map;
      // The shrinks inside the dX GEMM launch, on CTA pairs its round count leaves idle: job 1 =
      // S_b (g . B_i, needed by the dX tiles), job 2 = S_f (x . A_i^T, read by the dB gram) unless
      // the forward's is reused.
      const int spare =
          cosched_allowed(ds) && !cosched_prologue() ? pair_spare_pairs(T, K, ds->num_sms, info->n_shrink_units) : 0;
      if (!drop && cosched_allowed(ds) && (spare > 0 || cosched_prologue())) {
        PairShrink sh{};
        sh.a_map = bt_map;
        sh.s_ext = s_b;
        sh.unit_ready = reinterpret_cast<uint64_t*>(ws + 2 * sb);
        sh.gen = next_generation();
        sh.wait_gen = wait_generation(sh.gen);
        sh.n_pairs = spare;
        sh.prologue = cosched_prologue();
        sh.job2 = !reuse_sf;
        sh.p2_map = p_x;
        sh.a2_map = a_map;
        sh.s_ext2 = s_f;
        sh.K2 = K;
        e = tc_gemm_pair(dt, true, dx, T, K, N, lora, tb, grad_x_dev, K, ds->num_sms, st, &sh, &tail, nullptr, mx4p);
        if (e == cudaSuccess) {
          planes = 2;
          gemm_done = true;
        } else {
          refuse_cosched(ds, e);  // cooperative launch refused: nothing ran
        }
      }
      if (!gemm_done && drop) {
        // the mask is of grad_x's adapters' part alone: it is added to g W.  S_f and m x, which dA and dB read, are computed
        // on CTA pairs that this GEMM's rounds leave idle, or ahead of it.
        CUtensorMap x_map, delta_map;
        float* delta = reinterpret_cast<float*>(opt.scratch + drop_scratch_mask(prob));
        const PairDelta d{delta, nullptr, K};
        if (!make_map(&x_map, dt, prob->x_dev, K, T, K * es, 64, 128) ||
            !make_map(&delta_map, LF_F32, delta, K, T, static_cast<uint64_t>(K) * 4, 32, 32))
          return LF_ERR_UNSUPPORTED;
        PairShrink sh{};
        sh.n_pairs = spare;
        sh.job2 = sh.job2_only = true;
        sh.p2_map = x_map;
        sh.a2_map = a_map;
        sh.a_map = p_x;
        sh.s_ext2 = s_f;
        sh.K2 = K;
        sh.drop = opt.drop;
        const bool two = spare == 0;
        if (two) e = tc_shrink(dt, x_map, a_map, K, tb, s_f, ds->num_sms, st, &opt.drop, &p_x, true, false);
        if (e == cudaSuccess) e = tc_shrink(dt, p_g, bt_map, N, tb, s_b, ds->num_sms, st, nullptr, nullptr, two, two);
        if (e == cudaSuccess) e = drop_expand(dt, sb_map, dx.l, delta_map, T, K, tb, opt.drop, ds->num_sms, st);
        if (e == cudaSuccess)
          e = tc_gemm_pair(dt, true, dx, T, K, N, false, tb, grad_x_dev, K, ds->num_sms, st, spare > 0 ? &sh : nullptr, nullptr,
                           &d, mx4p);
        if (e != cudaSuccess) return LF_ERR_CUDA;
        gemm_done = true;
      }
      if (!gemm_done) {
        if (!reuse_sf) {
          e = tc_shrink(dt, p_x, a_map, K, tb, s_f, ds->num_sms, st);
          if (e != cudaSuccess) return LF_ERR_CUDA;
        }
        e = tc_shrink(dt, p_g, bt_map, N, tb, s_b, ds->num_sms, st);
        if (e != cudaSuccess) return LF_ERR_CUDA;
      }
    } else {
      dx.s = dx.l = p_g;
    }
    if (!gemm_done) {
      const bool behind = lora && do_shrink;
      e = tc_gemm_pair(dt, true, dx, T, K, N, lora, tb, grad_x_dev, K, ds->num_sms, st, nullptr,
                       cosched_allowed(ds) ? &tail : nullptr, nullptr, mx4p, behind);
      if (e != cudaSuccess && cosched_allowed(ds)) {  // cooperative launch refused: nothing ran
        refuse_cosched(ds, e);
        e = tc_gemm_pair(dt, true, dx, T, K, N, lora, tb, grad_x_dev, K, ds->num_sms, st, nullptr, nullptr, nullptr, mx4p,
                         behind);
      }
      if (e != cudaSuccess) return LF_ERR_CUDA;
    }
    if (lora && do_gab) {  // dB and dA in one launch
      GramJobDesc jobs[2];
      jobs[0].d_map = p_g;
      jobs[0].s_map = sf_map;
      jobs[0].C = N;
      jobs[0].out = grad_b_dev;
      jobs[0].transpose_out = 0;
      jobs[0].out_f32 = grad_f32;
      jobs[1].d_map = p_x;
      jobs[1].s_map = sb_map;
      jobs[1].C = K;
      jobs[1].out = grad_a_dev;
      jobs[1].transpose_out = 1;
      jobs[1].out_f32 = grad_f32;
      void* scratch = gram_scratch;
      // the grams read hi and lo planes: 2 per K half
      const int f_planes = reuse_sf ? sf_planes : planes;
      if (f_planes == planes) {
        e = tc_gram(dt, jobs, 2, tb, ds->num_sms, st, 2 * planes, scratch, next_generation(), gpp);
      } else {  // S_f and S_b hold different plane counts: one launch each
        e = tc_gram(dt, &jobs[0], 1, tb, ds->num_sms, st, 2 * f_planes, scratch, next_generation(), gpp);
        if (e == cudaSuccess)
          e = tc_gram(dt, &jobs[1], 1, tb, ds->num_sms, st, 2 * planes, scratch, next_generation(), gpp);
      }
      if (e != cudaSuccess) return LF_ERR_CUDA;
    }
    return LF_OK;
  }

  if (drop) {
    e = drop_mask(dt, prob->x_dev, T, K, tb, opt.drop, opt.scratch, st);
    if (e != cudaSuccess) return LF_ERR_CUDA;
  }
  double* sf = reinterpret_cast<double*>(ws);  // the CUDA-core path computes its own f64 S_f
  double* sbp = static_cast<double*>(s_b);
  if (do_shrink) {
    e = simt_shrink(dt, xa, K, K, prob->a_pack_dev, tb, sf, st);
    if (e != cudaSuccess) return LF_ERR_CUDA;
    e = simt_shrink(dt, grad_out_dev, N, N, prob->bt_pack_dev, tb, sbp, st);
    if (e != cudaSuccess) return LF_ERR_CUDA;
  }
  if (do_gx) {  // grad_x = g W + S_b . A   (Q(c, m) = W[m][c])
    e = simt_gemm(dt, grad_out_dev, N, prob->w_dev, 1, K, T, K, N, sbp, prob->at_pack_dev, tb, grad_x_dev, K, opt.drop,
                  st);
    if (e != cudaSuccess) return LF_ERR_CUDA;
  }
  if (do_gab) {
    e = simt_gram(dt, grad_out_dev, N, N, sf, tb, grad_b_dev, 0, grad_f32, st);
    if (e != cudaSuccess) return LF_ERR_CUDA;
    e = simt_gram(dt, xa, K, K, sbp, tb, grad_a_dev, 1, grad_f32, st);
  }
  return to_status(e);
}
}  // namespace

extern "C" int lf_backward(const lf_problem* prob, const lf_plan_info* info, const int32_t* table_dev,
                           const void* grad_out_dev, void* grad_x_dev, void* grad_a_dev, void* grad_b_dev,
                           void* workspace_dev, size_t workspace_bytes, lf_stream_t stream) {
  return backward_impl(prob, info, table_dev, grad_out_dev, nullptr, 0, 0, grad_x_dev, grad_a_dev, grad_b_dev,
                       workspace_dev, workspace_bytes, stream);
}

extern "C" int lf_backward_sf(const lf_problem* prob, const lf_plan_info* info, const int32_t* table_dev,
                              const void* grad_out_dev, const void* s_f_dev, int32_t s_f_planes, void* grad_x_dev,
                              void* grad_a_dev, void* grad_b_dev, void* workspace_dev, size_t workspace_bytes,
                              lf_stream_t stream) {
  if (!s_f_dev || (s_f_planes != 1 && s_f_planes != 2)) return LF_ERR_INVALID_ARG;
  return backward_impl(prob, info, table_dev, grad_out_dev, s_f_dev, s_f_planes, 0, grad_x_dev, grad_a_dev,
                       grad_b_dev, workspace_dev, workspace_bytes, stream);
}

extern "C" int lf_backward_stages(const lf_problem* prob, const lf_plan_info* info, const int32_t* table_dev,
                                  const void* grad_out_dev, const void* s_f_dev, int32_t s_f_planes,
                                  int32_t grad_ab_dtype, void* grad_x_dev, void* grad_a_dev, void* grad_b_dev,
                                  void* workspace_dev, size_t workspace_bytes, int32_t stages, lf_stream_t stream) {
  if (!prob) return LF_ERR_INVALID_ARG;
  if (stages <= 0 || stages > (LF_BSTAGE_SHRINK | LF_BSTAGE_GRAD_X | LF_BSTAGE_GRAD_AB)) return LF_ERR_INVALID_ARG;
  if (s_f_dev && s_f_planes != 1 && s_f_planes != 2) return LF_ERR_INVALID_ARG;
  if (grad_ab_dtype != prob->dtype && grad_ab_dtype != LF_F32) return LF_ERR_INVALID_ARG;
  return backward_impl(prob, info, table_dev, grad_out_dev, s_f_dev, s_f_dev ? s_f_planes : 0,
                       grad_ab_dtype == LF_F32 ? 1 : 0, grad_x_dev, grad_a_dev, grad_b_dev, workspace_dev,
                       workspace_bytes, stream, stages);
}

extern "C" int lf_backward_ex(const lf_problem* prob, const lf_plan_info* info, const int32_t* table_dev,
                              const void* grad_out_dev, const void* s_f_dev, int32_t s_f_planes, int32_t grad_ab_dtype,
                              void* grad_x_dev, void* grad_a_dev, void* grad_b_dev, void* workspace_dev,
                              size_t workspace_bytes, lf_stream_t stream) {
  if (!prob) return LF_ERR_INVALID_ARG;
  if (s_f_dev && s_f_planes != 1 && s_f_planes != 2) return LF_ERR_INVALID_ARG;
  if (grad_ab_dtype != prob->dtype && grad_ab_dtype != LF_F32) return LF_ERR_INVALID_ARG;
  return backward_impl(prob, info, table_dev, grad_out_dev, s_f_dev, s_f_dev ? s_f_planes : 0,
                       grad_ab_dtype == LF_F32 ? 1 : 0, grad_x_dev, grad_a_dev, grad_b_dev, workspace_dev,
                       workspace_bytes, stream);
}

extern "C" int lf_backward_peer(const lf_problem* prob, const lf_plan_info* info, const int32_t* table_dev,
                                const void* grad_out_dev, const void* s_f_dev, int32_t s_f_planes,
                                int32_t grad_ab_dtype, void* grad_x_dev, void* grad_a_dev, void* grad_b_dev,
                                void* workspace_dev, size_t workspace_bytes, const lf_peer_reduce* peer,
                                lf_stream_t stream) {
  if (!prob || !peer) return LF_ERR_INVALID_ARG;
  if (s_f_dev && s_f_planes != 1 && s_f_planes != 2) return LF_ERR_INVALID_ARG;
  if (grad_ab_dtype != prob->dtype && grad_ab_dtype != LF_F32) return LF_ERR_INVALID_ARG;
  return backward_impl(prob, info, table_dev, grad_out_dev, s_f_dev, s_f_dev ? s_f_planes : 0,
                       grad_ab_dtype == LF_F32 ? 1 : 0, grad_x_dev, grad_a_dev, grad_b_dev, workspace_dev,
                       workspace_bytes, stream, 0, peer);
}

extern "C" int lf_backward_opt(const lf_problem* prob, const lf_plan_info* info, const int32_t* table_dev,
                               const lf_options* options, const void* grad_out_dev, const void* s_f_dev,
                               int32_t s_f_planes, int32_t grad_ab_dtype, void* grad_x_dev, void* grad_a_dev,
                               void* grad_b_dev, void* workspace_dev, size_t workspace_bytes, const lf_peer_reduce* peer,
                               lf_stream_t stream) {
  if (!prob) return LF_ERR_INVALID_ARG;
  if (s_f_dev && s_f_planes != 1 && s_f_planes != 2) return LF_ERR_INVALID_ARG;
  if (grad_ab_dtype != prob->dtype && grad_ab_dtype != LF_F32) return LF_ERR_INVALID_ARG;
  return backward_impl(prob, info, table_dev, grad_out_dev, s_f_dev, s_f_dev ? s_f_planes : 0,
                       grad_ab_dtype == LF_F32 ? 1 : 0, grad_x_dev, grad_a_dev, grad_b_dev, workspace_dev,
                       workspace_bytes, stream, 0, peer, options);
}

extern "C" size_t lf_peer_exchange_bytes(int32_t world, int32_t n_blocks, int32_t r_pad) {
  if (world < 1 || world > LF_MAX_PEERS || n_blocks < 0 || (r_pad != 16 && r_pad != 32 && r_pad != 64)) return 0;
  return 2 * peer_half_bytes(world, n_blocks, r_pad);
}

extern "C" int lf_peer_alloc(size_t bytes, void** dev_ptr) {
  if (!dev_ptr || bytes == 0) return LF_ERR_INVALID_ARG;
  *dev_ptr = nullptr;
  if (cudaMalloc(dev_ptr, bytes) != cudaSuccess) return LF_ERR_CUDA;
  if (cudaMemset(*dev_ptr, 0, bytes) != cudaSuccess) return LF_ERR_CUDA;  // flags start below any generation
  return LF_OK;
}

extern "C" int lf_peer_free(void* dev_ptr) { return cudaFree(dev_ptr) == cudaSuccess ? LF_OK : LF_ERR_CUDA; }

extern "C" int lf_ipc_handle(const void* dev_ptr, void* handle) {
  static_assert(sizeof(cudaIpcMemHandle_t) == LF_IPC_HANDLE_BYTES, "IPC handle size");
  if (!dev_ptr || !handle) return LF_ERR_INVALID_ARG;
  cudaIpcMemHandle_t h;
  if (cudaIpcGetMemHandle(&h, const_cast<void*>(dev_ptr)) != cudaSuccess) return LF_ERR_CUDA;
  memcpy(handle, &h, sizeof(h));
  return LF_OK;
}

extern "C" int lf_ipc_open(const void* handle, void** dev_ptr) {
  if (!handle || !dev_ptr) return LF_ERR_INVALID_ARG;
  cudaIpcMemHandle_t h;
  memcpy(&h, handle, sizeof(h));
  *dev_ptr = nullptr;
  return cudaIpcOpenMemHandle(dev_ptr, h, cudaIpcMemLazyEnablePeerAccess) == cudaSuccess ? LF_OK : LF_ERR_CUDA;
}

extern "C" int lf_ipc_close(void* dev_ptr) {
  return cudaIpcCloseMemHandle(dev_ptr) == cudaSuccess ? LF_OK : LF_ERR_CUDA;
}

// Workspace of lf_rows_forward: each row's adapter, S (two 16-bit halves, or one float32 array on the CUDA-core
// path: the same bytes), what the tensor-core path knows of the sorted rows, the adapters' part of the
// result.  Long batches run in chunks of rows, one after another in the same place.
struct RowsSpace {
  size_t eff, s_hi, s_lo, factor, perm, tiles, n_tiles, delta, bytes;
};
static RowsSpace rows_space(int32_t T, int32_t N, int32_t r_pad, int32_t dtype) {
  const size_t all = static_cast<size_t>(T), rows = T < kRowsChunk ? all : kRowsChunk;
  const bool tc = dtype != LF_F32;
  RowsSpace s{};
  size_t at = 0;
  auto take = [&](size_t& place, size_t bytes) {
    place = at;
    at += align256(bytes);
  };
  take(s.eff, all * 4);
  take(s.s_hi, all * r_pad * 2);
  take(s.s_lo, all * r_pad * 2);
  take(s.factor, tc ? rows * 4 : 0);
  take(s.perm, tc ? rows * 4 : 0);
  take(s.tiles, tc ? rows * 16 : 0);
  take(s.n_tiles, tc ? 4 : 0);
  take(s.delta, tc ? rows * ((static_cast<size_t>(N) + 15) / 16 * 16) * 4 : 0);
  s.bytes = at;
  return s;
}
extern "C" size_t lf_rows_workspace_bytes(int32_t T, int32_t N, int32_t r_pad, int32_t dtype) {
  return T < 0 || N < 0 || r_pad < 0 ? 0 : rows_space(T, N, r_pad, dtype).bytes;
}

extern "C" int lf_bank_load(const lf_bank_adapter* p, lf_stream_t stream) {
  if (!p || (p->dtype != LF_F32 && p->dtype != LF_BF16 && p->dtype != LF_F16)) return LF_ERR_INVALID_ARG;
  if (p->r_pad != 16 && p->r_pad != 32 && p->r_pad != 64 && p->r_pad != LF_BANK_MAX_RANK) return LF_ERR_INVALID_ARG;
  if (p->K <= 0 || p->N <= 0 || p->rank <= 0 || p->rank > p->r_pad) return LF_ERR_INVALID_ARG;
  if ((p->rank > 1 && p->lda < p->K) || (p->N > 1 && p->ldb < p->rank)) return LF_ERR_INVALID_ARG;
  if (!p->a_dev || !p->b_dev || !p->slot_a_dev || !p->slot_b_dev || !p->slot_rank_dev || !p->slot_scale_dev)
    return LF_ERR_INVALID_ARG;
  // threads zero and write the slot while others still read the adapter
  const uint64_t es = static_cast<uint64_t>(elem_bytes(p->dtype)), r_pad = p->r_pad, K = p->K, N = p->N;
  const uint64_t rows_a = p->rank - 1, rows_b = N - 1;  // beyond the first
  auto meet = [](const void* a, uint64_t na, const void* b, uint64_t nb) {
    const uint64_t a0 = reinterpret_cast<uint64_t>(a), b0 = reinterpret_cast<uint64_t>(b);
    return a0 < b0 + nb && b0 < a0 + na;
  };
  const uint64_t bytes_a = (rows_a * (rows_a ? p->lda : 0) + K) * es, bytes_b = (rows_b * (rows_b ? p->ldb : 0) + p->rank) * es;
  if (meet(p->a_dev, bytes_a, p->slot_a_dev, r_pad * K * es) || meet(p->a_dev, bytes_a, p->slot_b_dev, r_pad * N * es) ||
      meet(p->b_dev, bytes_b, p->slot_a_dev, r_pad * K * es) || meet(p->b_dev, bytes_b, p->slot_b_dev, r_pad * N * es))
    return LF_ERR_INVALID_ARG;
  DeviceState* ds = nullptr;
  if (device_state(&ds) != cudaSuccess) return LF_ERR_CUDA;
  const BankLoad b{p->a_dev, p->b_dev,  p->slot_a_dev, p->slot_b_dev, p->slot_rank_dev, p->slot_scale_dev, p->lda,
                   p->ldb,   p->K,      p->N,          p->r_pad,      p->rank,          p->scale};
  return to_status(bank_load(b, p->dtype, ds->num_sms, static_cast<cudaStream_t>(stream)));
}

extern "C" int lf_rows_launch_count(int32_t T, int32_t r_pad) {
  if (T <= 0) return 0;
  const int rest = T % kRowsChunk;
  return T / kRowsChunk * 4 + (rest > few_rows(r_pad) ? 4 : rest > 0 ? 2 : 0);
}

extern "C" int lf_rows_uses_pairs(int32_t T, int32_t K, int32_t N, int32_t num_sms) {
  return T > 0 && K > 0 && N > 0 && num_sms > 1 && rows_use_pairs(T, K, N, num_sms);
}

extern "C" int lf_rows_forward(const lf_rows_problem* p, void* y_dev, void* workspace_dev, size_t workspace_bytes,
                               lf_stream_t stream) {
  if (!p || p->T < 0 || p->K < 0 || p->N < 0 || p->n_slots < 0) return LF_ERR_INVALID_ARG;
  if (p->dtype != LF_F32 && p->dtype != LF_BF16 && p->dtype != LF_F16) return LF_ERR_INVALID_ARG;
  if (p->r_pad != 16 && p->r_pad != 32 && p->r_pad != 64 && p->r_pad != LF_BANK_MAX_RANK) return LF_ERR_INVALID_ARG;
  if (p->row_slot_bytes != 4 && p->row_slot_bytes != 8) return LF_ERR_INVALID_ARG;
  if (p->weight_format != LF_WEIGHT_DENSE && p->weight_format != LF_WEIGHT_MX4) return LF_ERR_INVALID_ARG;
  const bool mx4 = p->weight_format == LF_WEIGHT_MX4;
  // what 32-bit indices of elements and of bank rows hold
  if (p->K > (1 << 24) || p->N > (1 << 24) || p->n_slots >= (1 << 24) ||
      static_cast<int64_t>(p->n_slots) * (p->r_pad / 16) * (p->N > 16 ? p->N : 16) > INT32_MAX)
    return LF_ERR_UNSUPPORTED;
  if (p->T == 0 || p->N == 0) return LF_OK;
  if (p->ldx < p->K || !p->x_dev || !p->w_dev || !p->row_slot_dev || !y_dev) return LF_ERR_INVALID_ARG;
  if (p->n_slots > 0 && (!p->a_bank_dev || !p->b_bank_dev || !p->slot_rank_dev || !p->slot_scale_dev))
    return LF_ERR_INVALID_ARG;
  if (!workspace_dev || workspace_bytes < lf_rows_workspace_bytes(p->T, p->N, p->r_pad, p->dtype)) return LF_ERR_CAPACITY;
  if (!aligned16(workspace_dev) || !aligned16(p->b_bank_dev)) return LF_ERR_INVALID_ARG;
  const uint64_t es = static_cast<uint64_t>(elem_bytes(p->dtype)), T = p->T, K = p->K, N = p->N;
  const uint64_t ranks = static_cast<uint64_t>(p->n_slots) * p->r_pad, y0 = reinterpret_cast<uint64_t>(y_dev);
  auto meets_y = [&](const void* base, uint64_t bytes) {
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    return bytes > 0 && b < y0 + T * N * es && y0 < b + bytes;
  };
  const uint64_t n_slots = p->n_slots;
  if (meets_y(p->x_dev, ((T - 1) * p->ldx + K) * es) || meets_y(p->w_dev, mx4 ? mx4_bytes(p->N, p->K) : N * K * es) ||
      meets_y(p->a_bank_dev, ranks * K * es) || meets_y(p->b_bank_dev, ranks * N * es) ||
      meets_y(p->slot_rank_dev, n_slots * 4) || meets_y(p->slot_scale_dev, n_slots * 4) ||
      meets_y(p->row_slot_dev, T * p->row_slot_bytes))
    return LF_ERR_INVALID_ARG;
  DeviceState* ds = nullptr;
  if (device_state(&ds) != cudaSuccess) return LF_ERR_CUDA;
  RowsArgs a{};
  a.x = p->x_dev;
  a.w = p->w_dev;
  a.a_bank = p->a_bank_dev;
  a.b_bank = p->b_bank_dev;
  a.slot_rank = p->slot_rank_dev;
  a.slot_scale = p->slot_scale_dev;
  a.row_slot = p->row_slot_dev;
  a.y = y_dev;
  a.ldx = p->ldx;
  a.T = p->T;
  a.K = p->K;
  a.N = p->N;
  a.n_slots = p->n_slots;
  a.r_pad = p->r_pad;
  a.wide = p->row_slot_bytes == 8;
  a.err = ds->status;
  char* ws = static_cast<char*>(workspace_dev);
  const RowsSpace space = rows_space(p->T, p->N, p->r_pad, p->dtype);
  a.eff = reinterpret_cast<uint32_t*>(ws + space.eff);
  a.s_hi = ws + space.s_hi;
  a.s_lo = ws + space.s_lo;
  a.factor = reinterpret_cast<float*>(ws + space.factor);
  a.perm = reinterpret_cast<int*>(ws + space.perm);
  a.tiles = ws + space.tiles;
  a.n_tiles = reinterpret_cast<int*>(ws + space.n_tiles);
  a.delta = reinterpret_cast<float*>(ws + space.delta);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool tc = p->dtype != LF_F32 && p->K > 0 && p->K % 8 == 0 && p->N % 8 == 0 && p->ldx % 8 == 0 &&
                  aligned16(p->x_dev) && aligned16(p->w_dev) && aligned16(p->a_bank_dev) && aligned16(y_dev);
  if (mx4 && !tc) return LF_ERR_UNSUPPORTED;
  if (mx4) a.mx4 = mx4_view(p->w_dev, p->N, p->K);
  // chunks of rows share the workspace, one after another on the stream
  const char* x = static_cast<const char*>(p->x_dev);
  const char* slots = static_cast<const char*>(p->row_slot_dev);
  char* y = static_cast<char*>(y_dev);
  if (!tc) {
    for (int64_t t0 = 0; t0 < p->T; t0 += kRowsSimtChunk) {
      a.T = static_cast<int>(p->T - t0 < kRowsSimtChunk ? p->T - t0 : kRowsSimtChunk);
      a.x = x + t0 * p->ldx * static_cast<int64_t>(es);
      a.row_slot = slots + t0 * p->row_slot_bytes;
      a.y = y + t0 * p->N * static_cast<int64_t>(es);
      const int rc = to_status(rows_forward_simt(a, p->dtype, st));
      if (rc != LF_OK) return rc;
    }
    return LF_OK;
  }
  for (int64_t t0 = 0; t0 < p->T; t0 += kRowsChunk) {
    a.T = static_cast<int>(p->T - t0 < kRowsChunk ? p->T - t0 : kRowsChunk);
    a.x = x + t0 * p->ldx * 2;
    a.row_slot = slots + t0 * p->row_slot_bytes;
    a.y = y + t0 * p->N * 2;
    const uint64_t x_pitch = static_cast<uint64_t>(p->ldx) * 2, w_pitch = static_cast<uint64_t>(p->K) * 2;
    cudaError_t e;
    ManyMaps maps_of_many;
    ManyMaps* many = a.T > few_rows(a.r_pad) ? &maps_of_many : nullptr;
    if (many) {
      const uint64_t bank_rows = static_cast<uint64_t>(a.n_slots > 0 ? a.n_slots : 1) * a.r_pad;
      const uint64_t s_pitch = static_cast<uint64_t>(a.r_pad) * 2;
      const void* a_bank = a.n_slots > 0 ? a.a_bank : a.x;  // an empty bank: a map that nothing uses
      const void* b_bank = a.n_slots > 0 ? a.b_bank : a.x;
      if (!make_map(&many->a, p->dtype, a_bank, a.K, bank_rows, w_pitch, 64, 16) ||
          !make_map(&many->s_hi, p->dtype, a.s_hi, a.r_pad, a.T, s_pitch, 16, 128) ||
          !make_map(&many->s_lo, p->dtype, a.s_lo, a.r_pad, a.T, s_pitch, 16, 128) ||
          !make_map(&many->b, p->dtype, b_bank, 16, bank_rows / 16 * a.N, 32, 16, 256))
        return LF_ERR_UNSUPPORTED;
    }
    if (mx4 ? mx4_use_pairs(a.T, a.N, ds->num_sms) : rows_use_pairs(a.T, a.K, a.N, ds->num_sms)) {
      TcMaps maps;
      if (!make_map(&maps.p, p->dtype, a.x, a.K, a.T, x_pitch, 64, 128) ||
          (!mx4 && !make_map(&maps.q, p->dtype, a.w, a.K, a.N, w_pitch, 64, 128)) ||
          !make_map(&maps.o, p->dtype, a.y, a.N, a.T, static_cast<uint64_t>(a.N) * 2, 64, 32))
        return LF_ERR_UNSUPPORTED;
      maps.s = maps.l = maps.p;
      if (mx4) maps.q = maps.p;
      Tables tb{};
      tb.r_pad = 16;
      tb.err = ds->status;
      const PairDelta delta{a.delta, a.eff, (a.N + 15) / 16 * 16};
      e = rows_lora_part(a, p->dtype, many, ds->num_sms, st);
      if (e == cudaSuccess)
        e = tc_gemm_pair(p->dtype, false, maps, a.T, a.N, a.K, false, tb, a.y, a.N, ds->num_sms, st, nullptr, nullptr,
                         &delta, mx4 ? &a.mx4 : nullptr);
    } else {
      const RowsTiles tiles = rows_tiles(a.T, a.K, a.N, ds->num_sms);
      CUtensorMap w_map, x_map;
      if ((!mx4 && !make_map(&w_map, p->dtype, a.w, a.K, a.N, w_pitch, 64, 128)) ||
          !make_map(&x_map, p->dtype, a.x, a.K, a.T, x_pitch, 64, tiles.rows))
        return LF_ERR_UNSUPPORTED;
      if (mx4) w_map = x_map;
      e = rows_forward_tc(a, p->dtype, w_map, x_map, tiles, many, ds->num_sms, st);
    }
    if (e != cudaSuccess) return LF_ERR_CUDA;
  }
  return LF_OK;
}

// ------------------------------------------------------------------------------------- weights in 4 bits
extern "C" size_t lf_mx4_bytes(int32_t N, int32_t K) { return N < 0 || K < 0 ? 0 : mx4_bytes(N, K); }

namespace {
bool meet(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
  return na > 0 && nb > 0 && a0 < b0 + nb && b0 < a0 + na;
}
int mx4_check(int32_t dtype, int32_t N, int32_t K) {
  if (N < 0 || K < 0) return LF_ERR_INVALID_ARG;
  if (dtype != LF_BF16 && dtype != LF_F16) return dtype == LF_F32 ? LF_ERR_UNSUPPORTED : LF_ERR_INVALID_ARG;
  return N > (1 << 24) || K > (1 << 24) ? LF_ERR_UNSUPPORTED : LF_OK;
}
}  // namespace

extern "C" int lf_mx4_quantize(int32_t dtype, const void* w_dev, int32_t N, int32_t K, int64_t ldw, void* mx4_dev,
                               lf_stream_t stream) {
  const int rc = mx4_check(dtype, N, K);
  if (rc != LF_OK) return rc;
  if (N == 0 || K == 0) return LF_OK;
  if (!w_dev || !mx4_dev || !aligned16(mx4_dev) || (N > 1 && ldw < K)) return LF_ERR_INVALID_ARG;
  if (meet(w_dev, (static_cast<size_t>(N - 1) * (N > 1 ? ldw : 0) + K) * 2, mx4_dev, mx4_bytes(N, K)))
    return LF_ERR_INVALID_ARG;
  DeviceState* ds = nullptr;
  if (device_state(&ds) != cudaSuccess) return LF_ERR_CUDA;
  return to_status(mx4_quantize(dtype, w_dev, N, K, ldw, mx4_dev, ds->num_sms, static_cast<cudaStream_t>(stream)));
}

extern "C" int lf_mx4_dequantize(int32_t dtype, const void* mx4_dev, int32_t N, int32_t K, void* w_dev,
                                 lf_stream_t stream) {
  const int rc = mx4_check(dtype, N, K);
  if (rc != LF_OK) return rc;
  if (N == 0 || K == 0) return LF_OK;
  if (!w_dev || !mx4_dev || !aligned16(mx4_dev)) return LF_ERR_INVALID_ARG;
  if (meet(w_dev, static_cast<size_t>(N) * K * 2, mx4_dev, mx4_bytes(N, K))) return LF_ERR_INVALID_ARG;
  DeviceState* ds = nullptr;
  if (device_state(&ds) != cudaSuccess) return LF_ERR_CUDA;
  return to_status(mx4_dequantize(dtype, mx4_dev, N, K, w_dev, ds->num_sms, static_cast<cudaStream_t>(stream)));
}

extern "C" size_t lf_mx4_linear_workspace_bytes(int32_t K, int32_t N) {
  if (K <= 0 || N <= 0) return 0;
  return K % 8 || N % 8 ? align256(static_cast<size_t>(N) * static_cast<size_t>(K) * 2) : tail_scratch_bytes();
}

extern "C" int lf_mx4_linear_tail_parts(int32_t T, int32_t K, int32_t N, int32_t transpose, int32_t num_sms) {
  if (T <= 0 || K <= 0 || N <= 0 || K % 8 || N % 8 || num_sms < 2) return 0;
  if (!transpose && !mx4_use_pairs(T, N, num_sms)) return 0;
  return transpose ? pair_tail_parts(T, K, N, num_sms, true) : pair_tail_parts(T, N, K, num_sms, true);
}

extern "C" int lf_mx4_linear(const lf_mx4_problem* p, void* out_dev, void* workspace_dev, size_t workspace_bytes,
                             lf_stream_t stream) {
  if (!p || p->T < 0 || (p->transpose != 0 && p->transpose != 1)) return LF_ERR_INVALID_ARG;
  const int rc = mx4_check(p->dtype, p->N, p->K);
  if (rc != LF_OK) return rc;
  const int T = p->T, K = p->K, N = p->N, dt = p->dtype;
  const int in = p->transpose ? N : K, out = p->transpose ? K : N;
  if (T == 0 || out == 0) return LF_OK;
  if (!p->in_dev || !p->mx4_dev || !out_dev || p->ld < in) return LF_ERR_INVALID_ARG;
  if (in == 0 || !aligned16(p->mx4_dev) || !aligned16(workspace_dev)) return LF_ERR_INVALID_ARG;
  const size_t out_bytes = static_cast<size_t>(T) * out * 2;
  if (meet(out_dev, out_bytes, p->in_dev, (static_cast<size_t>(T - 1) * p->ld + in) * 2) ||
      meet(out_dev, out_bytes, p->mx4_dev, mx4_bytes(N, K)))
    return LF_ERR_INVALID_ARG;
  const bool cores = K % 8 || N % 8 || p->ld % 8 || !aligned16(p->in_dev) || !aligned16(out_dev);
  const size_t dense = static_cast<size_t>(N) * K * 2;
  if (cores && (!workspace_dev || workspace_bytes < dense)) return LF_ERR_CAPACITY;
  const size_t used = cores ? dense : workspace_bytes < tail_scratch_bytes() ? workspace_bytes : tail_scratch_bytes();
  if (workspace_dev && (meet(workspace_dev, used, p->in_dev, (static_cast<size_t>(T - 1) * p->ld + in) * 2) ||
                        meet(workspace_dev, used, p->mx4_dev, mx4_bytes(N, K)) ||
                        meet(workspace_dev, used, out_dev, out_bytes)))
    return LF_ERR_INVALID_ARG;
  DeviceState* ds = nullptr;
  if (device_state(&ds) != cudaSuccess) return LF_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cores) {
    cudaError_t e = mx4_dequantize(dt, p->mx4_dev, N, K, workspace_dev, ds->num_sms, st);
    const int64_t qsn = p->transpose ? 1 : K, qsk = p->transpose ? K : 1;
    if (e == cudaSuccess)
      e = simt_gemm(dt, p->in_dev, p->ld, workspace_dev, qsn, qsk, T, out, in, nullptr, nullptr, Tables{}, out_dev, out,
                    DropArgs{}, st);
    return to_status(e);
  }
  const PairMx4 mx4 = mx4_view(p->mx4_dev, N, K);
  const uint64_t pitch = static_cast<uint64_t>(p->ld) * 2;
  // The gradient takes the CTA pairs whatever T is: the kernel of few rows has W's rows as the M operand, whose reduction runs
  // along a row's codes; that of g V runs across them, and no tile of it is decoded that way.  1 row 4096 -> 4096 takes
  // 29 us so, the forward's kernel 14; 512 rows 33 and 27, 1024 rows 41 and 39.
  if (!p->transpose && !mx4_use_pairs(T, N, ds->num_sms)) {
    RowsArgs a{};
    a.x = p->in_dev;
    a.y = out_dev;
    a.ldx = p->ld;
    a.T = T, a.K = K, a.N = N, a.r_pad = 16;
    a.mx4 = mx4;
    a.err = ds->status;
    const RowsTiles tiles = rows_tiles(T, K, N, ds->num_sms);
    CUtensorMap x_map;
    if (!make_map(&x_map, dt, a.x, K, T, pitch, 64, tiles.rows)) return LF_ERR_UNSUPPORTED;
    return to_status(rows_forward_tc(a, dt, x_map, x_map, tiles, nullptr, ds->num_sms, st));
  }
  TcMaps maps;
  if (!make_map(&maps.p, dt, p->in_dev, in, T, pitch, 64, 128) ||
      !make_map(&maps.o, dt, out_dev, out, T, static_cast<uint64_t>(out) * 2, 64, 32))
    return LF_ERR_UNSUPPORTED;
  maps.q = maps.s = maps.l = maps.p;
  Tables tb{};
  tb.r_pad = 16;
  tb.err = ds->status;
  const PairTail tail = tail_scratch(workspace_dev, workspace_bytes, 0);
  const bool split = cosched_allowed(ds);
  if (fresh_flags(split && is_captured(st), tail.flags, kTailFlagBytes, st) != cudaSuccess) return LF_ERR_CUDA;
  cudaError_t e = tc_gemm_pair(dt, p->transpose != 0, maps, T, out, in, false, tb, out_dev, out, ds->num_sms, st, nullptr,
                               split ? &tail : nullptr, nullptr, &mx4);
  if (e != cudaSuccess && split) {  // cooperative launch refused: nothing ran
    refuse_cosched(ds, e);
    e = tc_gemm_pair(dt, p->transpose != 0, maps, T, out, in, false, tb, out_dev, out, ds->num_sms, st, nullptr, nullptr,
                     nullptr, &mx4);
  }
  return to_status(e);
}

extern "C" int lf_device_error(int32_t* code) {
  if (!code) return LF_ERR_INVALID_ARG;
  DeviceState* ds = nullptr;
  if (device_state(&ds) != cudaSuccess) return LF_ERR_CUDA;
  if (cudaDeviceSynchronize() != cudaSuccess) return LF_ERR_CUDA;
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_device_ctl, sizeof(int), offsetof(DeviceCtl, status)) != cudaSuccess)
    return LF_ERR_CUDA;
  const int zero = 0;
  if (cudaMemcpyToSymbol(g_device_ctl, &zero, sizeof(int), offsetof(DeviceCtl, status)) != cudaSuccess)
    return LF_ERR_CUDA;
  *code = v;
  return LF_OK;
}

extern "C" const char* lf_status_string(int status) {
  switch (status) {
    case LF_OK:
      return "ok";
    case LF_ERR_INVALID_ARG:
      return "invalid argument";
    case LF_ERR_ROUTING:
      return "routes do not tile the fused rows";
    case LF_ERR_UNSUPPORTED:
      return "unsupported dtype, rank or alignment";
    case LF_ERR_CUDA:
      return "CUDA call failed";
    case LF_ERR_CAPACITY:
      return "buffer too small";
    case LF_ERR_DEVICE:
      return "a kernel gave up waiting (device timeout)";
    default:
      return "unknown status";
  }
}

extern "C" const char* lf_version(void) { return "lorafusion_b200 0.1.0 sm_100a"; }
