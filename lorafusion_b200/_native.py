"""ctypes binding of the C ABI declared in ``include/lorafusion_b200.h``.

The shared library is built in-tree (``python -m lorafusion_b200.csrc.build``)
into ``lorafusion_b200/_lib/liblorafusion_b200.so``.  :func:`lib` loads it once
and raises ``RuntimeError`` when it is missing: the operator has no fallback.
"""

from __future__ import annotations

import ctypes
import importlib.util
import os
import re
import sysconfig
import threading
from contextlib import nullcontext

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "_lib", "liblorafusion_b200.so")
HEADER_PATH = os.path.join(os.path.dirname(_HERE), "include", "lorafusion_b200.h")

LF_OK = 0
LF_ERR_INVALID_ARG = 1
LF_ERR_ROUTING = 2
LF_ERR_UNSUPPORTED = 3
LF_ERR_CUDA = 4
LF_ERR_CAPACITY = 5
LF_ERR_DEVICE = 6

LF_F32, LF_BF16, LF_F16 = 0, 1, 2
LF_WEIGHT_DENSE, LF_WEIGHT_MX4 = 0, 1
LF_STAGE_SHRINK, LF_STAGE_EXPAND, LF_STAGE_BASE, LF_STAGE_SINGLE_CTA, LF_STAGE_SEPARATE = 1, 2, 4, 8, 16
LF_BSTAGE_SHRINK, LF_BSTAGE_GRAD_X, LF_BSTAGE_GRAD_AB = 1, 2, 4
TILE_ROWS = 128

_c_i32 = ctypes.c_int32
_c_p = ctypes.c_void_p


class PlanInfo(ctypes.Structure):
    _fields_ = [(name, _c_i32) for name in (
        "total_rows", "n_routes", "n_slots", "n_tiles", "n_segtiles", "r_pad", "max_rank", "rank_total",
        "n_shrink_units", "table_words",
        "off_tile_st", "off_st_tile", "off_st_lo", "off_st_hi", "off_st_slot", "off_st_route", "off_st_scale",
        "off_slot_st", "off_slot_list", "off_slot_rank", "off_rank_prefix", "off_slot_order",
        "off_unit_tile", "off_unit_st0", "off_unit_nst",
        "n_pair_lora", "off_pair_lora", "off_pl_a", "off_pl_b", "off_pl_slot", "off_tile_unit")]


class Problem(ctypes.Structure):
    _fields_ = [
        ("dtype", _c_i32), ("T", _c_i32), ("K", _c_i32), ("N", _c_i32),
        ("x_dev", _c_p), ("w_dev", _c_p), ("a_pack_dev", _c_p), ("b_pack_dev", _c_p),
        ("bt_pack_dev", _c_p), ("at_pack_dev", _c_p),
    ]


class RowRun(ctypes.Structure):
    _fields_ = [("src", ctypes.c_uint64), ("dst", ctypes.c_uint64), ("src_stride", ctypes.c_int64),
                ("dst_stride", ctypes.c_int64), ("rows", ctypes.c_int64), ("row0", ctypes.c_int64)]


MAX_PEERS = 8
IPC_HANDLE_BYTES = 64


class PeerReduce(ctypes.Structure):
    """lf_peer_reduce: the gram kernel's exchange of spanning adapters' blocks between GPUs."""
    _fields_ = [("world", ctypes.c_int32), ("rank", ctypes.c_int32), ("exchange", ctypes.c_void_p * MAX_PEERS),
                ("slot_span_dev", ctypes.c_void_p), ("span_info_dev", ctypes.c_void_p), ("n_span", ctypes.c_int32),
                ("r_pad_x", ctypes.c_int32), ("gen", ctypes.c_uint64)]


class HostChunk(ctypes.Structure):
    _fields_ = [("row0", ctypes.c_int32), ("rows", ctypes.c_int32), ("info", ctypes.POINTER(PlanInfo)),
                ("table_dev", ctypes.c_void_p)]


class RowsProblem(ctypes.Structure):
    _fields_ = [("dtype", _c_i32), ("T", _c_i32), ("K", _c_i32), ("N", _c_i32), ("n_slots", _c_i32),
                ("r_pad", _c_i32), ("row_slot_bytes", _c_i32), ("weight_format", _c_i32), ("ldx", ctypes.c_int64),
                ("x_dev", _c_p), ("w_dev", _c_p), ("a_bank_dev", _c_p), ("b_bank_dev", _c_p),
                ("slot_rank_dev", _c_p), ("slot_scale_dev", _c_p), ("row_slot_dev", _c_p)]


class BankAdapter(ctypes.Structure):
    _fields_ = [("dtype", _c_i32), ("K", _c_i32), ("N", _c_i32), ("r_pad", _c_i32), ("rank", _c_i32),
                ("scale", ctypes.c_float), ("lda", ctypes.c_int64), ("ldb", ctypes.c_int64), ("a_dev", _c_p),
                ("b_dev", _c_p), ("slot_a_dev", _c_p), ("slot_b_dev", _c_p), ("slot_rank_dev", _c_p),
                ("slot_scale_dev", _c_p)]


class Mx4Problem(ctypes.Structure):
    _fields_ = [("dtype", _c_i32), ("T", _c_i32), ("K", _c_i32), ("N", _c_i32), ("transpose", _c_i32),
                ("reserved", _c_i32), ("ld", ctypes.c_int64), ("in_dev", _c_p), ("mx4_dev", _c_p)]


class Dropout(ctypes.Structure):
    _fields_ = [("seed", ctypes.c_uint64), ("offset", ctypes.c_uint64), ("slot_threshold_dev", _c_p),
                ("scratch_dev", _c_p), ("scratch_bytes", ctypes.c_size_t)]


class Options(ctypes.Structure):
    """lf_options: how the base weight is held, and dropout in front of the adapters."""
    _fields_ = [("weight_format", _c_i32), ("reserved", _c_i32), ("dropout", ctypes.POINTER(Dropout))]


class AdamWArgs(ctypes.Structure):
    _fields_ = [("tensors", _c_p), ("tensors_dev", _c_p), ("chunk_tensor_dev", _c_p), ("grads", _c_p),
                ("hyper_dev", _c_p), ("steps_dev", _c_p), ("exp_avg_dev", _c_p), ("exp_avg_sq_dev", _c_p),
                ("master_dev", _c_p), ("norms_dev", _c_p), ("workspace_dev", _c_p),
                ("workspace_bytes", ctypes.c_size_t), ("n_chunks", ctypes.c_int64), ("beta1", ctypes.c_double),
                ("beta2", ctypes.c_double), ("eps", ctypes.c_double), ("max_norm", ctypes.c_double),
                ("n_tensors", _c_i32), ("n_groups", _c_i32), ("param_dtype", _c_i32), ("grad_dtype", _c_i32),
                ("skip_nonfinite", _c_i32), ("reserved", _c_i32)]


# numpy layouts of lf_grad_tensor and lf_adamw_tensor (arrays of records passed by pointer)
GRAD_TENSOR = [("ptr", "<u8"), ("numel", "<u8"), ("dtype", "<i4"), ("group", "<i4")]
ADAMW_TENSOR = [("param", "<u8"), ("state_off", "<i8"), ("numel", "<u4"), ("group", "<i4"), ("chunk0", "<i4"),
                ("n_chunks", "<i4")]
BANK_MAX_RANK = 128


_lock = threading.Lock()
_lib: ctypes.CDLL | None = None
_glue = None


def _declare(L: ctypes.CDLL) -> None:
    P = ctypes.POINTER
    L.lf_plan_table_words.argtypes = [_c_i32, _c_i32, _c_i32]
    L.lf_plan_table_words.restype = _c_i32
    L.lf_plan_tables.argtypes = [P(_c_i32), P(_c_i32), P(_c_i32), _c_i32, _c_i32, P(_c_i32),
                                 P(ctypes.c_float), _c_i32, P(_c_i32), _c_i32, P(PlanInfo)]
    L.lf_plan_tables.restype = ctypes.c_int
    L.lf_forward_workspace_bytes.argtypes = [P(PlanInfo), _c_i32]
    L.lf_forward_workspace_bytes.restype = ctypes.c_size_t
    L.lf_backward_workspace_bytes.argtypes = [P(PlanInfo), _c_i32]
    L.lf_backward_workspace_bytes.restype = ctypes.c_size_t
    L.lf_pack_adapters.argtypes = [_c_i32, _c_i32, _c_p, _c_p, _c_i32, _c_i32, _c_i32, _c_i32, _c_i32, _c_i32,
                                   _c_p, _c_p]
    L.lf_pack_adapters.restype = ctypes.c_int
    L.lf_copy_rows.argtypes = [_c_p, _c_i32, ctypes.c_int64, ctypes.c_int64, _c_p]
    L.lf_forward_host.argtypes = [P(Problem), P(HostChunk), _c_i32, _c_p, _c_p, _c_p, _c_p, _c_p, ctypes.c_size_t,
                                  _c_p, _c_p, _c_p]
    L.lf_forward_host.restype = ctypes.c_int
    L.lf_release.argtypes = []
    L.lf_release.restype = ctypes.c_int
    L.lf_copy_rows.restype = ctypes.c_int
    L.lf_greedy_pack.argtypes = [P(_c_i32), P(_c_i32), _c_i32, _c_i32, _c_i32, P(_c_i32), P(_c_i32), P(_c_i32),
                                 P(_c_i32), P(_c_i32)]
    L.lf_greedy_pack.restype = ctypes.c_int
    L.lf_assign_rows.argtypes = [P(_c_i32), P(_c_i32), P(_c_i32), _c_i32, _c_i32, _c_i32, _c_i32,
                                 P(ctypes.c_int64), P(ctypes.c_int64), P(_c_i32), P(_c_i32)]
    L.lf_assign_rows.restype = ctypes.c_int
    L.lf_forward.argtypes = [P(Problem), P(PlanInfo), _c_p, _c_p, _c_p, ctypes.c_size_t, _c_p]
    L.lf_forward.restype = ctypes.c_int
    L.lf_forward_stages.argtypes = [P(Problem), P(PlanInfo), _c_p, _c_p, _c_p, ctypes.c_size_t, _c_i32, _c_p]
    L.lf_forward_stages.restype = ctypes.c_int
    L.lf_forward_launch_count.argtypes = [P(Problem), P(PlanInfo)]
    L.lf_forward_launch_count.restype = ctypes.c_int
    L.lf_backward_launch_count.argtypes = [P(Problem), P(PlanInfo)]
    L.lf_backward_launch_count.restype = ctypes.c_int
    L.lf_set_co_scheduling.argtypes = [_c_i32]
    L.lf_set_co_scheduling.restype = ctypes.c_int
    L.lf_get_co_scheduling.argtypes = [P(_c_i32), P(_c_i32)]
    L.lf_get_co_scheduling.restype = ctypes.c_int
    L.lf_forward_sf.argtypes = [P(Problem), P(PlanInfo), _c_p, _c_p, _c_p, ctypes.c_size_t, _c_p, ctypes.c_size_t,
                                P(_c_i32), _c_p]
    L.lf_forward_sf.restype = ctypes.c_int
    L.lf_forward_fixed_workspace_bytes.argtypes = [P(PlanInfo), _c_i32]
    L.lf_forward_fixed_workspace_bytes.restype = ctypes.c_size_t
    L.lf_backward_ex.argtypes = [P(Problem), P(PlanInfo), _c_p, _c_p, _c_p, _c_i32, _c_i32, _c_p, _c_p, _c_p, _c_p,
                                 ctypes.c_size_t, _c_p]
    L.lf_backward_ex.restype = ctypes.c_int
    L.lf_backward_peer.argtypes = [P(Problem), P(PlanInfo), _c_p, _c_p, _c_p, _c_i32, _c_i32, _c_p, _c_p, _c_p,
                                   _c_p, ctypes.c_size_t, P(PeerReduce), _c_p]
    L.lf_backward_peer.restype = ctypes.c_int
    L.lf_peer_exchange_bytes.argtypes = [_c_i32, _c_i32, _c_i32]
    L.lf_peer_exchange_bytes.restype = ctypes.c_size_t
    L.lf_peer_alloc.argtypes = [ctypes.c_size_t, P(ctypes.c_void_p)]
    L.lf_peer_alloc.restype = ctypes.c_int
    L.lf_peer_free.argtypes = [_c_p]
    L.lf_peer_free.restype = ctypes.c_int
    L.lf_ipc_handle.argtypes = [_c_p, _c_p]
    L.lf_ipc_handle.restype = ctypes.c_int
    L.lf_ipc_open.argtypes = [_c_p, P(ctypes.c_void_p)]
    L.lf_ipc_open.restype = ctypes.c_int
    L.lf_ipc_close.argtypes = [_c_p]
    L.lf_ipc_close.restype = ctypes.c_int
    L.lf_backward_stages.argtypes = [P(Problem), P(PlanInfo), _c_p, _c_p, _c_p, _c_i32, _c_i32, _c_p, _c_p, _c_p,
                                     _c_p, ctypes.c_size_t, _c_i32, _c_p]
    L.lf_backward_stages.restype = ctypes.c_int
    L.lf_backward.argtypes = [P(Problem), P(PlanInfo), _c_p, _c_p, _c_p, _c_p, _c_p, _c_p, ctypes.c_size_t, _c_p]
    L.lf_backward.restype = ctypes.c_int
    L.lf_backward_sf.argtypes = [P(Problem), P(PlanInfo), _c_p, _c_p, _c_p, _c_i32, _c_p, _c_p, _c_p, _c_p,
                                 ctypes.c_size_t, _c_p]
    L.lf_backward_sf.restype = ctypes.c_int
    L.lf_forward_noalloc.argtypes = [P(Problem), P(PlanInfo), _c_p, _c_p, _c_p]
    L.lf_forward_noalloc.restype = ctypes.c_int
    L.lf_rows_workspace_bytes.argtypes = [_c_i32, _c_i32, _c_i32, _c_i32]
    L.lf_rows_workspace_bytes.restype = ctypes.c_size_t
    L.lf_rows_forward.argtypes = [P(RowsProblem), _c_p, _c_p, ctypes.c_size_t, _c_p]
    L.lf_rows_forward.restype = ctypes.c_int
    L.lf_bank_load.argtypes = [P(BankAdapter), _c_p]
    L.lf_bank_load.restype = ctypes.c_int
    L.lf_rows_launch_count.argtypes = [_c_i32, _c_i32]
    L.lf_rows_launch_count.restype = ctypes.c_int
    L.lf_rows_uses_pairs.argtypes = [_c_i32, _c_i32, _c_i32, _c_i32]
    L.lf_rows_uses_pairs.restype = ctypes.c_int
    L.lf_mx4_bytes.argtypes = [_c_i32, _c_i32]
    L.lf_mx4_bytes.restype = ctypes.c_size_t
    L.lf_mx4_quantize.argtypes = [_c_i32, _c_p, _c_i32, _c_i32, ctypes.c_int64, _c_p, _c_p]
    L.lf_mx4_quantize.restype = ctypes.c_int
    L.lf_mx4_dequantize.argtypes = [_c_i32, _c_p, _c_i32, _c_i32, _c_p, _c_p]
    L.lf_mx4_dequantize.restype = ctypes.c_int
    L.lf_mx4_linear_workspace_bytes.argtypes = [_c_i32, _c_i32]
    L.lf_mx4_linear_workspace_bytes.restype = ctypes.c_size_t
    L.lf_mx4_linear.argtypes = [P(Mx4Problem), _c_p, _c_p, ctypes.c_size_t, _c_p]
    L.lf_mx4_linear.restype = ctypes.c_int
    L.lf_mx4_linear_tail_parts.argtypes = [_c_i32, _c_i32, _c_i32, _c_i32, _c_i32]
    L.lf_mx4_linear_tail_parts.restype = ctypes.c_int
    L.lf_dropout_scratch_bytes.argtypes = [P(Problem), _c_i32]
    L.lf_dropout_scratch_bytes.restype = ctypes.c_size_t
    L.lf_forward_opt.argtypes = [P(Problem), P(PlanInfo), _c_p, P(Options), _c_p, _c_p, ctypes.c_size_t, _c_p,
                                 ctypes.c_size_t, P(_c_i32), _c_p]
    L.lf_forward_opt.restype = ctypes.c_int
    L.lf_backward_opt.argtypes = [P(Problem), P(PlanInfo), _c_p, P(Options), _c_p, _c_p, _c_i32, _c_i32, _c_p, _c_p,
                                  _c_p, _c_p, ctypes.c_size_t, P(PeerReduce), _c_p]
    L.lf_backward_opt.restype = ctypes.c_int
    L.lf_grad_clip_workspace_bytes.argtypes = [_c_p, _c_i32, _c_i32]
    L.lf_grad_clip_workspace_bytes.restype = ctypes.c_size_t
    L.lf_grad_clip.argtypes = [_c_p, _c_i32, _c_i32, _c_i32, _c_i32, ctypes.c_double, _c_p, _c_p, ctypes.c_size_t,
                               _c_p]
    L.lf_grad_clip.restype = ctypes.c_int
    L.lf_adamw_plan.argtypes = [_c_p, _c_i32, _c_i32, _c_p, ctypes.c_int64, P(ctypes.c_int64), P(ctypes.c_int64)]
    L.lf_adamw_plan.restype = ctypes.c_int
    L.lf_adamw_workspace_bytes.argtypes = [ctypes.c_int64, _c_i32]
    L.lf_adamw_workspace_bytes.restype = ctypes.c_size_t
    L.lf_adamw_step.argtypes = [P(AdamWArgs), _c_p]
    L.lf_adamw_step.restype = ctypes.c_int
    L.lf_set_wait_limit.argtypes = [ctypes.c_uint64]
    L.lf_set_wait_limit.restype = ctypes.c_int
    L.lf_inject_stale_ready.argtypes = [_c_i32]
    L.lf_inject_stale_ready.restype = ctypes.c_int
    L.lf_device_error.argtypes = [P(_c_i32)]
    L.lf_device_error.restype = ctypes.c_int
    L.lf_status_string.argtypes = [ctypes.c_int]
    L.lf_status_string.restype = ctypes.c_char_p
    L.lf_version.argtypes = []
    L.lf_version.restype = ctypes.c_char_p


def lib() -> ctypes.CDLL:
    """The loaded library; ``RuntimeError`` if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise RuntimeError(
                    f"lorafusion_b200 native library not found at {LIB_PATH}; "
                    "build it with `python -m lorafusion_b200.csrc.build` (needs nvcc for sm_100a)")
            L = ctypes.CDLL(LIB_PATH)
            _declare(L)
            _lib = L
    return _lib


def glue_path() -> str:
    """Where the Python module of ``csrc/lf_pyglue.cpp`` for this Python and this PyTorch is built.  It is C++
    against both, so one built for another version must not be loaded: the name holds the versions."""
    import torch
    tag = f"{sysconfig.get_config_var('SOABI')}.torch-{torch.__version__}"
    return os.path.join(_HERE, "_lib", f"lf_pyglue.{tag}.so")


def glue():
    """The Python module of ``csrc/lf_pyglue.cpp`` (tensor checks and calls without a Python step per
    tensor); ``RuntimeError`` if it has not been built for this Python and PyTorch."""
    global _glue
    if _glue is None:
        L = lib()
        with _lock:
            if _glue is None:
                path = glue_path()
                if not os.path.exists(path):
                    raise RuntimeError(f"{path} not found; build it with `python -m lorafusion_b200.csrc.build`")
                spec = importlib.util.spec_from_file_location("lf_pyglue", path)
                module = importlib.util.module_from_spec(spec)
                spec.loader.exec_module(module)
                _glue = module
        assert L is not None
    return _glue


def header_symbols() -> list[str]:
    """Names of every entry point the public header declares."""
    text = open(HEADER_PATH).read()
    return re.findall(r"^LF_API\s+[\w\s\*]+?\b(lf_\w+)\s*\(", text, flags=re.M)


def status_text(code: int) -> str:
    return lib().lf_status_string(code).decode()


def check(code: int, what: str) -> None:
    """Map a C status to the reference's exception types."""
    if code == LF_OK:
        return
    msg = f"{what}: {status_text(code)} (status {code})"
    if code in (LF_ERR_CUDA, LF_ERR_DEVICE):
        raise RuntimeError(msg)
    raise ValueError(msg)


def raw_stream(device_index: int) -> int:
    """cudaStream_t of the device's current stream (without building a Stream object: 0.1 us, not 2)."""
    import torch
    return torch._C._cuda_getCurrentRawStream(device_index)


_current_device = None
_HERE_ALREADY = nullcontext()


def on_device(device_index: int):
    """Context that makes a device current; nothing to do where it already is.  (CUDA has been initialised: the caller
    has a tensor there.)"""
    global _current_device
    if _current_device is None:
        import torch
        _current_device = torch._C._cuda_getDevice
    if _current_device() == device_index:
        return _HERE_ALREADY
    import torch
    return torch.cuda.device(device_index)


def co_scheduling() -> tuple[int, int]:
    """(process-wide co-scheduling mode, cudaError_t of a refused cooperative launch on the current
    device or 0)."""
    mode, refused = _c_i32(0), _c_i32(0)
    check(lib().lf_get_co_scheduling(ctypes.byref(mode), ctypes.byref(refused)), "lf_get_co_scheduling")
    return int(mode.value), int(refused.value)


ERR_ROW_SLOT = 0x106  # a row of fused_lora_forward_rows named a slot its bank does not have
# device status codes of bounded waits that ran out (lf_ptx.cuh DeviceErr)
ERR_TIMEOUT_FULL, ERR_TIMEOUT_EMPTY, ERR_TIMEOUT_ACC, ERR_TIMEOUT_DRAIN, ERR_TIMEOUT_FLAG = 0x101, 0x102, 0x103, 0x104, 0x105


def set_wait_limit(limit_ns: int) -> None:
    """Bound of every in-kernel wait on the current device (0: the default, about 1 s)."""
    check(lib().lf_set_wait_limit(int(limit_ns)), "lf_set_wait_limit")


def device_error() -> int:
    """Read and clear the kernels' device status word (synchronizes the device)."""
    v = _c_i32(0)
    check(lib().lf_device_error(ctypes.byref(v)), "lf_device_error")
    return int(v.value)
