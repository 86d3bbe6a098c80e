"""B200 backend of lorafusion's fused multi-adapter LoRA op.

Drop-in for ``lorafusion.ops.mock_ops`` / ``lorafusion.ops.triton_ops``: the same
two functions with the same signatures, return conventions and exceptions
(``lorafusion/ops/mock_ops.py:15-95``, ``lorafusion/ops/triton_ops.py:373-468``),
so ``Coordinator(backend=b200_ops)`` (``lorafusion/runtime/coordinator.py:32,58-65``)
runs it unchanged.  All arithmetic happens in the sm_100a library behind
``include/lorafusion_b200.h``; there is no CPU path and no fallback: CPU inputs
raise ``ValueError`` and a missing library raises ``RuntimeError``.

Per call, on the current CUDA stream (co-scheduled launches, the default on a B200):
  forward   1 launch: routed shrink on spare CTA pairs + fused base GEMM / LoRA expand
  backward  2 launches: fused dX GEMM (with the routed shrink g.B_i on spare CTA pairs),
            then one segmented gram launch for dA and dB
bf16/f16 problems whose K or N is not a multiple of 8, or whose buffers are not 16-byte
aligned, cannot use the tensor-core (TMA) path and run on CUDA cores with a
``CudaCorePathWarning``.

Host work is cached the way ``triton_ops._prepare`` caches its weight copies
(``triton_ops.py:114-145``): validated routes and routing tables per routing
object (re-checked against a snapshot of its route list), packed adapter slabs
per (tensor identity, storage pointer, version counter) of every adapter
tensor, converted base weights likewise.  A repeated call with unchanged inputs
costs a few identity and version comparisons per adapter, so batches of hundreds
of adapters stay ahead of the GPU.
"""

from __future__ import annotations

import ctypes
import threading
import warnings
import weakref
from collections import OrderedDict

import numpy as np
import torch

from lorafusion_b200 import _native as nat
from lorafusion_b200.config import AdapterDropout
from lorafusion_b200.quant import MX4Weight

_DTYPE_CODE = {torch.float32: nat.LF_F32, torch.bfloat16: nat.LF_BF16, torch.float16: nat.LF_F16}

__all__ = ["AdapterDropout", "fused_lora_forward", "fused_lora_backward", "fused_lora_forward_host", "prepare_forward",
           "PreparedForward", "prepare_backward", "PreparedBackward", "clear_weight_cache", "release",
           "last_launch_count", "use_cooperative_launch", "CudaCorePathWarning"]


class CudaCorePathWarning(UserWarning):
    """A bf16/f16 problem the tensor-core path cannot address runs on the (much slower) CUDA cores."""


_WARNED_SHAPES: set = set()


def _warn_if_cuda_core(dtype, K: int, N: int, tensors, stacklevel: int = 3) -> None:
    """Warn once per (dtype, K, N) when a bf16/f16 call must run on CUDA cores: TMA needs K and N
    multiples of 8 and every buffer 16-byte aligned (the same test the library makes)."""
    if dtype == torch.float32:
        return
    ok = K > 0 and N > 0 and K % 8 == 0 and N % 8 == 0 and all(t.data_ptr() % 16 == 0 for t in tensors)
    if ok:
        return
    key = (dtype, K, N)
    if key not in _WARNED_SHAPES:
        _WARNED_SHAPES.add(key)
        warnings.warn(f"{dtype} problem with in_features={K}, out_features={N} runs on the CUDA-core path: the "
                      "tensor-core path needs both to be multiples of 8 and 16-byte aligned buffers",
                      CudaCorePathWarning, stacklevel=stacklevel)


# --------------------------------------------------------------------------- caches
# Held by every call while it looks things up in the caches, fills them and enqueues its launches: calls of several threads
# take turns on the host.
_LOCK = threading.RLock()
_ROUTE_CACHE: dict[int, "_Routes"] = {}
# adapter records by (slots, id of the first A, id of the first B), least recently used first; a
# model calls the op with one routing and many adapter sets (layers x projections), so every set
# keeps its record and packed slabs until _ADAPTER_CACHE_MAX sets are cached
_ADAPTER_CACHE: "OrderedDict[tuple, _AdapterSet]" = OrderedDict()
_ADAPTER_CACHE_MAX = 4096
_WEIGHT_CACHE: dict[tuple, tuple] = {}
_PLAN_BY_CONTENT: dict[tuple, "_Plan"] = {}
_CACHE_MAX = 256
_last_launches = 0
# S_f = s x A^T left by forwards, for a backward on the same inputs (what autograd would save as
# the activation x A^T): (id(x), id(route record), id(adapter record)) -> (weakref x, x version,
# route record, plan, adapter record, workspace, planes, capture), least recently used first; entries whose
# x has died are dropped on the next insertion
_SAVED_SF: "OrderedDict[tuple, tuple]" = OrderedDict()
_SAVED_MAX = 1024
# per capture into a CUDA graph: plans, packed slabs and base weights by id, which its replays read whatever the caches
# drop, for as long as the graph (or one instantiated from it) lives
_CAPTURED: dict[int, dict] = {}
_VERSION = torch.Tensor._version.__get__
_DATA_PTR = torch.Tensor.data_ptr


def use_cooperative_launch(enabled: bool, shrink_prologue: bool = False) -> None:
    """Allow (default) or forbid the co-scheduled cooperative launches (process-wide).

    When allowed, the routed shrinks run inside the GEMM's launch (forward: 1 launch;
    backward: 2): by default on CTA pairs the GEMM's round count leaves idle (when there are at
    least four; otherwise forward 2 launches, backward 3-4); with ``shrink_prologue`` every CTA
    instead computes its share of the shrink items before its GEMM tiles.  Profilers and
    SM-partitioned GPUs refuse cooperative launches; forbid them there and every shrink runs as
    a launch of its own (forward: 2 launches; backward: 4).
    """
    mode = (2 if shrink_prologue else 1) if enabled else 0
    nat.check(nat.lib().lf_set_co_scheduling(mode), "lf_set_co_scheduling")


def clear_weight_cache() -> None:
    """Drop every cached table, packed adapter slab and converted weight.  What captured calls read stays for as long as
    their graphs live."""
    with _LOCK:
        _ROUTE_CACHE.clear()
        _ADAPTER_CACHE.clear()
        _PLAN_BY_CONTENT.clear()
        _SAVED_SF.clear()
        _WEIGHT_CACHE.clear()
        _drop_ended()


def release() -> None:
    """Drop every host cache (``clear_weight_cache``) and what the library holds on the devices
    (``lf_release``: the host-streamed forward's events); later calls rebuild what they need."""
    with _LOCK:
        clear_weight_cache()
        _SIDE_STREAMS.clear()
        nat.check(nat.lib().lf_release(), "lf_release")


def last_launch_count() -> int:
    """Kernel launches issued by the most recent op call (0 for empty problems)."""
    return _last_launches


class _Routes:
    """A routing object's routes, validated for ``valid_rows`` rows, as the arrays the table
    builder takes, plus the routing plans built from them."""

    __slots__ = ("ref", "snapshot", "valid_rows", "starts", "ends", "route_slot", "slots", "plans", "chunk_plans")

    def __init__(self, routing, routes, total_rows):
        self.ref = weakref.ref(routing)
        self.snapshot = list(routes)
        self.valid_rows = total_rows
        n = len(routes)
        self.starts = np.fromiter((r.row_start for r in routes), dtype=np.int32, count=n)
        self.ends = np.fromiter((r.row_end for r in routes), dtype=np.int32, count=n)
        slot_of: dict[int, int] = {}
        self.route_slot = np.fromiter((slot_of.setdefault(r.adapter_id, len(slot_of)) for r in routes),
                                      dtype=np.int32, count=n)
        self.slots = tuple(slot_of)
        self.plans: list = []
        self.chunk_plans: list = []


def _routes(routing, total_rows: int) -> _Routes:
    """Validate ``routing`` for ``total_rows`` rows (``TileRoutingConfig.validate``,
    lorafusion/ops/config.py:55-69, raising its ``ValueError``) and return its arrays.

    A routing object already seen is re-validated only when its route list differs from the
    snapshot taken then (routes are immutable records, so comparing the list is enough) or the
    row count changed.
    """
    routes = routing.routes
    hit = _ROUTE_CACHE.get(id(routing))
    if hit is not None and hit.ref() is routing and routes == hit.snapshot:
        if hit.valid_rows != total_rows:
            routing.validate(total_rows)
            hit.valid_rows = total_rows
        return hit
    routing.validate(total_rows)
    rec = _Routes(routing, routes, total_rows)
    if len(_ROUTE_CACHE) >= _CACHE_MAX:
        _ROUTE_CACHE.clear()
    try:
        _ROUTE_CACHE[id(routing)] = rec
    except TypeError:  # pragma: no cover - routing object without weakref support
        pass
    return rec


MAX_SLOT_RANK = 64  # lf_plan_tables carries a slot of larger rank as several virtual slots


def _virtual_slots(ranks):
    """(slot index, first rank row, rank) of every virtual slot, in table order: a slot of rank
    r > 64 becomes ceil(r/64) chunks of 64 ranks and a remainder (lf_plan_tables' rule)."""
    return tuple((i, c0, min(MAX_SLOT_RANK, r - c0)) for i, r in enumerate(ranks) for c0 in range(0, r, MAX_SLOT_RANK))


def _plan_tables(starts, ends, route_slot, total_rows, ranks, scales, n_slots):
    """lf_plan_tables into a pinned host buffer (grown once when high ranks need more words)."""
    L = nat.lib()
    n_routes = len(starts)
    cap = L.lf_plan_table_words(n_routes, total_rows, n_slots)
    if cap < 0:
        raise ValueError("routing too large for int32 tables")
    rk = np.asarray(ranks, dtype=np.int32)
    sc = np.asarray(scales, dtype=np.float32)
    i32p = ctypes.POINTER(ctypes.c_int32)
    for _ in range(2):
        table = torch.empty(max(cap, 1), dtype=torch.int32, pin_memory=True)
        info = nat.PlanInfo()
        rc = L.lf_plan_tables(
            starts.ctypes.data_as(i32p), ends.ctypes.data_as(i32p), route_slot.ctypes.data_as(i32p), n_routes,
            total_rows, rk.ctypes.data_as(i32p), sc.ctypes.data_as(ctypes.POINTER(ctypes.c_float)), n_slots,
            ctypes.cast(table.data_ptr(), i32p), cap, ctypes.byref(info))
        if rc == nat.LF_ERR_CAPACITY and info.table_words > cap:
            cap = info.table_words
            continue
        nat.check(rc, "lf_plan_tables")
        return info, table
    raise RuntimeError("lf_plan_tables: table size did not converge")


class _Made:
    """Cached device memory and the stream that fills it.  A call on another stream comes after that, and the memory is
    used for nothing else before that call has run, whatever the caches drop meanwhile; the host waits for nothing (but
    within a capture)."""

    __slots__ = ("tensors", "stream", "event", "others")

    def __init__(self, device, *tensors):
        stream = torch.cuda.current_stream(device)
        self.tensors = tensors
        self.stream = stream.cuda_stream
        self.event = torch.cuda.Event()
        self.event.record(stream)
        self.others: set = set()  # streams that have waited

    def use(self, device, at) -> None:
        raw, captured = at
        if captured:  # replays may run on any stream
            nat.glue().wait_event(self.event.cuda_event)
        elif raw != self.stream and raw not in self.others:
            stream = torch.cuda.current_stream(device)
            stream.wait_event(self.event)
            for t in self.tensors:
                t.record_stream(stream)
            self.others.add(raw)


class _Plan:
    __slots__ = ("info", "table_dev", "slots", "ranks", "vslots", "thresholds", "made", "sizes")

    def __init__(self, info, table_dev, slots, ranks, thresholds=0):
        self.info = info
        self.table_dev = table_dev
        self.slots = slots
        self.ranks = ranks
        self.vslots = _virtual_slots(ranks)
        self.thresholds = thresholds  # address of the virtual slots' dropout thresholds, behind the table's words
        self.made = _Made(table_dev.device, table_dev)
        self.sizes: dict = {}  # dtype code -> bytes of a forward's fixed workspace, of its tail's, of a backward's

    def workspace(self, code: int) -> tuple[int, int, int]:
        sizes = self.sizes.get(code)
        if sizes is None:
            L, info = nat.lib(), ctypes.byref(self.info)
            fixed = int(L.lf_forward_fixed_workspace_bytes(info, code))
            sizes = self.sizes[code] = (max(fixed, 256), max(int(L.lf_forward_workspace_bytes(info, code)) - fixed, 256),
                                        max(int(L.lf_backward_workspace_bytes(info, code)), 256))
        return sizes


class _AdapterSet:
    """The A and B tensors of one call's adapter slots (in slot order) with the identity,
    storage pointer and version counter of each, their ranks and scalings, and the padded
    slabs packed from them (``packs``, per dtype and shape)."""

    __slots__ = ("a", "b", "a_ids", "b_ids", "a_ver", "b_ver", "a_ptr", "b_ptr", "ranks", "spec_ids", "scales",
                 "packs")

    def __init__(self, a_list, b_list, a_ids, b_ids, specs):
        self.a, self.b, self.a_ids, self.b_ids = a_list, b_list, a_ids, b_ids
        self.a_ver = list(map(_VERSION, a_list))
        self.b_ver = list(map(_VERSION, b_list))
        self.a_ptr = list(map(_DATA_PTR, a_list))
        self.b_ptr = list(map(_DATA_PTR, b_list))
        self.ranks = tuple(int(t.shape[0]) if t.dim() == 2 else -1 for t in a_list)
        self.spec_ids = list(map(id, specs))
        self.scales = tuple(float(sp.scaling) for sp in specs)
        self.packs: dict = {}

    def unchanged(self, a_list, b_list) -> bool:
        return (list(map(_VERSION, a_list)) == self.a_ver and list(map(_VERSION, b_list)) == self.b_ver
                and list(map(_DATA_PTR, a_list)) == self.a_ptr and list(map(_DATA_PTR, b_list)) == self.b_ptr)


def _adapters(rts: _Routes, lora_a, lora_b, adapters) -> _AdapterSet:
    """The adapter record of this call's slots: reused while every A/B tensor is the same object
    with the same storage and version counter, rebuilt (slabs repacked) otherwise.  A missing
    adapter raises ``KeyError`` like the reference's dict lookups (mock_ops.py:40-42)."""
    slots = rts.slots
    specs = list(map(adapters.__getitem__, slots))
    a_list = list(map(lora_a.__getitem__, slots))
    b_list = list(map(lora_b.__getitem__, slots))
    a_ids = list(map(id, a_list))
    b_ids = list(map(id, b_list))
    # the record holds the tensors, so an id in a live record cannot be reused by another tensor
    key = (slots, a_ids[0], b_ids[0]) if slots else (slots,)
    rec = _ADAPTER_CACHE.get(key)
    if rec is not None and rec.a_ids == a_ids and rec.b_ids == b_ids:
        _ADAPTER_CACHE.move_to_end(key)
        if not rec.unchanged(a_list, b_list):
            rec = _ADAPTER_CACHE[key] = _AdapterSet(a_list, b_list, a_ids, b_ids, specs)  # same tensors, updated
        elif list(map(id, specs)) != rec.spec_ids:
            rec.spec_ids = list(map(id, specs))
            rec.scales = tuple(float(sp.scaling) for sp in specs)
        return rec
    rec = _ADAPTER_CACHE[key] = _AdapterSet(a_list, b_list, a_ids, b_ids, specs)
    _ADAPTER_CACHE.move_to_end(key)
    while len(_ADAPTER_CACHE) > _ADAPTER_CACHE_MAX:
        _ADAPTER_CACHE.popitem(last=False)
    return rec


def _drop_ended() -> None:
    """Lets go of what captures held whose graphs are gone."""
    if _CAPTURED:
        for capture in nat.glue().ended():
            _CAPTURED.pop(capture, None)
            for k in [k for k, v in _SAVED_SF.items() if v[-1] == capture]:
                del _SAVED_SF[k]


def _at(device) -> tuple[int, int]:
    """The device's current stream, and the capture into a CUDA graph that it is in (0: none)."""
    _drop_ended()
    return nat.glue().at(device.index)


def _hold(captured: int, device, *read) -> None:
    """Keeps what a captured call reads for as long as its graph lives."""
    held = _CAPTURED.get(captured)
    if held is None:
        held = _CAPTURED[nat.glue().hold_capture(device.index)] = {}
    held.update((id(o), o) for o in read)


def _building(what: str, device) -> None:
    """Refuses to fill a cache within a capture: nothing runs there, so later calls would find it empty, and replays would
    fill it again from host memory that is gone by then."""
    if nat.glue().at(device.index)[1]:
        raise RuntimeError(f"{what} would be made within a CUDA graph capture: make the same call once before it")


def _plan(rts: _Routes, aset: _AdapterSet, total_rows: int, device: torch.device, at, drop=None) -> _Plan:
    """The routing's tables for this adapter set and, with ``drop``, its factors and thresholds (``at``: ``_at(device)``)."""
    ranks, scales, thresholds = aset.ranks, aset.scales, None
    if drop is not None:
        scales, thresholds = drop.scales(scales), drop.thresholds
    for pr, ps, pt, pd, plan in rts.plans:
        if pd == device and pr == ranks and ps == scales and pt == thresholds:
            plan.made.use(device, at)
            return plan
    if any(r <= 0 for r in ranks):
        bad = rts.slots[next(i for i, r in enumerate(ranks) if r <= 0)]
        raise ValueError(f"adapter {bad}: lora_a must be a non-empty [rank, in_features] matrix")
    # a new routing object with the same routes (a runtime that re-packs every batch) reuses the plan
    content = (rts.starts.tobytes(), rts.ends.tobytes(), rts.route_slot.tobytes(), rts.slots, total_rows, device,
               ranks, scales, thresholds)
    plan = _PLAN_BY_CONTENT.get(content)
    if plan is None:
        _building("the routing's tables", device)
        plan = _build_plan(rts, ranks, scales, thresholds, total_rows, device)
        if len(_PLAN_BY_CONTENT) >= _CACHE_MAX:
            _PLAN_BY_CONTENT.clear()
        _PLAN_BY_CONTENT[content] = plan
    else:
        plan.made.use(device, at)
    rts.plans.insert(0, (ranks, scales, thresholds, device, plan))
    del rts.plans[4:]
    return plan


def _build_plan(rts: _Routes, ranks, scales, thresholds, total_rows: int, device) -> _Plan:
    info, table = _plan_tables(rts.starts, rts.ends, rts.route_slot, total_rows, ranks, scales, len(rts.slots))
    words = max(info.table_words, 1)
    table = table[:words]
    if thresholds is not None:  # behind them, in the same copy
        more = [thresholds[i] for i, _, _ in _virtual_slots(ranks)]
        both = torch.empty(words + len(more), dtype=torch.int32, pin_memory=True)
        both[:words] = table
        both[words:] = torch.tensor(more, dtype=torch.int32)
        table = both
    table_dev = table.to(device, non_blocking=True)
    return _Plan(info, table_dev, rts.slots, ranks, table_dev.data_ptr() + 4 * words)


def _pack(plan: _Plan, aset: _AdapterSet, dtype: torch.dtype, K: int, N: int, device, at, backward: bool) -> dict:
    """Zero-padded adapter slabs in the layouts the kernels read (cached in the adapter record)."""
    key = (dtype, K, N, device, plan.info.r_pad)
    entry = aset.packs.get(key)
    want = ("a", "b", "bt", "at") if backward else ("a", "b")
    if entry is None or any(w not in entry for w in want):
        _building("the adapters' slabs", device)
    if entry is None:
        for aid, a, b, r in zip(plan.slots, aset.a, aset.b, plan.ranks):
            if a.dim() != 2 or a.shape[1] != K or b.dim() != 2 or b.shape != (N, r):
                raise ValueError(
                    f"adapter {aid}: lora_a {tuple(a.shape)} / lora_b {tuple(b.shape)} do not match "
                    f"in_features={K}, out_features={N}")
            if a.device != device or b.device != device:
                raise ValueError(f"adapter {aid}: LoRA weights must live on {device}")
        # one source matrix per virtual slot: A_i's rank rows [c0, c0 + r), B_i's columns likewise
        a_src, b_src = [], []
        for i, c0, r in plan.vslots:
            a, b = aset.a[i], aset.b[i]
            if r != a.shape[0]:
                a, b = a[c0:c0 + r], b[:, c0:c0 + r]
            a_src.append(a if a.is_contiguous() else a.contiguous())
            b_src.append(b if b.is_contiguous() else b.contiguous())
        entry = aset.packs[key] = {"src": (a_src, b_src)}
    for made in entry.get("made", ()):
        made.use(device, at)
    missing = [w for w in want if w not in entry]
    if missing:
        _fill_packs(entry, plan, dtype, K, N, device, missing)
        entry.setdefault("made", []).append(_Made(device, *(entry[w] for w in missing)))
    return entry


def _fill_packs(entry, plan: _Plan, dtype, K, N, device, which) -> None:
    L = nat.lib()
    a_src, b_src = entry["src"]
    n = len(plan.vslots)
    rp = plan.info.r_pad
    vranks = [r for _, _, r in plan.vslots]
    ranks_dev = torch.tensor(vranks if n else [0], dtype=torch.int32).to(device, non_blocking=True)
    stream = torch.cuda.current_stream(device).cuda_stream
    dst_code = _DTYPE_CODE[dtype]
    for w in which:
        srcs = a_src if w in ("a", "at") else b_src
        src_code = _DTYPE_CODE.get(srcs[0].dtype) if n else dst_code
        if n and any(t.dtype != srcs[0].dtype for t in srcs):
            srcs = [t.to(srcs[0].dtype) for t in srcs]
            entry.setdefault("converted", []).append(srcs)
        if src_code is None:
            raise ValueError(f"unsupported LoRA weight dtype {srcs[0].dtype}")
        ptrs = torch.tensor([t.data_ptr() for t in srcs] if n else [0], dtype=torch.int64).to(
            device, non_blocking=True)
        # (rank_dim, other_dim, transpose, d0, d1)
        spec = {
            "a": (0, K, 0, rp, K),   # A_i [r, K]  -> [slot, r_pad, K]
            "at": (0, K, 1, K, rp),  # A_i [r, K]  -> [slot, K, r_pad]
            "b": (1, N, 0, N, rp),   # B_i [N, r]  -> [slot, N, r_pad]
            "bt": (1, N, 1, rp, N),  # B_i [N, r]  -> [slot, r_pad, N]
        }[w]
        dst = torch.empty((max(n, 1), spec[3], spec[4]), dtype=dtype, device=device)
        rc = L.lf_pack_adapters(src_code, dst_code, ptrs.data_ptr(), ranks_dev.data_ptr(), n, spec[0], spec[1],
                                spec[2], spec[3], spec[4], dst.data_ptr(), stream)
        nat.check(rc, "lf_pack_adapters")
        entry[w] = dst
        entry.setdefault("ptr_bufs", []).append((ptrs, ranks_dev))


def _weight(base_weight: torch.Tensor, dtype, device, at) -> torch.Tensor:
    """Base weight as a contiguous tensor of the activation dtype (converted copies cached)."""
    if isinstance(base_weight, MX4Weight):
        raise ValueError("this call takes a dense base_weight (MX4Weight.dequantize)")
    if base_weight.device != device:
        raise ValueError(f"base_weight must live on {device}")
    if base_weight.dtype == dtype and base_weight.is_contiguous():
        return base_weight
    key = (id(base_weight), dtype)
    hit = _WEIGHT_CACHE.get(key)
    if hit is not None:
        ref, ptr, ver, conv, made = hit
        if ref() is base_weight and ptr == base_weight.data_ptr() and ver == base_weight._version:
            made.use(device, at)
            return conv
    _building("a copy of base_weight", device)
    conv = base_weight.to(dtype).contiguous()
    if len(_WEIGHT_CACHE) >= _CACHE_MAX:
        _WEIGHT_CACHE.clear()
    try:
        _WEIGHT_CACHE[key] = (weakref.ref(base_weight), base_weight.data_ptr(), base_weight._version, conv,
                              _Made(device, conv))
    except TypeError:  # pragma: no cover
        pass
    return conv


def _activation(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor: lorafusion_b200 has no CPU path")
    if t.dtype not in _DTYPE_CODE:
        raise ValueError(f"{name}: unsupported dtype {t.dtype} (float32, bfloat16, float16)")
    return t if t.is_contiguous() else t.contiguous()


def _problem(code, T, K, N, x, w, packs) -> nat.Problem:
    p = nat.Problem()
    p.dtype, p.T, p.K, p.N = code, T, K, N
    p.x_dev = x.data_ptr()
    p.w_dev = w.data_ptr()
    p.a_pack_dev = packs["a"].data_ptr()
    p.b_pack_dev = packs["b"].data_ptr()
    if "bt" in packs:
        p.bt_pack_dev = packs["bt"].data_ptr()
        p.at_pack_dev = packs["at"].data_ptr()
    return p


def _base(base_weight, x: torch.Tensor, at):
    """(tensor that holds the base weight, whether it is the data of one in 4 bits).  A problem the tensor-core path
    cannot address takes a dense copy of a weight in 4 bits, made within the call."""
    if not isinstance(base_weight, MX4Weight):
        return _weight(base_weight, x.dtype, x.device, at), False
    if base_weight.dtype is not x.dtype:
        raise ValueError(f"x ({x.dtype}) must have the dtype of the weight in 4 bits ({base_weight.dtype})")
    if base_weight.device != x.device:
        raise ValueError(f"base_weight must live on {x.device}")
    N, K = base_weight.shape
    if N % 8 or K % 8:
        return base_weight.dequantize(), False
    return base_weight.data, True


def _shape_of(base_weight, K: int) -> int:
    """out_features of a base weight that fits activations of K features."""
    shape = tuple(base_weight.shape)
    if len(shape) != 2 or shape[1] != K:
        raise ValueError(f"base_weight {shape} does not match x of {K} features")
    return shape[0]


class _Drop:
    """Dropout of one call: thresholds of its slots and the factors that go with them."""

    __slots__ = ("thresholds", "seed", "offset")

    def __init__(self, thresholds, seed, offset):
        self.thresholds, self.seed, self.offset = thresholds, seed, offset

    def scales(self, scales):
        return tuple(s * (65536.0 / (65536 - t)) for s, t in zip(scales, self.thresholds))

    def args(self, plan: _Plan, prob, backward: bool, device):
        """lf_dropout, and the scratch that it points at."""
        n = int(nat.lib().lf_dropout_scratch_bytes(ctypes.byref(prob), int(backward)))
        scratch = torch.empty(n, dtype=torch.uint8, device=device) if n else None
        return nat.Dropout(self.seed, self.offset, plan.thresholds, scratch.data_ptr() if n else None, n), scratch


# A float16 rank product s / (1 - p) x A^T must stay below 65504: factors beyond this one, which float16 training would
# hardly survive, are refused there rather than turned into infinities.
_F16_MAX_FACTOR = 64.0


def _drop(dropout, rts: _Routes, dtype) -> _Drop | None:
    """The call's dropout, or None where no adapter of the call has any."""
    if dropout is None:
        return None
    if not isinstance(dropout, AdapterDropout):
        raise ValueError(f"dropout must be an AdapterDropout or None, got {type(dropout).__name__}")
    thresholds = tuple(map(dropout.threshold, rts.slots))
    if dtype == torch.float16 and any(t > 65536 - 65536 / _F16_MAX_FACTOR for t in thresholds):
        raise ValueError(f"float16 calls take dropout rates up to {1 - 1 / _F16_MAX_FACTOR}")
    return _Drop(thresholds, dropout.seed, dropout.offset) if any(thresholds) else None


def fused_lora_forward(x, base_weight, lora_a, lora_b, adapters, routing, *,
                       dropout: AdapterDropout | None = None) -> torch.Tensor:
    """``y = x W^T + s_i (x A_i^T) B_i^T`` per routed row range.

    Same contract as ``mock_ops.fused_lora_forward`` (mock_ops.py:15-48):
    ``routing.validate`` runs first (``ValueError``); the result is a new
    ``[T, out_features]`` tensor in ``x.dtype``.

    Two things have no counterpart in the reference.  ``base_weight`` may be a ``quant.MX4Weight`` of x's dtype
    and device.  ``dropout`` (keyword only) puts a mask in front of the adapters: ``y = x W^T + s_i / (1 - p_i) (m x)
    A_i^T B_i^T``, a dropped element being zero whatever it was.

    A call can be captured into a CUDA graph once the same call has run (``RuntimeError`` before): replays read x and the
    base weight as they are then, repeat the mask, and keep the adapters' values of the capture.
    """
    with _LOCK:
        return _forward(x, base_weight, lora_a, lora_b, adapters, routing, dropout)


def _forward(x, base_weight, lora_a, lora_b, adapters, routing, dropout) -> torch.Tensor:
    global _last_launches
    rts = _routes(routing, x.shape[0])
    _last_launches = 0
    x_in = x
    x = _activation(x, "x")
    device = x.device
    T, K = x.shape
    N = _shape_of(base_weight, K)
    dtype = x.dtype
    code = _DTYPE_CODE[dtype]
    drop = _drop(dropout, rts, dtype)
    aset = _adapters(rts, lora_a, lora_b, adapters)
    at = stream, captured = _at(device)
    w, mx4 = _base(base_weight, x, at)
    if mx4 and x.data_ptr() % 16:
        x = x.detach().clone()
    plan = _plan(rts, aset, T, device, at, drop)
    packs = _pack(plan, aset, dtype, K, N, device, at, backward=False)
    y = torch.empty((T, N), dtype=dtype, device=device)
    if T == 0 or N == 0:
        return y
    _warn_if_cuda_core(dtype, K, N, (x, w, y), 4)
    L = nat.lib()
    info = ctypes.byref(plan.info)
    # S_ext and flags in one buffer (kept for the backward), the K-split tail's scratch in another
    # (back to the allocator's cache once the launch is enqueued)
    fixed, rest, _ = plan.workspace(code)
    ws = torch.empty(fixed, dtype=torch.uint8, device=device)
    tail = torch.empty(rest, dtype=torch.uint8, device=device)
    prob = _problem(code, T, K, N, x, w, packs)
    planes = ctypes.c_int32(0)
    opt, keep = _options(mx4, drop, plan, prob, False, device)
    with nat.on_device(device.index):
        rc = L.lf_forward_opt(ctypes.byref(prob), info, plan.table_dev.data_ptr(), opt, y.data_ptr(), ws.data_ptr(),
                              ws.numel(), tail.data_ptr(), tail.numel(), ctypes.byref(planes), stream)
    nat.check(rc, "lf_forward_opt")
    if captured:
        _hold(captured, device, plan, packs, base_weight.data if isinstance(base_weight, MX4Weight) else w)
    # 2 K-half planes: shrink inside the GEMM launch (1 launch); 1: shrink launched on its own
    _last_launches = {2: 1, 1: 2}.get(planes.value) or int(L.lf_forward_launch_count(ctypes.byref(prob), info))
    if drop is not None:
        _last_launches += planes.value == 0  # the masked copy on CUDA cores
    elif planes.value > 0 and plan.info.n_segtiles > 0:
        _save_sf(x_in, rts, plan, aset, ws, planes.value, captured)
    return y


def _options(mx4: bool, drop: _Drop | None, plan: _Plan, prob, backward: bool, device):
    """lf_options of a call (None for a plain one), and what must live until it is enqueued."""
    if not mx4 and drop is None:
        return None, None
    opt = nat.Options(nat.LF_WEIGHT_MX4 if mx4 else nat.LF_WEIGHT_DENSE, 0, None)
    keep = None
    if drop is not None:
        args, keep = drop.args(plan, prob, backward, device)
        opt.dropout = ctypes.pointer(args)
    return ctypes.byref(opt), (opt, keep)


def _save_sf(x, rts, plan, aset, ws, planes: int, captured: int = 0) -> None:
    """Remember this forward's S_f (the fixed part of its workspace: S_ext planes and flags, not
    the K-split tail's scratch) for a backward on the same inputs."""
    dead = [k for k, v in _SAVED_SF.items() if v[0]() is None]
    for k in dead:
        del _SAVED_SF[k]
    while len(_SAVED_SF) >= _SAVED_MAX:
        _SAVED_SF.popitem(last=False)
    try:
        key = (id(x), id(rts), id(aset))
        _SAVED_SF[key] = (weakref.ref(x), x._version, rts, plan, aset, ws, planes, captured)
        _SAVED_SF.move_to_end(key)
    except TypeError:  # pragma: no cover - objects without weakref support
        pass


def _saved_sf(x, rts, plan, aset, captured: int = 0):
    """(workspace, planes) of a forward on this very x (unchanged since), with the same validated
    routes, plan and adapter record (every A and B tensor unchanged since), or None.  A captured
    backward takes that of a forward of the same capture alone: replays find another x."""
    hit = _SAVED_SF.get((id(x), id(rts), id(aset)))
    if hit is None:
        return None
    xref, ver, r0, p0, a0, ws, planes, c0 = hit
    if c0 != captured or xref() is not x or x._version != ver or r0 is not rts or p0 is not plan or a0 is not aset:
        return None
    return ws, planes


class PreparedForward:
    """A forward call with routing tables, adapter slabs and workspace resolved once.

    ``launch(y, stages)`` enqueues the selected stages (``LF_STAGE_*`` bits of
    ``lf_forward_stages``) on the current stream with no Python-side checks,
    for callers that replay the same batch layout (benchmarks, CUDA graphs).
    The caller keeps ``x`` and the weights alive and unchanged.
    """

    def __init__(self, x, base_weight, lora_a, lora_b, adapters, routing):
        rts = _routes(routing, x.shape[0])
        self.x = _activation(x, "x")
        self.device = self.x.device
        self.T, self.K = self.x.shape
        self.N = base_weight.shape[0]
        dtype = self.x.dtype
        self.dtype = dtype
        aset = _adapters(rts, lora_a, lora_b, adapters)
        at = _at(self.device)
        self.w = _weight(base_weight, dtype, self.device, at)
        self.plan = _plan(rts, aset, self.T, self.device, at)
        self.packs = _pack(self.plan, aset, dtype, self.K, self.N, self.device, at, backward=False)
        code = _DTYPE_CODE[dtype]
        L = nat.lib()
        ws_bytes = L.lf_forward_workspace_bytes(ctypes.byref(self.plan.info), code)
        self.ws = torch.empty(max(ws_bytes, 256), dtype=torch.uint8, device=self.device)
        self.prob = _problem(code, self.T, self.K, self.N, self.x, self.w, self.packs)

    def launch_count(self) -> int:
        """Kernel launches of the default forward (1: shrink co-scheduled in the GEMM launch)."""
        return int(nat.lib().lf_forward_launch_count(ctypes.byref(self.prob), ctypes.byref(self.plan.info)))

    def new_output(self) -> torch.Tensor:
        return torch.empty((self.T, self.N), dtype=self.dtype, device=self.device)

    def launch(self, y: torch.Tensor, stages: int = nat.LF_STAGE_SHRINK | nat.LF_STAGE_EXPAND) -> None:
        stream = torch.cuda.current_stream(self.device).cuda_stream
        rc = nat.lib().lf_forward_stages(ctypes.byref(self.prob), ctypes.byref(self.plan.info),
                                         self.plan.table_dev.data_ptr(), y.data_ptr(), self.ws.data_ptr(),
                                         self.ws.numel(), stages, stream)
        nat.check(rc, "lf_forward_stages")


def prepare_forward(x, base_weight, lora_a, lora_b, adapters, routing) -> PreparedForward:
    """Resolve a forward call once (see :class:`PreparedForward`)."""
    with _LOCK:
        return PreparedForward(x, base_weight, lora_a, lora_b, adapters, routing)


def fused_lora_backward(grad_out, x, base_weight, lora_a, lora_b, adapters, routing, *, grad_dtype=None,
                        peer=None, dropout: AdapterDropout | None = None):
    """Return ``(grad_x, grad_lora_a, grad_lora_b)`` as ``mock_ops.fused_lora_backward``.

    mock_ops.py:51-95: the base weight is frozen (no gradient); the dicts hold
    one entry per adapter that owns a route, in order of first appearance,
    each summed over that adapter's routes; tensors are in ``x.dtype``.
    ``grad_dtype=torch.float32`` (keyword only, no counterpart in the reference) returns the
    adapter gradients in float32, unrounded, for a caller that sums them across GPUs first.
    ``peer`` (keyword only, a ``sharding.PeerExchange``; no counterpart in the reference) sums the
    gradients of adapters whose rows span GPUs inside the dA/dB kernel, over NVLink: every rank
    calls it for its own rows, and each rank's dicts then hold the summed gradients of every
    spanning adapter, held here or not (``lf_backward_peer``).
    ``base_weight`` and ``dropout`` as in :func:`fused_lora_forward`: with the forward's ``dropout`` these are the
    gradients of its result, ``grad_x = g W + m (s_i / (1 - p_i) g B_i A_i)``.
    """
    with _LOCK:
        return _backward(grad_out, x, base_weight, lora_a, lora_b, adapters, routing, grad_dtype, peer, dropout)


def _backward(grad_out, x, base_weight, lora_a, lora_b, adapters, routing, grad_dtype, peer, dropout):
    global _last_launches
    rts = _routes(routing, x.shape[0])
    _last_launches = 0
    x_in = x
    x = _activation(x, "x")
    g = _activation(grad_out, "grad_out")
    device = x.device
    T, K = x.shape
    N = _shape_of(base_weight, K)
    if g.shape != (T, N):
        raise ValueError(f"grad_out {tuple(g.shape)} does not match [{T}, {N}]")
    dtype = x.dtype
    if g.dtype != dtype:
        g = g.to(dtype)
    code = _DTYPE_CODE[dtype]
    gdt = dtype if grad_dtype is None else grad_dtype
    if gdt not in (dtype, torch.float32):
        raise ValueError(f"grad_dtype must be None, x.dtype or torch.float32, got {grad_dtype}")
    drop = _drop(dropout, rts, dtype)
    aset = _adapters(rts, lora_a, lora_b, adapters)
    at = stream, captured = _at(device)
    if captured and peer is not None:  # every call numbers its blocks; replays would repeat the number
        raise RuntimeError("a call with peer cannot be captured into a CUDA graph")
    w, mx4 = _base(base_weight, x, at)
    if mx4:
        x, g = (t.detach().clone() if t.data_ptr() % 16 else t for t in (x, g))
    plan = _plan(rts, aset, T, device, at, drop)
    packs = _pack(plan, aset, dtype, K, N, device, at, backward=True)
    info = plan.info
    rtot = info.rank_total
    ext = _peer_layout(plan, peer, device) if peer is not None else None
    rows = rtot + (ext.extra_rows if ext is not None else 0)  # + spanning adapters not held here
    grad_x = torch.empty((T, K), dtype=dtype, device=device)
    ga_flat = torch.empty(max(rows * K, 1), dtype=gdt, device=device)
    gb_flat = torch.empty(max(rows * N, 1), dtype=gdt, device=device)
    _warn_if_cuda_core(dtype, K, N, (x, w, g, grad_x), 4)
    L = nat.lib()
    ws = torch.empty(plan.workspace(code)[2], dtype=torch.uint8, device=device)
    prob = _problem(code, T, K, N, x, w, packs)
    saved = _saved_sf(x_in, rts, plan, aset, captured) if dtype != torch.float32 and drop is None else None
    sf_ptr, sf_planes = (saved[0].data_ptr(), saved[1]) if saved is not None else (None, 0)
    # S_f from the forward on these inputs, when there was one: no second s x A^T shrink
    pr = None
    if ext is not None:
        peer.ensure(len(peer.vslots) * (-(-N // 128) + -(-K // 128)))
        pr = nat.PeerReduce(world=peer.world, rank=peer.rank, n_span=len(peer.vslots), r_pad_x=peer.r_pad_x,
                            gen=peer.next_gen())
        for r, ptr in enumerate(peer.ptrs):
            pr.exchange[r] = ptr
        pr.slot_span_dev = ext.slot_span.data_ptr()
        pr.span_info_dev = ext.span_info.data_ptr()
    opt, keep = _options(mx4, drop, plan, prob, True, device)
    with nat.on_device(device.index):
        rc = L.lf_backward_opt(ctypes.byref(prob), ctypes.byref(info), plan.table_dev.data_ptr(), opt, g.data_ptr(),
                               sf_ptr, sf_planes, _DTYPE_CODE[gdt], grad_x.data_ptr(), ga_flat.data_ptr(),
                               gb_flat.data_ptr(), ws.data_ptr(), ws.numel(), pr and ctypes.byref(pr), stream)
    if saved is not None:
        saved[0].record_stream(torch.cuda.current_stream(device))
    nat.check(rc, "lf_backward_opt")
    if captured:
        _hold(captured, device, plan, packs, base_weight.data if isinstance(base_weight, MX4Weight) else w)
    n_launch = max(0, int(L.lf_backward_launch_count(ctypes.byref(prob), ctypes.byref(info))))
    _last_launches = n_launch - 1 if saved is not None and n_launch == 4 else n_launch
    if drop is not None:
        # S_b, (S_f,) expand, grad_x (with S_f), dA and dB; on CUDA cores mask, S_f, S_b, grad_x, dA, dB
        _last_launches = {2: 4, 4: 5}.get(n_launch, 6)
    grad_a, grad_b = _grad_dicts(plan, ga_flat, gb_flat, K, N)
    if ext is not None:  # spanning adapters not held here: their summed blocks after the local ones
        for aid, parts in ext.nonheld.items():
            pre, r = parts[0][0], sum(rv for _, rv in parts)
            grad_a[aid] = ga_flat[pre * K:(pre + r) * K].view(r, K)
            blocks = [gb_flat[p0 * N:(p0 + rv) * N].view(N, rv) for p0, rv in parts]
            grad_b[aid] = blocks[0] if len(blocks) == 1 else torch.cat(blocks, dim=1)
    return grad_x, grad_a, grad_b


class _PeerLayout:
    __slots__ = ("slot_span", "span_info", "extra_rows", "nonheld")


_PEER_LAYOUTS: "OrderedDict[tuple, tuple]" = OrderedDict()


def _peer_layout(plan: _Plan, peer, device) -> _PeerLayout:
    """Device tables of lf_peer_reduce for one plan: each local virtual slot's index among the
    spanning virtual slots (-1: not spanning, or no rows here), and per spanning virtual slot its
    first gradient row in this call's layout (slots not held here follow rank_total), rank and
    holder mask.  Cached per (plan, exchange)."""
    key = (id(plan), id(peer))
    hit = _PEER_LAYOUTS.get(key)
    if hit is not None and hit[0] is plan and hit[1] is peer:
        return hit[2]
    me = 1 << peer.rank
    held: dict[int, int] = {}
    slot_span = []
    prefix = 0
    for si, c0, r in plan.vslots:
        i = peer.index.get((plan.slots[si], c0), -1)
        if i >= 0 and not peer.masks[i] & me:  # routes of this adapter here are all empty
            i = -1
        slot_span.append(i)
        if i >= 0:
            held[i] = prefix
        prefix += r
    info, extra, nonheld = [], 0, {}
    for i, (aid, c0, r) in enumerate(peer.vslots):
        if i in held:
            pre = held[i]
        else:
            pre = plan.info.rank_total + extra
            extra += r
            nonheld.setdefault(aid, []).append((pre, r))
        info += [pre, r, peer.masks[i]]
    lay = _PeerLayout()
    lay.slot_span = torch.tensor(slot_span or [-1], dtype=torch.int32, device=device)
    lay.span_info = torch.tensor(info, dtype=torch.int32, device=device)
    lay.extra_rows = extra
    lay.nonheld = nonheld
    while len(_PEER_LAYOUTS) >= 256:
        _PEER_LAYOUTS.popitem(last=False)
    _PEER_LAYOUTS[key] = (plan, peer, lay)
    return lay


class PreparedBackward:
    """A backward call with tables, slabs, outputs and workspace resolved once.

    ``launch(stages)`` enqueues ``lf_backward_stages`` (``LF_BSTAGE_*`` bits: routed shrinks,
    grad_x GEMM, dA/dB grams, each a launch of its own) on the current stream with no Python-side
    checks, so a caller can time the stages or order them around other work (a gradient
    all-reduce that overlaps the grad_x GEMM).  ``grads()`` returns ``(grad_x, grad_a, grad_b)``
    views of the outputs in the layout ``fused_lora_backward`` returns.  The caller keeps the
    inputs alive and unchanged.
    """

    def __init__(self, grad_out, x, base_weight, lora_a, lora_b, adapters, routing, grad_dtype=None):
        rts = _routes(routing, x.shape[0])
        self.x = _activation(x, "x")
        self.g = _activation(grad_out, "grad_out")
        self.device = self.x.device
        T, K = self.x.shape
        N = base_weight.shape[0]
        self.T, self.K, self.N = T, K, N
        dtype = self.x.dtype
        if self.g.dtype != dtype:
            self.g = self.g.to(dtype)
        gdt = dtype if grad_dtype is None else grad_dtype
        if gdt not in (dtype, torch.float32):
            raise ValueError(f"grad_dtype must be None, x.dtype or torch.float32, got {grad_dtype}")
        aset = _adapters(rts, lora_a, lora_b, adapters)
        at = _at(self.device)
        self.w = _weight(base_weight, dtype, self.device, at)
        self.plan = _plan(rts, aset, T, self.device, at)
        self.packs = _pack(self.plan, aset, dtype, K, N, self.device, at, backward=True)
        code = _DTYPE_CODE[dtype]
        self.gcode = _DTYPE_CODE[gdt]
        rtot = self.plan.info.rank_total
        self.grad_x = torch.empty((T, K), dtype=dtype, device=self.device)
        self.ga_flat = torch.empty(max(rtot * K, 1), dtype=gdt, device=self.device)
        self.gb_flat = torch.empty(max(rtot * N, 1), dtype=gdt, device=self.device)
        ws_bytes = nat.lib().lf_backward_workspace_bytes(ctypes.byref(self.plan.info), code)
        self.ws = torch.empty(max(ws_bytes, 256), dtype=torch.uint8, device=self.device)
        self.prob = _problem(code, T, K, N, self.x, self.w, self.packs)

    def launch(self, stages: int) -> None:
        stream = torch.cuda.current_stream(self.device).cuda_stream
        rc = nat.lib().lf_backward_stages(
            ctypes.byref(self.prob), ctypes.byref(self.plan.info), self.plan.table_dev.data_ptr(), self.g.data_ptr(),
            None, 0, self.gcode, self.grad_x.data_ptr(), self.ga_flat.data_ptr(), self.gb_flat.data_ptr(),
            self.ws.data_ptr(), self.ws.numel(), stages, stream)
        nat.check(rc, "lf_backward_stages")

    def grads(self):
        return self.grad_x, *_grad_dicts(self.plan, self.ga_flat, self.gb_flat, self.K, self.N)


def prepare_backward(grad_out, x, base_weight, lora_a, lora_b, adapters, routing, grad_dtype=None) -> PreparedBackward:
    """Resolve a backward call once (see :class:`PreparedBackward`)."""
    with _LOCK:
        return PreparedBackward(grad_out, x, base_weight, lora_a, lora_b, adapters, routing, grad_dtype)


def _grad_dicts(plan: _Plan, ga_flat, gb_flat, K: int, N: int):
    """Per-adapter views of the packed gradients: dA_i rows [rank_prefix_i, +r_i) of a
    [rank_total, K] matrix, dB_i the [N, r_i] block at element rank_prefix_i * N.  One split per
    run of equal ranks keeps the view count per call, not per adapter, in Python.  An adapter of
    rank > 64 (several virtual slots) gets its dB blocks joined along the rank dimension."""
    slots, ranks = plan.slots, plan.ranks
    rtot = plan.info.rank_total
    if not slots:
        return {}, {}
    grad_a = dict(zip(slots, ga_flat[:rtot * K].view(rtot, K).split(ranks)))
    if len(plan.vslots) != len(slots):
        grad_b, off = {}, 0
        for aid, r in zip(slots, ranks):
            blocks = []
            for c0 in range(0, r, MAX_SLOT_RANK):
                rv = min(MAX_SLOT_RANK, r - c0)
                blocks.append(gb_flat[off * N:(off + rv) * N].view(N, rv))
                off += rv
            grad_b[aid] = blocks[0] if len(blocks) == 1 else torch.cat(blocks, dim=1)
        return grad_a, grad_b
    grad_b: dict[int, torch.Tensor] = {}
    i, off, n = 0, 0, len(slots)
    while i < n:
        r = ranks[i]
        j = i + 1
        while j < n and ranks[j] == r:
            j += 1
        grad_b.update(zip(slots[i:j], gb_flat[off * N:(off + (j - i) * r) * N].view((j - i) * N, r).split(N)))
        off += (j - i) * r
        i = j
    return grad_a, grad_b


# ----------------------------------------------------------------------------- host-resident batches
_SIDE_STREAMS: dict[int, tuple] = {}


class _ChunkPlans:
    """Row chunks of one routing for the host-streamed forward: per chunk, tables of its routes
    (rebased to the chunk) over the whole batch's slots, as the C ABI's chunk array."""

    __slots__ = ("array", "n", "infos", "tables", "ws_bytes", "launches", "made")

    def __init__(self, rts: _Routes, ranks, scales, total_rows: int, chunk_rows: int, device, code: int):
        L = nat.lib()
        rk = np.asarray(ranks, dtype=np.int32)
        sc = np.asarray(scales, dtype=np.float32)
        n_slots = len(rts.slots)
        bounds = _chunk_bounds(total_rows, chunk_rows)
        self.n = len(bounds)
        self.array = (nat.HostChunk * max(self.n, 1))()
        self.infos, self.tables, self.ws_bytes, self.launches = [], [], 256, 0
        for i, c0 in enumerate(bounds):
            c1 = bounds[i + 1] if i + 1 < len(bounds) else total_rows
            sel = (rts.starts < c1) & (rts.ends > c0)
            starts = np.ascontiguousarray(np.maximum(rts.starts[sel], c0) - c0, dtype=np.int32)
            ends = np.ascontiguousarray(np.minimum(rts.ends[sel], c1) - c0, dtype=np.int32)
            rslot = np.ascontiguousarray(rts.route_slot[sel], dtype=np.int32)
            info, table = _plan_tables(starts, ends, rslot, c1 - c0, rk, sc, n_slots)
            table_dev = table[: max(info.table_words, 1)].to(device, non_blocking=True)
            self.infos.append(info)
            self.tables.append(table_dev)
            self.array[i].row0, self.array[i].rows = c0, c1 - c0
            self.array[i].info = ctypes.pointer(info)
            self.array[i].table_dev = table_dev.data_ptr()
            self.ws_bytes = max(self.ws_bytes, int(L.lf_forward_workspace_bytes(ctypes.byref(info), code)))
        self.made = _Made(device, *self.tables)


EDGE_CHUNK_ROWS = 256


def _chunk_bounds(total_rows: int, chunk_rows: int) -> list[int]:
    """First row of every chunk of the host-streamed forward, all on the 128-row tile grid.  The
    first and the last chunk are short (EDGE_CHUNK_ROWS): the GPU work starts once the first
    chunk is copied in, and only the last chunk's copy back follows the last GEMM, so short edge
    chunks shorten the part of the call that the copies in both directions do not overlap.
    Batches too small for that are cut every chunk_rows."""
    edge = EDGE_CHUNK_ROWS
    if total_rows <= 2 * edge + chunk_rows:
        return list(range(0, total_rows, chunk_rows))
    bounds, cur = [0], edge
    last = (total_rows - edge) // 128 * 128
    while cur < last:
        bounds.append(cur)
        cur += chunk_rows
    bounds.append(last)
    return bounds


def _chunk_plans(rts: _Routes, aset: _AdapterSet, total_rows: int, chunk_rows: int, device, code: int,
                 at) -> _ChunkPlans:
    key = (chunk_rows, total_rows, aset.ranks, aset.scales, device, code)
    for k, v in rts.chunk_plans:
        if k == key:
            v.made.use(device, at)
            return v
    _building("the chunks' tables", device)
    plans = _ChunkPlans(rts, aset.ranks, aset.scales, total_rows, chunk_rows, device, code)
    rts.chunk_plans.insert(0, (key, plans))
    del rts.chunk_plans[4:]
    return plans


def fused_lora_forward_host(x_host, base_weight, lora_a, lora_b, adapters, routing, out=None,
                            chunk_rows: int = 1024):
    """``fused_lora_forward`` of a batch that lives in host memory; the result lands in host memory.

    One native call (``lf_forward_host``) enqueues everything: the rows travel in chunks of
    ``chunk_rows`` (a multiple of 256) between a short first and a short last chunk; chunk i is
    copied to the GPU on one stream while chunk i-1 is computed on the caller's current stream and
    chunk i-2 is copied back on a third, so both PCIe directions and the GPU work overlap.  Each output row depends only on its own input
    row, chunks start on the 128-row tile grid and their tables use the whole batch's slots, so
    the result equals one ``fused_lora_forward`` over the whole batch (bit for bit whenever the
    chunks and the whole batch run the routed shrink the same way: both co-scheduled, or both as
    separate launches).  ``x_host`` should be pinned (``pin_memory()``); ``out`` (pinned,
    ``[T, N]``, x's dtype) is allocated when omitted.  The copies back are enqueued, not waited
    for: synchronize the current stream before reading the result.  No counterpart in the
    reference (its ops take device tensors).
    """
    with _LOCK:
        return _forward_host(x_host, base_weight, lora_a, lora_b, adapters, routing, out, chunk_rows)


def _forward_host(x_host, base_weight, lora_a, lora_b, adapters, routing, out, chunk_rows):
    global _last_launches
    rts = _routes(routing, x_host.shape[0])
    if isinstance(base_weight, MX4Weight):
        raise ValueError("this call takes a dense base_weight (MX4Weight.dequantize)")
    if x_host.is_cuda or not base_weight.is_cuda:
        raise ValueError("x_host must be a host tensor and base_weight a CUDA tensor")
    if chunk_rows <= 0 or chunk_rows % 256:
        raise ValueError("chunk_rows must be a positive multiple of 256")
    if x_host.dim() != 2 or x_host.dtype not in _DTYPE_CODE:
        raise ValueError(f"x_host must be a 2-D float32/bfloat16/float16 tensor, got {tuple(x_host.shape)} "
                         f"{x_host.dtype}")
    device = base_weight.device
    T, K = x_host.shape
    N = base_weight.shape[0]
    if base_weight.dim() != 2 or base_weight.shape[1] != K:
        raise ValueError(f"base_weight {tuple(base_weight.shape)} does not match x {tuple(x_host.shape)}")
    dtype = x_host.dtype
    y_host = out if out is not None else torch.empty((T, N), dtype=dtype, pin_memory=True)
    if y_host.shape != (T, N) or y_host.dtype != dtype or y_host.is_cuda or not y_host.is_contiguous():
        raise ValueError("out must be a contiguous host tensor [T, N] of x's dtype")
    _last_launches = 0
    if T == 0:
        return y_host
    if not x_host.is_contiguous():
        x_host = x_host.contiguous()
    code = _DTYPE_CODE[dtype]
    aset = _adapters(rts, lora_a, lora_b, adapters)
    at = _at(device)
    w = _weight(base_weight, dtype, device, at)
    plan = _plan(rts, aset, T, device, at)
    packs = _pack(plan, aset, dtype, K, N, device, at, backward=False)
    chunks = _chunk_plans(rts, aset, T, chunk_rows, device, code, at)
    x_dev = torch.empty((T, K), dtype=dtype, device=device)
    y_dev = torch.empty((T, N), dtype=dtype, device=device)
    ws = torch.empty(chunks.ws_bytes, dtype=torch.uint8, device=device)
    prob = _problem(code, T, K, N, x_dev, w, packs)
    compute = torch.cuda.current_stream(device)
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx not in _SIDE_STREAMS:
        _SIDE_STREAMS[idx] = (torch.cuda.Stream(device), torch.cuda.Stream(device))
    s_in, s_out = _SIDE_STREAMS[idx]
    L = nat.lib()
    rc = L.lf_forward_host(ctypes.byref(prob), chunks.array, chunks.n, x_host.data_ptr(), y_host.data_ptr(),
                           x_dev.data_ptr(), y_dev.data_ptr(), ws.data_ptr(), ws.numel(), compute.cuda_stream,
                           s_in.cuda_stream, s_out.cuda_stream)
    nat.check(rc, "lf_forward_host")
    # the current stream waits for the last copy back, so the allocator may reuse these after it
    pc = nat.Problem.from_buffer_copy(prob)
    for info in chunks.infos:
        pc.T = info.total_rows
        _last_launches += int(L.lf_forward_launch_count(ctypes.byref(pc), ctypes.byref(info)))
    return y_host
