"""Training: what follows ``b200_ops.fused_lora_backward`` in a step of many adapters.

Every adapter of a fused batch is a job of its own: its gradients have a norm of their own, and its
step count, learning rate and decay are its own.  :func:`clip_adapter_grads` computes the norms
over all projections and clips, :class:`AdapterAdamW` updates the weights (and can clip on the way,
without a pass that writes the gradients back).  Both take gradients in the form the backward
returns them: dicts of adapter id -> tensor, one dict for each ``lora_a`` and each ``lora_b``.  A step
makes two or three launches whatever the number of adapters.

No counterpart in the reference (it has no optimizer).
"""

from __future__ import annotations

import ctypes
import math
from collections.abc import Mapping, Sequence

import numpy as np
import torch

from lorafusion_b200 import _native as nat
from lorafusion_b200 import b200_ops

__all__ = ["AdapterAdamW", "clip_adapter_grads"]

_CODE = b200_ops._DTYPE_CODE
# descriptors called through map(): one C call a tensor keeps hundreds of tensors cheap
_DTYPE = torch.Tensor.dtype.__get__
_SHAPE = torch.Tensor.shape.__get__
_NUMEL = torch.Tensor.numel
_DATA_PTR = torch.Tensor.data_ptr
_CONTIGUOUS = torch.Tensor.is_contiguous
_DEVICE_INDEX = torch.Tensor.get_device  # -1 on the CPU

_GRAD_TENSOR = np.dtype(nat.GRAD_TENSOR)
_ADAMW_TENSOR = np.dtype(nat.ADAMW_TENSOR)
_MAX_NUMEL = (1 << 32) - 8192


def _one_device(tensors, what: str) -> int:
    devices = set(map(_DEVICE_INDEX, tensors))
    if -1 in devices:
        raise ValueError(f"{what} must be CUDA tensors: lorafusion_b200 has no CPU path")
    if len(devices) > 1:
        raise ValueError(f"{what} must live on one device, got {sorted(devices)}")
    return devices.pop()


def clip_adapter_grads(grads: Sequence[Mapping], max_norm: float | None, *, norm_type: float = 2.0,
                       per_adapter: bool = True) -> torch.Tensor:
    """Norm of each adapter's gradients over all dicts of ``grads``, and the gradients clipped in place.

    ``grads`` is a sequence of dicts adapter id -> gradient, such as the ``grad_lora_a`` and
    ``grad_lora_b`` of every projection; the tensors are contiguous float32, bfloat16 or float16 CUDA
    tensors of one device that share no memory.  ``norm_type`` is 2 or ``inf``.  Each adapter's gradients are
    multiplied by ``min(1, max_norm / (norm + 1e-6))``; with ``per_adapter=False`` one norm over all
    adapters clips them together.  ``max_norm=None`` computes the norms only.  A norm that is NaN makes its
    gradients NaN, an infinite one makes them zero, and NaN where they were infinite.

    Returns the norms before clipping as a float32 tensor on the gradients' device: one per adapter,
    in order of first appearance in ``grads``, or a 0-dim tensor with ``per_adapter=False``.  The sums are
    float64 in a fixed order.  Three launches for up to 1500 tensors; nothing is read back.
    """
    if max_norm is not None and not max_norm >= 0.0:
        raise ValueError(f"max_norm must be non-negative, got {max_norm}")
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    grads = list(grads)
    norms = nat.glue().clip(grads, per_adapter, norm_type != 2.0, None if max_norm is None else float(max_norm))
    if norms is not None:
        return norms
    # anything that is an error, or a mapping that is not a dict
    tensors: list[torch.Tensor] = []
    ids: list = []
    for d in grads:
        tensors += d.values()
        ids += d
    if not tensors:
        raise ValueError("no gradients")
    index = _one_device(tensors, "gradients")
    codes = list(map(_CODE.get, map(_DTYPE, tensors)))
    if None in codes:
        raise ValueError("gradients must be float32, bfloat16 or float16")
    if not all(map(_CONTIGUOUS, tensors)):
        raise ValueError("gradients must be contiguous")
    n = len(tensors)
    rec = np.empty(n, dtype=_GRAD_TENSOR)
    rec["ptr"] = list(map(_DATA_PTR, tensors))
    rec["numel"] = list(map(_NUMEL, tensors))
    rec["dtype"] = codes
    if per_adapter:
        order = dict.fromkeys(ids)
        for i, aid in enumerate(order):
            order[aid] = i
        rec["group"] = list(map(order.__getitem__, ids))
        n_groups = len(order)
    else:
        rec["group"] = 0
        n_groups = 1
    if int(rec["numel"].max()) >= _MAX_NUMEL:
        raise ValueError(f"a gradient has {int(rec['numel'].max())} elements: at most {_MAX_NUMEL - 1} are supported")
    L = nat.lib()
    device = torch.device("cuda", index)
    at = rec.ctypes.data
    ws = torch.empty(max(16, L.lf_grad_clip_workspace_bytes(at, n, n_groups)), dtype=torch.uint8, device=device)
    norms = torch.empty(n_groups, dtype=torch.float32, device=device)
    with nat.on_device(index):
        rc = L.lf_grad_clip(at, n, n_groups, int(norm_type != 2.0), int(max_norm is not None),
                            0.0 if max_norm is None else float(max_norm), norms.data_ptr(), ws.data_ptr(), ws.numel(),
                            nat.raw_stream(index))
    if rc == nat.LF_ERR_INVALID_ARG:
        raise ValueError("gradients share memory: each may be named once")
    nat.check(rc, "lf_grad_clip")
    if max_norm is not None:
        torch.autograd.graph.increment_version(tensors)
    return norms if per_adapter else norms[0]


class AdapterAdamW:
    """AdamW over the LoRA weights of many adapters, each adapter a job with its own step count.

    ``params`` is a sequence of dicts adapter id -> weight (``lora_a`` and ``lora_b`` of every projection):
    contiguous CUDA tensors of one device and one dtype (float32, bfloat16, float16), updated in place.
    ``lr`` and ``weight_decay`` are one value or a dict by adapter id (``set_adapter`` changes them
    later).  16-bit weights keep float32 masters, from which they are rounded after each step.

    ``step(grads)`` takes dicts in the order of ``params``.  An adapter that a dict lacks (the backward
    returns only adapters with rows in the batch) keeps that weight and its state, and its step count
    when no dict has it.  With ``max_norm`` each adapter's gradients are scaled by
    ``min(1, max_norm / (norm + 1e-6))`` on the way, norm over all its gradients (the gradient tensors are
    not written); ``skip_nonfinite`` leaves an adapter whose norm is NaN or infinite as it is, so one
    diverged job does not spoil its weights.

    State: ``exp_avg``, ``exp_avg_sq`` and ``master`` are flat float32 tensors (each weight's block starts
    at a multiple of 8 elements, in the order of ``params``; ``state(adapter_id)`` has the views) and
    ``steps`` an int32 tensor, one count per adapter of ``ids``.  ``state_dict`` / ``load_state_dict``
    carry all of it.  A weight written by other code is taken up by ``refresh_masters()``.
    """

    def __init__(self, params: Sequence[Mapping], *, lr=1e-3, weight_decay=0.0, betas=(0.9, 0.999), eps: float = 1e-8,
                 max_norm: float | None = None, skip_nonfinite: bool = False):
        self.params = [dict(d) for d in params]
        self._tensors = [t for d in self.params for t in d.values()]
        self._names = [(j, aid) for j, d in enumerate(self.params) for aid in d]
        if not self._tensors:
            raise ValueError("no weights")
        index = _one_device(self._tensors, "weights")
        dtypes = set(map(_DTYPE, self._tensors))
        if len(dtypes) > 1 or next(iter(dtypes)) not in _CODE:
            raise ValueError(f"weights must share one dtype (float32, bfloat16, float16), got {dtypes}")
        if not all(map(_CONTIGUOUS, self._tensors)):
            raise ValueError("weights must be contiguous")
        common = self._common_hyper(betas, eps, max_norm, skip_nonfinite)
        self.device = torch.device("cuda", index)
        self.dtype = dtypes.pop()
        self.betas, self.eps, self.max_norm, self.skip_nonfinite = common
        self.ids = list(dict.fromkeys(aid for _, aid in self._names))
        self._group = {aid: i for i, aid in enumerate(self.ids)}
        self._hyper = np.empty((len(self.ids), 2))
        for column, (name, value) in enumerate((("lr", lr), ("weight_decay", weight_decay))):
            for i, aid in enumerate(self.ids):
                self._hyper[i, column] = self._hyper_value(name, value[aid] if isinstance(value, Mapping) else value)
        n = len(self._tensors)
        rec = np.zeros(n, dtype=_ADAMW_TENSOR)
        rec["param"] = list(map(_DATA_PTR, self._tensors))
        numel = np.array(list(map(_NUMEL, self._tensors)), dtype=np.int64)
        if int(numel.max()) >= _MAX_NUMEL:
            raise ValueError(f"a weight has {int(numel.max())} elements: at most {_MAX_NUMEL - 1} are supported")
        rec["numel"] = numel
        rec["group"] = [self._group[aid] for _, aid in self._names]
        ends = rec["param"] + numel.astype(np.uint64) * np.uint64(self._tensors[0].element_size())
        order = np.argsort(rec["param"], kind="stable")
        order = order[numel[order] > 0]
        if (ends[order][:-1] > rec["param"][order][1:]).any():
            raise ValueError("weights share memory: each may be named once")
        L = nat.lib()
        n_chunks, elems = ctypes.c_int64(0), ctypes.c_int64(0)
        nat.check(L.lf_adamw_plan(rec.ctypes.data, n, len(self.ids), None, 0, ctypes.byref(n_chunks),
                                  ctypes.byref(elems)), "lf_adamw_plan")
        chunk_tensor = np.zeros(max(1, n_chunks.value), dtype=np.int32)
        nat.check(L.lf_adamw_plan(rec.ctypes.data, n, len(self.ids), chunk_tensor.ctypes.data, n_chunks.value,
                                  ctypes.byref(n_chunks), ctypes.byref(elems)), "lf_adamw_plan")
        self._rec, self._n_chunks = rec, n_chunks.value
        self._addresses = np.ascontiguousarray(rec["param"])
        self._ws_bytes = int(L.lf_adamw_workspace_bytes(self._n_chunks, len(self.ids)))
        self._rec_dev = torch.from_numpy(rec.view(np.uint8).copy()).to(self.device)
        self._chunk_dev = torch.from_numpy(chunk_tensor).to(self.device)
        self._hyper_dev = torch.from_numpy(self._hyper.copy()).to(self.device)
        self._hyper_changed = False
        self._shapes = list(map(_SHAPE, self._tensors))
        self._keys = [list(d) for d in self.params]
        state = dict(dtype=torch.float32, device=self.device)
        self.exp_avg = torch.zeros(elems.value, **state)
        self.exp_avg_sq = torch.zeros(elems.value, **state)
        self.master = None if self.dtype == torch.float32 else torch.zeros(elems.value, **state)
        self.steps = torch.zeros(len(self.ids), dtype=torch.int32, device=self.device)
        self.refresh_masters()

    @staticmethod
    def _hyper_value(name: str, value) -> float:
        value = float(value)
        if not 0.0 <= value < math.inf:
            raise ValueError(f"{name} must be finite and non-negative, got {value}")
        return value

    @staticmethod
    def _common_hyper(betas, eps, max_norm, skip_nonfinite):
        """(betas, eps, max_norm, skip_nonfinite), checked."""
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0) or not eps >= 0.0:
            raise ValueError(f"betas must be in [0, 1) and eps non-negative, got {betas}, {eps}")
        if max_norm is not None and not max_norm >= 0.0:
            raise ValueError(f"max_norm must be non-negative, got {max_norm}")
        return (float(betas[0]), float(betas[1])), float(eps), max_norm, bool(skip_nonfinite)

    def set_adapter(self, adapter_id, *, lr: float | None = None, weight_decay: float | None = None) -> None:
        """Change one adapter's learning rate or decay, from the next step on."""
        row = self._hyper[self._group[adapter_id]]
        row[:] = (row[0] if lr is None else self._hyper_value("lr", lr),
                  row[1] if weight_decay is None else self._hyper_value("weight_decay", weight_decay))
        self._hyper_changed = True

    def _block(self, flat: torch.Tensor, k: int) -> torch.Tensor:
        off = int(self._rec["state_off"][k])
        return flat[off:off + self._tensors[k].numel()].view(self._shapes[k])

    @torch.no_grad()
    def refresh_masters(self) -> None:
        """Take the float32 masters from the weights as they are now (16-bit weights only)."""
        if self.master is not None:
            masters = [self._block(self.master, k) for k in range(len(self._tensors))]
            torch._foreach_copy_(masters, self._tensors)

    def state(self, adapter_id) -> dict:
        """``{index into params: {"exp_avg", "exp_avg_sq"[, "master"]}}`` views of one adapter's state."""
        flats = {"exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq}
        if self.master is not None:
            flats["master"] = self.master
        return {j: {name: self._block(flat, k) for name, flat in flats.items()}
                for k, (j, aid) in enumerate(self._names) if aid == adapter_id}

    def state_dict(self) -> dict:
        """Copies of the state, step counts and hyperparameters (``load_state_dict`` takes them back), and
        ``layout``: dict index, adapter id and shape of the weight of each block, in the state's order."""
        return {"ids": list(self.ids), "layout": self._layout(), "exp_avg": self.exp_avg.clone(),
                "exp_avg_sq": self.exp_avg_sq.clone(), "master": None if self.master is None else self.master.clone(),
                "steps": self.steps.clone(), "hyper": self._hyper.tolist(), "betas": self.betas, "eps": self.eps,
                "max_norm": self.max_norm, "skip_nonfinite": self.skip_nonfinite}

    def _layout(self) -> list:
        return [(j, aid, tuple(shape)) for (j, aid), shape in zip(self._names, self._shapes)]

    @torch.no_grad()
    def load_state_dict(self, state: dict) -> None:
        """Restore ``state_dict()`` of an optimizer over the same adapters and shapes in the same order, with
        its hyperparameters; 16-bit weights are rounded from the restored masters.  A state of another layout is refused before anything
        is written; so is one without a ``layout`` (its blocks could belong to other weights)."""
        if "layout" not in state:
            raise ValueError("the state has no record of the weights its blocks belong to (\"layout\")")
        same = (state["ids"] == self.ids and [(j, aid, tuple(s)) for j, aid, s in state["layout"]] == self._layout()
                and state["exp_avg"].shape == self.exp_avg.shape
                and state["exp_avg_sq"].shape == self.exp_avg_sq.shape and state["steps"].shape == self.steps.shape
                and (state["master"] is None) == (self.master is None)
                and (self.master is None or state["master"].shape == self.master.shape)
                and np.shape(state["hyper"]) == self._hyper.shape)
        if not same:
            raise ValueError("the state belongs to other adapters, shapes, weight types or another order of them")
        hyper = [[self._hyper_value(name, v) for name, v in zip(("lr", "weight_decay"), row)] for row in state["hyper"]]
        common = self._common_hyper(*(state.get(name, getattr(self, name))
                                      for name in ("betas", "eps", "max_norm", "skip_nonfinite")))
        self.betas, self.eps, self.max_norm, self.skip_nonfinite = common
        self.exp_avg.copy_(state["exp_avg"])
        self.exp_avg_sq.copy_(state["exp_avg_sq"])
        self.steps.copy_(state["steps"])
        self._hyper[:] = hyper
        self._hyper_changed = True
        if self.master is not None:
            self.master.copy_(state["master"])
            masters = [self._block(self.master, k) for k in range(len(self._tensors))]
            torch._foreach_copy_(self._tensors, masters)

    def step(self, grads: Sequence[Mapping]) -> torch.Tensor | None:
        """One update; returns each adapter's gradient norm before clipping (float32, in the order of
        ``ids``, 0 for an adapter without gradients) when ``max_norm`` or ``skip_nonfinite`` needs it.

        ``grads`` holds one dict per dict of ``params``; its tensors are contiguous, shaped like the
        weights, all float32 or all of the weights' dtype.  The weights' version counters advance, so
        ``b200_ops`` repacks them; a step therefore cannot be captured into a CUDA graph
        (``RuntimeError``).  Enqueued on the current stream; nothing is read back.
        """
        if len(grads) != len(self.params):
            raise ValueError(f"expected {len(self.params)} dicts of gradients, got {len(grads)}")
        ptrs = np.empty(len(self._tensors), dtype=np.uint64)
        code = nat.glue().gather_step(grads, self._keys, self._tensors, self._addresses, ptrs)
        if code is None:
            code = self._gather(grads, ptrs)
        if code < 0:
            return self._no_gradients()
        if self._hyper_changed:
            with nat.on_device(self.device.index):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("AdapterAdamW.step cannot be captured into a CUDA graph")
                # a pinned copy of its own for each upload: the allocator hands it out again only after the copy, and
                # the host waits for nothing that is queued (from pageable memory it waits for all of it)
                self._hyper_dev.copy_(torch.from_numpy(self._hyper).pin_memory(), non_blocking=True)
            self._hyper_changed = False
        return nat.glue().adamw_step(
            self._tensors, ptrs, self._rec, self._rec_dev, self._chunk_dev, self._hyper_dev, self.steps, self.exp_avg,
            self.exp_avg_sq, self.master, self._n_chunks, len(self.ids), self._ws_bytes, self.betas, self.eps,
            self.max_norm, self.skip_nonfinite, _CODE[self.dtype], code)

    def _gather(self, grads, ptrs: np.ndarray) -> int:
        """``gather_step`` with every check on its own, for its error; dicts may be other mappings here."""
        dtypes, at = set(), 0
        for d, keys in zip(grads, self._keys):
            unknown = set(d) - set(keys)
            if unknown:
                raise ValueError(f"gradients of unknown adapters: {sorted(unknown, key=str)}")
            for aid in keys:
                w, g = self._tensors[at], d.get(aid)
                if w.data_ptr() != self._addresses[at]:
                    raise RuntimeError("a weight's storage was replaced: build a new AdapterAdamW")
                if g is not None:
                    if g.device != self.device:
                        raise ValueError(f"gradients must live on {self.device}, got {g.device}")
                    if not g.is_contiguous():
                        raise ValueError("gradients must be contiguous")
                    if g.shape != w.shape:
                        raise ValueError(f"gradient of adapter {aid} (dict {self._names[at][0]}) has shape "
                                         f"{tuple(g.shape)}, its weight {tuple(w.shape)}")
                    dtypes.add(g.dtype)
                ptrs[at] = 0 if g is None else g.data_ptr()
                at += 1
        if not dtypes:
            return -1
        gdt = dtypes.pop()
        if dtypes or (gdt != torch.float32 and gdt != self.dtype):
            raise ValueError(f"gradients must all be float32 or all {self.dtype}, got {dtypes | {gdt}}")
        return _CODE[gdt]

    def _no_gradients(self):
        if self.max_norm is None and not self.skip_nonfinite:
            return None
        return torch.zeros(len(self.ids), dtype=torch.float32, device=self.device)
