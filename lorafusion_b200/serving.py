"""Serving: one shared projection for rows of many requests, each row with its own adapter.

``b200_ops.fused_lora_forward`` takes a batch whose rows a scheduler has packed into contiguous
routes, every row with an adapter.  A decoding server has neither: each step brings one token of
every running request, in the requests' order, some without an adapter, and the choice changes every
step.  Here the adapters stay resident in an :class:`AdapterBank` and
:func:`fused_lora_forward_rows` reads each row's slot from a device tensor, so nothing is planned on
the host and a captured call follows later changes of the slots and of the bank.

No counterpart in the reference (``lorafusion/ops/mock_ops.py:15-48`` is the packed form).
"""

from __future__ import annotations

import torch

from lorafusion_b200 import _native as nat
from lorafusion_b200 import b200_ops
from lorafusion_b200.quant import MX4Weight

__all__ = ["AdapterBank", "fused_lora_forward_rows"]

_DTYPE_CODE = b200_ops._DTYPE_CODE
_MAX_ROWS = (1 << 31) - 1


def _launches(rows: int, r_pad: int, tensor_cores: bool) -> int:
    if not tensor_cores:
        return 2 * -(-rows // (32 * 65535))
    return 2 if rows <= 256 else nat.lib().lf_rows_launch_count(rows, r_pad)


class AdapterBank:
    """Resident low-rank adapters of one projection, in ``n_slots`` slots of rank up to ``max_rank``.

    A slot holds ``lora_a [r, in_features]``, ``lora_b [out_features, r]`` and the factor ``scaling``
    (``alpha / r``); an empty slot adds nothing to its rows.  Memory: ``n_slots * r_pad *
    (in_features + out_features)`` elements of ``dtype``, ``r_pad`` being ``max_rank`` rounded up to 16,
    32, 64 or 128.  ``load`` and ``unload`` copy on the device's current stream: a forward enqueued
    there earlier still sees the old contents, a later one the new.  On another stream than the forwards', order
    them with events: the rows of a slot that changes under a running forward are undefined.
    """

    def __init__(self, n_slots: int, max_rank: int, in_features: int, out_features: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("an adapter bank lives on a CUDA device: lorafusion_b200 has no CPU path")
        if dtype not in _DTYPE_CODE:
            raise ValueError(f"unsupported dtype {dtype} (float32, bfloat16, float16)")
        if not 0 < n_slots < 1 << 24:
            raise ValueError(f"n_slots must be 1 .. {(1 << 24) - 1}, got {n_slots}")
        if not 0 < max_rank <= nat.BANK_MAX_RANK:
            raise ValueError(f"max_rank must be 1 .. {nat.BANK_MAX_RANK}, got {max_rank}")
        if not (0 < in_features <= 1 << 24 and 0 < out_features <= 1 << 24):
            raise ValueError(f"in_features and out_features must be 1 .. {1 << 24}, got {in_features}, {out_features}")
        self.r_pad = next(r for r in (16, 32, 64, nat.BANK_MAX_RANK) if max_rank <= r)
        if n_slots * (self.r_pad // 16) * max(out_features, 16) >= 1 << 31:
            raise ValueError(f"{n_slots} slots of rank {self.r_pad} and {out_features} features are too many for one "
                             "bank: n_slots * padded rank / 16 * out_features must stay below 2**31")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.n_slots, self.max_rank = n_slots, max_rank
        self.in_features, self.out_features = in_features, out_features
        self.dtype, self.device = dtype, device
        self.lora_a = torch.zeros(n_slots, self.r_pad, in_features, dtype=dtype, device=device)
        # B_i in steps of 16 ranks: what a kernel reads of an adapter is contiguous whatever its rank
        self.lora_b = torch.zeros(n_slots, self.r_pad // 16, out_features, 16, dtype=dtype, device=device)
        self.ranks = torch.zeros(n_slots, dtype=torch.int32, device=device)
        self.scales = torch.zeros(n_slots, dtype=torch.float32, device=device)

    def _check_slot(self, slot: int) -> None:
        if not 0 <= slot < self.n_slots:
            raise ValueError(f"slot {slot} is outside the bank's 0 .. {self.n_slots - 1}")

    def load(self, slot: int, lora_a: torch.Tensor, lora_b: torch.Tensor, scaling: float) -> None:
        """Copy an adapter into ``slot``, over what it held (converted to the bank's dtype)."""
        self._check_slot(slot)
        r = lora_a.shape[0] if lora_a.dim() == 2 else 0
        if lora_a.shape != (r, self.in_features) or lora_b.shape != (self.out_features, r):
            raise ValueError(f"slot {slot}: lora_a {tuple(lora_a.shape)} / lora_b {tuple(lora_b.shape)} do not match "
                             f"in_features={self.in_features}, out_features={self.out_features}")
        if not 0 < r <= self.max_rank:
            raise ValueError(f"slot {slot}: rank {r} is outside 1 .. {self.max_rank}")
        scaling = float(scaling)
        if nat.glue().bank_load(self.lora_a, self.lora_b, self.ranks, self.scales, slot, lora_a, lora_b, scaling):
            return
        # another dtype or device, rows that are not dense, parts of the slot itself: a copy as the bank has them, then
        # the same call
        lora_a, lora_b = (t.to(self.device, self.dtype, copy=True).contiguous() for t in (lora_a, lora_b))
        if not nat.glue().bank_load(self.lora_a, self.lora_b, self.ranks, self.scales, slot, lora_a, lora_b, scaling):
            raise ValueError(f"slot {slot}: the adapter cannot be copied into the bank's tensors")

    def unload(self, slot: int) -> None:
        """Empty ``slot``: its rows get the shared projection alone."""
        self._check_slot(slot)
        self.ranks[slot] = 0


def fused_lora_forward_rows(x: torch.Tensor, base_weight: torch.Tensor | MX4Weight, bank: AdapterBank,
                            row_slot: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``y[t] = x[t] W^T + s_i (x[t] A_i^T) B_i^T`` with ``i = row_slot[t]``, a slot of ``bank``.

    ``x [T, in_features]`` (rows may be strided), ``base_weight [out_features, in_features]`` and the
    bank share one dtype (float32, bfloat16, float16) and device.  ``base_weight`` may be a ``quant.MX4Weight``
    (bfloat16, float16), whose values W then are.  ``row_slot [T]`` is an int32 or int64
    tensor on that device, in any order; a negative entry means no adapter, and so does an
    empty slot.  An entry at or above ``bank.n_slots`` also gets the shared projection alone and is
    reported by ``_native.device_error()`` (``ERR_ROW_SLOT``): the slots are never read on the host.  Until the call
    has run, ``row_slot`` and the bank must not change on another stream (the result would be undefined).
    ``out`` (contiguous, ``[T, out_features]``) receives the result in place of a new tensor; it must not
    overlap ``x``, ``base_weight``, the bank or ``row_slot``, and not require a gradient unless under
    ``torch.no_grad()``.  Autograd does not record the call: the result has no gradient, whatever ``x`` and the
    weights require (``b200_ops.fused_lora_forward`` and ``fused_lora_backward`` are the pair for training).

    The same call gives the same bits every time.  In a batch of four launches (below) a row's bits do not depend on the
    rows beside it; in a shorter one its last bit may.

    Two launches on the current stream of ``x``'s device; long batches (above 256 rows, or 512 where the
    bank's padded rank is at most 32) run in chunks of 8192 rows of four launches each.  bf16/f16
    problems whose in_features or out_features is not a multiple of 8, or whose buffers are not 16-byte
    aligned, run on CUDA cores with a ``CudaCorePathWarning``.
    """
    mx4 = isinstance(base_weight, MX4Weight)
    y = None
    if bank is not None and not (mx4 and (base_weight.dtype is not x.dtype or base_weight.shape != (
            bank.out_features, bank.in_features))):
        y = nat.glue().rows_forward(
            x, base_weight.data if mx4 else base_weight, bank.lora_a, bank.lora_b, bank.ranks, bank.scales, row_slot,
            out, bank.r_pad, bank.out_features, int(mx4))
    if y is not None:
        b200_ops._last_launches = _launches(x.shape[0], bank.r_pad, x.dtype is not torch.float32)
        return y
    # anything that needs a copy, a warning or an error
    if x.dim() != 2:
        raise ValueError(f"x must be 2-D, got shape {tuple(x.shape)}")
    device, dtype = x.device, x.dtype
    if device.type != "cuda":
        raise ValueError("x must be a CUDA tensor: lorafusion_b200 has no CPU path")
    T, K = x.shape
    N = bank.out_features
    if T > _MAX_ROWS:
        raise ValueError(f"x has {T} rows: at most {_MAX_ROWS} are supported")
    if K != bank.in_features or base_weight.shape != (N, K):
        raise ValueError(f"x {tuple(x.shape)}, base_weight {tuple(base_weight.shape)} and a bank of "
                         f"{bank.in_features} -> {N} features do not match")
    if dtype != bank.dtype or base_weight.dtype != dtype:
        raise ValueError(f"x ({dtype}), base_weight ({base_weight.dtype}) and the bank ({bank.dtype}) must share one "
                         "dtype")
    if row_slot.shape != (T,):
        raise ValueError(f"row_slot must have shape ({T},), got {tuple(row_slot.shape)}")
    slot_dtype = row_slot.dtype
    if slot_dtype is not torch.int32 and slot_dtype is not torch.int64:
        raise ValueError(f"row_slot must be int32 or int64, got {slot_dtype}")
    if base_weight.device != device or bank.device != device or row_slot.device != device:
        raise ValueError(f"base_weight, the bank and row_slot must live on {device}")
    if not mx4 and not base_weight.is_contiguous():
        raise ValueError("base_weight must be contiguous")
    if not row_slot.is_contiguous():
        row_slot = row_slot.contiguous()
    ldx = K
    if not x.is_contiguous():
        ldx = x.stride(0)
        if x.stride(1) != 1 or ldx < K:
            x, ldx = x.contiguous(), K
    if out is None:
        out = torch.empty((T, N), dtype=dtype, device=device)
    elif out.shape != (T, N) or out.dtype != dtype or out.device != device or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {dtype} tensor of shape ({T}, {N}) on {device}")
    elif out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out requires a gradient, and this operator records none: call it under torch.no_grad()")
    b200_ops._last_launches = 0
    if T == 0:
        return out
    if mx4 and (K % 8 or N % 8 or out.data_ptr() % 16):  # CUDA cores: from a dense copy, made within the call
        base_weight, mx4 = base_weight.dequantize(), False
    weight = base_weight.data if mx4 else base_weight
    p = nat.RowsProblem(_DTYPE_CODE[dtype], T, K, N, bank.n_slots, bank.r_pad, 4 if slot_dtype is torch.int32 else 8,
                        int(mx4), ldx, x.data_ptr(), weight.data_ptr(), bank.lora_a.data_ptr(), bank.lora_b.data_ptr(),
                        bank.ranks.data_ptr(), bank.scales.data_ptr(), row_slot.data_ptr())
    tensor_cores = dtype is not torch.float32
    if tensor_cores and (K % 8 or N % 8 or ldx % 8 or
                         (p.x_dev | p.w_dev | p.a_bank_dev | p.b_bank_dev | out.data_ptr()) % 16):
        if ldx % 8 or p.x_dev % 16:  # only x's rows: a dense copy of x is far cheaper than CUDA cores
            x = x.clone(memory_format=torch.contiguous_format)
            p.x_dev, p.ldx = x.data_ptr(), K
        tensor_cores = not (K % 8 or N % 8 or (p.w_dev | p.a_bank_dev | p.b_bank_dev | out.data_ptr()) % 16)
        b200_ops._warn_if_cuda_core(dtype, K, N, (x, weight, bank.lora_a, bank.lora_b, out))
    L = nat.lib()
    ws = torch.empty(L.lf_rows_workspace_bytes(T, N, bank.r_pad, p.dtype), dtype=torch.uint8, device=device)
    with nat.on_device(device.index):
        rc = L.lf_rows_forward(p, out.data_ptr(), ws.data_ptr(), ws.numel(), nat.raw_stream(device.index))
    nat.check(rc, "lf_rows_forward")
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)
    b200_ops._last_launches = _launches(T, bank.r_pad, tensor_cores)
    return out
