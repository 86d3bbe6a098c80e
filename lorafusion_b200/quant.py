"""A frozen base weight held in 4 bits, and its products.

Adapters train and serve over a weight that does not change.  :class:`MX4Weight` holds it in microscaled
4-bit floating point (17/32 byte an element instead of 2) and stands in the place of the dense
``base_weight`` of ``b200_ops.fused_lora_forward`` / ``fused_lora_backward``, of ``serving.fused_lora_forward_rows``
and of ``Coordinator``.  :func:`mx4_linear` and :func:`mx4_linear_backward` are the products alone.  The kernels
decode the weight on its way into the tensor cores: no dense copy of it is made.

Format (OCP MXFP4): 32 neighbours along ``in_features`` share a power of two ``2**E`` with ``E = floor(log2(largest
magnitude)) - 2``, at least -127; a value is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it, with its sign, ties to
the even code, and 6 for what is larger.  A block that holds an infinity or NaN becomes NaN.  Every product takes the
values that the codes stand for, which the weight's own dtype holds exactly.

No counterpart in the reference (its base weight is dense, ``lorafusion/ops/mock_ops.py:15-48``).
"""

from __future__ import annotations

import torch

from lorafusion_b200 import _native as nat

__all__ = ["MX4Weight", "quantize_weight", "mx4_linear", "mx4_linear_backward"]

_CODE = {torch.bfloat16: nat.LF_BF16, torch.float16: nat.LF_F16}
_MAX = 1 << 24


class MX4Weight:
    """A weight ``[out_features, in_features]`` in 4 bits, made by :func:`quantize_weight`.

    ``data`` is its only tensor: uint8, in an order of its own that goes with ``dtype``, to be saved and restored as it is
    (``MX4Weight(data, out_features, in_features, dtype)``).  ``dtype`` (bfloat16 or float16) is that of the weight it was
    made from and of the activations it is multiplied with.  Its products read ``data`` on their stream: keep it
    unchanged until they have run.  Another tensor of the same bytes may be put in its place (``weight.data = saved``);
    the sizes and the dtype are fixed.
    """

    def __init__(self, data: torch.Tensor, out_features: int, in_features: int, dtype: torch.dtype):
        if dtype not in _CODE:
            raise ValueError(f"a weight in 4 bits serves bfloat16 or float16, not {dtype}")
        if not (0 < out_features <= _MAX and 0 < in_features <= _MAX):
            raise ValueError(f"out_features and in_features must be 1 .. {_MAX}, got {out_features}, {in_features}")
        self.out_features, self.in_features = out_features, in_features
        self.dtype = dtype
        self.data = data

    def __setattr__(self, name: str, value) -> None:
        # the kernels go by the sizes: what they read has to hold them
        if name == "data":
            if value.device.type != "cuda":
                raise ValueError("data must be a CUDA tensor: lorafusion_b200 has no CPU path")
            need = nat.lib().lf_mx4_bytes(self.out_features, self.in_features)
            if value.dtype is not torch.uint8 or value.shape != (need,) or not value.is_contiguous() or value.data_ptr() % 16:
                raise ValueError(f"data must be a contiguous, 16-byte aligned uint8 tensor of shape ({need},), got "
                                 f"{value.dtype} {tuple(value.shape)}")
        elif name in ("out_features", "in_features", "dtype") and name in self.__dict__:
            raise AttributeError(f"the {name} of a weight in 4 bits is fixed")
        object.__setattr__(self, name, value)

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.out_features, self.in_features))

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    def dequantize(self) -> torch.Tensor:
        """The values that the codes stand for, dense ``[out_features, in_features]`` in ``dtype``."""
        return nat.glue().mx4_dequantize(self.data, self.out_features, self.in_features, _CODE[self.dtype])

    def __repr__(self) -> str:
        return (f"MX4Weight(out_features={self.out_features}, in_features={self.in_features}, dtype={self.dtype}, "
                f"device={self.device})")


def quantize_weight(weight: torch.Tensor) -> MX4Weight:
    """``weight [out_features, in_features]`` (bfloat16 or float16, CUDA, rows may be strided) in 4 bits.

    One launch on the current stream of its device; nothing is read back.
    """
    code = _CODE.get(weight.dtype)
    data = nat.glue().mx4_quantize(weight, code) if code is not None else None
    if data is None:  # a copy, or an error
        if weight.dim() != 2 or 0 in weight.shape or max(weight.shape) > _MAX:
            raise ValueError(f"weight must be 2-D with sizes 1 .. {_MAX}, got shape {tuple(weight.shape)}")
        if weight.device.type != "cuda":
            raise ValueError("weight must be a CUDA tensor: lorafusion_b200 has no CPU path")
        if code is None:
            raise ValueError(f"weight must be bfloat16 or float16 (convert a {weight.dtype} one to the activations' dtype "
                             "first)")
        data = nat.glue().mx4_quantize(weight.detach().contiguous(), code)
    out = MX4Weight.__new__(MX4Weight)
    N, K = weight.shape
    out.__dict__.update(data=data, out_features=N, in_features=K, dtype=weight.dtype)
    return out


def _product(x: torch.Tensor, weight: MX4Weight, transpose: bool, name: str) -> torch.Tensor:
    if not isinstance(weight, MX4Weight):
        raise ValueError(f"weight must be an MX4Weight (quantize_weight), got {type(weight).__name__}")
    y = nat.glue().mx4_linear(x, weight.data, weight.out_features, weight.in_features, _CODE[weight.dtype],
                              int(transpose))
    if y is not None:
        return y
    # anything that needs a copy, a warning or an error
    N, K = weight.shape
    width = N if transpose else K
    if x.dim() != 2 or x.shape[1] != width:
        raise ValueError(f"{name} must have shape [rows, {width}], got {tuple(x.shape)}")
    if x.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor: lorafusion_b200 has no CPU path")
    if x.dtype is not weight.dtype:
        raise ValueError(f"{name} ({x.dtype}) must have the weight's dtype ({weight.dtype})")
    if x.device != weight.device:
        raise ValueError(f"{name} must live on {weight.device}")
    if x.shape[0] >= 1 << 31:
        raise ValueError(f"{name} has {x.shape[0]} rows: at most {(1 << 31) - 1} are supported")
    device = x.device
    x = x.detach()
    out = torch.empty((x.shape[0], K if transpose else N), dtype=x.dtype, device=device)
    if x.shape[0] == 0:
        return out
    if not x.is_contiguous() or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    from lorafusion_b200 import b200_ops
    b200_ops._warn_if_cuda_core(x.dtype, K, N, (x, weight.data, out))
    L = nat.lib()
    p = nat.Mx4Problem(_CODE[x.dtype], x.shape[0], K, N, int(transpose), 0, width, x.data_ptr(), weight.data.data_ptr())
    ws = torch.empty(L.lf_mx4_linear_workspace_bytes(K, N), dtype=torch.uint8, device=device)
    with nat.on_device(device.index):
        rc = L.lf_mx4_linear(p, out.data_ptr(), ws.data_ptr(), ws.numel(), nat.raw_stream(device.index))
    nat.check(rc, "lf_mx4_linear")
    return out


def mx4_linear(x: torch.Tensor, weight: MX4Weight) -> torch.Tensor:
    """``y = x V^T``, V the values of ``weight``: ``x [T, in_features]`` of the weight's dtype and device.

    One launch on the current stream of ``x``'s device; rows of ``x`` may be strided.  Autograd does not record the call
    (:func:`mx4_linear_backward` is its gradient; the weight has none).  The same call gives the same bits every
    time.  Problems whose in_features or out_features is not a multiple of 8 run on CUDA cores, from a dense copy of
    the weight made within the call, with a ``CudaCorePathWarning``.
    """
    return _product(x, weight, False, "x")


def mx4_linear_backward(grad_out: torch.Tensor, weight: MX4Weight) -> torch.Tensor:
    """``grad_x = grad_out V``, the gradient of :func:`mx4_linear`: ``grad_out [T, out_features]``."""
    return _product(grad_out, weight, True, "grad_out")
