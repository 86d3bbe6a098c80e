"""lf_mx4_linear by the C ABI and at sizes its tests leave out, against 64-bit arithmetic.  A 16-bit result is off by at most
half a step and ``n 2^-24`` of its sum of n magnitudes; the values of the weight are exact."""

import pytest
import torch

from lorafusion_b200 import _native as nat
from lorafusion_b200.quant import mx4_linear, mx4_linear_backward, quantize_weight

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def rand(*shape, seed=0, scale=1.0, dtype=BF16):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


def check(got, left, right):
    ref, mag = left.double() @ right, left.double().abs() @ right.abs()
    half = torch.finfo(got.dtype).eps / 2
    bound = half * ref.abs() + (left.shape[1] * 2.0 ** -24) * mag * (1 + half)
    assert torch.isfinite(got).all() and ((got.double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("transpose", [0, 1])
def test_a_pitch_that_only_cuda_cores_take(transpose):
    """K and N are multiples of 8, the rows' pitch is not: the workspace is a dense copy's."""
    T, K, N = 30, 256, 320
    q = quantize_weight(rand(N, K, seed=1, scale=1 / 16))
    v = q.dequantize().double()
    width, out = (N, K) if transpose else (K, N)
    x = rand(T, width + 3, seed=2)[:, :width]
    y = torch.empty(T, out, dtype=BF16, device=DEV)
    p = nat.Mx4Problem(nat.LF_BF16, T, K, N, transpose, 0, x.stride(0), x.data_ptr(), q.data.data_ptr())
    ws = torch.empty(2 * K * N, dtype=torch.uint8, device=DEV)
    stream = nat.raw_stream(0)
    assert nat.lib().lf_mx4_linear(p, y.data_ptr(), ws.data_ptr(), ws.numel() - 1, stream) == nat.LF_ERR_CAPACITY
    nat.check(nat.lib().lf_mx4_linear(p, y.data_ptr(), ws.data_ptr(), ws.numel(), stream), "lf_mx4_linear")
    torch.cuda.synchronize()
    check(y, x, v if transpose else v.t())
    # operands of the tensor cores need none
    x = x.contiguous()
    p.ld, p.in_dev = width, x.data_ptr()
    nat.check(nat.lib().lf_mx4_linear(p, y.data_ptr(), None, 0, stream), "lf_mx4_linear")
    torch.cuda.synchronize()
    check(y, x, v if transpose else v.t())
    assert nat.device_error() == 0


@pytest.mark.parametrize("transpose", [False, True])
def test_more_rows_than_one_dimension_of_a_grid(transpose):
    """4,194,240 rows are 65,535 tiles of 64 on CUDA cores."""
    T, K, N = 4_194_240 + 150, 9, 10
    q = quantize_weight(rand(N, K, seed=3))
    v = q.dequantize().double()
    x = rand(T, N if transpose else K, seed=4)
    y = (mx4_linear_backward if transpose else mx4_linear)(x, q)
    check(y, x, v if transpose else v.t())
    assert nat.device_error() == 0


@pytest.mark.parametrize("T,red,out,parts,transpose", [
    (1792, 384, 3584, 3, 0), (2048, 1000, 3328, 2, 0), (2300, 640, 2552, 3, 0), (2304, 256, 2560, 2, 0), (2304, 192, 2560, 1, 0),
    (1792, 384, 3584, 3, 1), (2048, 1000, 3328, 2, 1), (2300, 640, 2552, 3, 1), (2304, 256, 2560, 2, 1),
    (1024, 512, 1536, 3, 1), (1280, 2048, 1536, 2, 1), (3, 4096, 1000, 3, 1)])
def test_a_last_round_cut_along_the_reduction(T, red, out, parts, transpose):
    """Two and three parts in either direction, and the same sizes without the scratch for it."""
    K, N = (out, red) if transpose else (red, out)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert nat.lib().lf_mx4_linear_tail_parts(T, K, N, transpose, sms) == parts
    q = quantize_weight(rand(N, K, seed=5, scale=red ** -0.5))
    v = q.dequantize().double()
    x = rand(T, red, seed=6)
    call = mx4_linear_backward if transpose else mx4_linear
    y = call(x, q)
    check(y, x, v if transpose else v.t())
    assert torch.equal(call(x, q), y)
    whole = torch.empty_like(y)
    p = nat.Mx4Problem(nat.LF_BF16, T, K, N, transpose, 0, red, x.data_ptr(), q.data.data_ptr())
    nat.check(nat.lib().lf_mx4_linear(p, whole.data_ptr(), None, 0, nat.raw_stream(0)), "lf_mx4_linear")
    torch.cuda.synchronize()
    check(whole, x, v if transpose else v.t())
    assert nat.device_error() == 0
