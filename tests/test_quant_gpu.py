"""A base weight in 4 bits: the format, its products and the fused ops over it, against 64-bit arithmetic.

Tolerances.  A 16-bit result is off by at most half a step, ``eps / 2`` of its value, plus what a float32 sum of n
products can lose: ``n 2^-24`` of the sum of their magnitudes, in whatever order they are added.  The values of the weight
are exact.
"""

import numpy as np
import pytest
import torch

from lorafusion_b200 import _native as nat
from lorafusion_b200 import b200_ops
from lorafusion_b200.config import AdapterSpec, TileRoute, TileRoutingConfig
from lorafusion_b200.coordinator import Coordinator
from lorafusion_b200.quant import MX4Weight, mx4_linear, mx4_linear_backward, quantize_weight
from lorafusion_b200.scheduler import Request
from lorafusion_b200.serving import AdapterBank, fused_lora_forward_rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16


def values(w: torch.Tensor) -> torch.Tensor:
    """The format's definition in 64 bits, element by element on the CPU."""
    v = w.detach().double().cpu().numpy()
    n, k = v.shape
    out = np.empty_like(v)
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    for lo in range(0, k, 32):
        b = v[:, lo:lo + 32]
        top = np.abs(b).max(axis=1)
        bad = ~np.isfinite(top)
        _, e = np.frexp(np.where(bad | (top == 0), 2.0 ** -150, top))
        unit = np.ldexp(1.0, np.maximum(e - 3, -127))[:, None]
        a = np.abs(np.where(np.isfinite(b), b, 0.0)) / unit
        q = np.zeros(a.shape, dtype=int)
        for i, t in enumerate(ties):  # a tie goes to the even code: i is below it, i + 1 above
            q += (a > t) | ((a == t) & (i % 2 == 1))
        out[:, lo:lo + 32] = np.copysign(np.asarray(grid)[q] * unit, np.where(np.isfinite(b), b, 0.0))
        out[bad, lo:lo + 32] = np.nan
    return torch.from_numpy(out).to(w.device)


def rand(*shape, seed=0, scale=1.0, dtype=BF16):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


def check(got, ref, bound):
    """|got - ref| within half a step of got's type and `bound` (of the sums)."""
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - ref).abs()
    tol = half * ref.abs() + bound * (1 + half) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    worst = (err - tol).max().item()
    assert not torch.isnan(got).any() and worst <= 0, f"worst excess {worst:.3g}"


# ------------------------------------------------------------------------------------------- format
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 33), (3, 31), (128, 64), (130, 128), (129, 200), (257, 1000), (5, 4097)])
def test_values(shape, dtype):
    w = rand(*shape, seed=1, dtype=dtype)
    q = quantize_weight(w)
    assert q.shape == shape and q.dtype == dtype and q.nbytes == nat.lib().lf_mx4_bytes(*shape)
    assert torch.equal(q.dequantize().double(), values(w))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_values_of_every_magnitude(dtype):
    """Blocks at every power of two the type has, subnormals, zeros and ties among them."""
    fi = torch.finfo(dtype)
    lowest = -133 if dtype == BF16 else -24
    highest = 127 if dtype == BF16 else 15
    steps = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 1.96875, .125], device=DEV).double()
    rows = [torch.cat([steps, -steps])[:32] * 2.0 ** (e - 2) for e in range(lowest, highest + 1)]
    w = torch.stack(rows + [torch.zeros(32, device=DEV).double(), torch.full((32,), fi.max, device=DEV).double(),
                            torch.full((32,), -fi.smallest_normal, device=DEV).double()]).to(dtype)
    got = quantize_weight(w).dequantize()
    assert torch.equal(got.double(), values(w))
    assert torch.equal(torch.signbit(got), torch.signbit(w))  # of zeros too


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_blocks_that_are_not_finite(dtype):
    w = rand(4, 96, seed=2, dtype=dtype)
    w[0, 5], w[1, 40], w[2, 95] = float("inf"), float("nan"), -float("inf")
    got, ref = quantize_weight(w).dequantize(), values(w)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.isnan(got[0, :32]).all() and torch.isnan(got[1, 32:64]).all() and torch.isnan(got[2, 64:]).all()
    assert torch.equal(torch.nan_to_num(got.double()), torch.nan_to_num(ref))
    assert torch.isfinite(got[3]).all()


def test_strided_rows_and_transposed_weights():
    w = rand(70, 200, seed=3)
    for v in (w[:, 8:136], w[:, 3:100], w.t(), w[::2]):
        assert torch.equal(quantize_weight(v).dequantize(), quantize_weight(v.contiguous()).dequantize())


def test_values_are_their_own():
    """The values of a weight come back unchanged (a block's largest stays within its factor of two), and a restored
    weight is the same."""
    q = quantize_weight(rand(150, 300, seed=4))
    w = q.dequantize()
    again = quantize_weight(w).dequantize()
    assert torch.equal(again, w)
    copy = MX4Weight(q.data.clone(), 150, 300, BF16)
    assert torch.equal(copy.dequantize(), w)


# ------------------------------------------------------------------------------------------- products
SIZES = [(1, 64, 128), (1, 8, 8), (3, 72, 136), (16, 256, 64), (17, 200, 264), (33, 1000, 1048), (64, 512, 384),
         (100, 4096, 256), (129, 328, 520), (256, 1024, 1024), (257, 192, 320), (300, 2048, 4104), (777, 520, 1000),
         (1030, 1024, 512)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,K,N", SIZES)
def test_linear(T, K, N, dtype):
    x, g = rand(T, K, seed=5, dtype=dtype), rand(T, N, seed=6, dtype=dtype)
    q = quantize_weight(rand(N, K, seed=7, scale=K ** -0.5, dtype=dtype))
    v = q.dequantize().double()
    y = mx4_linear(x, q)
    assert y.shape == (T, N) and y.dtype == dtype
    check(y, x.double() @ v.t(), K * 2.0 ** -24 * (x.double().abs() @ v.abs().t()))
    gx = mx4_linear_backward(g, q)
    assert gx.shape == (T, K) and gx.dtype == dtype
    check(gx, g.double() @ v, N * 2.0 ** -24 * (g.double().abs() @ v.abs()))
    assert torch.equal(mx4_linear(x, q), y) and torch.equal(mx4_linear_backward(g, q), gx)
    assert nat.device_error() == 0


@pytest.mark.parametrize("T,K,N", [(1, 33, 7), (5, 100, 50), (70, 65, 130)])
def test_linear_odd_sizes(T, K, N):
    x, g = rand(T, K, seed=8), rand(T, N, seed=9)
    q = quantize_weight(rand(N, K, seed=10, scale=K ** -0.5))
    v = q.dequantize().double()
    with pytest.warns(b200_ops.CudaCorePathWarning) if (BF16, K, N) not in b200_ops._WARNED_SHAPES else _quiet():
        y = mx4_linear(x, q)
    check(y, x.double() @ v.t(), K * 2.0 ** -24 * (x.double().abs() @ v.abs().t()))
    check(mx4_linear_backward(g, q), g.double() @ v, N * 2.0 ** -24 * (g.double().abs() @ v.abs()))


def _quiet():
    from contextlib import nullcontext
    return nullcontext()


def test_linear_many_rounds_and_split_tails():
    """Sizes whose tiles take several rounds of the CTA pairs, and whose last round is cut along K in 2 to 4 parts."""
    for T, K, N in ((4096, 320, 4096), (5000, 192, 5120), (2048, 1024, 3584), (512, 4096, 4096), (2304, 640, 2560)):
        x, g = rand(T, K, seed=11), rand(T, N, seed=12)
        q = quantize_weight(rand(N, K, seed=13, scale=K ** -0.5))
        v = q.dequantize().float()
        y, gx = mx4_linear(x, q), mx4_linear_backward(g, q)
        rows = torch.arange(0, T, 37, device=DEV)
        check(y[rows], x[rows].double() @ v.double().t(),
              K * 2.0 ** -24 * (x[rows].double().abs() @ v.double().abs().t()))
        check(gx[rows], g[rows].double() @ v.double(), N * 2.0 ** -24 * (g[rows].double().abs() @ v.double().abs()))
    assert nat.device_error() == 0


@pytest.mark.parametrize("T", [1, 20, 50, 100, 250, 600])
def test_codes_that_come_late(T):
    """The weight from memory, not from L2, many K blocks: loads arrive late and out of order."""
    K, N = 4096, 1024
    x, g = rand(T, K, seed=80), rand(T, N, seed=81)
    q = quantize_weight(rand(N, K, seed=82, scale=K ** -0.5))
    v = q.dequantize().double()
    y, gx = mx4_linear(x, q), mx4_linear_backward(g, q)
    check(y, x.double() @ v.t(), K * 2.0 ** -24 * (x.double().abs() @ v.abs().t()))
    check(gx, g.double() @ v, N * 2.0 ** -24 * (g.double().abs() @ v.abs()))
    flush = torch.empty(256 << 20, dtype=torch.uint8, device=DEV)
    for _ in range(20):
        flush.fill_(0)
        assert torch.equal(mx4_linear(x, q), y)
        flush.fill_(1)
        assert torch.equal(mx4_linear_backward(g, q), gx)
    assert nat.device_error() == 0


def test_linear_strided_misaligned_and_empty():
    q = quantize_weight(rand(256, 512, seed=14))
    x = rand(40, 1024, seed=15)
    ref = mx4_linear(x[:, :512].contiguous(), q)
    assert torch.equal(mx4_linear(x[:, :512], q), ref)
    assert torch.equal(mx4_linear(x[:, :512].t().contiguous().t(), q), ref)
    flat = torch.zeros(40 * 512 + 1, dtype=BF16, device=DEV)
    flat[1:] = x[:, :512].reshape(-1)
    assert torch.equal(mx4_linear(flat[1:].view(40, 512), q), ref)
    assert mx4_linear(x[:0, :512], q).shape == (0, 256)
    assert mx4_linear_backward(x[:0, :256], q).shape == (0, 512)
    one = mx4_linear(x[3:4, :512], q)  # one row of a strided matrix
    check(one, x[3:4, :512].double() @ q.dequantize().double().t(),
          512 * 2.0 ** -24 * (x[3:4, :512].double().abs() @ q.dequantize().double().abs().t()))


def test_values_that_are_not_finite_stay_in_their_rows():
    x, w = rand(70, 256, seed=16), rand(304, 256, seed=17)
    w[37, 100] = float("nan")
    x[11, 3] = float("inf")
    y = mx4_linear(x, quantize_weight(w))
    nan = torch.isnan(y)
    assert nan[:, 37].all() and not torch.isfinite(y[11]).any()
    keep = torch.ones(70, dtype=torch.bool, device=DEV)
    keep[11] = False
    assert torch.isfinite(y[keep][:, torch.arange(304, device=DEV) != 37]).all()
    g = rand(70, 304, seed=18)
    gx = mx4_linear_backward(g, quantize_weight(w))
    assert torch.isnan(gx[:, 96:128]).all() and torch.isfinite(gx[:, :96]).all() and torch.isfinite(gx[:, 128:]).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scales_far_from_one(dtype):
    """Blocks of very small and very large scales beside ordinary ones."""
    exps = [-110, -60, -20, 0, 8, 30, 100] if dtype == BF16 else [-22, -14, -8, 0, 4, 8]
    K, N = 256, 64 * len(exps)
    w = rand(N, K, seed=19, dtype=torch.float32)
    w *= torch.tensor([2.0 ** e for e in exps], device=DEV).repeat_interleave(64)[:, None]
    q = quantize_weight(w.to(dtype))
    v = q.dequantize().double()
    x = rand(20, K, seed=20, scale=2.0 ** -6, dtype=dtype)
    ref, mag = x.double() @ v.t(), x.double().abs() @ v.abs().t()
    got = mx4_linear(x, q)
    fits = ref.abs() < torch.finfo(dtype).max / 2
    check(torch.where(fits, got, torch.zeros_like(got)), torch.where(fits, ref, 0.0),
          K * 2.0 ** -24 * mag + 2.0 ** -126)  # float32 sums below its normal range may lose the last 2^-149 steps


# ------------------------------------------------------------------------------------------- the fused ops over it
def adapters_of(K, N, ranks, dtype, seed=30):
    a = {i: rand(r, K, seed=seed + 2 * i, scale=K ** -0.5, dtype=dtype) for i, r in enumerate(ranks)}
    b = {i: rand(N, r, seed=seed + 2 * i + 1, scale=0.1, dtype=dtype) for i, r in enumerate(ranks)}
    return a, b, {i: AdapterSpec(i, r, 8.0, K, N) for i, r in enumerate(ranks)}


def same_as_dense(T, K, N, ranks, cuts, dtype):
    """Over a weight in 4 bits the fused ops give what they give over its dense values: the same bits of dA and dB (the
    same launches), y and grad_x up to the order of their sums, which a tile split along K may change."""
    q = quantize_weight(rand(N, K, seed=21, scale=K ** -0.5, dtype=dtype))
    dense = q.dequantize()
    x, g = rand(T, K, seed=22, dtype=dtype), rand(T, N, seed=23, dtype=dtype)
    a, b, specs = adapters_of(K, N, ranks, dtype)
    ends = list(cuts) + [T]
    routing = TileRoutingConfig(128, [TileRoute(lo, hi, i % len(ranks)) for i, (lo, hi) in
                                      enumerate(zip([0] + list(cuts), ends))])
    y = b200_ops.fused_lora_forward(x, q, a, b, specs, routing)
    gx, ga, gb = b200_ops.fused_lora_backward(g, x, q, a, b, specs, routing)
    b200_ops.clear_weight_cache()
    y0 = b200_ops.fused_lora_forward(x, dense, a, b, specs, routing)
    gx0, ga0, gb0 = b200_ops.fused_lora_backward(g, x, dense, a, b, specs, routing)
    for got, ref, left, right, n in ((y, y0, x, dense.t(), K), (gx, gx0, g, dense, N)):
        # each is off by its sum's error and half a step; the adapters' part, at most as large here, is summed with it
        mag = left.double().abs() @ right.double().abs() + ref.double().abs()
        tol = torch.finfo(dtype).eps * ref.double().abs() + 2 * (n + 64) * 2.0 ** -24 * 2 * mag
        assert ((got.double() - ref.double()).abs() <= tol + torch.finfo(dtype).smallest_normal).all()
    assert ga.keys() == ga0.keys() and all(torch.equal(ga[i], ga0[i]) and torch.equal(gb[i], gb0[i]) for i in ga)
    assert nat.device_error() == 0
    return y, x, dense, a, b, specs, routing


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,K,N,ranks,cuts", [
    (1, 64, 64, [4], []), (130, 256, 320, [8, 16], [60]), (515, 512, 1024, [8, 33, 64], [3, 200, 401]),
    (1024, 1024, 768, [16] * 6, [100, 128, 500, 512, 900]), (300, 200, 136, [100, 16], [129])])
def test_fused_ops(T, K, N, ranks, cuts, dtype):
    y, x, dense, a, b, specs, routing = same_as_dense(T, K, N, ranks, cuts, dtype)
    ref = x.double() @ dense.double().t()
    mag = x.double().abs() @ dense.double().abs().t()
    bound = (K + max(ranks)) * 2.0 ** -24 * mag
    for r in routing.routes:
        s = slice(r.row_start, r.row_end)
        i, sc = r.adapter_id, specs[r.adapter_id].scaling
        low = sc * x[s].double() @ a[i].double().t()
        ref[s] += low @ b[i].double().t()
        # S is rounded to the type before the second product
        bound[s] += (torch.finfo(dtype).eps / 2 + (K + ranks[i]) * 2.0 ** -24) * (
            (sc * x[s].double().abs() @ a[i].double().abs().t()) @ b[i].double().abs().t())
    check(y, ref, bound)


def test_fused_ops_co_scheduled_modes():
    """Every way the routed shrink is scheduled gives the dense op's bits of the same mode."""
    try:
        for mode in (1, 2, 0):
            nat.check(nat.lib().lf_set_co_scheduling(mode), "mode")
            same_as_dense(4096, 256, 4096, [16] * 9, [i * 455 for i in range(1, 9)], BF16)
    finally:
        nat.lib().lf_set_co_scheduling(1)


def test_fused_ops_odd_sizes():
    same_as_dense(40, 100, 60, [8], [], BF16)


def test_coordinator():
    K, N = 256, 384
    q = quantize_weight(rand(N, K, seed=24))
    a, b, specs = adapters_of(K, N, [8, 16], BF16)
    reqs = [Request(0, 0, 20), Request(1, 1, 150), Request(2, 0, 7)]
    xs = {r.request_id: rand(r.num_rows, K, seed=25 + r.request_id) for r in reqs}
    got = Coordinator(q, specs, a, b).run_batch(reqs, xs)
    ref = Coordinator(q.dequantize(), specs, a, b).run_batch(reqs, xs)
    assert got.keys() == ref.keys() and all(torch.equal(got[i], ref[i]) for i in got)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,K,N", [(1, 256, 256), (5, 328, 136), (64, 1024, 4096), (200, 512, 512), (300, 1024, 768),
                                   (700, 256, 1024), (9000, 128, 256)])
def test_rows(T, K, N, dtype):
    q = quantize_weight(rand(N, K, seed=40, scale=K ** -0.5, dtype=dtype))
    bank = AdapterBank(5, 32, K, N, dtype)
    a, b, _ = adapters_of(K, N, [8, 32, 16, 20], dtype)
    for i in a:
        bank.load(i, a[i], b[i], 0.5 + i)
    gen = torch.Generator(device=DEV).manual_seed(41)
    slot = torch.randint(-1, 5, (T,), generator=gen, device=DEV)
    x = rand(T, K, seed=42, dtype=dtype)
    y = fused_lora_forward_rows(x, q, bank, slot)
    v = q.dequantize().double()
    ref, bound = x.double() @ v.t(), K * 2.0 ** -24 * (x.double().abs() @ v.abs().t())
    for i in a:
        at = (slot == i).nonzero().view(-1)
        s = (0.5 + i) * x[at].double() @ a[i].double().t()
        ref[at] += s @ b[i].double().t()
        # S keeps 2^-16, its sums and products float32's error
        bound[at] += (2.0 ** -15 + (K + 32) * 2.0 ** -23) * (
            ((0.5 + i) * x[at].double().abs() @ a[i].double().abs().t()) @ b[i].double().abs().t())
    check(y, ref, bound)
    out = torch.empty_like(y)
    assert fused_lora_forward_rows(x, q, bank, slot.int(), out=out) is out and torch.equal(out, y)
    assert nat.device_error() == 0


def test_rows_odd_sizes_and_misaligned_output():
    q = quantize_weight(rand(60, 100, seed=43))
    bank = AdapterBank(1, 8, 100, 60)
    x, slot = rand(9, 100, seed=44), torch.full((9,), -1, device=DEV)
    ref = fused_lora_forward_rows(x, q.dequantize(), bank, slot)
    assert torch.equal(fused_lora_forward_rows(x, q, bank, slot), ref)
    q, bank = quantize_weight(rand(64, 128, seed=45)), AdapterBank(1, 8, 128, 64)
    x = rand(9, 128, seed=46)
    out = torch.empty(9 * 64 + 1, dtype=BF16, device=DEV)[1:].view(9, 64)
    y = fused_lora_forward_rows(x, q, bank, slot, out=out)
    v = q.dequantize().double()
    check(y, x.double() @ v.t(), 128 * 2.0 ** -24 * (x.double().abs() @ v.abs().t()))


# ------------------------------------------------------------------------------------------- streams, graphs, refusals
def test_another_stream_and_a_captured_graph():
    q = quantize_weight(rand(512, 256, seed=50, scale=1 / 16))
    x = rand(300, 256, seed=51)
    ref = mx4_linear(x, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = mx4_linear(x, q)
        w = quantize_weight(q.dequantize()).dequantize()
    side.synchronize()
    assert torch.equal(y, ref) and torch.isfinite(w).all()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = mx4_linear(x, q)
            back = mx4_linear_backward(out, q)
        graphs.append((gr, out, back))
    for n in range(6):  # replays follow what x holds
        x.copy_(rand(300, 256, seed=52 + n))
        ref, refb = mx4_linear(x, q), mx4_linear_backward(mx4_linear(x, q), q)
        for gr, out, back in graphs + graphs:
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ref) and torch.equal(back, refb)
    assert nat.device_error() == 0


@pytest.mark.parametrize("mx4", [False, True])
def test_captured_fused_ops_follow_their_inputs(mx4):
    """Sizes whose launches wait for parts of themselves: co-scheduled shrink, split tails, slots cut into parts."""
    T, K, N = 4096, 512, 4096
    w = quantize_weight(rand(N, K, seed=70, scale=K ** -0.5))
    w = w if mx4 else w.dequantize()
    x, g = rand(T, K, seed=71), rand(T, N, seed=72)
    a, b, specs = adapters_of(K, N, [16, 8, 16], BF16)
    routing = TileRoutingConfig(128, [TileRoute(0, 2500, 0), TileRoute(2500, 2600, 1), TileRoute(2600, T, 2)])

    def step():
        y = b200_ops.fused_lora_forward(x, w, a, b, specs, routing)
        return y, b200_ops.fused_lora_backward(g, x, w, a, b, specs, routing)

    step()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y, (gx, ga, gb) = step()  # (its packed adapters and tables live in the caches, which stay as they are)
    for n in range(4):
        x.copy_(rand(T, K, seed=73 + 2 * n))
        g.copy_(rand(T, N, seed=74 + 2 * n))
        for _ in range(2):
            gr.replay()
            torch.cuda.synchronize()
            ry, (rgx, rga, rgb) = step()
            assert torch.equal(y, ry) and torch.equal(gx, rgx)
            for i in rga:
                assert torch.equal(ga[i], rga[i]) and torch.equal(gb[i], rgb[i])
    assert nat.device_error() == 0


def test_a_wait_that_runs_out_reports_and_the_next_call_is_right():
    """The co-scheduled launch over a weight in 4 bits waits for a shrink that never reports (the test hook)."""
    T, K, N = 1024, 512, 768
    q = quantize_weight(rand(N, K, seed=90, scale=K ** -0.5))
    x = rand(T, K, seed=91)
    a, b, specs = adapters_of(K, N, [16, 8], BF16)
    routing = TileRoutingConfig(128, [TileRoute(0, 600, 0), TileRoute(600, T, 1)])
    y = b200_ops.fused_lora_forward(x, q, a, b, specs, routing)
    if b200_ops.last_launch_count() != 1:
        pytest.skip("the shrink does not run inside the GEMM launch on this device")
    assert nat.device_error() == 0
    nat.set_wait_limit(50_000_000)
    try:
        nat.check(nat.lib().lf_inject_stale_ready(1), "lf_inject_stale_ready")
        b200_ops.fused_lora_forward(x, q, a, b, specs, routing)
        assert nat.device_error() in (nat.ERR_TIMEOUT_FULL, nat.ERR_TIMEOUT_EMPTY, nat.ERR_TIMEOUT_ACC,
                                      nat.ERR_TIMEOUT_DRAIN, nat.ERR_TIMEOUT_FLAG)
    finally:
        nat.check(nat.lib().lf_inject_stale_ready(0), "lf_inject_stale_ready")
        nat.set_wait_limit(0)
    assert torch.equal(b200_ops.fused_lora_forward(x, q, a, b, specs, routing), y)
    assert nat.device_error() == 0


def test_random_sizes():
    rng = np.random.default_rng(92)
    for i in range(40):
        T, K, N = int(2 ** rng.uniform(0, 11)), 8 * int(2 ** rng.uniform(0, 8)), 8 * int(2 ** rng.uniform(0, 8))
        dtype = BF16 if i % 2 else F16
        q = quantize_weight(rand(N, K, seed=93 + i, scale=K ** -0.5, dtype=dtype))
        v = q.dequantize().double()
        x, g = rand(T, K, seed=200 + i, dtype=dtype), rand(T, N, seed=300 + i, dtype=dtype)
        check(mx4_linear(x, q), x.double() @ v.t(), K * 2.0 ** -24 * (x.double().abs() @ v.abs().t()))
        check(mx4_linear_backward(g, q), g.double() @ v, N * 2.0 ** -24 * (g.double().abs() @ v.abs()))
    assert nat.device_error() == 0


def test_two_streams_at_once():
    """Products of several sizes side by side give what each gives alone."""
    qs = [quantize_weight(rand(n, 512, seed=95 + n)) for n in (1024, 264)]
    xs = [rand(t, 512, seed=96 + t) for t in (900, 40)]
    alone = [mx4_linear(x, q) for x, q in zip(xs, qs)]
    streams = [torch.cuda.Stream() for _ in qs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(mx4_linear(xs[i], qs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, alone[i]) for i in range(2) for y in got[i])


def test_refusals():
    q = quantize_weight(rand(64, 128, seed=60))
    x = rand(4, 128, seed=61)
    with pytest.raises(ValueError, match="dtype"):
        mx4_linear(x.half(), q)
    with pytest.raises(ValueError, match="shape"):
        mx4_linear(x[:, :64], q)
    with pytest.raises(ValueError, match="shape"):
        mx4_linear(x[0], q)
    with pytest.raises(ValueError, match="CUDA"):
        mx4_linear(x.cpu(), q)
    with pytest.raises(ValueError, match="MX4Weight"):
        mx4_linear(x, q.dequantize())
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        quantize_weight(torch.zeros(4, 4, device=DEV))
    with pytest.raises(ValueError, match="2-D"):
        quantize_weight(torch.zeros(4, 0, dtype=BF16, device=DEV))
    with pytest.raises(ValueError, match="uint8"):
        MX4Weight(q.data[:-1], 64, 128, BF16)
    a, b, specs = adapters_of(128, 64, [8], BF16)
    routing = TileRoutingConfig(128, [TileRoute(0, 4, 0)])
    with pytest.raises(ValueError, match="dtype"):
        b200_ops.fused_lora_forward(x.float(), q, a, b, specs, routing)
    with pytest.raises(ValueError, match="does not match"):
        b200_ops.fused_lora_forward(x, quantize_weight(rand(64, 256)), a, b, specs, routing)
    with pytest.raises(ValueError, match="dense"):
        b200_ops.prepare_forward(x, q, a, b, specs, routing)
    with pytest.raises(ValueError, match="dense"):
        b200_ops.prepare_backward(rand(4, 64), x, q, a, b, specs, routing)
    with pytest.raises(ValueError, match="dense"):
        b200_ops.fused_lora_forward_host(x.cpu(), q, a, b, specs, routing)
    bank = AdapterBank(1, 8, 128, 64)
    slot = torch.zeros(4, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="share one"):
        fused_lora_forward_rows(x, quantize_weight(rand(64, 128).half()), bank, slot)
    with pytest.raises(ValueError, match="do not match"):
        fused_lora_forward_rows(x, quantize_weight(rand(64, 256)), bank, slot)
    with pytest.raises(ValueError):  # an output that lies in the weight
        out = q.data[:4 * 64 * 2].view(BF16).view(4, 64)
        fused_lora_forward_rows(x, q, bank, slot, out=out)
