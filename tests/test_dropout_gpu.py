"""Dropout in front of the adapters, its mask never stored: forward, backward and refusals against 64-bit arithmetic.

Tolerances.  A result is off by at most half a step of its type, plus: ``n 2^-24`` of the sum of magnitudes for a float32
sum of n products; the rank product S, which the forward on tensor cores rounds to the type (half a step, of S or of its
two halves along K, which share out the reduction) and the backward keeps to 2^-15 (two 16-bit halves; the lower of float16
no finer than 2^-25); in float32 everything is summed in 64 bits and only the factor s / (1 - p) and the result are rounded.
"""

import numpy as np
import pytest
import torch

from oracle.dropout_oracle import kept
from lorafusion_b200 import _native as nat
from lorafusion_b200 import b200_ops
from lorafusion_b200.b200_ops import fused_lora_backward, fused_lora_forward
from lorafusion_b200.config import AdapterDropout, AdapterSpec, TileRoute, TileRoutingConfig
from lorafusion_b200.quant import quantize_weight

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def rand(*shape, seed=0, scale=1.0, dtype=BF16):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


class Problem:
    def __init__(self, T, K, N, ranks, cuts, rates, dtype, seed=5, offset=3, mx4=False):
        self.T, self.K, self.N, self.dtype = T, K, N, dtype
        self.x, self.g = rand(T, K, seed=1, dtype=dtype), rand(T, N, seed=2, dtype=dtype)
        self.w = rand(N, K, seed=3, scale=K ** -0.5, dtype=dtype)
        self.a = {i: rand(r, K, seed=10 + 2 * i, scale=K ** -0.5, dtype=dtype) for i, r in enumerate(ranks)}
        self.b = {i: rand(N, r, seed=11 + 2 * i, scale=0.3, dtype=dtype) for i, r in enumerate(ranks)}
        self.specs = {i: AdapterSpec(i, r, 12.0, K, N) for i, r in enumerate(ranks)}
        ends = list(cuts) + [T]
        self.routing = TileRoutingConfig(128, [TileRoute(lo, hi, i % len(ranks)) for i, (lo, hi) in
                                               enumerate(zip([0] + list(cuts), ends))])
        self.dropout = AdapterDropout(dict(enumerate(rates)), seed, offset)
        self.base = quantize_weight(self.w) if mx4 else self.w
        self.v = (self.base.dequantize() if mx4 else self.w).double()

    def forward(self, **kw):
        return fused_lora_forward(self.x, self.base, self.a, self.b, self.specs, self.routing,
                                  **{"dropout": self.dropout, **kw})

    def backward(self, **kw):
        return fused_lora_backward(self.g, self.x, self.base, self.a, self.b, self.specs, self.routing,
                                   **{"dropout": self.dropout, **kw})

    def mask(self):
        th = np.zeros(self.T, dtype=np.int64)
        for r in self.routing.routes:
            th[r.row_start:r.row_end] = round(self.dropout.rates[r.adapter_id] * 65536)
        return torch.from_numpy(kept(self.T, self.K, th, self.dropout.seed, self.dropout.offset)).to(DEV)

    def reference(self):
        """(value, bound) of y, grad_x and every dA_i, dB_i."""
        one, f32 = 2.0 ** -24, self.dtype == F32
        half = torch.finfo(self.dtype).eps / 2
        m = self.mask()
        x, g = self.x.double(), self.g.double()
        xm = torch.where(m, x, 0.0)
        y, gx = x @ self.v.t(), g @ self.v
        by = torch.zeros_like(y) if f32 else self.K * one * (x.abs() @ self.v.abs().t())
        bgx = torch.zeros_like(gx) if f32 else self.N * one * (g.abs() @ self.v.abs())
        ga, gb, bga, bgb = {}, {}, {}, {}
        for r in self.routing.routes:
            i, s = r.adapter_id, slice(r.row_start, r.row_end)
            t = round(self.dropout.rates[i] * 65536)
            f = self.specs[i].scaling / (1 - t / 65536)
            a, b = self.a[i].double(), self.b[i].double()
            S, G = f * xm[s] @ a.t(), f * g[s] @ b
            mS, mG = f * xm[s].abs() @ a.abs().t(), f * g[s].abs() @ b.abs()
            if f32:
                eS, eG, fwd = 2 * one * mS, 2 * one * mG, 2 * one * mS
                n = 0.0
            else:
                eS = 2.0 ** -15 * S.abs() + self.K * one * mS + 2.0 ** -24
                eG = 2.0 ** -15 * G.abs() + self.N * one * mG + 2.0 ** -24
                # the forward takes S as one rounded number, or as two, of the halves of K (in blocks of 64)
                k = (-(-self.K // 64) + 1) // 2 * 64
                S0, S1 = f * xm[s, :k] @ a[:, :k].t(), f * xm[s, k:] @ a[:, k:].t()
                fwd = half * (S0.abs() + S1.abs()) + self.K * one * mS + torch.finfo(self.dtype).smallest_normal
                n = (a.shape[0] + self.T) * one
            y[s] += S @ b.t()
            by[s] += fwd @ b.abs().t() + n * (S.abs() @ b.abs().t())
            gx[s] += torch.where(m[s], G @ a, 0.0)
            bgx[s] += eG @ a.abs() + n * (G.abs() @ a.abs())
            parts = (G.t() @ xm[s], g[s].t() @ S, eG.t() @ xm[s].abs() + n * (G.abs().t() @ xm[s].abs()),
                     g[s].abs().t() @ eS + n * (g[s].abs().t() @ S.abs()))
            for d, v in zip((ga, gb, bga, bgb), parts):
                d[i] = d[i] + v if i in d else v
        return (y, by), (gx, bgx), {i: (ga[i], bga[i]) for i in ga}, {i: (gb[i], bgb[i]) for i in gb}


def check(got, ref, what):
    value, bound = ref
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * value.abs() + bound * (1 + fi.eps) + fi.smallest_normal * fi.eps
    excess = ((got.double() - value).abs() - tol).max().item()
    assert not torch.isnan(got).any() and excess <= 0, f"{what}: worst excess {excess:.3g}"


def check_all(p):
    y, (gx, ga, gb) = p.forward(), p.backward()
    ry, rgx, rga, rgb = p.reference()
    assert y.dtype == p.dtype and gx.dtype == p.dtype and ga.keys() == rga.keys() == gb.keys()
    check(y, ry, "y")
    check(gx, rgx, "grad_x")
    for i in rga:
        check(ga[i], rga[i], f"dA {i}")
        check(gb[i], rgb[i], f"dB {i}")
    # the same call, the same bits
    assert torch.equal(p.forward(), y)
    again = p.backward()
    assert torch.equal(again[0], gx) and all(torch.equal(again[1][i], ga[i]) and torch.equal(again[2][i], gb[i]) for i in ga)
    assert nat.device_error() == 0


CASES = [  # T, K, N, ranks, cuts, rates
    (1, 64, 64, [4], [], [0.5]),
    (3, 72, 40, [1], [], [0.1]),
    (130, 256, 320, [8, 16], [60], [0.1, 0.0]),
    (300, 200, 136, [100, 16], [129], [0.25, 0.05]),       # an adapter of several virtual slots
    (515, 512, 264, [8, 33, 64], [3, 200, 401], [0.0, 0.9, 65535 / 65536]),
    (700, 136, 1024, [16] * 5, [128, 128, 256, 600], [0.1, 0.2, 0.3, 0.4, 0.5]),  # a route without rows
    (256, 1024, 256, [64], [], [0.05]),
]


@pytest.mark.parametrize("mx4", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,K,N,ranks,cuts,rates", CASES)
def test_tensor_cores(T, K, N, ranks, cuts, rates, dtype, mx4):
    p = Problem(T, K, N, ranks, cuts, rates, dtype, mx4=mx4)
    if dtype == F16 and max(rates) > 63 / 64:  # s / (1 - p) g B is beyond float16 there
        for call in (p.forward, p.backward):
            with pytest.raises(ValueError, match="float16"):
                call()
        return
    check_all(p)


@pytest.mark.parametrize("T,K,N,ranks,cuts,rates", CASES[:5])
def test_float32(T, K, N, ranks, cuts, rates):
    check_all(Problem(T, K, N, ranks, cuts, rates, F32))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,K,N", [(5, 33, 7), (140, 67, 50)])
def test_odd_sizes_on_cuda_cores(T, K, N, dtype):
    check_all(Problem(T, K, N, [3, 8], [T // 2], [0.3, 0.1], dtype))


def test_odd_sizes_over_a_weight_in_4_bits():
    check_all(Problem(20, 100, 60, [8], [], [0.3], BF16, mx4=True))


@pytest.mark.parametrize("seed,offset", [(0, 0), ((1 << 64) - 1, (1 << 64) - 1), (1 << 32, 7), (7, 1 << 32)])
def test_seeds_and_offsets(seed, offset):
    check_all(Problem(40, 80, 64, [8], [], [0.5], BF16, seed=seed, offset=offset))


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_co_scheduling_modes(mode):
    """Sizes whose shrink can share the GEMM's launch, in every mode."""
    try:
        nat.check(nat.lib().lf_set_co_scheduling(mode), "mode")
        p = Problem(4096, 64, 4096, [16] * 4, [1000, 2047, 3001], [0.1, 0.0, 0.3, 0.5], BF16)
        y, (gx, ga, gb) = p.forward(), p.backward()
    finally:
        nat.lib().lf_set_co_scheduling(1)
    ry, rgx, rga, rgb = p.reference()
    check(y, ry, "y")
    check(gx, rgx, "grad_x")
    for i in rga:
        check(ga[i], rga[i], f"dA {i}")
        check(gb[i], rgb[i], f"dB {i}")


@pytest.mark.parametrize("mx4", [False, True])
@pytest.mark.parametrize("mode", [0, 1])
def test_shrinks_beside_one_another(mode, mx4):
    """More row tiles than half of the SMs and K blocks enough to cut: the backward's two shrinks share the GPU (mode 1: its
    GEMM's rounds leave no pairs idle)."""
    try:
        nat.check(nat.lib().lf_set_co_scheduling(mode), "mode")
        check_all(Problem(9400, 512, 576, [64, 20], [4000], [0.1, 0.3], BF16, mx4=mx4))
    finally:
        nat.lib().lf_set_co_scheduling(1)


def test_rows_and_gradients_at_odd_addresses():
    """Views of x and of the gradient that start in the middle of 16 bytes."""
    p = Problem(150, 128, 192, [16], [], [0.2], BF16, mx4=True)
    y, (gx, ga, gb) = p.forward(), p.backward()
    for name in ("x", "g"):
        t = getattr(p, name)
        flat = torch.zeros(t.numel() + 1, dtype=BF16, device=DEV)
        flat[1:] = t.reshape(-1)
        setattr(p, name, flat[1:].view(t.shape))
    assert torch.equal(p.forward(), y)
    again = p.backward()
    assert torch.equal(again[0], gx) and torch.equal(again[1][0], ga[0]) and torch.equal(again[2][0], gb[0])


def test_two_streams_at_once():
    """Calls of different masks, weights and sizes side by side give what each gives alone."""
    ps = [Problem(700, 512, 640, [16, 8], [300], [0.1, 0.4], BF16, seed=i, mx4=bool(i)) for i in range(2)]
    alone = [(p.forward(), p.backward()) for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, (p, s) in enumerate(zip(ps, streams)):
            with torch.cuda.stream(s):
                got[i].append((p.forward(), p.backward()))
    torch.cuda.synchronize()
    for i, calls in enumerate(got):
        for y, (gx, ga, gb) in calls:
            ry, (rgx, rga, rgb) = alone[i]
            assert torch.equal(y, ry) and torch.equal(gx, rgx)
            assert all(torch.equal(ga[k], rga[k]) and torch.equal(gb[k], rgb[k]) for k in rga)
    assert nat.device_error() == 0


def test_under_inference_mode_and_with_leaves():
    """Operands that require gradients, or inference tensors: the same results, no graph."""
    p = Problem(90, 64, 64, [8], [], [0.3], BF16, mx4=True)
    y = p.forward()
    p.x.requires_grad_(True)
    again = p.forward()
    assert torch.equal(again, y) and not again.requires_grad
    with torch.inference_mode():
        assert torch.equal(p.forward(), y)


def test_float32_gradients():
    p = Problem(300, 256, 128, [16, 8], [170], [0.2, 0.1], BF16)
    _, ga, gb = p.backward(grad_dtype=F32)
    _, _, rga, rgb = p.reference()
    for i in rga:
        assert ga[i].dtype == F32
        check(ga[i], rga[i], f"dA {i}")
        check(gb[i], rgb[i], f"dB {i}")


def test_rate_zero_is_no_dropout():
    p = Problem(200, 256, 128, [16, 8], [70], [0.0, 0.0], BF16)
    plain = p.forward(dropout=None)
    b200_ops.clear_weight_cache()
    assert torch.equal(p.forward(), plain)
    for got, ref in zip(p.backward(), p.backward(dropout=None)):
        if isinstance(got, dict):
            assert all(torch.equal(got[i], ref[i]) for i in ref)
        else:
            assert torch.equal(got, ref)


def test_masks_follow_seed_offset_and_position():
    """With x of ones and A = I / B = I, y - x W^T shows the mask itself."""
    K = 256
    x = torch.ones(300, K, device=DEV)
    a, b = {0: torch.eye(K, device=DEV)}, {0: torch.eye(K, device=DEV)}
    specs, routing = {0: AdapterSpec(0, K, float(K), K, K)}, TileRoutingConfig(128, [TileRoute(0, 300, 0)])
    w = torch.zeros(K, K, device=DEV)
    shown = {}
    for seed, offset in ((1, 0), (2, 0), (1, 1), (1, 1 << 40)):
        y = fused_lora_forward(x, w, a, b, specs, routing, dropout=AdapterDropout(0.25, seed, offset))
        m = torch.from_numpy(kept(300, K, [16384] * 300, seed, offset)).to(DEV)
        assert torch.equal(y > 0, m) and torch.allclose(y[m], torch.full_like(y[m], 4 / 3), rtol=1e-6)
        share = m.double().mean().item()
        assert abs(share - 0.75) < 5 * (0.75 * 0.25 / m.numel()) ** 0.5
        shown[seed, offset] = m
    masks = list(shown.values())
    for i in range(len(masks)):
        for j in range(i):
            agree = (masks[i] == masks[j]).double().mean().item()
            assert abs(agree - 0.625) < 5 * (0.625 * 0.375 / masks[i].numel()) ** 0.5


def test_the_backward_knows_no_other_forward():
    """A plain forward on the same x, or one of another offset, leaves nothing that a backward with dropout takes."""
    p = Problem(260, 128, 192, [16], [], [0.4], BF16)
    ref = p.backward()
    p.forward(dropout=None)
    p.forward(dropout=AdapterDropout(0.4, 99, 1))
    for got, want in zip(p.backward(), ref):
        assert torch.equal(got[0], want[0]) if isinstance(got, dict) else torch.equal(got, want)
    plain = p.backward(dropout=None)
    b200_ops.clear_weight_cache()
    assert torch.allclose(p.backward(dropout=None)[0].float(), plain[0].float())


def test_a_dropped_element_is_zero_whatever_it_was():
    p = Problem(50, 64, 64, [8], [], [0.5], BF16)
    m = p.mask()
    p.x[~m] = float("nan")
    _, ga, gb = p.backward()
    assert torch.isfinite(ga[0]).all() and torch.isfinite(gb[0]).all()
    assert torch.isfinite(p.backward()[0]).all()


def test_gradients_against_differences():
    """The loss sum(c * y) along random directions: float32 forwards, sums in 64 bits."""
    p = Problem(20, 40, 24, [4, 6], [9], [0.3, 0.1], F32)
    gx, ga, gb = p.backward()
    c = p.g.double()
    base = (p.x, {**p.a}, {**p.b})
    eps = 2.0 ** -7
    for kind in ("x", "a", "b"):
        for n in range(3):
            d = {"x": rand(20, 40, seed=70 + n, dtype=F32)} if kind == "x" else \
                {i: rand(*t.shape, seed=80 + n + i, dtype=F32) for i, t in (p.a if kind == "a" else p.b).items()}
            side = []
            for sign in (1, -1):
                p.x, p.a, p.b = base[0], {**base[1]}, {**base[2]}
                if kind == "x":
                    p.x = base[0] + sign * eps * d["x"]
                elif kind == "a":
                    p.a = {i: t + sign * eps * d[i] for i, t in base[1].items()}
                else:
                    p.b = {i: t + sign * eps * d[i] for i, t in base[2].items()}
                side.append((c * p.forward().double()).sum().item())
            got = (side[0] - side[1]) / (2 * eps)
            grads = {"x": gx} if kind == "x" else ga if kind == "a" else gb
            want = sum((grads[i].double() * d[i].double()).sum().item() for i in d)
            # y is linear in each of x, A and B, so differences are exact up to rounding: 2^-24 of every y and of the
            # moved operands (whose error of 2^-24 is divided by eps), sums of magnitudes below 1e4 here
            assert abs(got - want) <= 1e4 * 2.0 ** -24 * 4 / eps, (kind, got, want)
    p.x, p.a, p.b = base


def test_a_large_batch():
    """4096 rows, 16 adapters, over a weight in 4 bits."""
    cuts = [i * 256 + 17 * (i % 3) for i in range(1, 16)]
    check_all(Problem(4096, 1024, 512, [16] * 16, cuts, [0.05 * (i % 4) for i in range(16)], BF16, mx4=True))


def test_captured_graphs_and_streams():
    p = Problem(300, 256, 192, [16, 8], [100], [0.2, 0.1], BF16, mx4=True)
    y, back = p.forward(), p.backward()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, back2 = p.forward(), p.backward()
    side.synchronize()
    assert torch.equal(y2, y) and torch.equal(back2[0], back[0])
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = p.forward(), p.backward()
        graphs.append((gr, out))
    for gr, out in graphs + graphs:
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], y) and torch.equal(out[1][0], back[0])
        assert all(torch.equal(out[1][1][i], back[1][i]) and torch.equal(out[1][2][i], back[2][i]) for i in back[1])
    assert nat.device_error() == 0


@pytest.mark.parametrize("mx4,drop", [(True, True), (True, False), (False, True)])
def test_a_captured_call_keeps_what_its_replays_read(mx4, drop):
    """Other routings, rates and adapters push its tables out of the caches; a captured backward does not take what an
    eager forward left."""
    p = Problem(300, 256, 192, [16, 8], [100], [0.2, 0.1], BF16, mx4=mx4)
    kw = {} if drop else {"dropout": None}
    a0, b0 = dict(p.a), dict(p.b)
    p.forward(**kw), p.backward(**kw)
    graphs = []
    for call in (p.forward, p.backward):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = call(**kw)
        graphs.append((gr, out))
    p.x.copy_(rand(300, 256, seed=90))
    y = p.forward(**kw)
    b200_ops._SAVED_SF.clear()
    gx, ga, gb = p.backward(**kw)
    for n in range(300):
        q = Problem(8 + n, 64, 64, [4], [], [n / 1000 + 0.1], BF16)
        q.forward()
        p.a[0], p.b[0] = a0[0] + n, b0[0] + n
        p.forward(**kw)
    (fw, y1), (bw, (gx1, ga1, gb1)) = graphs
    bw.replay()
    fw.replay()
    torch.cuda.synchronize()
    assert torch.equal(y1, y) and torch.equal(gx1, gx)
    assert all(torch.equal(ga1[i], ga[i]) and torch.equal(gb1[i], gb[i]) for i in b0)
    assert nat.device_error() == 0


@pytest.mark.parametrize("mx4,drop", [(True, True), (True, False), (False, True), (False, False)])
def test_a_gemm_that_starts_beside_its_shrink(mx4, drop):
    """As many tiles as CTA pairs, so that none is left for the shrink: eager, on two streams at once and captured."""
    p = Problem(18944, 512, 256, [16, 8, 64, 33], [37, 5000, 5003, 12800], [0.1, 0.0, 0.3, 0.05], BF16, mx4=mx4)
    kw = {} if drop else {"dropout": None}
    if drop:
        check_all(p)

    def step():
        y = p.forward(**kw)
        gx, ga, gb = p.backward(**kw)
        return [y, gx, *ga.values(), *gb.values()]

    b200_ops._SAVED_SF.clear()
    want = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(step())
    torch.cuda.synchronize()
    if mx4 or drop:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        for _ in range(3):
            for t in out:
                t.zero_()
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    for res in got:
        assert all(torch.equal(a, b) for a, b in zip(res, want))
    assert nat.device_error() == 0


@pytest.mark.parametrize("mx4", [False, True])
def test_nothing_is_built_within_a_capture(mx4):
    p = Problem(64, 64, 64, [8], [], [0.5], BF16, mx4=mx4)
    for before, call in ((None, p.forward), (p.forward, p.backward)):
        if before is not None:
            before()
        with pytest.raises(RuntimeError, match="once before"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    torch.cuda.synchronize()
    check_all(p)


@pytest.mark.filterwarnings("ignore::lorafusion_b200.b200_ops.CudaCorePathWarning")
def test_a_weight_at_an_odd_address():
    """CUDA cores, sixteen-bit types: the mask is applied to a copy of x, by vectors and element by element."""
    for K, shift in ((64, 1), (68, 0), (33, 0)):
        p = Problem(70, K, 40, [8, 5], [30], [0.3, 0.0], BF16)
        store = torch.zeros(p.w.numel() + 1, dtype=BF16, device=DEV)
        p.w = p.base = store[shift:shift + p.w.numel()].view_as(p.w).copy_(p.w)
        check_all(p)


def test_empty_batches_and_refusals():
    p = Problem(64, 64, 64, [8], [], [0.5], BF16)
    empty = TileRoutingConfig(128, [])
    y = fused_lora_forward(p.x[:0], p.w, p.a, p.b, p.specs, empty, dropout=p.dropout)
    assert y.shape == (0, 64)
    with pytest.raises(KeyError):
        p.forward(dropout=AdapterDropout({1: 0.5}, 0))
    with pytest.raises(ValueError, match="AdapterDropout"):
        p.forward(dropout=0.5)


@pytest.mark.parametrize("mx4", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("T,K,N,ranks,cuts", [
    (300, 256, 192, [16, 8], [100]), (1030, 200, 1024, [64, 33, 100], [3, 140, 400, 401]),
    (18944, 128, 256, [16, 8], [37, 5000, 12800])])
def test_the_rank_product_enters_the_forward_in_two_halves(T, K, N, ranks, cuts, dtype, mode, mx4):
    """Over a weight of zeros y is S B^T alone.  S is held as hi + lo, each of the type: |S - hi| is at most half a step,
    eps / 2 |S|, and that rounded again leaves (eps / 2)^2 |S| (float16's low half ends at 2^-25), of S or of its two halves
    along K.  Freed memory is full of NaN, so that a zero tile which nothing wrote shows."""
    try:
        nat.check(nat.lib().lf_set_co_scheduling(mode), "mode")
        p = Problem(T, K, N, ranks, cuts, [0.1, 0.0, 0.3][:len(ranks)], dtype)
        p.base = torch.zeros_like(p.w)
        if mx4:
            p.base = quantize_weight(p.base)
        p.forward()
        torch.cuda.empty_cache()
        torch.full((64 << 20,), float("nan"), dtype=dtype, device=DEV)
        y = p.forward()
    finally:
        nat.lib().lf_set_co_scheduling(1)
    one, half = 2.0 ** -24, torch.finfo(dtype).eps / 2
    xm = torch.where(p.mask(), p.x.double(), 0.0)
    ref, bound = torch.zeros(T, N, dtype=torch.float64, device=DEV), torch.zeros(T, N, dtype=torch.float64, device=DEV)
    for r in p.routing.routes:
        i, s = r.adapter_id, slice(r.row_start, r.row_end)
        f = p.specs[i].scaling / (1 - round(p.dropout.rates[i] * 65536) / 65536)
        a, b = p.a[i].double(), p.b[i].double()
        k = (-(-K // 64) + 1) // 2 * 64
        S0, S1 = f * xm[s, :k] @ a[:, :k].t(), f * xm[s, k:] @ a[:, k:].t()
        mag = f * xm[s].abs() @ a.abs().t()
        eS = half * half * (S0.abs() + S1.abs()) + (K + 2) * one * mag + 2 * 2.0 ** -25
        ref[s] = (S0 + S1) @ b.t()
        # (two products a half and rank, summed in float32)
        bound[s] = eS @ b.abs().t() + 4 * a.shape[0] * one * ((S0.abs() + S1.abs()) @ b.abs().t())
    check(y, (ref, bound), "y")
    assert nat.device_error() == 0
