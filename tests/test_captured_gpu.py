"""Calls captured into CUDA graphs: what they may take from eager calls, and eager calls from them."""

import gc
import time
import weakref

import pytest
import torch

from lorafusion_b200 import _native as nat
from lorafusion_b200 import b200_ops as ops
from lorafusion_b200.config import AdapterDropout, AdapterSpec, TileRoute, TileRoutingConfig
from lorafusion_b200.quant import quantize_weight

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def rand(*shape, seed=0, scale=1.0, dtype=BF16):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


class Problem:
    def __init__(self, mx4=False, rate=0.0, T=300, K=256, N=192, seed=0, alpha=16.0):
        self.x, self.g = rand(T, K, seed=seed + 1), rand(T, N, seed=seed + 2)
        w = rand(N, K, seed=seed + 3, scale=K ** -0.5)
        self.w = quantize_weight(w) if mx4 else w
        self.a = {i: rand(r, K, seed=seed + 4 + i, scale=K ** -0.5) for i, r in enumerate((16, 8))}
        self.b = {i: rand(N, r, seed=seed + 6 + i, scale=0.2) for i, r in enumerate((16, 8))}
        self.specs = {i: AdapterSpec(i, r, alpha if i == 0 else 16.0, K, N) for i, r in enumerate((16, 8))}
        self.routing = TileRoutingConfig(128, [TileRoute(0, 100, 0), TileRoute(100, T, 1)])
        self.kw = {"dropout": AdapterDropout(rate, 5, 7)} if rate else {}

    def forward(self, **kw):
        return ops.fused_lora_forward(self.x, self.w, self.a, self.b, self.specs, self.routing, **{**self.kw, **kw})

    def backward(self, **kw):
        return ops.fused_lora_backward(self.g, self.x, self.w, self.a, self.b, self.specs, self.routing, **{**self.kw, **kw})

    def fresh(self):
        """The backward on its own, no forward's S at hand."""
        ops._SAVED_SF.clear()
        return self.backward()


def captured(call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


def same(got, want):
    for x, y in zip(got, want):
        if isinstance(x, dict):
            assert x.keys() == y.keys() and all(torch.equal(x[i], y[i]) for i in y)
        else:
            assert torch.equal(x, y)


ALL = [(False, 0.0), (False, 0.3), (True, 0.0), (True, 0.3)]


@pytest.mark.parametrize("mx4,rate", ALL)
def test_a_captured_backward_takes_nothing_from_an_eager_forward(mx4, rate):
    """Its replays find another x than that forward did."""
    p = Problem(mx4, rate)
    p.forward(), p.backward()
    graph, out = captured(p.backward)
    for n in range(2):
        p.x.copy_(rand(*p.x.shape, seed=20 + n))
        want = p.fresh()
        graph.replay()
        torch.cuda.synchronize()
        same(out, want)
    assert nat.device_error() == 0


@pytest.mark.parametrize("mx4,rate", ALL)
def test_an_eager_backward_takes_nothing_from_a_captured_forward(mx4, rate):
    """A capture runs nothing, and replays run whenever they are launched."""
    p = Problem(mx4, rate)
    p.forward(), p.backward()
    want = p.fresh()
    captured(p.forward)
    same(p.backward(), want)
    # nor does another capture
    one, _ = captured(p.forward)
    two, out = captured(p.backward)
    two.replay()
    torch.cuda.synchronize()
    same(out, want)
    assert nat.device_error() == 0


@pytest.mark.parametrize("mx4,rate", ALL)
def test_forward_and_backward_of_one_capture(mx4, rate):
    p = Problem(mx4, rate)
    p.forward(), p.backward()
    graph, (y, back) = captured(lambda: (p.forward(), p.backward()))
    for n in range(2):
        p.x.copy_(rand(*p.x.shape, seed=30 + n))
        wy, want = p.forward(), p.backward()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, wy)
        same(back, want)
    assert nat.device_error() == 0


@pytest.mark.parametrize("mx4,rate", ALL)
def test_nothing_is_built_within_a_capture(mx4, rate):
    """What a capture would build no later call could use: tables, slabs, a converted weight."""
    p = Problem(mx4, rate, seed=50)
    ops.clear_weight_cache()
    for before, call in ((None, p.forward), (p.forward, p.backward)):
        if before is not None:
            before()
        with pytest.raises(RuntimeError, match="once before"):
            captured(call)
    torch.cuda.synchronize()
    want = p.fresh()
    y = p.forward()
    same(p.backward(), want)
    if not mx4 and not rate:
        wide = p.w.float()
        with pytest.raises(RuntimeError, match="copy of base_weight"):
            captured(lambda: ops.fused_lora_forward(p.x, wide, p.a, p.b, p.specs, p.routing))
        torch.cuda.synchronize()
        assert torch.equal(ops.fused_lora_forward(p.x, wide, p.a, p.b, p.specs, p.routing), y)
        for prepare in (lambda: ops.prepare_forward(p.x, p.w, p.a, p.b, p.specs, TileRoutingConfig(128, [TileRoute(0, 300, 1)])),):
            with pytest.raises(RuntimeError, match="once before"):
                captured(prepare)
    assert nat.device_error() == 0


def test_a_call_with_peer_is_not_captured():
    p = Problem()
    p.forward(), p.backward()

    class Peer:
        """Never reached."""

    with pytest.raises(RuntimeError, match="peer"):
        captured(lambda: p.backward(peer=Peer()))
    torch.cuda.synchronize()


def test_nine_rates_of_an_adapter_whose_factor_stays_zero():
    """With alpha = 0 its factor is 0 whatever its rate: calls of other rates share all but the thresholds, and push
    nothing out that a captured call reads."""
    p = Problem(alpha=0.0)

    def drop(n):
        return AdapterDropout({0: n / 16, 1: 0.25}, 11, 3)

    p.forward(dropout=drop(1)), p.backward(dropout=drop(1))
    fw, y = captured(lambda: p.forward(dropout=drop(1)))
    bw, back = captured(lambda: p.backward(dropout=drop(1)))
    for n in range(2, 16):
        p.forward(dropout=drop(n)), p.backward(dropout=drop(n))
        torch.full((4096,), -1, dtype=torch.int32, device=DEV)
    filler = [torch.full((n,), -1, dtype=torch.int32, device=DEV) for n in (1, 2, 64, 128, 500, 512, 1024) for _ in range(64)]
    want_y, want = p.forward(dropout=drop(1)), p.backward(dropout=drop(1))
    fw.replay()
    bw.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want_y)
    same(back, want)
    del filler
    # adapter 1's rate is 1/4 whatever adapter 0's is
    for n in (1, 9):
        assert torch.equal(p.forward(dropout=drop(n))[100:], want_y[100:])
    assert nat.device_error() == 0


def busy(stream, ms=200):
    """Work of some length on the stream; an event behind it."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(int(ms * 1e6 * 1.9))
        event = torch.cuda.Event()
        event.record(stream)
    return event


@pytest.mark.parametrize("mx4", [False, True])
def test_a_new_routing_does_not_wait_for_the_gpu(mx4):
    """A trainer packs other rows every step: its calls enqueue behind what is queued."""
    p = Problem(mx4, 0.3)
    p.forward(), p.backward()
    for n in range(4):  # what the first new routing allocates is cached from here on
        p.routing = TileRoutingConfig(128, [TileRoute(0, 110 + n, 0), TileRoute(110 + n, 300, 1)])
        p.forward(), p.backward()
    torch.cuda.synchronize()
    done = busy(torch.cuda.current_stream())
    for n in range(2):
        p.routing = TileRoutingConfig(128, [TileRoute(0, 120 + n, 0), TileRoute(120 + n, 300, 1)])
        y, back = p.forward(), p.backward()
    assert not done.query()
    torch.cuda.synchronize()
    want_y, want = p.forward(), p.fresh()
    assert torch.equal(y, want_y)
    same(back, want)


@pytest.mark.parametrize("mx4,rate", ALL)
def test_tables_and_slabs_made_on_a_stream_that_is_behind(mx4, rate):
    """The first call's tables and slabs are still to be written when a call on another stream takes them from the caches,
    and the caches drop them before that has run."""
    p = Problem(mx4, rate, seed=60)
    want_y, want = p.forward(), p.fresh()
    torch.cuda.synchronize()
    ops.clear_weight_cache()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    done = busy(first)
    with torch.cuda.stream(first):
        p.forward(), p.fresh()
    with torch.cuda.stream(second):
        y, back = p.forward(), p.fresh()
    ops.clear_weight_cache()
    with torch.cuda.stream(first):
        filler = [torch.full((n,), -1, dtype=torch.int32, device=DEV) for n in (64, 128, 500, 512, 4096, 1 << 16) for _ in range(16)]
    assert not done.query()
    torch.cuda.synchronize()
    assert torch.equal(y, want_y)
    same(back, want)
    del filler
    assert nat.device_error() == 0


def gone(count=0, seconds=20.0):
    """Waits until captures are let go of (CUDA tells from a thread of its own)."""
    end = time.monotonic() + seconds
    while len(ops._CAPTURED) > count and time.monotonic() < end:
        time.sleep(0.01)
        ops._drop_ended()
    return len(ops._CAPTURED)


@pytest.mark.parametrize("mx4", [False, True])
def test_a_capture_holds_what_it_reads_as_long_as_its_graph_lives(mx4):
    """Once for the graph, however many calls are in it, and nothing of a graph that is gone."""
    gc.collect()
    torch.cuda.synchronize()
    before = gone()
    assert before == 0
    p = Problem(mx4, 0.3, seed=70)
    p.forward(), p.backward()
    want_y, want = p.forward(), p.fresh()
    graph, (y, back) = captured(lambda: [(p.forward(), p.backward()) for _ in range(6)][-1])
    held, = ops._CAPTURED.values()
    # one plan, one entry of slabs, one weight
    assert len(held) == 3
    ref = weakref.ref(next(v for v in held.values() if isinstance(v, torch.Tensor)))
    # dropped caches, and other calls over the same memory, do not touch what it reads
    ops.clear_weight_cache()
    p.w = quantize_weight(rand(192, 256, seed=99)) if mx4 else rand(192, 256, seed=99)
    p.a, p.b = {i: t * 2 for i, t in p.a.items()}, {i: t * 2 for i, t in p.b.items()}
    for n in range(20):
        Problem(mx4, 0.2, T=140 + n, seed=100 + n).forward()
    assert ref() is not None
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want_y)
    same(back, want)
    del held, y, back
    graph.replay()
    graph.reset()
    assert gone() == 0 and ref() is None
    assert not any(v[-1] for v in ops._SAVED_SF.values())
    assert nat.device_error() == 0


def test_many_captures_leave_nothing_behind():
    p = Problem(True, 0.3, seed=80)
    p.forward(), p.backward()
    for _ in range(12):
        captured(lambda: (p.forward(), p.backward()))
    gc.collect()
    torch.cuda.synchronize()
    assert gone() == 0
    # a capture that fails is let go of as well
    other = Problem(True, 0.3, T=140, seed=81)
    with pytest.raises(RuntimeError, match="once before"):
        captured(lambda: (p.forward(), other.forward()))
    gc.collect()
    torch.cuda.synchronize()
    assert gone() == 0
