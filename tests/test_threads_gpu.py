"""Calls of several threads at once, each on a stream of its own."""

import threading

import pytest
import torch

from lorafusion_b200 import _native as nat
from lorafusion_b200 import b200_ops as ops
from lorafusion_b200.config import AdapterDropout, AdapterSpec, TileRoute, TileRoutingConfig
from lorafusion_b200.quant import quantize_weight

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(*shape, seed=0, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(torch.bfloat16)


def test_threads_that_share_adapters():
    """The same adapters, weights and routings from four threads, new activations every time: no call fails, and each
    result is what the call gives alone."""
    K, N, T = 256, 320, 200
    w = rand(N, K, seed=1, scale=1 / 16)
    bases = [w, quantize_weight(w)]
    a = {i: rand(r, K, seed=2 + i, scale=1 / 16) for i, r in enumerate((16, 8))}
    b = {i: rand(N, r, seed=4 + i, scale=0.1) for i, r in enumerate((16, 8))}
    specs = {i: AdapterSpec(i, r, 16.0, K, N) for i, r in enumerate((16, 8))}
    routings = [TileRoutingConfig(128, [TileRoute(0, n, 0), TileRoute(n, T, 1)]) for n in (10, 100, 128)]
    x, g = rand(T, K, seed=8), rand(T, N, seed=9)
    cases = [(base, rt, d) for base in bases for rt in routings for d in (None, AdapterDropout(0.25, 3, 4))]

    def step(x, base, rt, d):
        y = ops.fused_lora_forward(x, base, a, b, specs, rt, dropout=d)
        gx, ga, gb = ops.fused_lora_backward(g, x, base, a, b, specs, rt, dropout=d)
        return [y, gx, *ga.values(), *gb.values()]

    want = [step(x.clone(), *c) for c in cases]
    torch.cuda.synchronize()
    ops.clear_weight_cache()
    failed = []

    def work(n):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for i in range(300):
                    k = (5 * n + i) % len(cases)
                    got = step(x.clone(), *cases[k])
                    if i % 100 == 99 and n == 0:
                        ops.clear_weight_cache()
                    if not all(torch.equal(p, q) for p, q in zip(got, want[k])):
                        failed.append((n, i, k))
        except Exception as e:  # noqa: BLE001 - told below
            failed.append((n, repr(e)))

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed[:3]
    assert nat.device_error() == 0
