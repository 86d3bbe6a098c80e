"""The backward's exchange of spanning adapters together with dropout and a weight in 4 bits, on one GPU.

The spanning adapters are held by this rank alone, so its kernel pushes their blocks into both ranks' buffers (both here) and
sums its own: no launch waits for another.  The sums are those of the call without an exchange, bit for bit.
"""

import pytest
import torch

from lorafusion_b200 import _native as nat
from lorafusion_b200 import b200_ops as ops
from lorafusion_b200.config import AdapterDropout, AdapterSpec, TileRoute, TileRoutingConfig
from lorafusion_b200.quant import quantize_weight

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(*shape, seed=0, scale=1.0, dtype=torch.bfloat16):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


class OneHolder:
    """Rank 0 of two, whose other rank holds no row of any adapter."""

    def __init__(self, ranks, K, N):
        self.world, self.rank, self.gen = 2, 0, 0
        self.vslots = [(a, c0, min(64, r - c0)) for a, r in ranks.items() for c0 in range(0, r, 64)]
        self.index = {(a, c0): i for i, (a, c0, _) in enumerate(self.vslots)}
        self.masks = [1] * len(self.vslots)
        self.r_pad_x = 64
        self.blocks = len(self.vslots) * (-(-N // 128) + -(-K // 128))
        need = nat.lib().lf_peer_exchange_bytes(2, self.blocks, 64)
        self.buffers = [torch.zeros(need, dtype=torch.uint8, device=DEV) for _ in range(2)]
        self.ptrs = [t.data_ptr() for t in self.buffers]

    def ensure(self, n_blocks):
        assert n_blocks == self.blocks

    def next_gen(self):
        self.gen += 1
        return self.gen


@pytest.mark.parametrize("rate", [0.0, 0.3])
@pytest.mark.parametrize("mx4", [False, True])
@pytest.mark.parametrize("T", [300, 9400])
def test_with_dropout_and_a_weight_in_4_bits(T, mx4, rate):
    K, N, ranks = 512, 576, {0: 100, 1: 8, 2: 16}
    x, g = rand(T, K, seed=1), rand(T, N, seed=2)
    w = rand(N, K, seed=3, scale=K ** -0.5)
    w = quantize_weight(w) if mx4 else w
    a = {i: rand(r, K, seed=4 + i, scale=K ** -0.5) for i, r in ranks.items()}
    b = {i: rand(N, r, seed=8 + i, scale=0.1) for i, r in ranks.items()}
    specs = {i: AdapterSpec(i, r, 16.0, K, N) for i, r in ranks.items()}
    routing = TileRoutingConfig(128, [TileRoute(0, 130, 0), TileRoute(130, 200, 1), TileRoute(200, T, 2)])
    kw = {"dropout": AdapterDropout(rate, 5, 7)} if rate else {}
    kw["grad_dtype"] = torch.float32
    ops._SAVED_SF.clear()
    gx, ga, gb = ops.fused_lora_backward(g, x, w, a, b, specs, routing, **kw)
    peer = OneHolder({0: 100, 2: 16}, K, N)
    for _ in range(3):  # both halves of the buffers
        px, pa, pb = ops.fused_lora_backward(g, x, w, a, b, specs, routing, peer=peer, **kw)
        torch.cuda.synchronize()
        assert nat.device_error() == 0
        assert torch.equal(px, gx) and pa.keys() == ga.keys()
        for i in ga:
            assert torch.equal(pa[i], ga[i]) and torch.equal(pb[i], gb[i]), i
    assert torch.equal(*peer.buffers) and peer.buffers[0].any()
