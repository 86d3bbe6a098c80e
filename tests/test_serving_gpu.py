"""Rows with an adapter each (serving.fused_lora_forward_rows) against the formula in 64 bits.

Error bound per element, from the arithmetic: the result is rounded once (half a step of the output
type); sums run in float32 over K products of the base and r products of the adapter, each addition
off by at most 2^-23 of the magnitudes summed (a truncating accumulator); S enters the expand as two
halves of the input type after scaling by its row's largest magnitude, off by 2^-16 (bf16) or
2^-21 (f16) of that magnitude, and is itself a float32 sum over K.
"""

import numpy as np
import pytest
import torch

from lorafusion_b200 import _native as nat
from lorafusion_b200 import b200_ops
from lorafusion_b200.serving import AdapterBank, fused_lora_forward_rows

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
S_HALVES = {BF16: 2.0 ** -16, F16: 2.0 ** -21, F32: 2.0 ** -24}


def make(dtype, T, K, N, ranks, max_rank, seed=0, slots=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x = rnd(T, K).to(dtype)
    w = (rnd(N, K) / K ** 0.5).to(dtype)
    bank = AdapterBank(len(ranks), max_rank, K, N, dtype, "cuda")
    adapters = []
    for i, r in enumerate(ranks):
        a, b, s = (rnd(r, K) / K ** 0.5).to(dtype), (0.1 * rnd(N, r)).to(dtype), 0.5 + 0.25 * i % 3
        if r:
            bank.load(i, a, b, s)
        adapters.append((a, b, s))
    if slots is None:
        slots = torch.randint(-1, len(ranks), (T,), generator=gen, device="cuda", dtype=torch.int32)
    return x, w, bank, adapters, slots


def reference(x, w, adapters, slots):
    """(y, bound on the error) in 64 bits."""
    xd, wd = x.double(), w.double()
    K = x.shape[1]
    y = xd @ wd.T
    size = xd.abs() @ wd.abs().T
    slack = torch.zeros_like(y)
    for i in range(len(adapters)):
        at = (slots == i).nonzero().view(-1)
        if not len(at) or adapters[i][0].shape[0] == 0:
            continue
        a, b, s = adapters[i][0].double(), adapters[i][1].double(), adapters[i][2]
        S = xd[at] @ a.T
        y[at] += s * S @ b.T
        size[at] += abs(s) * S.abs() @ b.T.abs()
        off = S_HALVES[x.dtype] * S.abs().amax(1, keepdim=True) + (K + 32) * 2.0 ** -23 * (xd[at].abs() @ a.T.abs())
        slack[at] += abs(s) * off @ b.T.abs()
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    return y, half * y.abs() + (K + 200) * 2.0 ** -23 * size + 1.01 * slack + tiny


def check(y, x, w, adapters, slots):
    ref, bound = reference(x, w, adapters, slots)
    over = (y.double() - ref).abs() - bound
    assert y.shape == ref.shape and y.dtype == x.dtype
    assert torch.isfinite(y).all()
    assert over.max() <= 0, f"{int((over > 0).sum())} of {over.numel()} over the bound, worst by {over.max():.3g}"


CASES = [  # dtype, T, K, N, ranks, max_rank
    (BF16, 1, 64, 128, [16], 16),
    (BF16, 1, 4096, 4096, [16, 8], 16),
    (F16, 2, 8, 8, [1], 1),
    (BF16, 7, 72, 136, [3, 16, 0, 1], 16),
    (F16, 16, 1000, 520, [16, 5], 20),
    (BF16, 17, 264, 2048, [32] * 5, 32),
    (BF16, 33, 4096, 1024, [64, 8, 33, 17], 64),
    (F16, 64, 520, 776, [128, 100, 1], 128),
    (BF16, 65, 1024, 14336, [16] * 80, 16),
    (BF16, 130, 2048, 264, [8, 16, 32, 64] * 10, 64),
    (F16, 256, 512, 512, [16] * 300, 16),
    (BF16, 257, 328, 392, [48, 20], 48),
    (BF16, 1031, 640, 1288, [16, 40, 64], 64),
    (F16, 300, 1032, 2056, [16, 3, 33, 64, 0], 64),
    (BF16, 700, 520, 1032, [128, 90, 16], 128),
    (F16, 2000, 264, 4104, [16] * 200, 16),
    (BF16, 8500, 72, 264, [8, 24, 16], 32),  # more rows than one chunk
    (F32, 1, 37, 53, [4], 4),
    (F32, 128, 256, 256, [8] * 4, 8),
    (F32, 45, 300, 129, [16, 1, 70], 70),
    (BF16, 19, 37, 61, [5, 2], 8),   # K, N no multiples of 8: CUDA cores
    (F16, 40, 64, 30, [5, 2], 8),
]


@pytest.mark.filterwarnings("ignore::lorafusion_b200.b200_ops.CudaCorePathWarning")
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{str(c[0])[6:]}-{c[1]}x{c[2]}x{c[3]}-r{c[5]}")
def test_rows_against_64_bits(case):
    dtype, T, K, N, ranks, max_rank = case
    x, w, bank, adapters, slots = make(dtype, T, K, N, ranks, max_rank)
    y = fused_lora_forward_rows(x, w, bank, slots)
    if dtype is torch.float32 or K % 8 or N % 8:
        launches = 2
    else:  # per chunk of 8192 rows
        launches = sum(4 if n > (512 if max_rank <= 32 else 256) else 2 for n in [8192] * (T // 8192) + [T % 8192] if n)
    assert b200_ops.last_launch_count() == launches
    check(y, x, w, adapters, slots)
    again = fused_lora_forward_rows(x, w, bank, slots.to(torch.int64))
    assert torch.equal(y, again)  # the same bits on every run, for either index type
    assert nat.device_error() == 0


def test_orders_and_absent_adapters():
    T, K, N = 300, 512, 640
    x, w, bank, adapters, _ = make(BF16, T, K, N, [16, 8, 12], 16)
    sorted_slots = torch.arange(T, device="cuda", dtype=torch.int32) // 100
    y_sorted = fused_lora_forward_rows(x, w, bank, sorted_slots)
    check(y_sorted, x, w, adapters, sorted_slots)
    none = torch.full((T,), -7, device="cuda", dtype=torch.int32)
    base = fused_lora_forward_rows(x, w, bank, none)
    check(base, x, w, adapters, none)
    one = torch.zeros(T, device="cuda", dtype=torch.int32)
    check(fused_lora_forward_rows(x, w, bank, one), x, w, adapters, one)
    bank.unload(1)
    y = fused_lora_forward_rows(x, w, bank, sorted_slots)
    assert torch.equal(y[100:200], base[100:200]) and torch.equal(y[:100], y_sorted[:100])


@pytest.mark.parametrize("dtype, T, ranks, max_rank", [(BF16, 1500, [16] * 700, 16), (F16, 700, [64, 16, 33] * 3, 64),
                                                       (BF16, 1100, [100], 128)])
def test_long_batches_in_any_order(dtype, T, ranks, max_rank):
    """A row's result has the same bits wherever it stands and however often it is computed."""
    K, N = 200, 328
    x, w, bank, adapters, _ = make(dtype, T, K, N, ranks, max_rank)
    slots = torch.arange(T, device="cuda") * 7 % len(ranks)
    slots[::11] = -1
    y = fused_lora_forward_rows(x, w, bank, slots)
    check(y, x, w, adapters, slots)
    for _ in range(3):
        order = torch.randperm(T, device="cuda")
        assert torch.equal(fused_lora_forward_rows(x[order], w, bank, slots[order]), y[order])


@pytest.mark.parametrize("dtype, r", [(BF16, 16), (F16, 32), (BF16, 64), (BF16, 128)])
def test_prompts(dtype, r):
    """Long runs of one adapter, short ones and rows without any, across the tiles of a long batch."""
    lengths = [1, 300, 7, 8, 9, 511, 64, 33, 128, 40, 2, 900]
    slots = torch.cat([torch.full((n,), i % 4 - 1, dtype=torch.int32) for i, n in enumerate(lengths)]).cuda()
    x, w, bank, adapters, slots = make(dtype, len(slots), 776, 1544, [r, r - 3, r // 2], r, slots=slots)
    y = fused_lora_forward_rows(x, w, bank, slots)
    check(y, x, w, adapters, slots)
    order = torch.randperm(len(slots), device="cuda")
    shuffled = fused_lora_forward_rows(x[order].contiguous(), w, bank, slots[order].contiguous())
    check(shuffled, x[order], w, adapters, slots[order])
    assert nat.device_error() == 0


def test_agrees_with_the_packed_forward():
    from lorafusion_b200.config import AdapterSpec, TileRoute, TileRoutingConfig
    T, K, N = 200, 256, 384
    x, w, bank, adapters, _ = make(BF16, T, K, N, [16, 8], 16)
    slots = (torch.arange(T, device="cuda") >= 90).to(torch.int32)
    specs = {i: AdapterSpec(i, a.shape[0], s * a.shape[0], K, N) for i, (a, _, s) in enumerate(adapters)}
    routing = TileRoutingConfig(128, [TileRoute(0, 90, 0), TileRoute(90, T, 1)])
    packed = b200_ops.fused_lora_forward(x, w, {i: a for i, (a, _, _) in enumerate(adapters)},
                                         {i: b for i, (_, b, _) in enumerate(adapters)}, specs, routing)
    rows = fused_lora_forward_rows(x, w, bank, slots)
    check(rows, x, w, adapters, slots)
    torch.testing.assert_close(rows.float(), packed.float(), rtol=2e-2, atol=2e-2)


def test_empty_batch_out_and_strided_rows():
    x, w, bank, adapters, slots = make(BF16, 40, 256, 264, [16, 4], 16)
    assert fused_lora_forward_rows(x[:0], w, bank, slots[:0]).shape == (0, 264)
    out = torch.full((42, 264), 3.0, dtype=BF16, device="cuda")
    y = fused_lora_forward_rows(x, w, bank, slots, out=out[:40])
    assert y.data_ptr() == out.data_ptr() and bool((out[40:] == 3.0).all())  # rows behind the last stay
    check(y, x, w, adapters, slots)
    wide = torch.zeros(40, 264, dtype=BF16, device="cuda")
    for x2 in (wide[:, :256], wide[:, 8:], wide[:, 3:259], torch.zeros(256, 40, dtype=BF16, device="cuda").T,
               torch.zeros(40, 2 * 256, dtype=BF16, device="cuda")[:, ::2], wide.new_zeros(80, 256)[::2]):
        x2.copy_(x)
        assert torch.equal(fused_lora_forward_rows(x2, w, bank, slots), y)
    odd = torch.zeros(40 * 259, dtype=BF16, device="cuda").view(40, 259)[:, :256]  # row pitch no multiple of 8
    odd.copy_(x)
    assert torch.equal(fused_lora_forward_rows(odd, w, bank, slots), y)
    one_row = x[5].expand(40, 256)  # stride 0
    y1 = fused_lora_forward_rows(one_row, w, bank, slots)
    check(y1, one_row.contiguous(), w, adapters, slots)


def test_slots_out_of_range_are_reported():
    x, w, bank, adapters, slots = make(BF16, 24, 128, 128, [16, 16], 16)
    bad = slots.to(torch.int64)
    bad[3], bad[20] = 2, (1 << 32) + 1
    nat.device_error()
    y = fused_lora_forward_rows(x, w, bank, bad)
    assert nat.device_error() == nat.ERR_ROW_SLOT
    as_none = slots.clone()
    as_none[3] = as_none[20] = -1
    check(y, x, w, adapters, as_none)
    assert nat.device_error() == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T", [24, 1500])
def test_values_that_are_not_finite_stay_with_their_rows(dtype, T):
    K, N = 256, 256
    x, w, bank, adapters, _ = make(dtype, T, K, N, [16, 9, 16], 16)
    slots = torch.arange(T, device="cuda", dtype=torch.int32) % 3
    good = fused_lora_forward_rows(x, w, bank, slots)
    bank.load(1, torch.full((9, K), float("nan"), device="cuda"), torch.full((N, 9), float("inf"), device="cuda"), 1.0)
    x[2, 5] = float("inf")
    x[4, 7] = float("nan")
    y = fused_lora_forward_rows(x, w, bank, slots)
    bad = (slots == 1)
    bad[2] = bad[4] = True
    assert torch.equal(y[~bad], good[~bad])
    assert not torch.isfinite(y[bad]).any()


def test_float16_rank_products_beyond_its_range():
    """S far above 65504 and far below float16's smallest value, with results inside the range."""
    T, K, N = 9, 512, 128
    x, w, bank, adapters, _ = make(F16, T, K, N, [16, 16], 16)
    x *= 100
    slots = torch.arange(T, device="cuda", dtype=torch.int32) % 2
    big = (adapters[0][0] * 400, (adapters[0][1] * 1e-3).to(F16), 1.0)
    small = ((adapters[1][0] * 1e-4).to(F16), adapters[1][1], 300.0)
    for i, (a, b, s) in enumerate((big, small)):
        bank.load(i, a, b, s)
    S = x.double() @ big[0].double().T
    assert S.abs().max() > 65504
    y = fused_lora_forward_rows(x, w, bank, slots)
    check(y, x, w, [big, small], slots)


@pytest.mark.parametrize("T", [12, 200, 1100])
def test_captured_call_follows_slots_and_bank(T):
    K, N = 512, 512
    x, w, bank, adapters, slots = make(BF16, T, K, N, [16, 8], 16)
    out = torch.empty(T, N, dtype=BF16, device="cuda")
    fused_lora_forward_rows(x, w, bank, slots, out=out)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    out2 = torch.empty_like(out)
    with torch.cuda.graph(graph):
        fused_lora_forward_rows(x, w, bank, slots, out=out)
    with torch.cuda.graph(other, pool=graph.pool()):
        fused_lora_forward_rows(x, w, bank, slots, out=out2)
    for k in range(3):
        slots.copy_(torch.randint(-1, 2, (T,), dtype=torch.int32))
        a, b, _ = adapters[1]
        adapters[1] = (a * 0.5, b, 1.0 + k)
        bank.load(1, *adapters[1])
        x.copy_(torch.randn(T, K))
        graph.replay()
        other.replay()
        check(out, x, w, adapters, slots)
        assert torch.equal(out, out2)


def test_two_streams_at_once():
    x, w, bank, adapters, slots = make(BF16, 64, 2048, 2048, [16] * 64, 16)
    alone = fused_lora_forward_rows(x, w, bank, slots)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(fused_lora_forward_rows(x, w, bank, slots))
    torch.cuda.synchronize()
    assert all(torch.equal(y, alone) for ys in got for y in ys)


def test_refusals():
    x, w, bank, _, slots = make(BF16, 8, 64, 64, [16], 16)
    bad = [
        dict(x=x[0]), dict(x=x.cpu()), dict(x=x.half()), dict(x=x[:, :56]), dict(w=w[:56]), dict(w=w.float()),
        dict(w=w.T.contiguous().T), dict(w=w.cpu()), dict(slots=slots[:7]), dict(slots=slots.cpu()),
        dict(slots=slots.to(torch.int16)), dict(slots=slots.float()), dict(out=torch.empty(8, 65, device="cuda")),
        dict(out=torch.empty(8, 64, device="cuda")), dict(out=torch.empty(64, 8, dtype=BF16, device="cuda").T),
        dict(out=torch.empty(8, 64, dtype=BF16)), dict(out=x), dict(out=w[8:16]),
        dict(out=bank.lora_a[0, :8]), dict(out=bank.lora_b.view(-1, 64)[4:12]),
    ]
    for b in bad:
        with pytest.raises(ValueError):
            fused_lora_forward_rows(b.get("x", x), b.get("w", w), bank, b.get("slots", slots), out=b.get("out"))
    a, b = torch.zeros(4, 64, device="cuda"), torch.zeros(64, 4, device="cuda")
    for args in ((1, a, b, 1.0), (-1, a, b, 1.0), (0, a[:, :60], b, 1.0), (0, a, b[:60], 1.0), (0, a, b[:, :3], 1.0),
                 (0, a[:0], b[:, :0], 1.0), (0, a[0], b, 1.0), (0, a.repeat(5, 1), b.repeat(1, 5), 1.0)):
        with pytest.raises(ValueError):
            bank.load(*args)
    with pytest.raises(ValueError):
        bank.unload(1)


def test_load_converts_and_clears_past_the_rank():
    _, _, bank, _, _ = make(BF16, 8, 64, 72, [16], 16)
    a, b = torch.randn(5, 64, device="cuda"), torch.randn(72, 5, device="cuda")
    bank.load(0, a, b, 2.0)
    assert torch.equal(bank.lora_a[0, :5], a.to(BF16)) and not bank.lora_a[0, 5:].any()
    assert torch.equal(bank.lora_b[0, 0, :, :5], b.to(BF16)) and not bank.lora_b[0, :, :, 5:].any()
    assert bank.ranks.tolist() == [5] and bank.scales.tolist() == [2.0]
    assert np.isclose(bank.lora_a.element_size(), 2)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("r, max_rank", [(1, 16), (16, 16), (17, 32), (33, 64), (64, 64), (100, 128)])
def test_load_of_dense_strided_and_foreign_tensors(dtype, r, max_rank):
    K, N = 75, 41
    bank = AdapterBank(3, max_rank, K, N, dtype, "cuda")
    bank.lora_a.fill_(float("nan"))
    bank.lora_b.fill_(float("nan"))
    a, b = torch.randn(2 * r, K + 3, device="cuda"), torch.randn(N, 2 * r, device="cuda")
    sources = [(a[:r, :K].to(dtype).contiguous(), b[:, :r].to(dtype).contiguous()),  # dense
               (a.to(dtype)[:r, 1:K + 1], b.to(dtype)[:, :r]),  # rows apart
               (a[::2, :K], b[:, ::2]),  # float32 and no dense rows
               (a[:r, :K].cpu().double(), b[:, :r].cpu().double()),  # another device
               (a[:r, :K].to(dtype).t().contiguous().t(), b[:, :r].to(dtype).t().contiguous().t())]
    for i, (sa, sb) in enumerate(sources):
        bank.load(1, sa, sb, 0.5 + i)
        assert torch.equal(bank.lora_a[1, :r], sa.to("cuda", dtype)) and not bank.lora_a[1, r:].any()
        ranks = bank.lora_b[1].transpose(0, 1).reshape(N, -1)
        assert torch.equal(ranks[:, :r], sb.to("cuda", dtype)) and not ranks[:, r:].any()
        assert bank.ranks.tolist() == [0, r, 0] and bank.scales.tolist() == [0.0, 0.5 + i, 0.0]
    assert bank.lora_a[::2].isnan().all() and bank.lora_b[::2].isnan().all()  # the neighbours


@pytest.mark.parametrize("T", [40, 1100])
def test_rows_apart_without_adapters_and_out_of_range(T):
    K, N = 136, 264
    x, w, bank, adapters, slots = make(BF16, T, K, N, [64, 8, 0], 64)
    wide = torch.full((T, K + 24), float("nan"), dtype=BF16, device="cuda")
    wide[:, 8:K + 8] = x
    y = fused_lora_forward_rows(x, w, bank, slots)
    assert torch.equal(fused_lora_forward_rows(wide[:, 8:K + 8], w, bank, slots), y)
    off = torch.full((T, K + 3), float("nan"), dtype=BF16, device="cuda")  # rows that are not 16-byte aligned
    off[:, 1:K + 1] = x
    assert torch.equal(fused_lora_forward_rows(off[:, 1:K + 1], w, bank, slots), y)
    none = fused_lora_forward_rows(x, w, bank, torch.full((T,), -1, device="cuda"))
    check(none, x, w, adapters, torch.full((T,), -1, device="cuda"))
    assert torch.equal(fused_lora_forward_rows(x, w, bank, torch.full((T,), 2, device="cuda")), none)  # an empty slot
    assert nat.device_error() == 0
    assert torch.equal(fused_lora_forward_rows(x, w, bank, torch.full((T,), 3, device="cuda")), none)
    assert nat.device_error() == nat.ERR_ROW_SLOT and nat.device_error() == 0


def test_long_batches_on_two_streams():
    first = make(BF16, 1300, 512, 1024, [16, 64, 33], 64, seed=1)
    second = make(BF16, 900, 1024, 512, [100, 16], 128, seed=2)
    want = [fused_lora_forward_rows(x, w, bank, slots) for x, w, bank, _, slots in (first, second)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (x, w, bank, _, slots) in enumerate((first, second)):
            with torch.cuda.stream(streams[i]):
                got[i].append(fused_lora_forward_rows(x, w, bank, slots))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])
    assert nat.device_error() == 0


def test_a_single_slot_and_a_single_feature_block():
    """One adapter on every row of a long batch, eight output features, K below one block."""
    T, K, N = 1025, 8, 8
    x, w, bank, adapters, _ = make(F16, T, K, N, [7], 8)
    slots = torch.zeros(T, dtype=torch.int32, device="cuda")
    check(fused_lora_forward_rows(x, w, bank, slots), x, w, adapters, slots)


@pytest.mark.parametrize("T", [40, 1100])
def test_an_output_buffer_advances_its_version(T):
    x, w, bank, _, slots = make(BF16, T, 256, 264, [16, 4], 16)
    out = torch.empty(T, 264, dtype=BF16, device="cuda")
    odd = torch.zeros(T, 259, dtype=BF16, device="cuda")[:, :256]  # needs a dense copy: checked in Python
    odd.copy_(x)
    for rows in (x, odd):
        before = out._version
        assert fused_lora_forward_rows(rows, w, bank, slots, out=out) is out
        assert out._version == before + 1
    with torch.inference_mode():  # such tensors have no version
        fused_lora_forward_rows(x, w, bank, slots, out=torch.empty_like(out))
        fused_lora_forward_rows(odd, w, bank, slots, out=torch.empty_like(out))


def test_packed_backward_after_its_input_was_overwritten_by_rows():
    """The packed backward may keep x A^T of a forward only while x holds what that forward read."""
    from lorafusion_b200.config import AdapterSpec, TileRoute, TileRoutingConfig
    T, K = 200, 256
    x, w, bank, adapters, slots = make(BF16, T, K, K, [16, 8], 16)
    lora_a, lora_b = ({i: ad[k] for i, ad in enumerate(adapters)} for k in (0, 1))
    specs = {i: AdapterSpec(i, a.shape[0], 2.0 * a.shape[0], K, K) for i, a in lora_a.items()}
    routing = TileRoutingConfig(128, [TileRoute(0, 90, 0), TileRoute(90, T, 1)])
    g = torch.randn(T, K, device="cuda").to(BF16)
    buf = torch.randn(T, K, device="cuda").to(BF16)
    b200_ops.fused_lora_forward(buf, w, lora_a, lora_b, specs, routing)
    fused_lora_forward_rows(x, w, bank, slots, out=buf)
    _, got_a, got_b = b200_ops.fused_lora_backward(g, buf, w, lora_a, lora_b, specs, routing)
    _, want_a, want_b = b200_ops.fused_lora_backward(g, buf.clone(), w, lora_a, lora_b, specs, routing)
    for got, want in ((got_a, want_a), (got_b, want_b)):
        # both compute S anew: one in the backward's own launches, so the same bits
        assert all(torch.equal(got[i], want[i]) for i in want)


def test_load_and_unload_advance_the_versions_of_the_bank():
    _, _, bank, adapters, _ = make(BF16, 4, 64, 64, [16, 16], 16)
    tensors = (bank.lora_a, bank.lora_b, bank.ranks, bank.scales)
    for a in (adapters[0][0], adapters[0][0].float()):  # as it is, and converted first
        before = [t._version for t in tensors]
        bank.load(1, a, adapters[0][1], 1.0)
        assert [t._version for t in tensors] == [v + 1 for v in before]
    before = bank.ranks._version
    bank.unload(1)
    assert bank.ranks._version > before


def test_packed_forward_with_a_view_of_the_bank_follows_a_load():
    """The packed operator keeps packed copies of weights whose version has not changed."""
    from lorafusion_b200.config import AdapterSpec, TileRoute, TileRoutingConfig
    T, K = 64, 128
    x, w, bank, adapters, _ = make(BF16, T, K, K, [16, 16], 16)
    view = bank.lora_a[0]
    b, specs = {0: adapters[0][1]}, {0: AdapterSpec(0, 16, 16.0, K, K)}
    routing = TileRoutingConfig(64, [TileRoute(0, T, 0)])
    b200_ops.fused_lora_forward(x, w, {0: view}, b, specs, routing)
    bank.load(0, 4 * adapters[1][0], adapters[1][1], 1.0)
    got = b200_ops.fused_lora_forward(x, w, {0: view}, b, specs, routing)
    assert torch.equal(got, b200_ops.fused_lora_forward(x, w, {0: view.clone()}, b, specs, routing))


def whole_numbers(*shape, most):
    return torch.randint(-most, most + 1, shape, device="cuda").float()


def one_adapter(dtype, T, w, a, b, s=1.0):
    """(a bank that holds it, slots that name it); W beside it."""
    bank = AdapterBank(1, a.shape[0], a.shape[1], w.shape[0], dtype, "cuda")
    bank.load(0, a, b, s)
    return bank, torch.zeros(T, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("T", [3, 200, 1500])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_small_and_large_rank_products_in_one_row(T, dtype):
    """One S 2^-18 of the other, which B takes no part of.  S is exact (sums of whole numbers times powers of two), so
    the bound is: two halves of S (2^-16 or 2^-22 of it, and 2^-35 of the row's largest), the float32 sums, one
    rounding."""
    K, N = 64, 136
    x = whole_numbers(T, K, most=4).to(dtype)
    a = whole_numbers(2, K, most=4) * torch.tensor([[2.0 ** 6], [2.0 ** -12]], device="cuda")
    a, b = a.to(dtype), torch.zeros(N, 2, dtype=dtype, device="cuda")
    b[:, 1] = 4 * torch.randn(N, device="cuda")
    w = torch.zeros(N, K, dtype=dtype, device="cuda")
    bank, slots = one_adapter(dtype, T, w, a, b)
    S = x.double() @ a.double().T
    want = S @ b.double().T
    off = (2.0 ** -16 if dtype is BF16 else 2.0 ** -22) * S.abs() + 2.0 ** -35 * S.abs().amax(1, keepdim=True)
    bound = off @ b.double().abs().T + (torch.finfo(dtype).eps / 2 + 200 * 2.0 ** -23) * want.abs()
    bound += torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    got = fused_lora_forward_rows(x, w, bank, slots).double()
    assert ((got - want).abs() <= bound).all()


def check_not_finite(y, x, a, b, s=1.0):
    """Infinities and NaN of y where the formula (in 64 bits, term by term) has them."""
    S = (x.double()[:, None] * a.double()[None]).sum(2)
    want = s * (S[:, None] * b.double()[None]).sum(2)
    for kind in (torch.isposinf, torch.isneginf, torch.isnan):
        assert torch.equal(kind(y), kind(want))
    return want


@pytest.mark.parametrize("T", [9, 1100])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_infinite_rank_product(T, dtype):
    """S of one rank is infinite, of another beyond float16's range: the infinities of the result are the first's."""
    K, N = 64, 72
    x = (torch.rand(T, K, device="cuda") + 0.5).to(dtype)
    a = torch.full((3, K), 400.0, device="cuda")
    a[1] *= -50  # S up to 2e6
    a[0, 5] = float("inf")
    b = torch.randn(N, 3, device="cuda")
    b[:, 0] = torch.where(b[:, 0] < 0, -1.0, 1.0)  # x 0 would be NaN
    a, b = a.to(dtype), b.to(dtype)
    w = torch.zeros(N, K, dtype=dtype, device="cuda")
    for A in (a, -a):
        bank, slots = one_adapter(dtype, T, w, A, b, 0.5)
        y = fused_lora_forward_rows(x, w, bank, slots)
        want = check_not_finite(y, x, A, b, 0.5)
        assert torch.isposinf(want).any() and torch.isneginf(want).any()


@pytest.mark.parametrize("T", [9, 1100])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("r", [1, 16, 40])
def test_infinite_entries_of_b(T, dtype, r):
    """S (whole numbers: those one half holds, those it does not, zero) times an infinite entry of B."""
    K, N = 64, 136
    x = whole_numbers(T, K, most=9).to(dtype)
    x[0] = 0.0
    x[1], x[2, 1:] = 0.0, 0.0
    a = whole_numbers(r, K, most=9)
    a[:, 0] = 1.0
    x[1, 0], x[2, 0] = 1.0, -4.0  # S of one and of minus four
    a, b = a.to(dtype), torch.randn(N, r, device="cuda").to(dtype)
    b[::3, 0], b[1::3, r // 2], b[4, r - 1] = float("inf"), -float("inf"), float("nan")
    w = torch.zeros(N, K, dtype=dtype, device="cuda")
    a2 = a.clone()
    a2[0, 0] = float("inf")  # S of rank 0 infinite (NaN where x is zero)
    for A in (a, a2):
        bank, slots = one_adapter(dtype, T, w, A, b, -2.0)
        y = fused_lora_forward_rows(x, w, bank, slots)
        want = check_not_finite(y, x, A, b, -2.0)
        assert torch.isposinf(want).any() and torch.isneginf(want).any()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T, N, ranks", [(1, 136, [16]), (40, 264, [3, 16, 1]), (200, 520, [40, 64, 17]),
                                         (300, 264, [16, 9, 30]), (700, 392, [128, 90, 16]), (1500, 136, [16, 33, 64])])
def test_whole_numbers_are_exact_before_the_rounding(dtype, T, N, ranks):
    """x, W, A and B of whole numbers whose sums all fit float32 and whose S (up to 2^14) both halves hold: what is left
    is the one rounding of y.  S alone needs more bits than one half has, so this sees the low ones."""
    K = 512
    torch.manual_seed(T)
    x = whole_numbers(T, K, most=15).to(dtype)
    w = whole_numbers(N, K, most=3).to(dtype)
    bank = AdapterBank(len(ranks), max(ranks), K, N, dtype, "cuda")
    slots = torch.arange(T, device="cuda") * 5 % (len(ranks) + 1) - 1
    if T == 1:
        slots += 1
    want = x.double() @ w.double().T
    for i, r in enumerate(ranks):
        a, b = whole_numbers(r, K, most=15).to(dtype), whole_numbers(N, r, most=1).to(dtype)
        b *= (torch.arange(r, device="cuda") < 16).to(dtype)  # y stays in float16's range
        bank.load(i, a, b, 0.5)
        S = x.double() @ a.double().T
        assert S.abs().max() < 2 ** 14 and (T == 1 or S.abs().max() > 2 ** 11)
        want += torch.where((slots == i)[:, None], 0.5 * S @ b.double().T, 0.0)
    assert want.abs().max() < 65504
    y = fused_lora_forward_rows(x, w, bank, slots)
    assert torch.equal(y, want.to(dtype))


TALL_TILES = [  # dtype, T, K, N, ranks, max_rank: above 256 rows and not through the CTA-pair GEMM
    (BF16, 300, 4096, 1024, [64, 33], 64),       # K in 8 parts, sorted rows
    (F16, 512, 4096, 4096, [16] * 40, 16),       # in 2, the single launch of few rows
    (BF16, 400, 4096, 1032, [16, 3, 30], 32),    # in 4, a last tile of 8 features
    (BF16, 1000, 4096, 1024, [128, 16], 128),    # in 4, four row tiles
    (F16, 2048, 4096, 1024, [64] * 5, 64),       # in 2, eight
    (BF16, 400, 14336, 4096, [16, 8], 16),
    (BF16, 300, 4096, 4096, [16, 64], 64),       # two adapters: few tiles, K of x A_i in 8 parts
]


@pytest.mark.parametrize("case", TALL_TILES, ids=lambda c: f"{str(c[0])[6:]}-{c[1]}x{c[2]}x{c[3]}-r{c[5]}")
def test_row_tiles_beside_one_another(case):
    dtype, T, K, N, ranks, max_rank = case
    assert nat.lib().lf_rows_uses_pairs(T, K, N, torch.cuda.get_device_properties(0).multi_processor_count) == 0
    x, w, bank, adapters, slots = make(dtype, T, K, N, ranks, max_rank)
    y = fused_lora_forward_rows(x, w, bank, slots)
    check(y, x, w, adapters, slots)
    order = torch.randperm(T, device="cuda")
    moved = fused_lora_forward_rows(x[order], w, bank, slots[order])
    if nat.lib().lf_rows_launch_count(T, bank.r_pad) == 4:
        assert torch.equal(moved, y[order])
    else:  # how many warps share K depends on the adapters beside a row there: the order of a sum may change
        check(moved, x[order], w, adapters, slots[order])
    none = torch.full_like(slots, -1)
    check(fused_lora_forward_rows(x, w, bank, none), x, w, adapters, none)
    assert nat.device_error() == 0


def test_an_output_over_the_slots_is_refused():
    x, w, bank, _, slots = make(BF16, 8, 64, 64, [16], 16)
    memory = torch.zeros(8 * 64, dtype=BF16, device="cuda")
    for shared in (memory[16:32].view(torch.int32), memory[-32:].view(torch.int64)):
        shared.copy_(slots)
        with pytest.raises(ValueError):
            fused_lora_forward_rows(x, w, bank, shared, out=memory.view(8, 64))
        assert torch.equal(shared, slots.to(shared.dtype))


def test_more_rows_than_32_bits_count_are_refused():
    _, w, bank, _, _ = make(BF16, 8, 64, 64, [16], 16)
    for T in (2 ** 31, 2 ** 32 + 5):
        x = torch.zeros(1, 64, dtype=BF16, device="cuda").expand(T, 64)
        with pytest.raises(ValueError):
            fused_lora_forward_rows(x, w, bank, torch.zeros(1, dtype=torch.int32, device="cuda").expand(T))


@pytest.mark.filterwarnings("ignore::lorafusion_b200.b200_ops.CudaCorePathWarning")
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_rows_on_cuda_cores_than_one_grid_covers(dtype):
    T, K, N = 32 * 65535 + 37, 5, 3
    x, w, bank, adapters, slots = make(dtype, T, K, N, [2, 1], 2)
    out = torch.full((T + 1, N), 7.0, dtype=dtype, device="cuda")
    fused_lora_forward_rows(x, w, bank, slots, out=out[:T])
    assert b200_ops.last_launch_count() == 4
    check(out[:T], x, w, adapters, slots)
    assert bool((out[T] == 7).all())


@pytest.mark.parametrize("T", [1, 64, 400])
def test_slots_that_change_under_a_call_leave_no_wait_behind(T):
    """Not allowed, and the rows are undefined; but the CTAs of a cluster, which then disagree about the batches, end."""
    ranks = [16, 8, 32, 3] * 40
    x, w, bank, adapters, slots = make(BF16, T, 4096, 512, ranks, 32)
    patterns = [torch.full_like(slots, -1), slots.clone(), torch.arange(T, device="cuda", dtype=torch.int32) % 160,
                torch.zeros_like(slots)]
    changing, writer = slots.clone(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for k in range(200):
        with torch.cuda.stream(writer):
            for p in patterns:
                changing.copy_(p)
            bank.ranks[k % 4::4] = ranks[k % 4]  # as they are
        fused_lora_forward_rows(x, w, bank, changing)
    torch.cuda.synchronize()
    check(fused_lora_forward_rows(x, w, bank, slots), x, w, adapters, slots)
    assert nat.device_error() == 0


def test_nothing_is_recorded_and_an_output_that_requires_a_gradient_is_refused():
    x, w, bank, adapters, slots = make(BF16, 8, 64, 64, [16], 16)
    y = fused_lora_forward_rows(x, w, bank, slots)
    xg, wg = x.clone().requires_grad_(), torch.nn.Parameter(w)
    got = fused_lora_forward_rows(xg, wg, bank, slots)
    assert torch.equal(got, y) and not got.requires_grad
    leaf = torch.zeros_like(y).requires_grad_()
    for out in (leaf, leaf * 2):
        kept = out.detach().clone()
        with pytest.raises(ValueError):
            fused_lora_forward_rows(x, w, bank, slots, out=out)
        assert torch.equal(out, kept)
        with torch.no_grad():
            assert torch.equal(fused_lora_forward_rows(x, w, bank, slots, out=out), y)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_load_of_parts_of_the_slot_itself(dtype):
    """Half of an adapter's ranks, moved to the front, while the kernel zeroes the others."""
    K, N = 8192, 4096
    bank = AdapterBank(2, 16, K, N, dtype, "cuda")
    for _ in range(3):
        a, b = torch.randn(16, K, device="cuda").to(dtype), torch.randn(N, 16, device="cuda").to(dtype)
        bank.load(1, a, b, 1.0)
        bank.load(1, bank.lora_a[1, 8:], bank.lora_b[1, 0][:, 8:], 2.0)
        assert torch.equal(bank.lora_a[1, :8], a[8:]) and not bank.lora_a[1, 8:].any()
        assert torch.equal(bank.lora_b[1, 0, :, :8], b[:, 8:]) and not bank.lora_b[1, 0, :, 8:].any()
        assert bank.ranks.tolist() == [0, 8] and not bank.lora_a[0].any()
        bank.load(0, bank.lora_a[1, :8], bank.lora_b[1, 0][:, :8], 2.0)  # from another slot: no copy between
        assert torch.equal(bank.lora_a[0], bank.lora_a[1]) and torch.equal(bank.lora_b[0], bank.lora_b[1])
        bank.unload(0)
        bank.lora_a[0].zero_()
