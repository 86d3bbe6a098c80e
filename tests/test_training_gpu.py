"""Gradient clipping and AdamW of many adapters (training.py) against the formulas in 64 bits.

Bounds: a norm is a float64 sum rounded once to float32 (2^-24), its square root and the few float64
operations around it are far below that.  A clipped gradient is the float32 product of the gradient
with the factor (rounded to float32: 2^-24), rounded once more to its type.  AdamW runs in float32: each
value below is bounded by the roundings on its way (counted at the check).
"""

import math

import pytest
import torch

from lorafusion_b200 import b200_ops
from lorafusion_b200.training import AdapterAdamW, clip_adapter_grads

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def make_grads(dtype, layers, ranks, seed=0, gain=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for K, N in layers:
        for shape in (lambda r: (r, K), lambda r: (N, r)):
            out.append({i: (randn(gen, *shape(r)) * (gain[i] if gain else 1.0)).to(dtype) for i, r in ranks.items()})
    return out


def norms64(dicts, ids, inf=False):
    vals = []
    for i in ids:
        parts = [d[i].double().flatten() for d in dicts if i in d and d[i].numel()]
        flat = torch.cat(parts) if parts else torch.zeros(1, device="cuda", dtype=torch.float64)
        vals.append(flat.abs().max() if inf else flat.square().sum().sqrt())
    return torch.stack(vals)


def check_scaled(got, before, factor, dtype):
    want = before.double() * factor
    half = torch.finfo(dtype).eps / 2
    bound = (half + 3 * U) * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("layers, ranks", [
    ([(1, 1)], {0: 1}),
    ([(8, 24)], {3: 2}),
    ([(255, 33), (7, 1001)], {5: 3, 1: 1, 9: 16}),       # odd sizes: blocks that start off 16 bytes
    ([(4096, 1024)], {i: 16 for i in range(20)}),
    ([(4097, 2050), (64, 64), (513, 129)], {i: 1 + i % 5 for i in range(90)}),
], ids=["one", "tiny", "odd", "sixteen", "many"])
def test_clip_each_adapter(dtype, layers, ranks):
    gain = {i: [1e-3, 5.0, 0.3][k % 3] for k, i in enumerate(ranks)}
    dicts = make_grads(dtype, layers, ranks, gain=gain)
    before = [{i: t.clone() for i, t in d.items()} for d in dicts]
    ref = norms64(before, ranks)
    norms = clip_adapter_grads(dicts, 1.0)
    assert norms.dtype == F32 and norms.shape == (len(ranks),)
    assert ((norms.double() - ref).abs() <= 1.01 * U * ref).all()
    factors = (1.0 / (ref + 1e-6)).clamp(max=1.0).tolist()
    for d, b in zip(dicts, before):
        for i, f in zip(ranks, factors):
            if f == 1.0:
                assert torch.equal(d[i], b[i])
            else:
                check_scaled(d[i], b[i], f, dtype)


@pytest.mark.parametrize("per_adapter", [True, False])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_norm_kinds(per_adapter, norm_type):
    ranks = {"a": 3, "b": 16, "c": 1}
    dicts = make_grads(F32, [(100, 60), (33, 20)], ranks, gain={"a": 2.0, "b": 0.01, "c": 1.0})
    del dicts[2]["b"], dicts[3]["b"], dicts[0]["c"]  # dicts need not name the same adapters
    before = [{i: t.clone() for i, t in d.items()} for d in dicts]
    order = list(dict.fromkeys(i for d in dicts for i in d))
    ref = norms64(before, order, math.isinf(norm_type))
    if not per_adapter:
        ref = ref.max() if math.isinf(norm_type) else ref.square().sum().sqrt()
    only = clip_adapter_grads(dicts, None, norm_type=norm_type, per_adapter=per_adapter)
    assert all(torch.equal(d[i], b[i]) for d, b in zip(dicts, before) for i in d)
    norms = clip_adapter_grads(dicts, 0.5, norm_type=norm_type, per_adapter=per_adapter)
    assert torch.equal(only, norms) and norms.shape == ref.shape
    assert ((norms.double() - ref).abs() <= 1.01 * U * ref).all()
    f = (0.5 / (ref + 1e-6)).clamp(max=1.0).expand(len(order)).tolist()
    for d, b in zip(dicts, before):
        for i in d:
            check_scaled(d[i], b[i], f[order.index(i)], F32)


def test_norm_holds_where_float32_squares_do_not():
    g = {0: torch.full((5000,), 1e25, device="cuda"), 1: torch.full((5000,), 1e-30, device="cuda")}
    norms = clip_adapter_grads([g], None)
    ref = torch.tensor([1e25, 1e-30], dtype=F32).double().cuda() * math.sqrt(5000)
    assert ((norms.double() - ref).abs() <= 1.01 * U * ref).all()


def test_norms_that_are_not_finite():
    g = {i: torch.ones(3000, device="cuda") for i in range(3)}
    g[0][2999], g[1][0] = float("nan"), float("-inf")
    for norm_type in (2.0, math.inf):
        h = {i: t.clone() for i, t in g.items()}
        norms = clip_adapter_grads([h], 0.5, norm_type=norm_type)
        assert torch.isnan(norms[0]) and torch.isinf(norms[1]) and torch.isfinite(norms[2])
        assert torch.isnan(h[0]).all()
        assert torch.isnan(h[1][0]) and not h[1][1:].any()
        assert torch.isfinite(h[2]).all()


def test_mixed_types_empty_tensors_and_many_launches():
    gen = torch.Generator(device="cuda").manual_seed(3)
    types = [F32, BF16, F16]
    d = {i: randn(gen, 17 + i % 40).to(types[i % 3]) for i in range(3300)}  # over two launches of 1500
    d[7] = torch.empty(0, 5, device="cuda")
    before = {i: t.clone() for i, t in d.items()}
    ref = norms64([before], list(d))
    norms = clip_adapter_grads([d], 0.25)
    assert ((norms.double() - ref).abs() <= 1.01 * U * ref).all() and norms[7] == 0
    f = (0.25 / (ref + 1e-6)).clamp(max=1.0).tolist()
    for k, i in enumerate(d):
        check_scaled(d[i], before[i], f[k], d[i].dtype)
    whole = clip_adapter_grads([d], None, per_adapter=False)
    ref = norms64([d], list(d)).square().sum().sqrt()
    assert abs(whole.double() - ref) <= 1.01 * U * ref


def test_clip_is_repeatable_and_captures():
    dicts = make_grads(BF16, [(2048, 777)], {i: 16 for i in range(9)})
    before = [{i: t.clone() for i, t in d.items()} for d in dicts]
    first = clip_adapter_grads(dicts, 1.0)
    want = [{i: t.clone() for i, t in d.items()} for d in dicts]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norms = clip_adapter_grads(dicts, 1.0)
    for _ in range(3):
        for d, b in zip(dicts, before):
            for i in d:
                d[i].copy_(b[i])
        graph.replay()
        assert torch.equal(norms, first)
        assert all(torch.equal(d[i], w[i]) for d, w in zip(dicts, want) for i in d)


def test_clip_refusals():
    g = torch.ones(40, 4, device="cuda")
    for grads, max_norm, kw in (([], 1.0, {}), ([{}], 1.0, {}), ([{0: g.cpu()}], 1.0, {}), ([{0: g.double()}], 1.0, {}),
                                ([{0: g.T}], 1.0, {}), ([{0: g}], -1.0, {}), ([{0: g}], float("nan"), {}),
                                ([{0: g}], 1.0, {"norm_type": 1.0}), ([{0: g}, {0: g}], 1.0, {}),
                                ([{0: g}, {1: g.view(-1)[4:80]}], 1.0, {})):
        with pytest.raises(ValueError):
            clip_adapter_grads(grads, max_norm, **kw)
    assert bool((g == 1).all())
    clip_adapter_grads([{0: g}, {0: g}], None)  # norms alone may name a tensor twice
    halves = [{0: g[:20]}, {0: g[20:]}]
    assert abs(clip_adapter_grads(halves, 0.0).item() - math.sqrt(160)) < 1e-5
    assert not g.any()


# ------------------------------------------------------------------------------------------- AdamW
class Adam64:
    """The formula in 64 bits, from an optimizer's state."""

    def __init__(self, opt):
        self.opt = opt
        self.w = [{i: (s[j]["master"] if opt.master is not None else opt.params[j][i]).double().clone()
                   for i in opt.params[j] for s in [opt.state(i)]} for j in range(len(opt.params))]
        self.m = [{i: opt.state(i)[j]["exp_avg"].double().clone() for i in opt.params[j]}
                  for j in range(len(opt.params))]
        self.v = [{i: opt.state(i)[j]["exp_avg_sq"].double().clone() for i in opt.params[j]}
                  for j in range(len(opt.params))]
        self.t = dict(zip(opt.ids, opt.steps.tolist()))

    def step_and_check(self, grads):
        opt = self.opt
        b1, b2 = opt.betas
        norms = norms64(grads, opt.ids)
        got = opt.step(grads)
        if got is not None:
            assert ((got.double() - norms).abs() <= 1.01 * U * norms).all()
        seen = {i for d in grads for i in d}
        for k, i in enumerate(opt.ids):
            skip = opt.skip_nonfinite and not bool(torch.isfinite(norms[k]))
            if i in seen and not skip:
                self.t[i] += 1
        assert opt.steps.tolist() == [self.t[i] for i in opt.ids]
        for j, d in enumerate(grads):
            for i in opt.params[j]:
                state = opt.state(i)[j]
                w32 = state["master"] if opt.master is not None else opt.params[j][i]
                k = opt.ids.index(i)
                skip = opt.skip_nonfinite and not bool(torch.isfinite(norms[k]))
                if i not in d or skip:  # untouched, bit for bit
                    assert torch.equal(state["exp_avg"].double(), self.m[j][i])
                    assert torch.equal(state["exp_avg_sq"].double(), self.v[j][i])
                    assert torch.equal(w32.double(), self.w[j][i])
                    continue
                lr, wd = opt._hyper[k]
                f = min(1.0, opt.max_norm / (float(norms[k]) + 1e-6)) if opt.max_norm is not None else 1.0
                g = d[i].double() * f
                # g': factor and product rounded (2 U); then two products, a sum, a rounded constant each
                m = b1 * self.m[j][i] + (1 - b1) * g
                m_off = 6 * U * (b1 * self.m[j][i].abs() + (1 - b1) * g.abs()) + 1e-44
                v = b2 * self.v[j][i] + (1 - b2) * g * g
                v_off = 9 * U * v + 1e-44
                assert ((state["exp_avg"].double() - m).abs() <= m_off).all()
                assert ((state["exp_avg_sq"].double() - v).abs() <= v_off).all()
                # the weight from the moments as they were rounded: their own errors carry over
                mm, vv = state["exp_avg"].double(), state["exp_avg_sq"].double()
                size, root = lr / (1 - b1 ** self.t[i]), math.sqrt(1 - b2 ** self.t[i])
                denom = vv.sqrt() / root + opt.eps
                move = size * mm / denom
                w = self.w[j][i] * (1 - lr * wd) - move
                # decay: constant and product; move: size, product, sqrt, root, quotient, eps, sum, quotient; sum
                off = 3 * U * self.w[j][i].abs() + 10 * U * move.abs() + U * w.abs() + 1e-44
                assert ((w32.double() - w).abs() <= off).all()
                if opt.master is not None:
                    assert torch.equal(opt.params[j][i], w32.to(opt.dtype))
                self.m[j][i], self.v[j][i], self.w[j][i] = mm.clone(), vv.clone(), w32.double().clone()


def make_params(dtype, layers, ranks, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for K, N in layers:
        out.append({i: (0.05 * randn(gen, r, K)).to(dtype) for i, r in ranks.items()})
        out.append({i: (0.05 * randn(gen, N, r)).to(dtype) for i, r in ranks.items()})
    return out


@pytest.mark.parametrize("dtype, gdt", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)])
@pytest.mark.parametrize("layers, ranks", [
    ([(1, 3)], {0: 1}),
    ([(255, 33), (7, 1001)], {5: 3, 1: 1, 9: 16}),
    ([(4096, 1000)], {i: 16 for i in range(12)}),
    ([(520, 264)] * 3, {i: 1 + i % 4 for i in range(100)}),
], ids=["one", "odd", "sixteen", "many"])
@pytest.mark.parametrize("max_norm", [None, 1.0])
def test_adamw_against_64_bits(dtype, gdt, layers, ranks, max_norm):
    opt = AdapterAdamW(make_params(dtype, layers, ranks), lr={i: 1e-3 * (1 + k % 3) for k, i in enumerate(ranks)},
                       weight_decay={i: 0.1 * (k % 2) for k, i in enumerate(ranks)}, max_norm=max_norm)
    ref = Adam64(opt)
    for k in range(3):
        gain = {i: [0.01, 3.0][(n + k) % 2] for n, i in enumerate(ranks)}
        ref.step_and_check(make_grads(gdt, layers, ranks, seed=k, gain=gain))
    first = next(iter(ranks))
    opt.set_adapter(first, lr=5e-2, weight_decay=0.3)
    ref.step_and_check(make_grads(gdt, layers, ranks, seed=9))


def test_adapters_without_rows_keep_weights_and_counts():
    layers, ranks = [(64, 48), (40, 72)], {0: 4, 1: 8, 2: 3}
    opt = AdapterAdamW(make_params(BF16, layers, ranks), lr=1e-2, max_norm=1.0)
    ref = Adam64(opt)
    for absent in ((1,), (), (0, 2)):
        grads = make_grads(F32, layers, ranks, seed=len(absent))
        for i in absent:
            for d in grads:
                del d[i]
        ref.step_and_check(grads)
    partly = make_grads(F32, layers, ranks, seed=5)
    del partly[0][1], partly[3][1]  # one adapter, some of its weights
    ref.step_and_check(partly)
    before = opt.steps.tolist()
    assert not opt.step([{} for _ in opt.params]).any() and opt.steps.tolist() == before


def test_a_diverged_adapter_is_left_alone():
    layers, ranks = [(64, 48)], {0: 4, 1: 8, 2: 3}
    opt = AdapterAdamW(make_params(BF16, layers, ranks), lr=1e-2, skip_nonfinite=True)
    ref = Adam64(opt)
    grads = make_grads(BF16, layers, ranks)
    grads[1][1][3, 2], grads[0][2][0, 0] = float("nan"), float("inf")
    norms = opt.step([{i: t.clone() for i, t in d.items()} for d in grads])
    assert torch.isfinite(norms).tolist() == [True, False, False]
    assert opt.steps.tolist() == [1, 0, 0]
    for j in range(2):
        for i in (1, 2):
            assert torch.equal(opt.state(i)[j]["master"].double(), ref.w[j][i])
        assert not torch.equal(opt.state(0)[j]["master"].double(), ref.w[j][0])


def test_state_travels():
    layers, ranks = [(65, 31)], {0: 4, 7: 3}
    make = lambda: AdapterAdamW(make_params(BF16, layers, ranks), lr=1e-2, weight_decay=0.1)  # noqa: E731
    one = make()
    for k in range(2):
        one.step(make_grads(F32, layers, ranks, seed=k))
    two = make()
    two.load_state_dict(one.state_dict())
    for j in range(2):
        assert all(torch.equal(one.params[j][i], two.params[j][i]) for i in ranks)
    for opt in (one, two):
        opt.step(make_grads(F32, layers, ranks, seed=4))
    assert torch.equal(one.exp_avg, two.exp_avg) and torch.equal(one.master, two.master)
    assert all(torch.equal(one.params[j][i], two.params[j][i]) for i in ranks for j in range(2))
    with pytest.raises(ValueError):
        AdapterAdamW(make_params(BF16, layers, {0: 4})).load_state_dict(one.state_dict())


def test_many_tensors_over_several_launches():
    ranks = {i: 1 for i in range(4200)}  # more than one launch of 3840, more than 4096 groups
    opt = AdapterAdamW([make_params(F32, [(9, 5)], ranks)[0]], lr=1e-2, max_norm=1.0)
    Adam64(opt).step_and_check([make_grads(F32, [(9, 5)], ranks)[0]])


def test_adamw_refusals():
    layers, ranks = [(64, 48)], {0: 4, 1: 8}
    params = make_params(BF16, layers, ranks)
    for bad in ([], [{}], [{0: params[0][0].cpu()}], [{0: params[0][0].double()}], [{0: params[0][0].T}],
                [params[0], {0: params[1][0].float()}], [{0: params[0][0]}, {0: params[0][0]}]):
        with pytest.raises(ValueError):
            AdapterAdamW(bad)
    for kw in (dict(lr=-1.0), dict(lr=float("nan")), dict(weight_decay=-0.1), dict(betas=(1.0, 0.9)), dict(eps=-1.0),
               dict(max_norm=-1.0)):
        with pytest.raises(ValueError):
            AdapterAdamW(params, **kw)
    with pytest.raises(KeyError):
        AdapterAdamW(params, lr={0: 1e-3})
    opt = AdapterAdamW(params)
    good = make_grads(BF16, layers, ranks)
    shapes = [{i: t for i, t in d.items()} for d in good]
    shapes[0][1] = shapes[0][1].view(64, 8)
    mixed = [good[0], {i: t.float() for i, t in good[1].items()}]
    for bad in (good[:1], [good[0], {**good[1], 5: good[1][0]}], shapes, mixed,
                [good[0], {i: t.cpu() for i, t in good[1].items()}], [{i: t.half() for i, t in d.items()} for d in good],
                [good[0], {0: torch.empty(4, 48, dtype=BF16, device="cuda").T}]):
        with pytest.raises(ValueError):
            opt.step(bad)
    assert opt.steps.tolist() == [0, 0]
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step(good)
    params[0][0].data = params[0][0].data.clone()
    with pytest.raises(RuntimeError):
        opt.step(good)


def test_train_then_serve():
    """backward -> clip -> AdamW -> forward with the new weights -> bank -> a row at a time."""
    from lorafusion_b200.config import AdapterSpec, TileRoute, TileRoutingConfig
    from lorafusion_b200.serving import AdapterBank, fused_lora_forward_rows
    T, K, N = 96, 128, 136
    gen = torch.Generator(device="cuda").manual_seed(0)
    x, w = randn(gen, T, K).to(BF16), (randn(gen, N, K) / K ** 0.5).to(BF16)
    ranks = {4: 8, 2: 16, 9: 3}
    lora_a, lora_b = make_params(BF16, [(K, N)], ranks)
    specs = {i: AdapterSpec(i, r, 2.0 * r, K, N) for i, r in ranks.items()}
    routing = TileRoutingConfig(64, [TileRoute(0, 50, 4), TileRoute(50, T, 2)])  # adapter 9 has no rows
    opt = AdapterAdamW([lora_a, lora_b], lr=1e-2, max_norm=1.0)
    ref = Adam64(opt)
    outs = []
    for k in range(3):
        outs.append(b200_ops.fused_lora_forward(x, w, lora_a, lora_b, specs, routing))
        _, ga, gb = b200_ops.fused_lora_backward(randn(gen, T, N).to(BF16), x, w, lora_a, lora_b, specs, routing,
                                                 grad_dtype=F32 if k else None)
        ref.step_and_check([ga, gb])
    assert opt.steps.tolist() == [3, 3, 0]
    y = b200_ops.fused_lora_forward(x, w, lora_a, lora_b, specs, routing)
    assert not torch.equal(y, outs[0]) and not torch.equal(y, outs[-1])  # packed copies follow the step
    bank = AdapterBank(3, 16, K, N, BF16, "cuda")
    slot = {i: s for s, i in enumerate(ranks)}
    for i, s in slot.items():
        bank.load(s, lora_a[i], lora_b[i], specs[i].scaling)
    rows = torch.tensor([slot[4]] * 50 + [slot[2]] * (T - 50), dtype=torch.int32, device="cuda")
    served = fused_lora_forward_rows(x, w, bank, rows)
    want = x.double() @ w.double().T
    for lo, hi, i in ((0, 50, 4), (50, T, 2)):
        want[lo:hi] += 2.0 * (x[lo:hi].double() @ lora_a[i].double().T) @ lora_b[i].double().T
    for got in (served, y):
        torch.testing.assert_close(got.double(), want, rtol=2e-2, atol=2e-2)


def test_a_step_advances_the_versions_of_its_state():
    """Float32 masters used as weights of the packed operator, which keeps packed copies by version."""
    from lorafusion_b200.config import AdapterSpec, TileRoute, TileRoutingConfig
    K = 64
    opt = AdapterAdamW(make_params(BF16, [(K, K)], {0: 8}), lr=0.1)
    a, b = ({0: opt.state(0)[j]["master"]} for j in (0, 1))
    x, w = torch.randn(16, K, device="cuda"), torch.randn(K, K, device="cuda")
    forward = lambda a, b: b200_ops.fused_lora_forward(  # noqa: E731
        x, w, a, b, {0: AdapterSpec(0, 8, 8.0, K, K)}, TileRoutingConfig(64, [TileRoute(0, 16, 0)]))
    forward(a, b)
    state = (opt.exp_avg, opt.exp_avg_sq, opt.master, opt.steps)
    before = [t._version for t in state]
    opt.step(make_grads(F32, [(K, K)], {0: 8}))
    assert all(t._version > v for t, v in zip(state, before))
    assert torch.equal(forward(a, b), forward({0: a[0].clone()}, {0: b[0].clone()}))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_weights_that_require_gradients_leave_no_graph_in_the_state(dtype):
    import copy
    layers, ranks = [(64, 48)], {0: 4, 1: 8}
    params = [{i: torch.nn.Parameter(t) for i, t in d.items()} for d in make_params(dtype, layers, ranks)]
    opt = AdapterAdamW(params, lr=1e-2, max_norm=1.0)
    grads = make_grads(dtype, layers, ranks)
    for k in range(2):
        Adam64(opt).step_and_check(grads)
        saved = copy.deepcopy(opt.state_dict())
        opt.refresh_masters()
        opt.load_state_dict(saved)
        for t in (opt.exp_avg, opt.exp_avg_sq) + (() if opt.master is None else (opt.master,)):
            assert not t.requires_grad and t.grad_fn is None
        assert all(p.requires_grad and p.is_leaf for d in params for p in d.values())
    reader = opt.state(0)[0]["exp_avg"] * torch.ones(1, device="cuda", requires_grad=True)
    opt.load_state_dict({k: v.requires_grad_() if k == "exp_avg" else v for k, v in opt.state_dict().items()})
    assert not opt.exp_avg.requires_grad and reader.requires_grad


def test_state_of_another_layout_is_refused():
    """The same adapters and totals in another order: loading would give every block to another weight."""
    ranks = {0: 4, 1: 8}
    (a, b), (c, d) = (make_params(BF16, [shape], ranks, seed=k) for k, shape in enumerate([(64, 48), (48, 64)]))
    opt = AdapterAdamW([a, b], lr=1e-2)
    opt.step(make_grads(F32, [(64, 48)], ranks))
    saved = opt.state_dict()
    for params in ([c, d],                                   # [r, 48] and [64, r]: equal totals
                   [{i: t.view(64, -1) for i, t in a.items()}, b], [a, {1: b[1], 0: b[0]}]):
        other = AdapterAdamW([{i: t.clone() for i, t in p.items()} for p in params], lr=1e-2)
        assert other.ids == opt.ids and other.exp_avg.shape == opt.exp_avg.shape
        kept = [t.clone() for t in (other.exp_avg, other.master, other.steps)]
        weights = [t.clone() for p in other.params for t in p.values()]
        with pytest.raises(ValueError):
            other.load_state_dict(saved)
        assert all(torch.equal(t, k) for t, k in zip((other.exp_avg, other.master, other.steps), kept))
        assert all(torch.equal(t, k) for t, k in zip([t for p in other.params for t in p.values()], weights))
    twin = AdapterAdamW([a, b], lr=1e-2)
    with pytest.raises(ValueError):
        twin.load_state_dict({k: v for k, v in saved.items() if k != "layout"})
    assert not twin.exp_avg.any()
    twin.load_state_dict({**saved, "layout": [[j, aid, list(s)] for j, aid, s in saved["layout"]]})  # as JSON has it
    assert torch.equal(twin.exp_avg, opt.exp_avg) and torch.equal(twin.steps, opt.steps)


def test_state_carries_every_hyperparameter():
    layers, ranks = [(65, 31)], {0: 4, 7: 3}
    one = AdapterAdamW(make_params(BF16, layers, ranks), lr=1e-2, weight_decay=0.1, betas=(0.8, 0.97), eps=1e-5,
                       max_norm=0.5, skip_nonfinite=True)
    two = AdapterAdamW(make_params(BF16, layers, ranks))
    one.step(make_grads(F32, layers, ranks))
    saved = one.state_dict()
    for bad in (dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(max_norm=-1.0), dict(hyper=[[-1.0, 0.0]] * 2),
                dict(hyper=[[1.0, float("nan")]] * 2)):
        with pytest.raises(ValueError):
            two.load_state_dict({**saved, **bad})
    assert not two.exp_avg.any() and two.betas == (0.9, 0.999) and two.max_norm is None
    two.load_state_dict(saved)
    grads = make_grads(F32, layers, ranks, seed=4)
    grads[0][7][0, 0] = float("inf")
    norms = [opt.step(grads) for opt in (one, two)]
    assert torch.equal(*norms) and one.steps.tolist() == two.steps.tolist() == [2, 1]
    assert torch.equal(one.exp_avg, two.exp_avg) and torch.equal(one.master, two.master)


def test_set_adapter_writes_both_values_or_none():
    opt = AdapterAdamW(make_params(F32, [(16, 16)], {0: 4, 1: 4}), lr=1e-3, weight_decay=0.1)
    for kw in (dict(lr=0.5, weight_decay=-1.0), dict(lr=float("inf"), weight_decay=0.2), dict(lr=0.5, weight_decay="x")):
        with pytest.raises(ValueError):
            opt.set_adapter(1, **kw)
        assert opt.state_dict()["hyper"] == [[1e-3, 0.1], [1e-3, 0.1]]
    with pytest.raises(KeyError):
        opt.set_adapter(2, lr=0.5)
    opt.set_adapter(1, weight_decay=0.0)
    opt.set_adapter(0, lr=0.0)
    assert opt.state_dict()["hyper"] == [[0.0, 0.1], [1e-3, 0.0]]


def test_a_step_with_new_rates_does_not_wait_for_the_queue():
    """Every step gets rates of its own while the stream is busy: the host runs ahead, no upload overtakes another."""
    layers, ranks = [(64, 48)], {0: 4, 1: 8}
    ahead, behind = (AdapterAdamW(make_params(BF16, layers, ranks)) for _ in range(2))
    grads = [make_grads(F32, layers, ranks, seed=k) for k in range(8)]

    def steps(opt, wait):
        for k, g in enumerate(grads):
            opt.set_adapter(k % 2, lr=1e-3 * (k + 1), weight_decay=0.1 * (k % 3))
            opt.step(g)
            if wait:
                torch.cuda.synchronize()

    start = {k: v.clone() if torch.is_tensor(v) else v for k, v in ahead.state_dict().items()}
    steps(behind, True)
    steps(ahead, False)  # the pinned buffers and the launches' first use
    ahead.load_state_dict(start)
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    torch.cuda._sleep(2_000_000_000)  # about a second
    done.record()
    steps(ahead, False)
    assert not done.query()
    assert torch.equal(ahead.master, behind.master) and torch.equal(ahead.exp_avg_sq, behind.exp_avg_sq)
    assert ahead.state_dict()["hyper"] == behind.state_dict()["hyper"]
