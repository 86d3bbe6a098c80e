"""Cases of the operators around an adapter's life, in plain torch and through this package.

* ``rows``   one shared projection with the low-rank adapter of each row, the adapter's index read
             from a device tensor: ``y[t] = x[t] W^T + s_i (x[t] A_i^T) B_i^T``, ``i = slot[t]``,
             nothing added where ``slot[t] < 0`` (``serving.fused_lora_forward_rows``).
* ``clip``   gradient norms over all tensors of each adapter (or of all adapters together), and the
             gradients scaled by ``min(1, max_norm / (norm + 1e-6))`` (``training.clip_adapter_grads``).
* ``adamw``  AdamW of many adapters, each with its own step count, learning rate and decay, the
             gradients clipped per adapter first; 16-bit weights keep float32 masters
             (``training.AdapterAdamW``).

Adapters' gradients and weights are laid out as the backward returns them: for a projection K -> N,
one flat buffer of the [r_i, K] blocks and one of the [N, r_i] blocks, adapter after adapter.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BETA1, BETA2, EPS, MAX_NORM = 0.9, 0.999, 1e-8, 1.0

# The seven projections of a Llama-3-8B block, the workload with 64 adapters of mixed ranks.
BLOCK_8B = "4096x4096,4096x1024,4096x1024,4096x4096,4096x14336,4096x14336,14336x4096"


def listed():
    return [
        # one token of one request, the smallest call of a decoding server
        {"name": "rows_one_token", "op": "rows", "rows": 1, "K": 4096, "N": 4096, "slots": 16, "ranks": "16",
         "dtype": "bf16", "order": "tokens"},
        # a decode step of 64 requests through a gate projection, adapters of mixed ranks
        {"name": "rows_decode_64", "op": "rows", "rows": 64, "K": 4096, "N": 14336, "slots": 64,
         "ranks": "8,16,32,64", "dtype": "bf16", "order": "tokens"},
        # a large decode step: nearly every token brings another of 512 adapters
        {"name": "rows_decode_250_of_512", "op": "rows", "rows": 250, "K": 4096, "N": 4096, "slots": 512,
         "ranks": "16", "dtype": "f16", "order": "tokens"},
        # prompts and single tokens in one batch
        {"name": "rows_prompts_8192", "op": "rows", "rows": 8192, "K": 4096, "N": 4096, "slots": 64,
         "ranks": "8,16,32,64", "dtype": "bf16", "order": "prompts"},
        # the small float32 workload
        {"name": "rows_f32_128", "op": "rows", "rows": 128, "K": 256, "N": 256, "slots": 4, "ranks": "8",
         "dtype": "f32", "order": "prompts"},
        # the small float32 workload's gradients, one norm over all
        {"name": "clip_f32_small", "op": "clip", "shapes": "256x256", "adapters": 4, "ranks": "8", "dtype": "f32",
         "each": False},
        # one projection, 16 jobs, each with its own norm, unrounded gradients
        {"name": "clip_16_jobs", "op": "clip", "shapes": "4096x4096", "adapters": 16, "ranks": "16", "dtype": "f32",
         "each": True},
        # a whole block's gradients of 64 jobs
        {"name": "clip_block_64_jobs", "op": "clip", "shapes": BLOCK_8B, "adapters": 64, "ranks": "8,16,32,64",
         "dtype": "bf16", "each": True},
        # the small float32 workload's step
        {"name": "adamw_f32_small", "op": "adamw", "shapes": "256x256", "adapters": 4, "ranks": "8", "dtype": "f32",
         "grad": "f32", "clip": True},
        # one projection, 16 jobs, float32 gradients of bf16 weights
        {"name": "adamw_16_jobs", "op": "adamw", "shapes": "4096x4096", "adapters": 16, "ranks": "16",
         "dtype": "bf16", "grad": "f32", "clip": True},
        # a whole block's step of 64 jobs
        {"name": "adamw_block_64_jobs", "op": "adamw", "shapes": BLOCK_8B, "adapters": 64, "ranks": "8,16,32,64",
         "dtype": "bf16", "grad": "bf16", "clip": True},
        # a 70B gate projection with 256 jobs of rank 64, no clipping
        {"name": "adamw_256_jobs_r64", "op": "adamw", "shapes": "8192x28672", "adapters": 256, "ranks": "64",
         "dtype": "bf16", "grad": "bf16", "clip": False},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rows", "rows", "clip", "adamw"])
    if op == "rows":
        if rng.random() < 0.2:  # float32: small problems, any size
            return {"op": "rows", "rows": _log_int(rng, 1, 300), "K": rng.randint(60, 700), "N": rng.randint(60, 700),
                    "slots": rng.randint(1, 12), "ranks": rng.choice(["8", "3,8", "1,16"]), "dtype": "f32",
                    "order": rng.choice(["tokens", "prompts"])}
        K, N = 8 * _log_int(rng, 64, 1792), 8 * _log_int(rng, 64, 1792)
        ranks = rng.choice(["16", "8,16,32,64", "64", "4,8", "20,48", "1,16,33"])
        most = 8192 // max(_rank_list(ranks))
        T = min(_log_int(rng, 1, 8192), 8192 * 4096 * 4096 // (K * N))
        return {"op": "rows", "rows": T, "K": K, "N": N, "slots": _log_int(rng, 1, most), "ranks": ranks,
                "dtype": rng.choice(["bf16", "f16"]), "order": rng.choice(["tokens", "prompts"])}
    shapes = ",".join("%dx%d" % (8 * _log_int(rng, 32, 1792), 8 * _log_int(rng, 32, 1792))
                      for _ in range(rng.randint(1, 7)))
    case = {"op": op, "shapes": shapes, "adapters": _log_int(rng, 1, 100),
            "ranks": rng.choice(["16", "8,16,32,64", "4", "5,24", "64", "1,16"])}
    if op == "clip":
        return {**case, "dtype": rng.choice(["f32", "bf16", "f16"]), "each": rng.random() < 0.7}
    dtype = rng.choice(["f32", "bf16", "f16"])
    return {**case, "dtype": dtype, "grad": rng.choice(["f32", dtype]), "clip": rng.random() < 0.7}


def _rank_list(text):
    return [int(r) for r in text.split(",")]


def _ranks(case, n):
    cycle = _rank_list(case["ranks"])
    return [cycle[i % len(cycle)] for i in range(n)]


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


# ------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = _generator(seed)
    return (_prepare_rows if case["op"] == "rows" else _prepare_training)(case, gen)


def _prepare_rows(case, gen):
    T, K, N, n = case["rows"], case["K"], case["N"], case["slots"]
    dt = DTYPES[case["dtype"]]
    ranks = _ranks(case, n)
    r = max(ranks)
    keep = torch.arange(r, device="cuda")[None] < torch.tensor(ranks, device="cuda")[:, None]
    a = torch.empty(n, r, K, dtype=dt, device="cuda")
    b = torch.empty(n, N, r, dtype=dt, device="cuda")
    a.copy_(_randn(gen, n, r, K).mul_(keep[:, :, None]) / math.sqrt(K))
    b.copy_(_randn(gen, n, N, r).mul_(keep[:, None, :]) * 0.02)
    scale = torch.empty(n, device="cuda").uniform_(0.5, 2.0, generator=gen)
    # the last of every eight draws is a row (or a request) without an adapter
    if case["order"] == "tokens":
        slot = torch.randint(0, 8 * n, (T,), generator=gen, device="cuda")
    else:  # requests of many lengths, one after another
        cuts = torch.randint(0, T, (max(1, T // 80),), generator=gen, device="cuda").sort().values
        request = torch.searchsorted(cuts, torch.arange(T, device="cuda"), right=True)
        slot = torch.randint(0, 8 * n, (cuts.numel() + 1,), generator=gen, device="cuda")[request]
    slot = torch.where(slot % 8 == 7, -1, slot // 8).to(torch.int32)
    state = {"case": case, "x": _randn(gen, T, K).to(dt), "w": (_randn(gen, N, K) / math.sqrt(K)).to(dt), "a": a,
             "b": b, "scale": scale, "slot": slot, "bank": None}
    if own:
        from lorafusion_b200.serving import AdapterBank
        bank = AdapterBank(n, r, K, N, dt, "cuda")
        scales = scale.tolist()
        for i in range(n):
            bank.load(i, a[i, :ranks[i]], b[i, :, :ranks[i]], scales[i])
        state["bank"] = bank
    return state


def _views(flats, shapes, ranks):
    """One dict of adapter id -> block for each flat buffer: [r_i, K] blocks, then [N, r_i] blocks."""
    dicts = []
    for j, (K, N) in enumerate(shapes):
        fa, fb = flats[2 * j], flats[2 * j + 1]
        da, db, row = {}, {}, 0
        for i, r in enumerate(ranks):
            da[i] = fa[row * K:(row + r) * K].view(r, K)
            db[i] = fb[row * N:(row + r) * N].view(N, r)
            row += r
        dicts += [da, db]
    return dicts


def _prepare_training(case, gen):
    n = case["adapters"]
    ranks, shapes = _ranks(case, n), _shapes(case)
    row_of = torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor(ranks, device="cuda"))
    widths = [w for s in shapes for w in s]
    # jobs far from one another in gradient size; of every eight the last one's norm is below the limit
    gain = torch.empty(n, device="cuda").uniform_(math.log(0.1), math.log(10.0), generator=gen).exp_()
    gain[7::8] = 1e-6
    gdt = DTYPES[case["dtype" if case["op"] == "clip" else "grad"]]
    rows = row_of.numel()
    grads = [(_randn(gen, rows, w) * gain[row_of][:, None]).to(gdt).view(-1) for w in widths]
    state = {"case": case, "row_of": row_of, "widths": widths, "grads": grads,
             "grad_dicts": _views(grads, shapes, ranks)}
    if case["op"] == "clip":
        return state
    dt = DTYPES[case["dtype"]]
    lr = [1e-4 * (1 + i % 5) for i in range(n)]
    decay = [0.01 * (i % 3) for i in range(n)]
    steps = torch.randint(0, 500, (n,), generator=gen, device="cuda").to(torch.int32)
    master = [0.02 * _randn(gen, rows * w) for w in widths]
    params = [p if dt == torch.float32 else p.to(dt) for p in master]
    master = None if dt == torch.float32 else torch.cat(master)
    total = rows * sum(widths)
    exp_avg = _randn(gen, total).mul_(0.01)
    exp_avg_sq = _randn(gen, total).mul_(0.01).square_()
    state |= {"params": params, "sizes": [rows * w for w in widths], "lr": lr, "decay": decay, "opt": None}
    if own:
        from lorafusion_b200.training import AdapterAdamW
        opt = AdapterAdamW(_views(params, shapes, ranks), lr=dict(enumerate(lr)),
                           weight_decay=dict(enumerate(decay)), betas=(BETA1, BETA2), eps=EPS,
                           max_norm=MAX_NORM if case["clip"] else None)
        opt.exp_avg.copy_(exp_avg)
        opt.exp_avg_sq.copy_(exp_avg_sq)
        opt.steps.copy_(steps)
        if master is not None:
            opt.master.copy_(master)
        state["opt"] = opt
    else:
        state |= {"exp_avg": exp_avg, "exp_avg_sq": exp_avg_sq, "steps": steps, "master": master,
                  "lr_dev": torch.tensor(lr, device="cuda", dtype=torch.float64),
                  "decay_dev": torch.tensor(decay, device="cuda", dtype=torch.float64)}
    return state


# ------------------------------------------------------------------------------------- one pass
def run(state):
    return {"rows": _run_rows, "clip": _run_clip, "adamw": _run_adamw}[state["case"]["op"]](state)


def _run_rows(s):
    if own:
        from lorafusion_b200.serving import fused_lora_forward_rows
        return {"y": fused_lora_forward_rows(s["x"], s["w"], s["bank"], s["slot"])}
    n, r, K = s["a"].shape
    x = s["x"].float()
    y = x @ s["w"].float().t()
    low = (x @ s["a"].float().view(n * r, K).t()).view(-1, n, r)
    pick = (s["slot"][:, None] == torch.arange(n, device="cuda")) * s["scale"]
    y += (low * pick[:, :, None]).view(-1, n * r) @ s["b"].float().transpose(1, 2).reshape(n * r, -1)
    return {"y": y.to(s["x"].dtype)}


def _squares(grads, widths, row_of, n):
    """Sum of squares of each adapter's gradients, in 64 bits."""
    rows = row_of.numel()
    sums = [g.view(rows, w).float().square().sum(1, dtype=torch.float64) for g, w in zip(grads, widths)]
    return torch.zeros(n, dtype=torch.float64, device="cuda").index_add_(0, row_of, torch.stack(sums).sum(0))


def _run_clip(s):
    case = s["case"]
    if own:
        from lorafusion_b200.training import clip_adapter_grads
        return {"norms": clip_adapter_grads(s["grad_dicts"], MAX_NORM, per_adapter=case["each"]), "grads": s["grads"]}
    sums = _squares(s["grads"], s["widths"], s["row_of"], case["adapters"])
    norms = (sums if case["each"] else sums.sum()).sqrt()
    factor = (MAX_NORM / (norms + 1e-6)).clamp(max=1.0).float()
    rows = s["row_of"].numel()
    by_row = (factor[s["row_of"]] if case["each"] else factor.expand(rows))[:, None]
    [g.copy_((g.view(rows, w).float() * by_row).view(-1)) for g, w in zip(s["grads"], s["widths"])]
    return {"norms": norms.float(), "grads": s["grads"]}


def _run_adamw(s):
    case = s["case"]
    if own:
        opt = s["opt"]
        norms = opt.step(s["grad_dicts"])
        return {"params": s["params"], "exp_avg": opt.exp_avg, "exp_avg_sq": opt.exp_avg_sq, "steps": opt.steps,
                "master": opt.master if case["dtype"] != "f32" else None, "norms": norms if case["clip"] else None}
    row_of, rows = s["row_of"], s["row_of"].numel()
    norms, factor = None, torch.ones(case["adapters"], dtype=torch.float64, device="cuda")
    if case["clip"]:
        norms = _squares(s["grads"], s["widths"], row_of, case["adapters"]).sqrt()
        factor = (MAX_NORM / (norms + 1e-6)).clamp(max=1.0)
        norms = norms.float()
    s["steps"] += 1
    t = s["steps"].double()
    by_row = lambda v: v.float()[row_of][:, None]  # noqa: E731
    factor, shrink = by_row(factor), by_row(1.0 - s["lr_dev"] * s["decay_dev"])
    size, root = by_row(s["lr_dev"] / (1.0 - BETA1 ** t)), by_row((1.0 - BETA2 ** t).sqrt())
    masters = s["params"] if s["master"] is None else s["master"].split(s["sizes"])
    parts = zip(s["params"], s["grads"], masters, s["exp_avg"].split(s["sizes"]), s["exp_avg_sq"].split(s["sizes"]),
                s["widths"])
    [_update(p.view(rows, w), g.view(rows, w), q.view(rows, w), m.view(rows, w), v.view(rows, w), factor, shrink,
             size, root) for p, g, q, m, v, w in parts]
    return {"params": s["params"], "exp_avg": s["exp_avg"], "exp_avg_sq": s["exp_avg_sq"], "steps": s["steps"],
            "master": s["master"], "norms": norms}


def _update(p, g, q, m, v, factor, shrink, size, root):
    g = g.float() * factor
    m.mul_(BETA1).add_(g * (1.0 - BETA1))
    v.mul_(BETA2).add_(g * g * (1.0 - BETA2))
    q.copy_(q * shrink - size * m / (v.sqrt() / root + EPS))
    if p is not q and p.dtype != torch.float32:
        p.copy_(q)


# ------------------------------------------------------------------------------------- what it needs
def work(case):
    if case["op"] == "rows":
        T, K, N, n = case["rows"], case["K"], case["N"], case["slots"]
        ranks, size = _ranks(case, n), 4 if case["dtype"] == "f32" else 2
        mean = sum(ranks) / n
        chosen = T if case["order"] == "tokens" else max(1, T // 80) + 1
        active = n * (1.0 - (1.0 - 7.0 / (8.0 * n)) ** chosen)  # distinct adapters that the rows name
        return {"bytes": size * (T * K + N * K + T * N + active * mean * (K + N)) + 4 * T,
                "flops": 2.0 * T * K * N + 2.0 * T * 7 / 8 * mean * (K + N)}
    n = case["adapters"]
    ranks = _ranks(case, n)
    width = sum(K + N for K, N in _shapes(case))
    total = sum(ranks) * width
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "clip":
        clipped = sum(r for i, r in enumerate(ranks) if i % 8 != 7) * width if case["each"] else total
        return {"bytes": size[case["dtype"]] * (total + clipped), "flops": 3.0 * total}
    per = size[case["grad"]] + 16 + (8 if case["dtype"] == "f32" else 8 + 2)
    return {"bytes": per * total, "flops": 15.0 * total}


# ------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    return {"rows": _exact_rows, "clip": _exact_clip, "adamw": _exact_adamw}[case["op"]](s)


def _exact_rows(s):
    x = s["x"].double()
    y = x.mm(s["w"].double().t())
    for i in s["slot"].unique().tolist():
        if i >= 0:
            at = (s["slot"] == i).nonzero().view(-1)
            y[at] += s["scale"][i].double() * x[at].mm(s["a"][i].double().t()).mm(s["b"][i].double().t())
    return {"y": y}


def _exact_norms(s, blocks):
    sums = [sum(float(d[i].double().pow(2).sum()) for d in blocks) for i in range(s["case"]["adapters"])]
    return torch.tensor(sums, dtype=torch.float64, device="cuda")


def _exact_clip(s):
    case, dicts = s["case"], s["grad_dicts"]
    sums = _exact_norms(s, dicts)
    norms = sums.sqrt() if case["each"] else sums.sum().sqrt()
    factors = [min(1.0, MAX_NORM / (v + 1e-6)) for v in norms.expand(case["adapters"]).tolist()]
    return {"norms": norms, "grads": [torch.cat([d[i].double().view(-1) * f for i, f in enumerate(factors)])
                                      for d in dicts]}


def _exact_adamw(s):
    case, n = s["case"], s["case"]["adapters"]
    factors, norms = [1.0] * n, None
    if case["clip"]:
        norms = _exact_norms(s, s["grad_dicts"]).sqrt()
        factors = [min(1.0, MAX_NORM / (v + 1e-6)) for v in norms.tolist()]
    steps = [t + 1 for t in s["steps"].tolist()]
    master = torch.cat([p.double() for p in s["params"]]) if s["master"] is None else s["master"].double()
    m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    at = 0
    for d in s["grad_dicts"]:
        for i in range(n):
            here = slice(at, at + d[i].numel())
            at += d[i].numel()
            g = d[i].double().view(-1) * factors[i]
            m[here] = BETA1 * m[here] + (1 - BETA1) * g
            v[here] = BETA2 * v[here] + (1 - BETA2) * g * g
            mean, second = m[here] / (1 - BETA1 ** steps[i]), v[here] / (1 - BETA2 ** steps[i])
            old = master[here]
            master[here] = old - s["lr"][i] * s["decay"][i] * old - s["lr"][i] * mean / (second.sqrt() + EPS)
    return {"params": list(master.split(s["sizes"])), "exp_avg": m, "exp_avg_sq": v,
            "steps": torch.tensor(steps, dtype=torch.int32, device="cuda"),
            "master": None if s["master"] is None else master, "norms": norms}
