"""Cases of adapters trained and served over a frozen weight held in 4 bits, in plain torch and through this package.

* ``quant``   a weight [N, K] to microscaled 4-bit floating point and back: blocks of 32 along K share a power of two,
              ``2^(floor(log2(max |w|)) - 2)``, each element is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it, ties
              to the even code, larger ones 6 (``quant.quantize_weight`` and ``MX4Weight.dequantize``).
* ``linear``  the product with such a weight: ``y = x V^T`` and its gradient ``grad_x = g V``, V the values that the
              codes stand for (``quant.mx4_linear``, ``quant.mx4_linear_backward``).
* ``rows``    that product with the low-rank adapter of each row, ``y[t] = x[t] V^T + s_i (x[t] A_i^T) B_i^T``, the
              adapter's slot read from a device tensor (``serving.fused_lora_forward_rows``).
* ``train``   the packed adapters' forward and backward with dropout in front of each adapter,
              ``y = x W^T + s_i / (1 - p_i) (m x) A_i^T B_i^T``; the mask m comes from a counter-based generator and is
              never stored; W dense or in 4 bits (``b200_ops.fused_lora_forward`` / ``fused_lora_backward``).

Dropout's numbers: Philox 4x32 with ten rounds (Salmon et al., 2011), key the two halves of the seed, counter
(k // 8, row, the two halves of the offset).  Element k of a row takes 16 of the 128 bits: word (k % 8) // 2, the low
half where k is even.  It is kept where that number is at least ``round(65536 p_i)``, and p_i is that over 65536.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # a small projection of an odd size: its blocks and tiles end in the middle
        {"name": "quant_small_odd", "op": "quant", "N": 250, "K": 700, "dtype": "f16"},
        # a gate projection of an 8B block, once when the model is loaded
        {"name": "quant_gate_8b", "op": "quant", "N": 14336, "K": 4096, "dtype": "bf16"},
        # an uneven batch through an odd projection
        {"name": "linear_333_rows", "op": "linear", "pass": "forward", "rows": 333, "K": 1000, "N": 1048,
         "dtype": "f16"},
        # one fused batch of a 4096 projection
        {"name": "linear_4096", "op": "linear", "pass": "forward", "rows": 4096, "K": 4096, "N": 4096, "dtype": "bf16"},
        # ... and the gradient that flows back through the frozen weight
        {"name": "linear_4096_grad", "op": "linear", "pass": "backward", "rows": 4096, "K": 4096, "N": 4096,
         "dtype": "bf16"},
        # one token of one request, the smallest call of a decoding server
        {"name": "rows_one_token", "op": "rows", "rows": 1, "K": 4096, "N": 4096, "slots": 16, "ranks": "16",
         "dtype": "bf16"},
        # a decode step of 64 requests through a gate projection, adapters of mixed ranks
        {"name": "rows_decode_64", "op": "rows", "rows": 64, "K": 4096, "N": 14336, "slots": 64, "ranks": "8,16,32,64",
         "dtype": "bf16"},
        # the small float32 workload's step
        {"name": "train_f32_small", "op": "train", "pass": "both", "rows": 128, "K": 256, "N": 256, "adapters": 4,
         "ranks": "8", "rates": "0.1", "dtype": "f32", "base": "dense"},
        # a fused batch of 16 jobs, dense weight
        {"name": "train_dense_forward", "op": "train", "pass": "forward", "rows": 4096, "K": 4096, "N": 4096,
         "adapters": 16, "ranks": "16", "rates": "0.05,0.1", "dtype": "bf16", "base": "dense"},
        {"name": "train_dense_backward", "op": "train", "pass": "backward", "rows": 4096, "K": 4096, "N": 4096,
         "adapters": 16, "ranks": "16", "rates": "0.05,0.1", "dtype": "bf16", "base": "dense"},
        # 28 jobs of mixed ranks over a weight in 4 bits, some without dropout
        {"name": "train_mx4_forward", "op": "train", "pass": "forward", "rows": 8192, "K": 4096, "N": 4096,
         "adapters": 28, "ranks": "8,16,32,64", "rates": "0.05,0.1,0", "dtype": "bf16", "base": "mx4"},
        {"name": "train_mx4_backward", "op": "train", "pass": "backward", "rows": 8192, "K": 4096, "N": 4096,
         "adapters": 28, "ranks": "8,16,32,64", "rates": "0.05,0.1,0", "dtype": "bf16", "base": "mx4"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["quant", "linear", "linear", "rows", "train", "train"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "quant":
        K = _log_int(rng, 20, 14336)
        return {"op": op, "N": min(_log_int(rng, 20, 14336), 14336 * 4096 // K), "K": K, "dtype": dtype}
    K, N = 8 * _log_int(rng, 32, 1792), 8 * _log_int(rng, 32, 1792)
    rows = min(_log_int(rng, 1, 8192), 8192 * 4096 * 4096 // (K * N))
    ranks = rng.choice(["16", "8,16,32,64", "64", "4,8", "20,48", "1,16,33"])
    if op == "linear":
        if rng.random() < 0.15:  # odd sizes are small problems
            rows, K, N = _log_int(rng, 1, 300), rng.randint(33, 500), rng.randint(33, 500)
        return {"op": op, "pass": rng.choice(["forward", "forward", "backward"]), "rows": rows, "K": K, "N": N,
                "dtype": dtype}
    if op == "rows":
        most = max(1, min(4096, (1 << 25) // (K + N)) // max(_list(ranks)))
        return {"op": op, "rows": rows, "K": K, "N": N, "slots": _log_int(rng, 1, most), "ranks": ranks, "dtype": dtype}
    rates = rng.choice(["0.1", "0.05,0.1,0", "0.5", "0.01,0.3", "0.25"])
    case = {"op": op, "pass": rng.choice(["forward", "backward", "both"]), "rows": rows, "K": K, "N": N,
            "adapters": _log_int(rng, 1, 28), "ranks": ranks, "rates": rates, "dtype": dtype,
            "base": rng.choice(["dense", "mx4"])}
    if rng.random() < 0.2:
        case |= {"rows": _log_int(rng, 1, 300), "K": rng.randint(60, 500), "N": rng.randint(60, 500), "dtype": "f32",
                 "base": "dense", "adapters": rng.randint(1, 8)}
    return case | {"adapters": min(case["adapters"], case["rows"])}


def _list(text):
    return [int(r) for r in text.split(",")]


def _cycle(text, n, kind=int):
    cycle = [kind(v) for v in text.split(",")]
    return [cycle[i % len(cycle)] for i in range(n)]


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


# ------------------------------------------------------------------------------------- the formats, plainly
def _power(e):
    """2^e for whole e in -1022 .. 1023, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _encode(w):
    """Codes [N, K] (bit 3 the sign, bits 0-2 the index into VALUES) and the exponents [N, ceil(K / 32)] of w."""
    N, K = w.shape
    blocks = torch.zeros(N, -(-K // 32) * 32, dtype=w.dtype, device=w.device)
    blocks[:, :K] = w
    blocks = blocks.view(N, -1, 32)
    top = blocks.abs().amax(2).float()
    e = (torch.frexp(top).exponent - 3).clamp(min=-127)
    e = torch.where(top == 0, -127, e)
    v = blocks.double() * _power(-e)[:, :, None]
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = ((a / step).round() * step).clamp(max=6.0)
    code = sum((q > f).to(torch.uint8) for f in VALUES[:-1])
    code |= torch.signbit(v).to(torch.uint8) << 3
    return code.view(N, -1)[:, :K].contiguous(), e.to(torch.int16)


def _decode(code, e, dtype=torch.float32):
    """What codes and exponents stand for, in 32 bits (or 64)."""
    N, K = code.shape
    signed = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=dtype, device=code.device)
    scale = _power(e).to(dtype).repeat_interleave(32, dim=1)[:, :K]
    return signed[code.int()] * scale


M32 = 0xFFFFFFFF


def _keep(rows, K, thresholds, seed, offset):
    """Truth values [rows, K]: which elements dropout keeps; thresholds [rows] are whole numbers of 1/65536."""
    c0 = torch.arange(-(-K // 8), device="cuda")[None].expand(rows, -1).clone()
    c1 = torch.arange(rows, device="cuda")[:, None].expand_as(c0).clone()
    c2, c3 = torch.full_like(c0, offset & M32), torch.full_like(c0, offset >> 32)
    k0, k1 = seed & M32, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64 bits: the halves come out whatever the sign
        c0, c1, c2, c3 = ((p1 >> 32) & M32) ^ c1 ^ k0, p1 & M32, ((p0 >> 32) & M32) ^ c3 ^ k1, p0 & M32
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    words = torch.stack([c0, c1, c2, c3], 2)
    number = torch.stack([words & 0xFFFF, words >> 16], 3).view(rows, -1)[:, :K]
    return number >= thresholds[:, None]


# ------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    N, K = case["N"], case["K"]
    # rows of a trained weight differ in size
    w = (_randn(gen, N, K) / math.sqrt(K) * torch.exp(0.5 * _randn(gen, N, 1))).to(dt)
    if case["op"] == "quant":
        return {"case": case, "w": w}
    state = {"case": case, "w": w}
    if case.get("base", "mx4") == "mx4":
        if own:
            from lorafusion_b200.quant import quantize_weight
            state["mx4"] = quantize_weight(w)
        else:
            state["code"], state["e"] = _encode(w)
    T = case["rows"]
    state["x"] = _randn(gen, T, K).to(dt)
    state["g"] = _randn(gen, T, N).to(dt) if case.get("pass", "forward") != "forward" else None
    if case["op"] == "rows":
        return _prepare_rows(case, gen, dt, state)
    if case["op"] == "train":
        return _prepare_train(case, gen, dt, state, seed)
    return state


def _prepare_rows(case, gen, dt, state):
    n, N, K, T = case["slots"], case["N"], case["K"], case["rows"]
    ranks = _cycle(case["ranks"], n)
    a = [(_randn(gen, r, K) / math.sqrt(K)).to(dt) for r in ranks]
    b = [(_randn(gen, N, r) * 0.02).to(dt) for r in ranks]
    scale = torch.empty(n, device="cuda").uniform_(0.5, 2.0, generator=gen)
    # the last of every eight draws is a row without an adapter
    slot = torch.randint(0, 8 * n, (T,), generator=gen, device="cuda")
    slot = torch.where(slot % 8 == 7, -1, slot // 8).to(torch.int32)
    state |= {"a": a, "b": b, "scale": scale, "slot": slot}
    if own:
        from lorafusion_b200.serving import AdapterBank
        state["bank"] = AdapterBank(n, max(ranks), K, N, dt, "cuda")
        for i, s in enumerate(scale.tolist()):
            state["bank"].load(i, a[i], b[i], s)
    else:  # side by side: rank rows of all adapters, and whose they are
        state |= {"a_all": torch.cat(a), "b_all": torch.cat(b, 1),
                  "owner": torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor(ranks, device="cuda"))}
    return state


def _prepare_train(case, gen, dt, state, seed):
    n, N, K, T = case["adapters"], case["N"], case["K"], case["rows"]
    ranks, rates = _cycle(case["ranks"], n), _cycle(case["rates"], n, float)
    # jobs of many lengths, one after another
    cuts = torch.randperm(T - 1, generator=gen, device="cuda")[:n - 1].add(1).sort().values.tolist() if T > 1 else []
    spans = [(lo, hi, i) for i, (lo, hi) in enumerate(zip([0] + cuts, cuts + [T]))]
    a = {i: (_randn(gen, r, K) / math.sqrt(K)).to(dt) for i, r in enumerate(ranks)}
    b = {i: (_randn(gen, N, r) * 0.02).to(dt) for i, r in enumerate(ranks)}
    state |= {"a": a, "b": b, "spans": spans, "ranks": ranks, "rates": rates, "alpha": 16.0,
              "seed": 0x9E3779B97F4A7C15 * (seed + 1) & (1 << 63) - 1, "offset": (seed % 1000 << 33) + 5}
    if own:
        from lorafusion_b200.b200_ops import AdapterDropout
        from lorafusion_b200.config import AdapterSpec, TileRoute, TileRoutingConfig
        state["adapters"] = {i: AdapterSpec(i, r, 16.0, K, N) for i, r in enumerate(ranks)}
        state["routing"] = TileRoutingConfig(128, [TileRoute(*s) for s in spans])
        state["dropout"] = AdapterDropout(dict(enumerate(rates)), state["seed"], state["offset"])
    return state


# ------------------------------------------------------------------------------------- one pass
def run(state):
    one = {"quant": _run_quant, "linear": _run_linear, "rows": _run_rows, "train": _run_train}[state["case"]["op"]]
    return one(state)


def _run_quant(s):
    if own:
        from lorafusion_b200.quant import quantize_weight
        return {"values": quantize_weight(s["w"]).dequantize()}
    return {"values": _decode(*_encode(s["w"])).to(s["w"].dtype)}


def _run_linear(s):
    forward = s["case"]["pass"] == "forward"
    if own:
        from lorafusion_b200.quant import mx4_linear, mx4_linear_backward
        return {"y": mx4_linear(s["x"], s["mx4"])} if forward else {"grad_x": mx4_linear_backward(s["g"], s["mx4"])}
    v = _decode(s["code"], s["e"])
    if forward:
        return {"y": (s["x"].float() @ v.t()).to(s["x"].dtype)}
    return {"grad_x": (s["g"].float() @ v).to(s["g"].dtype)}


def _run_rows(s):
    if own:
        from lorafusion_b200.serving import fused_lora_forward_rows
        return {"y": fused_lora_forward_rows(s["x"], s["mx4"], s["bank"], s["slot"])}
    x = s["x"].float()
    y = x @ _decode(s["code"], s["e"]).t()
    low = (x @ s["a_all"].float().t()) * ((s["slot"][:, None] == s["owner"]) * s["scale"][s["owner"]])
    return {"y": (y + low @ s["b_all"].float().t()).to(s["x"].dtype)}


def _thresholds(s, n_rows):
    t = torch.zeros(n_rows, dtype=torch.int64, device="cuda")
    for lo, hi, i in s["spans"]:
        t[lo:hi] = int(round(s["rates"][i] * 65536))
    return t


def _run_train(s):
    which = s["case"]["pass"]
    if own:
        from lorafusion_b200.b200_ops import fused_lora_backward, fused_lora_forward
        w = s["mx4"] if "mx4" in s else s["w"]
        out = {}
        if which != "backward":
            out["y"] = fused_lora_forward(s["x"], w, s["a"], s["b"], s["adapters"], s["routing"], dropout=s["dropout"])
        if which != "forward":
            gx, ga, gb = fused_lora_backward(s["g"], s["x"], w, s["a"], s["b"], s["adapters"], s["routing"],
                                             dropout=s["dropout"])
            out |= {"grad_x": gx, "grad_a": list(ga.values()), "grad_b": list(gb.values())}
        return out
    dt = s["x"].dtype
    T, K = s["x"].shape
    w = _decode(s["code"], s["e"]) if "code" in s else s["w"].float()
    x = s["x"].float()
    kept = _keep(T, K, _thresholds(s, T), s["seed"], s["offset"])
    xm = x * kept
    y = x @ w.t() if which != "backward" else None
    g = s["g"].float() if which != "forward" else None
    gx = g @ w if which != "forward" else None
    ga, gb = [], []
    for lo, hi, i in s["spans"]:
        factor = s["alpha"] / s["ranks"][i] * 65536.0 / (65536 - int(round(s["rates"][i] * 65536)))
        a, b = s["a"][i].float(), s["b"][i].float()
        low = factor * (xm[lo:hi] @ a.t())
        if y is not None:
            y[lo:hi] += low @ b.t()
        if g is not None:
            glow = factor * (g[lo:hi] @ b)
            gx[lo:hi] += (glow @ a) * kept[lo:hi]
            ga.append((glow.t() @ xm[lo:hi]).to(dt))
            gb.append((g[lo:hi].t() @ low).to(dt))
    out = {"y": y.to(dt)} if y is not None else {}
    return out if g is None else out | {"grad_x": gx.to(dt), "grad_a": ga, "grad_b": gb}


# ------------------------------------------------------------------------------------- what it needs
def work(case):
    N, K, size = case["N"], case["K"], SIZE[case["dtype"]]
    if case["op"] == "quant":
        return {"bytes": 2 * size * N * K, "flops": 4.0 * N * K}
    T = case["rows"]
    held = N * K * 17 / 32 if case.get("base", "mx4") == "mx4" else size * N * K  # 4 bits, and 8 for 32 elements
    if case["op"] == "linear":
        return {"bytes": held + size * T * (N + K), "flops": 2.0 * T * N * K}
    ranks = _cycle(case["ranks"], case["slots" if case["op"] == "rows" else "adapters"])
    mean = sum(ranks) / len(ranks)
    if case["op"] == "rows":
        n = case["slots"]
        active = n * (1.0 - (1.0 - 7.0 / (8.0 * n)) ** T)  # distinct adapters that the rows name
        return {"bytes": held + size * (T * (N + K) + active * mean * (K + N)) + 4 * T,
                "flops": 2.0 * T * N * K + 2.0 * T * 7 / 8 * mean * (K + N)}
    adapters = size * sum(ranks) * (K + N)
    total = {"bytes": 0.0, "flops": 0.0}
    if case["pass"] != "backward":
        total["bytes"] += held + size * T * (N + K) + adapters
        total["flops"] += 2.0 * T * N * K + 2.0 * T * mean * (N + K)
    if case["pass"] != "forward":  # x, g and grad_x; the adapters and their gradients
        total["bytes"] += held + size * T * (N + 2 * K) + 2 * adapters
        total["flops"] += 2.0 * T * N * K + 2.0 * T * mean * (3 * K + 2 * N)
    return total


# ------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    if case["op"] == "quant":
        return {"values": _exact_values(s["w"])}
    v = _exact_values(s["w"]) if case.get("base", "mx4") == "mx4" else s["w"].double()
    x = s["x"].double()
    if case["op"] == "linear":
        return {"y": x.mm(v.t())} if case["pass"] == "forward" else {"grad_x": s["g"].double().mm(v)}
    if case["op"] == "rows":
        y = x.mm(v.t())
        for i in s["slot"].unique().tolist():
            if i >= 0:
                at = (s["slot"] == i).nonzero().view(-1)
                y[at] += s["scale"][i].double() * x[at].mm(s["a"][i].double().t()).mm(s["b"][i].double().t())
        return {"y": y}
    return _exact_train(case, s, x, v)


def _exact_values(w):
    """Each element becomes the nearest multiple of its block's unit; between two, the one of the even code."""
    N, K = w.shape
    out = torch.empty(N, K, dtype=torch.float64, device=w.device)
    grid = torch.tensor(VALUES, dtype=torch.float64, device=w.device)
    even = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=w.device)
    for lo in range(0, K, 32):
        block = w[:, lo:lo + 32].double()
        top = block.abs().max(1, keepdim=True).values
        # the largest power of two that is not above top, over four
        e = torch.floor(torch.log2(top.clamp(min=2.0 ** -140)))
        e = e + (torch.exp2(e + 1) <= top) - (torch.exp2(e) > top).double()
        unit = torch.exp2(e - 2).clamp(min=2.0 ** -127)
        a = block.abs() / unit
        low = torch.bucketize(a, even, right=False)  # a midpoint falls to the lower code
        at = torch.bucketize(a, even, right=True)    # ... and to the upper one
        q = torch.where(low % 2 == 0, grid[low], grid[at])
        out[:, lo:lo + 32] = torch.copysign(q * unit, block)
    return out


def _exact_train(case, s, x, v):
    T, K = s["x"].shape
    group = np.arange(-(-K // 8), dtype=np.uint64)[None, :]
    ctr = [np.broadcast_to(group, (T, group.size)).copy(),
           np.broadcast_to(np.arange(T, dtype=np.uint64)[:, None], (T, group.size)).copy(),
           np.full((T, group.size), s["offset"] % 2 ** 32, dtype=np.uint64),
           np.full((T, group.size), s["offset"] // 2 ** 32, dtype=np.uint64)]
    low32, shift = np.uint64(M32), np.uint64(32)
    key = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32]
    for r in range(10):
        k0, k1 = np.uint64((key[0] + r * 0x9E3779B9) % 2 ** 32), np.uint64((key[1] + r * 0xBB67AE85) % 2 ** 32)
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(b >> shift) ^ ctr[1] ^ k0, b & low32, (a >> shift) ^ ctr[3] ^ k1, a & low32]
    numbers = np.empty((T, group.size, 8), dtype=np.int32)
    for i, word in enumerate(ctr):
        numbers[:, :, 2 * i] = (word % np.uint64(65536)).astype(np.int32)
        numbers[:, :, 2 * i + 1] = (word // np.uint64(65536)).astype(np.int32)
    numbers = torch.from_numpy(numbers.reshape(T, -1)[:, :K]).to(x.device)
    which, out = case["pass"], {}
    y = x.mm(v.t()) if which != "backward" else None
    g = s["g"].double() if which != "forward" else None
    gx = g.mm(v) if which != "forward" else None
    ga, gb = [], []
    for lo, hi, i in s["spans"]:
        t = int(round(s["rates"][i] * 65536))
        xi = torch.where(numbers[lo:hi] < t, 0.0, x[lo:hi]) / (1.0 - t / 65536)
        a, b = s["a"][i].double(), s["b"][i].double()
        si = s["alpha"] / s["ranks"][i]
        if y is not None:
            y[lo:hi] += si * xi.mm(a.t()).mm(b.t())
        if g is not None:
            gi = si * g[lo:hi].mm(b)
            gx[lo:hi] += torch.where(numbers[lo:hi] < t, 0.0, gi.mm(a)) / (1.0 - t / 65536)
            ga.append(gi.t().mm(xi))
            gb.append(si * g[lo:hi].t().mm(xi.mm(a.t())))
    if y is not None:
        out["y"] = y
    return out if g is None else out | {"grad_x": gx, "grad_a": ga, "grad_b": gb}
