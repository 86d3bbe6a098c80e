"""What the serving and training operators refuse, and their host-side plans (no GPU needed)."""

import ctypes

import numpy as np
import pytest
import torch

from lorafusion_b200 import _native as nat
from lorafusion_b200.serving import AdapterBank, fused_lora_forward_rows
from lorafusion_b200.training import AdapterAdamW, clip_adapter_grads

C_TYPES = {"int32_t": 4, "uint32_t": 4, "float": 4, "int64_t": 8, "uint64_t": 8, "size_t": 8, "double": 8}


def _fields(name):
    """(field, bytes) of a struct of the public header; pointers are 8 bytes."""
    text = open(nat.HEADER_PATH).read()
    body = text.split("typedef struct %s {" % name)[1].split("} %s;" % name)[0]
    out = []
    for ln in body.splitlines():
        decl = ln.split("/*")[0].strip().rstrip(";")
        if not decl:
            continue
        kind = decl.split()[1] if decl.startswith("const") else decl.split()[0]
        size = 8 if "*" in decl else C_TYPES[kind]
        names = decl.split("*")[-1] if "*" in decl else decl.split(None, 1)[1]
        out += [(n.strip(), size) for n in names.split(",")]
    return out


@pytest.mark.parametrize("name, cls", [("lf_rows_problem", nat.RowsProblem), ("lf_adamw_args", nat.AdamWArgs),
                                       ("lf_bank_adapter", nat.BankAdapter)])
def test_structs_match_the_header(name, cls):
    assert _fields(name) == [(f, getattr(cls, f).size) for f, _ in cls._fields_]


@pytest.mark.parametrize("name, layout", [("lf_grad_tensor", nat.GRAD_TENSOR), ("lf_adamw_tensor", nat.ADAMW_TENSOR)])
def test_records_match_the_header(name, layout):
    dt = np.dtype(layout)
    assert _fields(name) == [(f, dt[f].itemsize) for f in dt.names]


def test_host_tensors_are_refused():
    x = torch.zeros(4, 16)
    with pytest.raises(ValueError):
        AdapterBank(2, 8, 16, 16, device="cpu")
    with pytest.raises(ValueError):
        fused_lora_forward_rows(x, torch.zeros(16, 16), None, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        clip_adapter_grads([{0: x}], 1.0)
    with pytest.raises(ValueError):
        AdapterAdamW([{0: x}])


@pytest.mark.parametrize("args", [(0, 8, 16, 16), (1 << 24, 8, 16, 16), (2, 0, 16, 16), (2, 129, 16, 16),
                                  (2, 8, 0, 16), (2, 8, 16, 0), (2, 8, 16, 16, torch.int8), (2, 8, (1 << 24) + 1, 16),
                                  (2, 8, 16, (1 << 24) + 1), (1 << 23, 128, 16, 64)])
def test_bank_sizes(args):
    with pytest.raises(ValueError):
        AdapterBank(*args, device="cuda:0")


def _rows(**kw):
    p = nat.RowsProblem(nat.LF_BF16, 4, 16, 16, 2, 16, 4, 0, 16, *([256] * 7))
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_rows_entry_refuses_before_any_launch():
    L = nat.lib()
    ws = L.lf_rows_workspace_bytes(4, 16, 16, nat.LF_BF16)
    assert ws == 8 * 256 and L.lf_rows_workspace_bytes(4, 16, 16, nat.LF_F32) == 3 * 256
    assert [L.lf_rows_launch_count(T, 64) for T in (0, 1, 256, 257, 8192, 8193, 16384)] == [0, 2, 2, 4, 4, 6, 8]
    assert [L.lf_rows_launch_count(T, 32) for T in (257, 512, 513)] == [2, 2, 4]
    call = lambda p, y=256, w=256, n=ws: L.lf_rows_forward(p, y, w, n, None)  # noqa: E731
    for kw in (dict(dtype=3), dict(dtype=-1), dict(T=-1), dict(K=-1), dict(N=-1), dict(n_slots=-1), dict(r_pad=8),
               dict(r_pad=256), dict(row_slot_bytes=2), dict(ldx=15), dict(x_dev=None), dict(w_dev=None),
               dict(row_slot_dev=None), dict(a_bank_dev=None), dict(b_bank_dev=None), dict(slot_rank_dev=None),
               dict(slot_scale_dev=None), dict(b_bank_dev=264)):
        assert call(_rows(**kw)) == nat.LF_ERR_INVALID_ARG, kw
    assert call(_rows(n_slots=1 << 24)) == nat.LF_ERR_UNSUPPORTED
    assert call(_rows(K=(1 << 24) + 1, ldx=1 << 25)) == call(_rows(N=(1 << 24) + 1), n=1 << 60) == nat.LF_ERR_UNSUPPORTED
    assert call(_rows(n_slots=(1 << 24) - 1, N=136), n=1 << 40) == nat.LF_ERR_UNSUPPORTED  # more than 31 bits of bank rows
    assert call(_rows(), y=None) == nat.LF_ERR_INVALID_ARG
    assert call(_rows(), w=264) == nat.LF_ERR_INVALID_ARG
    assert call(_rows(), w=None) == nat.LF_ERR_CAPACITY and call(_rows(), n=ws - 1) == nat.LF_ERR_CAPACITY
    assert L.lf_rows_forward(None, 256, 256, ws, None) == nat.LF_ERR_INVALID_ARG
    assert call(_rows(T=0, x_dev=None)) == nat.LF_OK and call(_rows(N=0)) == nat.LF_OK


def test_bank_load_refuses_before_any_launch():
    def call(**kw):
        d = dict(dtype=nat.LF_BF16, K=32, N=24, r_pad=16, rank=4, scale=1.0, lda=32, ldb=4, a_dev=256, b_dev=256,
                 slot_a_dev=256, slot_b_dev=256, slot_rank_dev=256, slot_scale_dev=256)
        return nat.lib().lf_bank_load(nat.BankAdapter(**{**d, **kw}), None)

    for kw in (dict(dtype=3), dict(K=0), dict(N=-1), dict(r_pad=8), dict(r_pad=256), dict(rank=0), dict(rank=17),
               dict(lda=31), dict(ldb=3), dict(a_dev=None), dict(b_dev=None), dict(slot_a_dev=None),
               dict(slot_b_dev=None), dict(slot_rank_dev=None), dict(slot_scale_dev=None)):
        assert call(**kw) == nat.LF_ERR_INVALID_ARG, kw
    assert nat.lib().lf_bank_load(None, None) == nat.LF_ERR_INVALID_ARG


def _grads(*rows):
    return np.array(list(rows), dtype=np.dtype(nat.GRAD_TENSOR))


def test_clip_entry_refuses_before_any_launch():
    L = nat.lib()
    good = _grads((4096, 100, nat.LF_F32, 0), (8192, 100, nat.LF_BF16, 1))

    def call(rec, groups=2, inf=0, scale=1, limit=1.0, norms=256, ws=256, n=None):
        need = L.lf_grad_clip_workspace_bytes(rec.ctypes.data, len(rec), groups)
        return L.lf_grad_clip(rec.ctypes.data, len(rec), groups, inf, scale, limit, norms, ws,
                              need if n is None else n, None)

    assert L.lf_grad_clip_workspace_bytes(good.ctypes.data, 2, 2) == 3 * 256
    for bad in (_grads((4096, 100, 3, 0)), _grads((4096, 100, 0, 2)), _grads((4096, 100, 0, -1)),
                _grads((0, 100, 0, 0)), _grads((4098, 100, nat.LF_F32, 0)), _grads((4097, 100, nat.LF_F16, 0)),
                _grads((4096, 1 << 32, 0, 0))):
        assert call(bad) == nat.LF_ERR_INVALID_ARG, bad
        assert L.lf_grad_clip_workspace_bytes(bad.ctypes.data, 1, 2) == 0
    for bad in (_grads((4096, 100, 0, 0), (4096, 100, 0, 1)), _grads((4400, 100, 0, 0), (4096, 100, 0, 1)),
                _grads((4096, 300, 0, 0), (4200, 10, 1, 1))):
        assert call(bad) == nat.LF_ERR_INVALID_ARG  # shared memory
    assert call(good, limit=-1.0) == nat.LF_ERR_INVALID_ARG
    assert call(good, limit=float("nan")) == nat.LF_ERR_INVALID_ARG
    assert call(good, norms=None) == nat.LF_ERR_INVALID_ARG
    assert call(good, ws=264) == nat.LF_ERR_INVALID_ARG
    assert call(good, ws=None) == nat.LF_ERR_CAPACITY and call(good, n=3 * 256 - 1) == nat.LF_ERR_CAPACITY
    assert call(_grads(), groups=0) == nat.LF_OK
    assert call(good, groups=0) == nat.LF_ERR_INVALID_ARG


def _plan(sizes, groups, n_groups, room=None):
    rec = np.zeros(len(sizes), dtype=np.dtype(nat.ADAMW_TENSOR))
    rec["param"], rec["numel"], rec["group"] = 4096, sizes, groups
    chunks, elems = ctypes.c_int64(0), ctypes.c_int64(0)
    table = np.full(4096, -1, dtype=np.int32)
    rc = nat.lib().lf_adamw_plan(rec.ctypes.data, len(sizes), n_groups, table.ctypes.data,
                                 4096 if room is None else room, ctypes.byref(chunks), ctypes.byref(elems))
    return rc, rec, table, chunks.value, elems.value


def test_adamw_plan():
    sizes = [1, 8192, 0, 8193, 20000, 7]
    rc, rec, table, chunks, elems = _plan(sizes, [0, 1, 1, 2, 0, 2], 3)
    assert rc == nat.LF_OK and chunks == 1 + 1 + 0 + 2 + 3 + 1
    assert table[:chunks].tolist() == [0, 1, 3, 3, 4, 4, 4, 5] and (table[chunks:] == -1).all()
    assert rec["chunk0"].tolist() == [0, 1, 2, 2, 4, 7] and rec["n_chunks"].tolist() == [1, 1, 0, 2, 3, 1]
    assert rec["state_off"].tolist() == [0, 8, 8200, 8200, 16400, 36400] and elems == 36408
    assert _plan(sizes, [0, 1, 1, 2, 0, 2], 3, room=7)[0] == nat.LF_ERR_CAPACITY
    assert _plan([5], [3], 3)[0] == nat.LF_ERR_INVALID_ARG
    assert _plan([5], [-1], 3)[0] == nat.LF_ERR_INVALID_ARG
    assert _plan([0xffffffff], [0], 1)[0] == nat.LF_ERR_INVALID_ARG


def test_adamw_entry_refuses_before_any_launch():
    L = nat.lib()
    _, rec, _, chunks, _ = _plan([100, 200], [0, 1], 2)
    grads = np.array([4096, 8192], dtype=np.uint64)

    def call(**kw):
        a = nat.AdamWArgs(rec.ctypes.data, 256, 256, grads.ctypes.data, 256, 256, 256, 256, 256, 256, 256,
                          L.lf_adamw_workspace_bytes(chunks, 2), chunks, 0.9, 0.999, 1e-8, 1.0, 2, 2, nat.LF_BF16,
                          nat.LF_F32, 0, 0)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.lf_adamw_step(ctypes.byref(a), None)

    for kw in (dict(n_tensors=-1), dict(n_groups=-1), dict(n_chunks=-1), dict(tensors=None), dict(tensors_dev=None),
               dict(grads=None), dict(hyper_dev=None), dict(steps_dev=None), dict(beta1=1.0), dict(beta2=-0.1),
               dict(beta1=float("nan")), dict(eps=-1.0), dict(max_norm=float("nan")), dict(norms_dev=None),
               dict(norms_dev=None, max_norm=-1.0, skip_nonfinite=1), dict(exp_avg_dev=None), dict(exp_avg_sq_dev=None),
               dict(master_dev=None), dict(chunk_tensor_dev=None), dict(exp_avg_dev=260), dict(workspace_dev=264),
               dict(n_groups=1)):
        assert call(**kw) == nat.LF_ERR_INVALID_ARG, kw
    for kw in (dict(param_dtype=3), dict(param_dtype=nat.LF_F32, grad_dtype=nat.LF_BF16),
               dict(grad_dtype=nat.LF_F16)):
        assert call(**kw) == nat.LF_ERR_UNSUPPORTED, kw
    assert call(workspace_bytes=8) == nat.LF_ERR_CAPACITY and call(workspace_dev=None) == nat.LF_ERR_CAPACITY
    assert call(n_tensors=0) == nat.LF_OK
    grads[1] = 8194  # float32 gradients off a multiple of 4 bytes
    assert call() == nat.LF_ERR_INVALID_ARG


def test_both_gemms_of_long_batches_are_chosen():
    """Which GEMM a long batch takes, at the 148 SMs of a B200: the sizes that the numeric tests rely on."""
    from tests.test_serving_gpu import CASES, TALL_TILES
    uses = nat.lib().lf_rows_uses_pairs
    assert all(uses(T, K, N, 148) == 0 for _, T, K, N, _, _ in TALL_TILES)
    long = [(T, K, N) for dtype, T, K, N, _, _ in CASES if T > 256 and dtype is not torch.float32]
    assert sum(uses(T, K, N, 148) for T, K, N in long) >= 5
    assert uses(256, 4096, 4096, 148) == uses(0, 4096, 4096, 148) == uses(1000, 4096, 4096, 0) == 0
    assert uses(8192, 4096, 4096, 148) == 1


def test_rows_output_may_not_share_memory_with_anything_read():
    """4 x 16 bf16 output at 4096; an operand whose last byte is its first, or the other way round."""
    L = nat.lib()
    ws = L.lf_rows_workspace_bytes(4, 16, 16, nat.LF_BF16)
    apart = dict(x_dev=1 << 20, w_dev=2 << 20, a_bank_dev=3 << 20, b_bank_dev=4 << 20, slot_rank_dev=5 << 20,
                 slot_scale_dev=6 << 20, row_slot_dev=7 << 20)
    sizes = dict(x_dev=4 * 16 * 2, w_dev=16 * 16 * 2, a_bank_dev=2 * 16 * 16 * 2, b_bank_dev=2 * 16 * 16 * 2,
                 slot_rank_dev=8, slot_scale_dev=8, row_slot_dev=16)
    for name, size in sizes.items():
        for at in (4096, 4096 + 4 * 16 * 2 - 16, 4096 - size + 16 if size > 16 else 4096):
            p = _rows(**{**apart, name: at})
            assert L.lf_rows_forward(p, 4096, 256, ws, None) == nat.LF_ERR_INVALID_ARG, (name, at)


def test_launch_count_of_the_largest_batches():
    count = nat.lib().lf_rows_launch_count
    assert count(2 ** 31 - 1, 64) == 4 * 2 ** 18 and count(2 ** 31 - 8192, 64) == 4 * (2 ** 18 - 1)
    assert count(-1, 64) == count(-2 ** 31, 16) == 0


def test_bank_load_from_its_own_slot_is_refused():
    def call(**kw):
        d = dict(dtype=nat.LF_BF16, K=32, N=24, r_pad=16, rank=4, scale=1.0, lda=40, ldb=6, a_dev=1 << 20, b_dev=2 << 20,
                 slot_a_dev=3 << 20, slot_b_dev=4 << 20, slot_rank_dev=256, slot_scale_dev=256)
        return nat.lib().lf_bank_load(nat.BankAdapter(**{**d, **kw}), None)

    last_a, last_b = 2 * (3 * 40 + 32) - 2, 2 * (23 * 6 + 4) - 2  # bytes to an operand's last element
    for slot, size in ((3 << 20, 16 * 32 * 2), (4 << 20, 16 * 24 * 2)):
        for name, last in (("a_dev", last_a), ("b_dev", last_b)):
            for at in (slot, slot + size - 2, slot - last):
                assert call(**{name: at}) == nat.LF_ERR_INVALID_ARG, (name, at)
