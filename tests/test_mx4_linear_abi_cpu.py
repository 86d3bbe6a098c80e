"""lf_mx4_linear's checks of its workspace, which come before the device is asked for anything (no GPU)."""

import pytest

from lorafusion_b200 import _native as nat

MB = 1 << 20


def linear(ws, n, out=256 * MB, **kw):
    d = dict(dtype=nat.LF_BF16, T=4, K=64, N=128, transpose=0, reserved=0, ld=64, in_dev=64 * MB, mx4_dev=128 * MB)
    return nat.lib().lf_mx4_linear(nat.Mx4Problem(**{**d, **kw}), out, ws, n, None)


CORES = [dict(ld=68), dict(in_dev=64 * MB + 2), dict(out=256 * MB + 8), dict(K=60), dict(N=100), dict(transpose=1, ld=132)]


@pytest.mark.parametrize("kw", CORES)
def test_products_on_cuda_cores_need_a_dense_copy(kw):
    """K and N may be multiples of 8: the operands' pitch and addresses decide as well."""
    dense = 2 * kw.get("K", 64) * kw.get("N", 128)
    assert linear(None, 0, **kw) == nat.LF_ERR_CAPACITY
    assert linear(512 * MB, dense - 1, **kw) == nat.LF_ERR_CAPACITY


@pytest.mark.parametrize("kw", [{}, dict(transpose=1, ld=128)] + CORES)
def test_a_workspace_that_meets_an_operand_is_refused(kw):
    bad = nat.LF_ERR_INVALID_ARG
    n = 32 * MB
    for at in (64 * MB, 128 * MB, 256 * MB):  # in, the weight, out
        assert linear(at, n, **kw) == bad, at
    # the last row's last element, and the first bytes of what the call uses
    width, ld = (128 if kw.get("transpose") else kw.get("K", 64)), kw.get("ld", 64)
    last = (kw.get("in_dev", 64 * MB) + 2 * (3 * ld + width) - 1) // 16 * 16
    assert linear(last, n, **kw) == bad


# rows, reduction, output features, parts on 148 SMs (74 pairs), forward and gradient alike
CUTS = [(1792, 384, 3584, 3),    # 98 tiles, 24 in the last round
        (2048, 1000, 3328, 2),   # 104, 30
        (4096, 4096, 4096, 2),   # 256, 34
        (2300, 640, 2552, 3),    # 90, 16: a fourth part has no room
        (2304, 256, 2560, 2),    # ... 4 blocks of the reduction are two parts
        (2304, 192, 2560, 1)]    # ... 3 are one


def test_where_the_last_round_is_cut():
    parts = nat.lib().lf_mx4_linear_tail_parts
    for T, red, out, n in CUTS:
        assert parts(T, red, out, 0, 148) == n and parts(T, out, red, 1, 148) == n, (T, red, out)
    assert parts(1024, 1536, 512, 1, 148) == 3 and parts(1280, 1536, 512, 1, 148) == 2  # 24 and 30 tiles, no full round
    assert parts(1024, 512, 1536, 0, 148) == 0 and parts(200, 512, 8192, 0, 148) == 0   # the tiles of W as the M operand
    assert parts(1024, 60, 64, 0, 148) == 0 and parts(0, 64, 64, 1, 148) == 0
