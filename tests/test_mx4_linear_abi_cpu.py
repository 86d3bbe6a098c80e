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
