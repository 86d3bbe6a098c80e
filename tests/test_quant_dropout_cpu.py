"""Refusals and definitions of the 4-bit weight and of the adapters' dropout that need no GPU."""

import ctypes

import pytest
import torch

from oracle.dropout_oracle import kept, philox
from lorafusion_b200 import _native as nat
from lorafusion_b200.config import AdapterDropout
from lorafusion_b200.quant import MX4Weight, mx4_linear, quantize_weight


def test_the_generator_gives_its_published_numbers():
    assert philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert philox((ones,) * 4, (ones,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert not kept(4, 9, [65536] * 4, 1, 2).any() and kept(4, 9, [0] * 4, 1, 2).all()
    seed, offset, at = 0x123456789ABCDEF0, (7 << 32) + 5, [40000, 1, 65535]
    got = kept(3, 21, at, seed, offset)
    for t in range(3):
        for k in range(21):
            words = philox((k // 8, t, offset & ones, offset >> 32), (seed & ones, seed >> 32))
            assert got[t, k] == ((words[k % 8 // 2] >> 16 * (k % 2) & 0xFFFF) >= at[t])


@pytest.mark.parametrize("rate", [-0.1, 1.0, 1.5, float("nan"), 1 - 2.0 ** -18])
def test_rates_outside_0_to_1_are_refused(rate):
    with pytest.raises(ValueError, match="rate"):
        AdapterDropout(rate, 0)
    with pytest.raises(ValueError, match="rate"):
        AdapterDropout({3: 0.1, 4: rate}, 0)


@pytest.mark.parametrize("bad", [-1, 1 << 64, 1.5, True, None])
def test_seeds_are_whole_numbers_of_64_bits(bad):
    with pytest.raises(ValueError, match="seed"):
        AdapterDropout(0.1, bad)
    with pytest.raises(ValueError, match="offset"):
        AdapterDropout(0.1, 0, bad)


def test_thresholds():
    d = AdapterDropout({1: 0.0, 2: 0.5, 3: 65535 / 65536}, 0)
    assert [d.threshold(i) for i in (1, 2, 3)] == [0, 32768, 65535]
    with pytest.raises(KeyError):
        d.threshold(9)
    assert AdapterDropout(0.1, 0).threshold(12345) == 6554


def test_sizes_of_a_weight_in_4_bits():
    L = nat.lib()
    assert L.lf_mx4_bytes(128, 128) == 128 * 128 * 17 // 32
    assert L.lf_mx4_bytes(1, 1) == L.lf_mx4_bytes(128, 128)
    assert L.lf_mx4_bytes(129, 128) == 2 * L.lf_mx4_bytes(128, 128) == L.lf_mx4_bytes(128, 129)
    assert L.lf_mx4_bytes(28672, 8192) == 28672 * 8192 * 17 // 32
    assert L.lf_mx4_bytes(-1, 8) == 0 and L.lf_mx4_bytes(0, 8) == 0
    assert L.lf_mx4_bytes(1 << 24, 1 << 24) == (1 << 48) * 17 // 32


def test_weights_on_the_cpu_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        quantize_weight(torch.zeros(4, 4, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA"):
        MX4Weight(torch.zeros(nat.lib().lf_mx4_bytes(4, 4), dtype=torch.uint8), 4, 4, torch.bfloat16)
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        MX4Weight(torch.zeros(1, dtype=torch.uint8), 4, 4, torch.float32)
    with pytest.raises(ValueError, match="MX4Weight"):
        mx4_linear(torch.zeros(4, 4), torch.zeros(4, 4))


def test_the_library_refuses_before_any_launch():
    """Every refusal comes before the device is asked for anything: none of these calls needs a GPU."""
    L, bad = nat.lib(), nat.LF_ERR_INVALID_ARG
    assert L.lf_mx4_quantize(nat.LF_F32, 256, 8, 8, 8, 4096, None) == nat.LF_ERR_UNSUPPORTED
    assert L.lf_mx4_quantize(7, 256, 8, 8, 8, 4096, None) == bad
    assert L.lf_mx4_quantize(nat.LF_BF16, 256, -1, 8, 8, 4096, None) == bad
    assert L.lf_mx4_quantize(nat.LF_BF16, None, 8, 8, 8, 4096, None) == bad
    assert L.lf_mx4_quantize(nat.LF_BF16, 256, 8, 8, 7, 4096, None) == bad      # rows that overlap
    assert L.lf_mx4_quantize(nat.LF_BF16, 256, 8, 8, 8, 4104, None) == bad      # not aligned
    assert L.lf_mx4_quantize(nat.LF_BF16, 4096, 8, 8, 8, 4096, None) == bad     # in place
    assert L.lf_mx4_quantize(nat.LF_BF16, 256, 1 << 25, 8, 8, 4096, None) == nat.LF_ERR_UNSUPPORTED
    assert L.lf_mx4_quantize(nat.LF_BF16, None, 0, 8, 8, None, None) == nat.LF_OK
    assert L.lf_mx4_dequantize(nat.LF_BF16, 4096, 8, 8, 4096, None) == bad
    assert L.lf_mx4_dequantize(nat.LF_BF16, None, 8, 8, 1 << 20, None) == bad

    def linear(out=1 << 30, ws=None, n=0, **kw):
        d = dict(dtype=nat.LF_BF16, T=4, K=64, N=128, transpose=0, reserved=0, ld=64, in_dev=1 << 20, mx4_dev=1 << 24)
        return L.lf_mx4_linear(nat.Mx4Problem(**{**d, **kw}), out, ws, n, None)

    assert L.lf_mx4_linear(None, 256, None, 0, None) == bad
    for kw in (dict(T=-1), dict(transpose=2), dict(ld=63), dict(in_dev=None), dict(mx4_dev=None), dict(out=None),
               dict(mx4_dev=(1 << 24) + 8), dict(out=1 << 20), dict(out=1 << 24), dict(transpose=1), dict(K=0, ld=0),
               dict(dtype=9), dict(ws=8, n=1 << 20)):
        assert linear(**kw) == bad, kw
    assert linear(dtype=nat.LF_F32) == nat.LF_ERR_UNSUPPORTED
    assert linear(T=0) == nat.LF_OK

    info = nat.PlanInfo(total_rows=4, n_slots=1, n_segtiles=1, r_pad=16)
    prob = nat.Problem(nat.LF_BF16, 4, 64, 64, 256, 256, 256, 256, 256, 256)
    drop = nat.Dropout(1, 2, 256, 256, 0)

    def forward(opt):
        return L.lf_forward_opt(prob, info, 256, opt, 256, 256, 1 << 40, None, 0, None, None)

    assert forward(nat.Options(5, 0, None)) == bad
    drop.slot_threshold_dev = None
    assert forward(nat.Options(0, 0, ctypes.pointer(drop))) == bad
    drop.slot_threshold_dev, drop.scratch_dev = 256, 8
    assert forward(nat.Options(0, 0, ctypes.pointer(drop))) == bad
    prob.dtype = nat.LF_F32
    assert forward(nat.Options(nat.LF_WEIGHT_MX4, 0, None)) == nat.LF_ERR_UNSUPPORTED
    def scratch(dtype, K, backward):
        return L.lf_dropout_scratch_bytes(nat.Problem(dtype, 128, K, 64, 256, 256), backward)

    assert L.lf_dropout_scratch_bytes(None, 0) == 0
    assert scratch(nat.LF_BF16, 64, 0) == 0 and scratch(nat.LF_BF16, 64, 1) == 128 * 64 * 6
    assert scratch(nat.LF_F32, 64, 0) == 128 * 64 * 4 == scratch(nat.LF_F32, 64, 1)
    assert scratch(nat.LF_BF16, 60, 0) == 128 * 60 * 2 == scratch(nat.LF_BF16, 60, 1)
    rows = nat.RowsProblem(dtype=nat.LF_BF16, T=1, K=64, N=64, n_slots=0, r_pad=16, row_slot_bytes=4, weight_format=2)
    assert L.lf_rows_forward(rows, 256, 256, 0, None) == bad
