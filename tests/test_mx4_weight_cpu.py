"""The fields of a weight in 4 bits: what the kernels would read past is refused (no GPU)."""

import copy
import pickle

import pytest
import torch

from lorafusion_b200 import _native as nat
from lorafusion_b200.quant import MX4Weight


class FakeCuda:
    """What the checks ask of a CUDA tensor."""
    device = torch.device("cuda", 0)
    dtype = torch.uint8

    def __init__(self, n, at=1 << 20, dense=True):
        self.shape, self.at, self.dense = torch.Size((n,)), at, dense

    def is_contiguous(self):
        return self.dense

    def data_ptr(self):
        return self.at


NEED = nat.lib().lf_mx4_bytes(200, 300)


def test_data_must_hold_the_weight():
    w = MX4Weight(FakeCuda(NEED), 200, 300, torch.bfloat16)
    first = w.data
    w.data = FakeCuda(NEED)
    assert w.data is not first
    for bad in (FakeCuda(NEED - 1), FakeCuda(NEED + 16), FakeCuda(0), FakeCuda(NEED, at=(1 << 20) + 8),
                FakeCuda(NEED, dense=False), torch.zeros(NEED, dtype=torch.uint8)):
        with pytest.raises(ValueError, match="data must be"):
            w.data = bad
        with pytest.raises(ValueError, match="data must be"):
            MX4Weight(bad, 200, 300, torch.bfloat16)


@pytest.mark.parametrize("name,value", [("out_features", 400), ("in_features", 600), ("dtype", torch.float16)])
def test_sizes_and_dtype_are_fixed(name, value):
    w = MX4Weight(FakeCuda(NEED), 200, 300, torch.bfloat16)
    with pytest.raises(AttributeError, match=name):
        setattr(w, name, value)
    assert w.shape == (200, 300) and w.dtype is torch.bfloat16


def test_copies():
    w = MX4Weight(FakeCuda(NEED), 200, 300, torch.bfloat16)
    for other in (copy.copy(w), copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
        assert other.shape == (200, 300) and other.dtype is torch.bfloat16 and other.data.shape == (NEED,)
