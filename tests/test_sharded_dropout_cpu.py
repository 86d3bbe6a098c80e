"""Dropout of rows sharded over GPUs: every rank's mask is its own (no GPU)."""

import numpy as np
import pytest

from oracle.dropout_oracle import kept
from lorafusion_b200.config import AdapterDropout
from lorafusion_b200.sharding import assign_bins, local_dropout


def test_ranks_and_offsets_have_masks_of_their_own():
    plan = assign_bins([[(0, 900), (1, 300)], [(2, 500)]], 4)
    d = AdapterDropout({0: 0.5, 1: 0.25, 2: 0.0}, 77, 5)
    masks = {}
    for step in (5, 6):
        for rank in range(4):
            local = local_dropout(d.at(step), plan, rank)
            assert local.seed == 77 and local.rates == d.rates
            assert [local.threshold(i) for i in range(3)] == [32768, 16384, 0]
            masks[step, rank] = kept(64, 256, [32768] * 64, local.seed, local.offset)
    assert len({(local_dropout(d.at(o), plan, r).offset) for o in range(50) for r in range(4)}) == 200
    keys = list(masks)
    for i, a in enumerate(keys):
        for b in keys[:i]:  # as like as two throws of 64 x 256 coins, five standard deviations
            assert abs(np.mean(masks[a] == masks[b]) - 0.5) < 5 * 0.5 / (64 * 256) ** 0.5
    assert local_dropout(d, plan, 3) == local_dropout(d, plan, 3)


def test_rates_are_those_of_the_first_object():
    rates = {0: 0.5}
    d = AdapterDropout(rates, 1, 2)
    rates[0] = 0.1
    assert d.at(9).threshold(0) == 32768 and d.at(9).offset == 9


def test_refusals():
    plan = assign_bins([[(0, 900)]], 2)
    d = AdapterDropout(0.5, 1, (1 << 63))
    with pytest.raises(ValueError, match="offset"):
        local_dropout(d, plan, 0)
    with pytest.raises(ValueError, match="rank"):
        local_dropout(d.at(1), plan, 2)
    with pytest.raises(ValueError, match="rank"):
        local_dropout(d.at(1), plan, -1)
    with pytest.raises(ValueError, match="offset"):
        d.at(-1)
