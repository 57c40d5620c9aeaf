"""Attention behind a shared prefix where it can go wrong: values that are not finite in parts of vanishing weight.  Restatement and bounds as in
test_shared_prefix_gpu.py."""

import math

import pytest
import torch

from test_shared_prefix_gpu import BF16, Batch, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q,groups", [(1, [0, 6]), (5, [0, 6]), (5, [0, 2, 6]), (24, [0, 6]), (150, [0, 6])])
@pytest.mark.parametrize("room", [0, 60000])
@pytest.mark.parametrize("low", ["prefix", "own"])
def test_values_that_are_not_finite_reach_rows_whose_weights_vanish(q, groups, room, low):
    """A visible NaN is in the sum however small its weight: the keys of the prefix, or the own ones, hundreds of units below the others."""
    import experiment_swa_kda_b200 as m
    b = Batch(4, 2, 64, 16, BF16, [q] * 6, [q + 40, q + 7, q + 100, q + 300, q, q + 64], [2500] * (len(groups) - 1), groups, seed=8, room=room)
    b.q = (b.q.abs() + 0.5).to(BF16)      # a key of -100 throughout scores -100 * 64 * 0.5 / 8 = -400 or less
    page = 16
    rows = {"prefix": [(b.prefix_table[g], 0, 2500) for g in range(len(groups) - 1)], "own": [(b.table[n], 2500, x) for n, x in enumerate(b.kv_lens)]}[low]
    for row, lo, hi in rows:
        for pos in range(lo, hi):
            b.k[int(row[pos // page]), pos % page] = -100.0
    row, pos = rows[0 if low == "prefix" else 3][0], 200 if low == "prefix" else 2600      # of group 0, or of sequence 3
    b.v[int(row[pos // page]), pos % page, 0, 7] = math.nan
    o = m.shared_prefix_attention(*b.device(), max_q_len=q)
    want, _, size = b.want()
    assert bool(torch.isnan(want[..., 7]).any()) and not bool(torch.isnan(want[..., 8]).any())
    close(o, want, size, BF16)
