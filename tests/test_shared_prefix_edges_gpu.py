"""Attention behind a shared prefix where it can go wrong: values that are not finite in parts of vanishing weight, tables that are rows of one pool's.
Restatement and bounds as in test_shared_prefix_gpu.py."""

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


def rows_of_one_table(args, width):
    """The tables of a batch as rows of one pool's, which are as wide as the longest sequence may become."""
    fit = lambda t: torch.cat((t, t.new_full((t.shape[0], width - t.shape[1]), -1)), 1)
    both = torch.cat((fit(args[3]), fit(args[5])))
    return [*args[:3], both[:args[3].shape[0]], args[4], both[args[3].shape[0]:], *args[6:]]


@pytest.mark.parametrize("q,n,own,groups", [(1, 40, 700, [0, 40]), (1, 9, 2000, [0, 4, 9]), (5, 20, 500, [0, 20]), (24, 6, 900, [0, 6]), (150, 4, 400, [0, 4])])
def test_tables_that_are_rows_of_one_pool(q, n, own, groups):
    """Both tables as wide: the widths say nothing of where prefixes end, and own keys may be many."""
    import experiment_swa_kda_b200 as m
    b = Batch(8, 4, 64, 16, BF16, [q] * n, [q + (own * (i + 1)) // n for i in range(n)], [600] * (len(groups) - 1), groups, seed=2)
    tight = b.device()
    for width in (tight[3].shape[1], 256, 4096):
        for bound in (q, 0):
            o, lse = m.shared_prefix_attention(*rows_of_one_table(tight, max(width, tight[3].shape[1])), max_q_len=bound, return_lse=True)
            b.check(o, lse)


@pytest.mark.parametrize("q,n,own", [(1, 32, 4096), (1, 256, 256), (5, 64, 640)])
def test_rows_of_one_pool_take_as_long_as_tables_cut_to_length(q, n, own):
    """A call with tables of 32,768 tokens takes less than twice the time of the same call with tables that end where the sequences do."""
    import experiment_swa_kda_b200 as m
    pages, prefix = 64, 2048
    gen = torch.Generator(device="cuda:0").manual_seed(1)
    k, v = (torch.randn(pages, 64, 4, 128, generator=gen, device="cuda:0").to(BF16) for _ in range(2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda:0")
    lens = [prefix + max(q, own * (i + 1) // n) for i in range(n)]
    table = torch.randint(0, pages, (n, -(-max(lens) // 64)), generator=gen, device="cuda:0", dtype=torch.int32)
    q_ = torch.randn(n * q, 16, 128, generator=gen, device="cuda:0").to(BF16)
    tight = [q_, k, v, table, i32(lens), table[:1, :prefix // 64].contiguous(), i32([prefix]), None, None]
    times = []
    for args in (tight, rows_of_one_table(tight, 512)):
        call = lambda: m.shared_prefix_attention(*args, max_q_len=q)
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(10):
                call()
        graph.replay()
        took = []
        for _ in range(7):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            begin.record()
            graph.replay()
            end.record()
            torch.cuda.synchronize()
            took.append(begin.elapsed_time(end))
        times.append(sorted(took)[3])
    assert times[1] <= 2 * times[0], times
