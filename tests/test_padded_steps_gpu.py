"""Steps of a fixed size that are not full: tokens behind the last sequence are padding in append and attention, and what `plan_pages` says of rows that wait can
be passed on.  Restatements and bounds as in test_attention_gpu.py and test_shared_prefix_gpu.py."""

import math

import pytest
import torch

import serving_oracle as S
import test_attention_gpu as P
import test_shared_prefix_gpu as X
from test_attention_gpu import BF16, DEV, F32

pytestmark = pytest.mark.gpu


def tail(t, rows):
    """The tensor with so many rows of NaN behind it."""
    return torch.cat((t, t.new_full((rows,) + t.shape[1:], math.nan)))


def poison(*shapes):
    """Memory that the next results are likely to get, full of NaN."""
    kept = [torch.full(shape, math.nan, dtype=dtype, device=DEV) for shape, dtype in shapes]
    del kept


def told():
    """Whether the calls so far have left an error."""
    import experiment_swa_kda_b200 as m
    nothing, table = torch.zeros(1, 0, 1, 128, device=DEV), torch.ones(4, 64, device=DEV)
    torch.cuda.synchronize()
    try:
        m.qk_norm_rope(nothing, nothing, table, table)
    except RuntimeError as e:
        return str(e)
    return None


def blank(o, lse, tokens):
    return bool((o[tokens:] == 0).all()) and bool((lse[tokens:] == -math.inf).all())


@pytest.mark.parametrize("q_lens,kv_lens,Hq,Hk,D,page,window,dtype,bound", [
    ([1], [700], 3, 3, 128, 16, 0, BF16, 1),                       # token steps: one sequence, whole ones, ones without a new token
    ([1, 0, 1, 0], [33, 20, 300, 0], 4, 2, 64, 16, 0, BF16, 1),
    ([1] * 60, [40 + n for n in range(60)], 16, 4, 128, 64, 0, BF16, 1),
    ([2, 0], [900, 5], 6, 2, 64, 16, 77, BF16, 2),
    ([0, 0], [4, 0], 4, 2, 128, 16, 0, BF16, 1),                   # no new token at all
    ([200, 9], [333, 1000], 12, 4, 64, 16, 0, BF16, 200),          # the tensor-core kernel, in parts and whole, with and without the bound
    ([200, 9], [333, 6000], 4, 2, 128, 16, 0, BF16, 0),
    ([30, 0, 41], [30, 3, 90], 5, 1, 96, 32, 0, BF16, 41),
    ([1] * 90, [500] * 90, 16, 4, 128, 64, 0, BF16, 0),
    ([20, 0], [50, 0], 2, 2, 200, 16, 0, BF16, 0),                 # the CUDA cores, in parts and whole
    ([17, 2], [90, 31], 3, 1, 100, 5, 0, F32, 17),
    ([3, 0], [700, 10], 2, 1, 64, 16, 0, F32, 0),
    ([200] * 4, [200] * 4, 16, 16, 64, 16, 0, F32, 200),
])
@pytest.mark.parametrize("more", [1, 300])
def test_paged_attention(q_lens, kv_lens, Hq, Hk, D, page, window, dtype, bound, more):
    import experiment_swa_kda_b200 as m
    b = P.Batch(q_lens, kv_lens, Hq, Hk, D, page, dtype, window, seed=D)
    tokens, q = sum(q_lens), tail(b.dq, more)
    poison((q.shape, dtype), (q.shape[:2], F32))
    o, lse = m.paged_attention(q, b.dk, b.dv, b.dtable, b.dlens, b.dcu, window=window, max_q_len=bound, return_lse=True, padded=True)
    want, _, size = b.oracle()
    P.close(o[:tokens], want, size, dtype)
    assert blank(o, lse, tokens) and told() is None
    m.paged_attention(q, b.dk, b.dv, b.dtable, b.dlens, b.dcu, window=window, max_q_len=bound)
    assert "cu_seqlens" in told()


@pytest.mark.parametrize("q,own,dtype", [(1, [1, 9, 300], BF16), (5, [5, 40, 9], BF16), (40, [60, 40, 90], BF16), (150, [150, 151, 400], BF16), (1, [4, 1, 9], F32), (33, [40, 33, 50], F32)])
@pytest.mark.parametrize("room", [0, 60000])
@pytest.mark.parametrize("more", [1, 300])
def test_shared_prefix_attention(q, own, dtype, room, more):
    import experiment_swa_kda_b200 as m
    b = X.Batch(8, 2, 64, 16, dtype, [q, 0, q, q, 0], [own[0], 7, own[1], own[2], 0], [300, 40], [0, 3, 5], room=room)
    args = b.device()
    args[0] = tail(args[0], more)
    for bound in (q, 0):
        poison((args[0].shape, dtype), (args[0].shape[:2], F32))
        o, lse = m.shared_prefix_attention(*args, max_q_len=bound, return_lse=True, padded=True)
        b.check(o[:3 * q], lse[:3 * q])
        assert blank(o, lse, 3 * q) and told() is None
        m.shared_prefix_attention(*args, max_q_len=bound)
        assert "cu_seqlens" in told()


@pytest.mark.parametrize("Hq,Hk,D,dtype", [(16, 4, 128, BF16), (3, 3, 64, F32), (2, 1, 34, BF16)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 0, 1], [9, 30, 17]), ([0, 0], [3, 0]), ([40, 1, 0], [60, 40, 20])])
@pytest.mark.parametrize("more", [1, 200])
def test_append(Hq, Hk, D, dtype, q_lens, kv_lens, more):
    import experiment_swa_kda_b200 as m
    b = P.Batch(q_lens, kv_lens, Hq, Hk, D, 16, dtype, reach=False)
    tokens = sum(q_lens)
    k, v = (torch.randn(tokens, Hk, D, generator=torch.Generator().manual_seed(s)).to(dtype).to(DEV) for s in (1, 2))
    cos, sin = (t.to(DEV) for t in P.tables(64, D))
    full, padded = [[t.clone() for t in (b.dk, b.dv)] for _ in range(2)]
    want = m.qk_norm_rope_append(b.dq, k, v, cos, sin, *full, b.dtable, b.dlens, b.dcu)
    poison((tail(b.dq, more).shape, dtype))
    got = m.qk_norm_rope_append(tail(b.dq, more), tail(k, more), tail(v, more), cos, sin, *padded, b.dtable, b.dlens, b.dcu, padded=True)
    assert torch.equal(got[:tokens], want) and bool((got[tokens:] == 0).all()) and told() is None
    for x, y in zip(full, padded):
        assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))
    m.qk_norm_rope_append(tail(b.dq, more), tail(k, more), tail(v, more), cos, sin, *padded, b.dtable, b.dlens, b.dcu)
    assert "cu_seqlens" in told()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shared", [False, True])
def test_a_captured_step_with_a_pool_that_runs_short(dtype, shared):
    """Pages, cache and attention of steps of a fixed size in one graph: rows wait, end and go on; nothing is reported, what waits keeps its keys and values, and
    the rows served get what the layer gives them alone."""
    import experiment_swa_kda_b200 as m
    torch.manual_seed(11)
    layer = m.PagedAttention(128, 4, 2, 32, max_positions=256).to(DEV)
    if dtype == F32:
        layer = layer.float()
    page, rows, prefix, most = 8, 4, 21 if shared else 0, 24
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    pages = 9 + (-(-prefix // page))
    pool = m.PagedCache.pool(rows + 1, 128, pages, page, 2, 32, DEV, dtype=dtype)      # the last row holds the prefix
    whole = m.PagedCache.zeros(rows, 128, page, 2, 32, DEV, dtype=dtype)
    if shared:
        text = torch.randn(1, prefix, 128, device=DEV).to(dtype)
        pool.kv_lens.copy_(i32([0] * rows + [prefix]))
        layer(text, pool, pool.plan(i32([0] * rows + [prefix]), prefix)[0], max_q_len=prefix)
        whole.kv_lens.fill_(prefix)
        layer(text.expand(rows, -1, -1), whole)
    serve = m.PagedCache(pool.k, pool.v, pool.block_table[:rows], pool.kv_lens[:rows],
                         prefix_table=pool.block_table[rows:] if shared else None, prefix_lens=pool.kv_lens[rows:] if shared else None)
    lens, new, starts = i32([0] * rows), i32([0] * (rows + 1)), i32([prefix] * rows + [0])
    x = torch.zeros(1, most, 128, device=DEV, dtype=dtype)

    def step():
        pool.kv_lens[:rows] = lens
        cu, positions, _ = pool.plan(new, most, starts=starts)
        return layer(x, serve, cu[:rows + 1], max_q_len=most, padded=True), cu, positions

    start = pool.block_table.clone(), pool.page_free.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    pool.block_table.copy_(start[0]), pool.page_free.copy_(start[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, cu, positions = step()
    waited = 0
    for own, add in (([3, 20, 0, 1], [3, 20, 0, 1]), ([4, 21, 40, 2], [1, 1, 40, 1]),      # place 2 asks for more than there is, 3 behind it waits as well
                     ([34, 22, 0, 2], [30, 1, 0, 1]),                                       # ... withdraws; more than a step takes in place 0: all wait
                     ([5, 22, 0, 2], [1, 1, 0, 1]), ([6, 0, 22, 3], [1, 0, 22, 1]),         # a row ends and 2 gets its pages
                     ([7, 0, 23, 3], [1, 0, 1, 1])):
        want_lens = [prefix + a if a else 0 for a in own]
        lens.copy_(i32(want_lens)), new.copy_(i32(add + [0]))
        table, before = pool.block_table.tolist(), (pool.k.clone(), pool.v.clone())
        _, got, _, want_cu, want_pos, _ = S.plan_pages(table, want_lens + [prefix], pool.page_free.tolist(), add + [0], page, most, [prefix] * rows + [0])
        x.copy_(torch.randn(1, most, 128, device=DEV))
        graph.replay()
        assert told() is None
        assert cu.tolist() == want_cu and positions.tolist() == want_pos and pool.kv_lens.tolist() == got
        served = [b - a for a, b in zip(want_cu, want_cu[1:])][:rows]
        total = sum(served)
        for n in range(rows):
            if served[n] == 0 and got[n] > 0:
                waited += add[n] > 0
                held = [p for p in table[n] if p >= 0 and p in pool.block_table[n].tolist()]
                for now, then in zip((pool.k, pool.v), before):
                    assert torch.equal(now[held], then[held])
        assert bool((y[0, total:] == 0).all())
        if total == 0:
            continue
        whole.kv_lens.copy_(i32(got[:rows]))
        want = layer(x[:, :total], whole, i32(want_cu[:rows + 1]), max_q_len=most)
        # one rounding of the outputs and one of the weights each, through one projection
        assert (y[0, :total].double() - want[0].double()).norm() <= (1e-2 if dtype == BF16 else 1e-5) * want.double().norm()
    assert waited == (5 if shared else 4)      # behind a prefix place 2 too has a length while it waits
