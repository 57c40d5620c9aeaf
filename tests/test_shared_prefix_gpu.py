"""Attention behind a shared prefix against a float64 restatement (oracle/serving_oracle.py).

Bounds, as for paged attention.  float32: 1e-5 of the relative 2-norm.  bfloat16 (unit roundoff u = 2^-8): one rounding of the
result, |err| <= u |y|; the softmax weights are rounded too, which moves o by at most u sum_j p_j |v_j|, and the sum they are divided
by as much again; 2^-12 of that scale covers float32 and second-order terms.  The log of the sums has no such rounding: 1e-4 absolute
(sums of float32 products of 128 bf16 values, a few units of 2^-24 of scores below 100)."""

import math

import pytest
import torch

import serving_oracle as S

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -8
F32, BF16 = torch.float32, torch.bfloat16


def close(got, want, size, dtype):
    got = got.detach().double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    fine = torch.isfinite(want)
    got, want, size = got[fine], want[fine], size[fine]
    if dtype == F32:
        assert (got - want).norm() <= 1e-5 * want.norm() + 1e-30
        return
    room = U * want.abs() + (2 * U + 2.0 ** -12) * size + 1e-30
    assert bool(((got - want).abs() <= room).all()), float(((got - want).abs() - room).max())


class Batch:
    """Sequences of groups, with garbage wherever nothing may be read."""

    def __init__(self, heads, kv_heads, dim, page, dtype, q_lens, own, prefix, cu_groups, seed=0, garbage=float("nan"), layout="dense", shares=None, room=0):
        """own[n]: tokens behind the prefix (the new ones among them); shares[n] false: own[n] tokens in all, none of them shared.  room:
        tokens that the sequences' tables have besides; which kernels take a call goes by the tables' widths."""
        gen = torch.Generator().manual_seed(seed)
        n = len(q_lens)
        group = [next((g for g in range(len(prefix)) if cu_groups[g] <= i < cu_groups[g + 1]), None) for i in range(n)]
        shares = [True] * n if shares is None else shares
        base = [prefix[g] if g is not None and s else 0 for g, s in zip(group, shares)]
        self.kv_lens = [b + o for b, o in zip(base, own)]
        self.q_lens, self.prefix, self.cu_groups, self.dtype = list(q_lens), list(prefix), list(cu_groups), dtype
        width = max(1, max(-(-x // page) for x in self.kv_lens)) + 1 + room // page
        pw = max(1, max(-(-x // page) for x in prefix))
        need = sum(max(0, -(-x // page) - b // page) for x, b in zip(self.kv_lens, base)) + sum(-(-x // page) for x in prefix)
        pages = need + 3
        order = torch.randperm(pages, generator=gen).tolist()
        bad = 2 ** 31 - 1
        self.table = torch.full((n, width), bad, dtype=torch.int32)
        self.prefix_table = torch.full((len(prefix), pw), -5, dtype=torch.int32)
        self.k, self.v = (torch.full((pages, page, kv_heads, dim), garbage) for _ in range(2))

        def put(row, lo, hi):
            for col in range(lo // page, -(-hi // page)):
                row[col] = order.pop()
                a, b = max(lo - col * page, 0), min(hi - col * page, page)
                for c in (self.k, self.v):
                    c[row[col], a:b] = torch.randn(b - a, kv_heads, dim, generator=gen)
        for g, x in enumerate(prefix):
            put(self.prefix_table[g], 0, x)
        for i in range(n):
            put(self.table[i], base[i], self.kv_lens[i])
        self.k, self.v = self.k.to(dtype), self.v.to(dtype)
        self.q = (1.5 * torch.randn(sum(q_lens), heads, dim, generator=gen)).to(dtype)
        self.layout = layout

    def device(self):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        q, k, v, table, ptable = (t.to(DEV) for t in (self.q, self.k, self.v, self.table, self.prefix_table))
        if self.layout == "strided":      # slices of larger buffers: one projection's q, k beside v, columns of wider tables
            wide = torch.empty(q.shape[0], q.shape[1] + 3, q.shape[2], dtype=q.dtype, device=DEV)
            wide[:, 1:1 + q.shape[1]] = q
            q = wide[:, 1:1 + q.shape[1]]
            both = torch.stack((k, v), 2).contiguous()
            k, v = both[:, :, 0], both[:, :, 1]
            table = torch.cat((torch.full_like(table, 7), table), 1)[:, table.shape[1]:]
            ptable = torch.cat((ptable, ptable), 1)[:, :ptable.shape[1]]
        return [q, k, v, table, i32(self.kv_lens), ptable, i32(self.prefix), i32(self.cu_groups), i32([0] + self.q_lens).cumsum(0).to(torch.int32)]

    def want(self, scale=None):
        return S.shared_prefix_attention(self.q, self.k, self.v, self.table, self.kv_lens, self.q_lens, self.prefix_table, self.prefix, self.cu_groups, scale)

    def check(self, out, lse=None, scale=None):
        o, want_lse, size = self.want(scale)
        close(out, o, size, self.dtype)
        if lse is not None:
            lse = lse.double().cpu()
            assert torch.equal(torch.isinf(lse), torch.isinf(want_lse)) and not bool(torch.isnan(lse).any())
            fine = torch.isfinite(want_lse)
            assert bool(((lse - want_lse).abs()[fine] <= 1e-4).all())


CASES = [  # heads, kv_heads, dim, page, dtype, q_lens, own, prefix, cu_groups
    (3, 3, 128, 16, BF16, [1], [1], [1], [0, 1]),
    (3, 3, 128, 16, BF16, [1] * 5, [1, 2, 17, 300, 16], [129], [0, 5]),
    (16, 4, 128, 64, BF16, [1] * 9, [5, 64, 65, 1, 127, 128, 1, 1000, 2], [1000], [0, 9]),
    (16, 16, 128, 16, BF16, [1] * 3, [33, 1, 8], [2049], [0, 3]),
    (16, 1, 128, 32, BF16, [1] * 20, list(range(1, 21)), [700], [0, 20]),
    (8, 1, 64, 128, BF16, [2] * 6, [2, 3, 70, 129, 4, 5], [257], [0, 6]),
    (6, 2, 96, 16, BF16, [5] * 4, [5, 9, 100, 6], [333], [0, 4]),
    (4, 2, 64, 8, BF16, [7, 1, 30, 1], [7, 40, 30, 1], [100, 5], [0, 2, 4]),
    (12, 4, 64, 16, BF16, [1] * 23, [(7 * i) % 40 + 1 for i in range(23)], [64, 1, 200, 15], [0, 10, 11, 20, 23]),
    (16, 4, 128, 64, BF16, [100, 33, 260], [130, 33, 261], [515], [0, 3]),
    (5, 1, 128, 64, BF16, [90, 1, 17], [100, 1, 20], [130], [0, 3]),
    (8, 2, 64, 16, BF16, [300], [301], [2100], [0, 1]),
    (4, 2, 128, 128, BF16, [200, 130], [260, 131], [1000, 127], [0, 1, 2]),
    (6, 1, 128, 16, BF16, [4] * 30, [4 + i for i in range(30)], [400], [0, 30]),
    (16, 4, 128, 16, BF16, [1] * 70, [1 + (i * 5) % 70 for i in range(70)], [900, 33], [0, 60, 70]),
    (8, 4, 64, 16, BF16, [1] * 50, [1 + i % 37 for i in range(50)], [20 + 3 * i for i in range(40)], list(range(40)) + [50]),
    (160, 1, 64, 16, BF16, [1, 2, 1], [40, 3, 1], [200], [0, 3]),
    (16, 8, 64, 64, BF16, [1] * 150, [1 + (i * 3) % 50 for i in range(150)], [200], [0, 150]),
    (4, 2, 8, 16, BF16, [1, 3], [4, 3], [31], [0, 2]),
    (4, 4, 128, 48, BF16, [1, 9, 2], [50, 9, 3], [97], [0, 3]),
    (2, 1, 200, 16, BF16, [1, 20], [10, 20], [70], [0, 2]),
    (4, 2, 64, 16, F32, [1, 33, 2], [5, 50, 3], [190], [0, 3]),
    (3, 3, 128, 16, F32, [1] * 7, [1, 9, 70, 3, 3, 3, 200], [300, 17], [0, 4, 7]),
    (2, 1, 50, 5, F32, [3, 1], [3, 2], [12], [0, 2]),
    (4, 1, 256, 16, F32, [1, 2], [1, 40], [65], [0, 2]),
]


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype,q_lens,own,prefix,cu_groups", CASES)
@pytest.mark.parametrize("bound", [True, False])
@pytest.mark.parametrize("room", [0, 60000])
def test_against_the_restatement(heads, kv_heads, dim, page, dtype, q_lens, own, prefix, cu_groups, bound, room):
    import experiment_swa_kda_b200 as m
    b = Batch(heads, kv_heads, dim, page, dtype, q_lens, own, prefix, cu_groups, layout="strided" if bound else "dense", room=room)
    o, lse = m.shared_prefix_attention(*b.device(), max_q_len=max(q_lens) if bound else 0, return_lse=True)
    b.check(o, lse)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q", [1, 3, 10, 40, 110])
@pytest.mark.parametrize("room", [0, 60000])
def test_sequences_that_do_not_share(dtype, q, room):
    """Places without a request, texts shorter than the prefix, sequences of no group, a group without sequences, a prefix of nothing."""
    import experiment_swa_kda_b200 as m
    n = 13
    own = [(11 * i) % 60 + q for i in range(n)]
    shares = [True] * n
    own[1], shares[1] = 0, False            # padding only
    own[4], shares[4] = max(q - 1, 0), False      # padding first, then tokens (q = 1: padding only)
    own[6], shares[6] = 20 + q, False       # shorter than its group's prefix
    own[9], shares[9] = 49 + q, False       # the prefix would begin behind its first new token
    b = Batch(4, 2, 64, 16, dtype, [q] * n, own, [50, 50, 0], [2, 8, 8, 12], shares=shares, room=room)
    for max_q in (q, 0):
        o, lse = m.shared_prefix_attention(*b.device(), max_q_len=max_q, return_lse=True)
        b.check(o, lse)


@pytest.mark.parametrize("room", [0, 60000])
def test_equal_groups_and_lengths_without_their_tables(room):
    import experiment_swa_kda_b200 as m
    for q in (1, 6, 70):
        b = Batch(8, 2, 128, 16, BF16, [q] * 6, [q, q + 1, 70, 79, 78, 100], [77, 128, 200], [0, 2, 4, 6], room=room)
        args = b.device()
        args[7] = args[8] = None
        o, lse = m.shared_prefix_attention(*args, return_lse=True, scale=0.2)
        b.check(o, lse, scale=0.2)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q", [1, 10, 24, 130])
@pytest.mark.parametrize("room", [0, 60000])
def test_values_that_are_not_finite(dtype, q, room):
    """Infinite and undefined values at keys that are seen, in the prefix and behind it; scores of -inf throughout."""
    import experiment_swa_kda_b200 as m
    for where in ("prefix_v", "prefix_k", "own_v", "last_v", "minus"):
        b = Batch(4, 2, 64, 16, dtype, [q] * 5, [q + 3, q, 30 + q, 2 + q, q], [150], [0, 5], seed=3, room=room)
        page = 16
        at = {"prefix_v": (int(b.prefix_table[0, 3]), 5), "prefix_k": (int(b.prefix_table[0, 9]), 2), "own_v": (int(b.table[2, (160) // page]), 160 % page),
              "last_v": (int(b.table[0, (b.kv_lens[0] - 1) // page]), (b.kv_lens[0] - 1) % page)}.get(where)
        if where == "minus":      # every key of the prefix and of sequence 0's first own key scores -inf against row 0
            b.q[0] = 1.0
            for p in range(150):
                b.k[int(b.prefix_table[0, p // page]), p % page] = -math.inf
            for p in range(150, b.kv_lens[0]):
                b.k[int(b.table[0, p // page]), p % page] = -math.inf
        elif where == "prefix_k":
            b.k[at[0], at[1], 1] = math.nan
        else:
            b.v[at[0], at[1], 0, 7], b.v[at[0], at[1], 1, 3], b.v[at[0], at[1], 1, 4] = math.inf, -math.inf, math.nan
        o = m.shared_prefix_attention(*b.device(), max_q_len=q)
        want, _, size = b.want()
        if where == "minus":
            # rows other than the first have scores of both signs and infinities: NaN in both, as the formula says
            assert bool(torch.isnan(want[0]).all()) and bool(torch.isnan(o[0]).all())
            continue
        close(o, want, size, dtype)


def test_equals_paged_attention_where_rows_hold_the_prefix():
    """Tables whose rows name the prefix's pages themselves: both operators say the same up to rounding."""
    import experiment_swa_kda_b200 as m
    b = Batch(16, 4, 128, 64, BF16, [1] * 40, [(37 * i) % 500 + 1 for i in range(40)], [1024], [0, 40])
    args = b.device()
    table = args[3].clone()
    table[:, :16] = args[5][0, :16]
    one, lse1 = m.shared_prefix_attention(*args, max_q_len=1, return_lse=True)
    two, lse2 = m.paged_attention(args[0], args[1], args[2], table, args[4], args[8], max_q_len=1, return_lse=True)
    assert (lse1 - lse2).abs().max() <= 1e-4
    # one rounding each, and the weights' of the tensor-core kernel
    assert (one.double() - two.double()).norm() <= 3 * U * two.double().norm()


@pytest.mark.parametrize("room", [0, 60000])
def test_inconsistent_arrays_are_bounded_and_told(room):
    import experiment_swa_kda_b200 as m
    fine = Batch(4, 2, 64, 16, BF16, [1] * 4, [3, 4, 5, 6], [40], [0, 4])
    for dtype in (BF16, F32):
        for at, bad, match in ((7, [0, 9], "cu_seqlens"), (7, [3, 1], "cu_seqlens|block table"), (7, [-2, 4], "cu_seqlens"), (6, [-1], "block table"), (6, [10 ** 6], "block table"),
                               (8, [0, 1, 2, 9, 4], "cu_seqlens"), (8, [0, 1, 2, 3, 3], "cu_seqlens"), (4, [43, 10 ** 6, 45, 46], "block table"),
                               (5, [[-1, 99, -7]], "block table")):
            args = Batch(4, 2, 64, 16, dtype, [1] * 4, [3, 4, 5, 6], [40], [0, 4], garbage=0.0, room=room).device()
            args[at] = torch.tensor(bad, dtype=torch.int32, device=DEV)
            for max_q in (1, 0):
                m.shared_prefix_attention(*args, max_q_len=max_q)
                torch.cuda.synchronize()
                with pytest.raises(RuntimeError, match=match):
                    m.shared_prefix_attention(*fine.device(), max_q_len=1)
    o = m.shared_prefix_attention(*fine.device(), max_q_len=1)
    fine.check(o)


@pytest.mark.parametrize("room", [0, 60000])
def test_captured_on_another_stream_and_graphs_at_once(room):
    import experiment_swa_kda_b200 as m
    batches = [Batch(16, 4, 128, 16, BF16, [q] * 12, [(13 * i) % 90 + q for i in range(12)], [600], [0, 12], seed=q, room=room) for q in (1, 6, 100)]
    args = [b.device() for b in batches]
    wants = [m.shared_prefix_attention(*a, max_q_len=q) for a, q in zip(args, (1, 6, 100))]
    for b, w in zip(batches, wants):
        b.check(w)
    graphs, outs = [], []
    for a, q in zip(args, (1, 6, 100)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(m.shared_prefix_attention(*a, max_q_len=q))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, wants):
        assert torch.equal(o, w)
    # the device arrays are followed: two tokens fewer in one sequence
    args[0][4][3] -= 2
    batches[0].kv_lens[3] -= 2
    graphs[0].replay()
    batches[0].check(outs[0])


def test_refusals():
    import experiment_swa_kda_b200 as m
    b = Batch(4, 2, 64, 16, BF16, [1] * 4, [3, 4, 5, 6], [40], [0, 4])
    for at, bad, match in ((5, torch.zeros(1, 3, device=DEV), "prefix_table"), (5, torch.zeros(5, 3, dtype=torch.int32, device=DEV), "prefix_table"),
                           (6, torch.zeros(2, dtype=torch.int32, device=DEV), "prefix_lens"), (7, torch.zeros(3, dtype=torch.int32, device=DEV), "cu_groups"),
                           (6, torch.zeros(1, dtype=torch.int32), "CPU"), (5, torch.zeros(1, 6, dtype=torch.int32, device=DEV)[:, ::2], "adjacent")):
        args = b.device()
        args[at] = bad
        with pytest.raises((ValueError, RuntimeError), match=match):
            m.shared_prefix_attention(*args, max_q_len=1)
    args = b.device()
    with pytest.raises(ValueError, match="scale"):
        m.shared_prefix_attention(*args, scale=0.0)
    with pytest.raises(ValueError, match="max_q_len"):
        m.shared_prefix_attention(*args, max_q_len=-1)
    args[5], args[6], args[7] = (torch.zeros(3, 3, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV), None)
    with pytest.raises(ValueError, match="cu_groups"):
        m.shared_prefix_attention(*args)
    args = b.device()
    args[0] = args[0].requires_grad_(True)
    with pytest.raises(RuntimeError, match="inference"):
        m.shared_prefix_attention(*args)
    args[0] = args[0].detach()[:0]
    args[8] = torch.zeros(5, dtype=torch.int32, device=DEV)
    assert m.shared_prefix_attention(*args).shape == (0, 4, 64)


def test_serving_with_a_pool_and_a_prefix():
    """A step as a scheduler makes it: pages are planned, keys and values appended, attention reads the prefix once."""
    import experiment_swa_kda_b200 as m
    torch.manual_seed(5)
    layer = m.PagedAttention(256, 4, 2, 64, max_positions=512).to(DEV)
    page, prefix = 16, 101
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    text = torch.randn(1, prefix, 256, device=DEV).bfloat16()
    # row 3 of the pool's table holds the prefix, rows 0 .. 2 are places for requests
    pool = m.PagedCache.pool(4, 300, 60, page, 2, 64, DEV)
    pool.kv_lens.copy_(i32([0, 0, 0, prefix]))
    cu, _, _ = pool.plan(i32([0, 0, 0, prefix]), prefix)
    layer(text, pool, cu, max_q_len=prefix)
    whole = m.PagedCache.zeros(3, 300, page, 2, 64, DEV)
    whole.kv_lens.fill_(prefix)
    layer(text.expand(3, -1, -1), whole)
    serve = m.PagedCache(pool.k, pool.v, pool.block_table[:3], pool.kv_lens[:3], prefix_table=pool.block_table[3:], prefix_lens=pool.kv_lens[3:])
    lens = [prefix] * 3
    for new in ([5, 40, 1], [1, 1, 1], [1, 1, 1], [2, 7, 30]):
        lens = [a + b for a, b in zip(lens, new)]
        pool.kv_lens.copy_(i32(lens + [prefix]))
        whole.kv_lens.copy_(i32(lens))
        cu, positions, slots = pool.plan(i32(new + [0]), sum(new), starts=i32([prefix] * 3 + [0]))
        x = torch.randn(1, sum(new), 256, device=DEV).bfloat16()
        got, want = layer(x, serve, cu[:4], max_q_len=max(new)), layer(x, whole, cu[:4], max_q_len=max(new))
        # two attention outputs of one rounding and one set of rounded weights each, through one projection
        assert (got.double() - want.double()).norm() <= 1e-2 * want.double().norm()
    assert int((~pool.page_free).sum()) == -(-prefix // page) + sum(-(-n // page) - prefix // page for n in lens)


def test_a_captured_step_of_a_scheduler():
    """Lengths, pages, cache and attention of a token step in one graph, replayed across page borders."""
    import experiment_swa_kda_b200 as m
    torch.manual_seed(6)
    layer = m.PagedAttention(256, 4, 2, 64, max_positions=512).to(DEV)
    page, prefix, rows = 8, 45, 3
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    text = torch.randn(1, prefix, 256, device=DEV).bfloat16()
    pool = m.PagedCache.pool(rows + 1, 200, 60, page, 2, 64, DEV)      # the last row holds the prefix
    pool.kv_lens.copy_(i32([0] * rows + [prefix]))
    layer(text, pool, pool.plan(i32([0] * rows + [prefix]), prefix)[0], max_q_len=prefix)
    whole = m.PagedCache.zeros(rows, 200, page, 2, 64, DEV)
    whole.kv_lens.fill_(prefix)
    layer(text.expand(rows, -1, -1), whole)
    serve = m.PagedCache(pool.k, pool.v, pool.block_table[:rows], pool.kv_lens[:rows], prefix_table=pool.block_table[rows:], prefix_lens=pool.kv_lens[rows:])
    pool.kv_lens[:rows] = prefix
    new, starts, x = i32([1] * rows + [0]), i32([prefix] * rows + [0]), torch.zeros(1, rows, 256, device=DEV, dtype=BF16)

    def step():
        pool.kv_lens[:rows] += 1
        cu, _, slots = pool.plan(new, rows, starts=starts)
        return layer(x, serve, cu[:rows + 1], max_q_len=1), slots

    kept = pool.block_table.clone(), pool.page_free.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):      # a first call outside of the graph
        step()
    torch.cuda.synchronize()
    pool.block_table.copy_(kept[0]), pool.page_free.copy_(kept[1]), pool.kv_lens[:rows].fill_(prefix)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, slots = step()
    for i in range(20):
        x.copy_(torch.randn(1, rows, 256, device=DEV))
        graph.replay()
        whole.kv_lens += 1
        want = layer(x[0][:, None], whole)
        assert (y[0].double() - want[:, 0].double()).norm() <= 1e-2 * want.double().norm()
        assert torch.equal(slots // page, pool.block_table[:rows, (prefix + i) // page].long()) and bool((slots % page == (prefix + i) % page).all())
    assert pool.kv_lens.tolist() == [prefix + 20] * rows + [prefix]


def test_calls_on_two_streams_at_once():
    """Two calls on two streams at once, each with a workspace of its own."""
    import experiment_swa_kda_b200 as m
    batches = [Batch(16, 4, 128, 64, BF16, [1] * 40, [(17 * i) % 300 + 1 for i in range(40)], [1500], [0, 40], seed=s, room=60000) for s in (1, 2)]
    args = [b.device() for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(m.shared_prefix_attention(*args[i], max_q_len=1))
    torch.cuda.synchronize()
    for b, of in zip(batches, outs):
        b.check(of[0])
        assert all(torch.equal(of[0], o) for o in of)


@pytest.mark.parametrize("q,room,dtype", [(1, 0, BF16), (1, 60000, BF16), (6, 60000, BF16), (100, 0, BF16), (100, 60000, BF16), (3, 0, F32)])
def test_inputs_written_just_before_the_call(q, room, dtype):
    """Kernels that start while the launch before them ends read what that one wrote."""
    import experiment_swa_kda_b200 as m
    two = [Batch(8, 2, 64, 16, dtype, [q] * 24, [(s + 11 * i) % 60 + q for i in range(24)], [300 + 16 * s], [0, 24], seed=s, room=room) for s in (1, 4)]
    width = max(b.table.shape[1] for b in two), max(b.prefix_table.shape[1] for b in two)
    pages = max(b.k.shape[0] for b in two)
    fit = lambda t, n, d: torch.cat((t, t.new_zeros((n - t.shape[d],) + t.shape[1:]) if d == 0 else t.new_full((t.shape[0], n - t.shape[1]), -1)), d)
    sets = []
    for b in two:
        a = b.device()
        a[1], a[2], a[3], a[5] = fit(a[1], pages, 0), fit(a[2], pages, 0), fit(a[3], width[0], 1), fit(a[5], width[1], 1)
        sets.append([t.contiguous() for t in a])
    live = [t.clone() for t in sets[0]]
    wants = [m.shared_prefix_attention(*a, max_q_len=q) for a in sets]
    for b, w in zip(two, wants):
        b.check(w)
    torch.cuda.synchronize()
    order = [0, 1, 1, 0] * 8
    outs = []
    for i in order:
        for t, src in zip(live, sets[i]):
            t.copy_(src)
        outs.append(m.shared_prefix_attention(*live, max_q_len=q))
    assert all(torch.equal(o, wants[i]) for o, i in zip(outs, order))
