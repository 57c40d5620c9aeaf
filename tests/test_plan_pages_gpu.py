"""Pages of a step against a restatement row by row (oracle/serving_oracle.py): whole numbers, all equal."""

import random

import pytest
import torch

import serving_oracle as S

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Pool:
    """The device's state beside the restatement's, compared after every step."""

    def __init__(self, rows, width, pages, page, wide=0, offset=0):
        self.page = page
        self.buffer = torch.full((rows, width + wide), -7, dtype=torch.int32, device=DEV)
        self.table = self.buffer[:, :width]
        self.table.fill_(-1)
        self.free = torch.ones(pages + offset, dtype=torch.bool, device=DEV)[offset:]
        self.want = ([[-1] * width for _ in range(rows)], [True] * pages)

    def step(self, lens, new, most, starts=None):
        import experiment_swa_kda_b200 as m
        kv = i32(lens)
        cu, pos, slots = m.plan_pages(self.table, kv, self.free, i32(new), page_size=self.page, max_tokens=most, starts=None if starts is None else i32(starts))
        self.check(lens, new, most, starts, kv, cu, pos, slots)
        return kv

    def check(self, lens, new, most, starts, kv, cu, pos, slots):
        table, want_lens, free, want_cu, want_pos, want_slots = S.plan_pages(self.want[0], lens, self.want[1], new, self.page, most, starts)
        self.want = (table, free)
        self.lens = want_lens
        assert cu.tolist() == want_cu and kv.tolist() == want_lens
        assert pos.dtype == torch.int32 and slots.dtype == torch.int64 and pos.tolist() == want_pos and slots.tolist() == want_slots
        assert self.table.tolist() == table and self.free.tolist() == free
        assert bool((self.buffer[:, self.table.shape[1]:] == -7).all())


@pytest.mark.parametrize("rows,width,pages,page,wide,offset", [
    (1, 1, 1, 1, 0, 0), (1, 512, 1024, 16, 0, 0), (2, 4, 5, 4, 3, 1), (3, 129, 250, 1, 0, 0), (17, 40, 300, 16, 5, 3), (64, 128, 5000, 8, 0, 16),
    (100, 130, 20000, 48, 0, 0), (257, 33, 4001, 64, 1, 7), (1025, 9, 9000, 16, 0, 0), (5, 1000, 16385, 32, 0, 0)])
def test_steps_of_a_scheduler(rows, width, pages, page, wide, offset):
    """Requests come, grow, take tokens back and leave; the pool runs short now and then."""
    rng = random.Random(rows * 1000 + width)
    pool, lens = Pool(rows, width, pages, page, wide, offset), [0] * rows
    room = width * page
    for step in range(7):
        new, starts, target = [0] * rows, [0] * rows, list(lens)
        for n in range(rows):
            what = rng.random()
            if lens[n] == 0 and what < 0.6:
                new[n] = min(room, max(1, round(rng.random() ** 3 * min(room, 3 * pages * page // rows + 1))))
                target[n] = new[n]
            elif what < 0.2:
                target[n] = 0
            elif what < 0.4:
                target[n] = rng.randint(0, lens[n])
                new[n] = rng.randint(0, min(target[n], 3))
            elif what < 0.9:
                new[n] = min(rng.choice((1, 1, 1, 4, page, 2 * page + 1)), room - lens[n])
                target[n] = lens[n] + new[n]
            starts[n] = rng.choice((0, 0, 0, target[n] // 2, max(target[n] - new[n], 0), target[n]))
        most = max(1, sum(new) - (step % 3 == 2) * rng.randint(0, max(new)))
        pool.step(target, new, most, starts if step % 2 else None)
        lens = list(pool.lens)


def test_a_step_done_again_changes_nothing():
    pool = Pool(6, 20, 80, 4)
    lens = [3, 0, 41, 80, 1, 16]
    pool.step(lens, lens, sum(lens))
    before = pool.table.clone(), pool.free.clone()
    pool.step(lens, [1, 0, 4, 1, 1, 16], 23)
    assert torch.equal(before[0], pool.table) and torch.equal(before[1], pool.free)


def test_short_of_pages_and_of_tokens():
    pool = Pool(4, 8, 6, 4)
    pool.step([8, 12, 9, 4], [8, 12, 9, 4], 64)      # 2 + 3 pages; row 2 would need 3 more and waits, row 3 behind it as well
    assert pool.lens == [8, 12, 0, 0]
    pool.step([8, 12, 9, 4], [0, 0, 9, 4], 64)       # rows that lack nothing are served
    assert pool.lens == [8, 12, 0, 0]
    pool.step([0, 12, 9, 4], [0, 0, 9, 4], 9)        # tokens for one of them
    assert pool.lens == [0, 12, 9, 0]
    pool.step([0, 12, 9, 4], [0, 0, 0, 0], 0)        # a length without new tokens and without pages waits too
    assert pool.lens == [0, 12, 9, 4] and pool.table[3].tolist() == [-1] * 8


def test_rows_that_wait_give_back_what_they_do_not_need():
    """A place in the batch changes hands: the next request finds its pages there, has to wait, and gives them back."""
    pool = Pool(2, 8, 5, 4)
    pool.step([12, 4], [12, 4], 16)
    pool.step([20, 4], [20, 0], 20)
    assert pool.lens == [0, 4] and pool.free.tolist() == [True, True, True, False, True]


def test_inconsistent_numbers_are_bounded_and_told():
    import experiment_swa_kda_b200 as m
    ok = lambda: m.plan_pages(torch.full((1, 1), -1, dtype=torch.int32, device=DEV), i32([0]), torch.ones(1, dtype=torch.bool, device=DEV), i32([0]),
                              page_size=1, max_tokens=0)
    big = 2 ** 31 - 1
    for lens, new, starts, entry, match in (([-5, 4], [2, 4], None, None, "block table"), ([33, 4], [3, 4], None, None, "block table"),
                                            ([big, 4], [big, 4], [big, -big], None, "block table"), ([8, 4], [9, -1], None, None, "cu_seqlens"),
                                            ([8, 4], [8, 4], [-3, 100], None, None), ([8, 4], [8, 4], None, 20, "block table"),
                                            ([8, 4], [8, 4], None, -2, None), ([0, 4], [0, 4], None, big, "block table")):
        pool = Pool(2, 8, 20, 4)
        if entry is not None:
            pool.table[0, 1] = entry
            pool.want[0][0][1] = entry
        pool.step(lens, new, 32, starts)
        torch.cuda.synchronize()
        if match is None:
            ok()
        else:
            with pytest.raises(RuntimeError, match=match):
                ok()
        ok()


def test_captured_and_on_another_stream():
    import experiment_swa_kda_b200 as m
    pool = Pool(5, 16, 50, 4)
    lens, new = i32([0] * 5), i32([0] * 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.plan_pages(pool.table, lens, pool.free, new, page_size=4, max_tokens=40)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.plan_pages(pool.table, lens, pool.free, new, page_size=4, max_tokens=40)
    for want, add in (([7, 0, 13, 4, 1], [7, 0, 13, 4, 1]), ([8, 9, 14, 0, 1], [1, 9, 1, 0, 0]), ([64, 9, 14, 64, 5], [56, 0, 0, 64, 4])):
        lens.copy_(i32(want))
        new.copy_(i32(add))
        graph.replay()
        pool.check(want, add, 40, None, lens, *out)


def test_as_many_rows_as_one_call_takes():
    rows = 16384
    pool = Pool(rows, 2, 2 * rows + 5, 4)
    lens = [(n * 5) % 9 for n in range(rows)]
    pool.step(lens, lens, sum(lens) + 100)
    with pytest.raises(RuntimeError, match="too large"):
        Pool(rows + 1, 1, 4, 4).step([0] * (rows + 1), [0] * (rows + 1), 0)


def test_a_cache_with_a_pool():
    import experiment_swa_kda_b200 as m
    torch.manual_seed(2)
    layer = m.PagedAttention(256, 4, 2, 64, max_positions=256).to(DEV)
    pool, whole = m.PagedCache.pool(3, 200, 20, 16, 2, 64, DEV), m.PagedCache.zeros(3, 200, 16, 2, 64, DEV)
    lens = [0, 0, 0]
    for new in ([40, 1, 70], [1, 30, 1], [17, 1, 5]):
        lens = [a + b for a, b in zip(lens, new)]
        for cache in (pool, whole):
            cache.kv_lens.copy_(i32(lens))
        cu, positions, slots = pool.plan(i32(new), sum(new))
        assert positions.tolist() == [p for a, b in zip(lens, new) for p in range(a - b, a)]
        x = torch.randn(1, sum(new), 256, device=DEV).bfloat16()
        got, want = (layer(x, cache, cu, max_q_len=max(new)) for cache in (pool, whole))
        assert torch.equal(got, want)
        qkv = layer.qkv_proj(x).reshape(-1, 8, 64)
        assert torch.equal(pool.v.view(-1, 2, 64)[slots], qkv[:, 6:])
