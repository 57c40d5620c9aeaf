"""Pages of a step where rows that have to wait hold up nobody: against the restatement row by row, whole numbers, all equal."""

import random

import pytest
import torch

import serving_oracle as S
from test_plan_pages_gpu import DEV, Pool, i32

pytestmark = pytest.mark.gpu


class Overtaking(Pool):
    def step(self, lens, new, most, starts=None):
        import experiment_swa_kda_b200 as m
        kv = i32(lens)
        out = m.plan_pages(self.table, kv, self.free, i32(new), page_size=self.page, max_tokens=most, starts=None if starts is None else i32(starts), overtake=True)
        self.check(lens, new, most, starts, kv, *out)

    def check(self, lens, new, most, starts, kv, cu, pos, slots):
        table, want_lens, free, want_cu, want_pos, want_slots = S.plan_pages(self.want[0], lens, self.want[1], new, self.page, most, starts, overtake=True)
        self.want, self.lens = (table, free), want_lens
        assert cu.tolist() == want_cu and kv.tolist() == want_lens and pos.tolist() == want_pos and slots.tolist() == want_slots
        assert self.table.tolist() == table and self.free.tolist() == free
        assert bool((self.buffer[:, self.table.shape[1]:] == -7).all())


def test_a_prompt_that_does_not_fit_holds_up_nobody():
    pool = Overtaking(4, 8, 6, 4)
    pool.step([0, 5, 3, 0], [0, 5, 3, 0], 32)
    pool.step([32, 6, 4, 0], [32, 1, 1, 0], 40)           # place 0 asks for eight pages of three
    assert pool.lens == [0, 6, 4, 0]
    pool.step([32, 7, 5, 12], [32, 1, 1, 12], 40)         # place 2 takes a page, place 3 lacks one
    assert pool.lens == [0, 7, 5, 0]
    pool.step([8, 8, 6, 0], [8, 1, 1, 0], 9)              # tokens run out behind place 1
    assert pool.lens == [8, 8, 5, 0]
    pool.step([0, 8, 8, 0], [0, 0, 0, 0], 0)
    assert pool.lens == [0, 8, 8, 0]


@pytest.mark.parametrize("rows,width,pages,page,wide,offset", [
    (1, 1, 1, 1, 0, 0), (2, 4, 5, 4, 3, 1), (31, 40, 200, 4, 0, 0), (33, 40, 300, 16, 5, 3), (64, 128, 700, 8, 0, 16), (257, 33, 1500, 16, 1, 7),
    (1025, 9, 2000, 16, 0, 0), (300, 20, 70000, 1, 0, 0)])
def test_steps_of_a_scheduler(rows, width, pages, page, wide, offset):
    """Requests come, grow, take tokens back and leave; the pool and the tokens are short nearly always."""
    rng = random.Random(rows * 1000 + width)
    pool, lens = Overtaking(rows, width, pages, page, wide, offset), [0] * rows
    room, waited = width * page, 0
    for step in range(8):
        new, starts, target = [0] * rows, [0] * rows, list(lens)
        for n in range(rows):
            what = rng.random()
            if lens[n] == 0 and what < 0.7:
                new[n] = min(room, max(1, round(rng.random() ** 2 * min(room, 8 * pages * page // rows + 1))))
                target[n] = new[n]
            elif what < 0.1:
                target[n] = 0
            elif what < 0.3:
                target[n] = rng.randint(0, lens[n])
                new[n] = rng.randint(0, min(target[n], 3))
            elif what < 0.9:
                new[n] = min(rng.choice((1, 1, 1, 4, page, 2 * page + 1)), room - lens[n])
                target[n] = lens[n] + new[n]
            starts[n] = rng.choice((0, 0, 0, target[n] // 2, max(target[n] - new[n], 0)))
        most = max(1, sum(new) if step % 3 else sum(new) // 2)
        pool.step(target, new, most, starts if step % 2 else None)
        waited += sum(a != b for a, b in zip(target, pool.lens))
        lens = list(pool.lens)
    assert waited or rows < 3


@pytest.mark.parametrize("seed", range(4))
def test_rows_that_just_fit_between_rows_that_do_not(seed):
    """Rows of one to seven pages and tokens against a pool and a step that run out little by little."""
    rng = random.Random(seed)
    rows = 200
    pool = Overtaking(rows, 8, 300, 2)
    asks = [rng.choice((0, 1, 2, 3, 9, 14)) for _ in range(rows)]
    pool.step(asks, asks, 500 if seed % 2 else 10 ** 6)
    lens = pool.lens
    asks = [min(16, a + rng.choice((0, 1, 2, 5))) for a in lens]
    pool.step(asks, [b - a for a, b in zip(lens, asks)], 150 if seed % 2 else 10 ** 6)


def test_numbers_at_the_edge_of_32_bits():
    """Rows that ask for as many tokens as fit in 32 bits, next to ones that ask for few."""
    big = 2 ** 31 - 2 ** 20
    pool = Overtaking(40, 1, 20, big)
    asks = [big if n % 3 else 1 for n in range(40)]
    pool.step(asks, asks, 30)
    assert pool.lens == [0 if n % 3 else 1 for n in range(40)]


def test_as_many_rows_as_one_call_takes():
    rows = 16384
    pool = Overtaking(rows, 2, rows // 2, 4)
    lens = [(n * 5) % 9 for n in range(rows)]
    pool.step(lens, lens, sum(lens) // 3)
    assert 0 < sum(pool.lens) < sum(lens)


def test_a_cache_whose_requests_overtake():
    import experiment_swa_kda_b200 as m
    cache = m.PagedCache.pool(3, 64, 4, 8, 1, 32, DEV)
    cache.kv_lens.copy_(i32([64, 9, 8]))
    cu, _, _ = cache.plan(i32([64, 9, 8]), 100, overtake=True)
    assert cu.tolist() == [0, 0, 9, 17] and cache.kv_lens.tolist() == [0, 9, 8]
    cache.kv_lens.copy_(i32([64, 9, 8]))
    assert cache.plan(i32([64, 0, 0]), 100)[0].tolist() == [0, 0, 0, 0]
