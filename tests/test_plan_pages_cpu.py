"""Pages of a step: refusals, and the restatement itself, without a GPU."""

import pytest
import torch

import experiment_swa_kda_b200 as m
import serving_oracle as S


def args():
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    return [torch.full((2, 4), -1, dtype=torch.int32), i32(5, 0), torch.ones(6, dtype=torch.bool), i32(5, 0)]


def test_refusals_name_the_argument():
    with pytest.raises(RuntimeError, match="CPU"):
        m.plan_pages(*args(), page_size=4, max_tokens=8)
    for at, bad, match in ((0, torch.zeros(2, 4), "block_table"), (0, torch.zeros(2, 0, dtype=torch.int32), "block_table"), (1, torch.zeros(3, dtype=torch.int32), "kv_lens"),
                           (2, torch.ones(6), "page_free"), (3, torch.zeros(2), "new_lens")):
        a = args()
        a[at] = bad
        with pytest.raises(ValueError, match=match):
            m.plan_pages(*a, page_size=4, max_tokens=8)
    with pytest.raises(ValueError, match="page_size"):
        m.plan_pages(*args(), page_size=0, max_tokens=8)
    with pytest.raises(ValueError, match="starts"):
        m.plan_pages(*args(), page_size=4, max_tokens=8, starts=torch.zeros(2))
    with pytest.raises(RuntimeError, match="pool"):
        m.PagedCache.zeros(2, 8, 4, 1, 16, "cpu").plan(torch.zeros(2, dtype=torch.int32), 4)


def test_abi_checks_run_before_any_launch():
    from experiment_swa_kda_b200 import _lib
    lib = _lib.load()
    s = _lib.PlanShape(rows=2, width=4, page_size=4, n_pages=6, max_tokens=8, table_stride=4)
    assert lib.kda_plan_pages(s, *([None] * 9), 0, None) == -5
    s.rows = 16385
    assert lib.kda_plan_pages(s, *([None] * 9), 0, None) == -2 and lib.kda_plan_pages_workspace_bytes(s) == 0
    s.rows, s.width, s.page_size = 2, 1 << 20, 1 << 12
    assert lib.kda_plan_pages(s, *([None] * 9), 0, None) == -1


def test_restatement_by_hand():
    """Two rows of four-token pages: growth, a hole, a row that waits, and what it gives back."""
    table, lens, free, cu, pos, slots = S.plan_pages([[-1] * 4, [-1] * 4], [5, 3], [True] * 6, [5, 3], 4, 8)
    assert (table, cu) == ([[0, 1, -1, -1], [2, -1, -1, -1]], [0, 5, 8]) and free == [False] * 3 + [True] * 3
    assert slots == [0, 1, 2, 3, 4, 8, 9, 10] and pos == [0, 1, 2, 3, 4, 0, 1, 2]
    # row 0 ends, row 1 grows into the pages that leaves; seven tokens are too many for a step of six
    table, lens, free, cu, pos, slots = S.plan_pages(table, [0, 10], free, [0, 7], 4, 6)
    assert (lens, cu, pos) == ([0, 3], [0, 0, 0], [-1] * 6) and table == [[-1] * 4, [2, -1, -1, -1]] and free == [True, True, False, True, True, True]
    table, lens, free, cu, pos, slots = S.plan_pages(table, [0, 10], free, [0, 7], 4, 7, starts=[0, 4])
    # a start inside the row: the page before it goes back
    table, lens, free, cu, pos, slots = S.plan_pages(table, [0, 10], free, [0, 6], 4, 7, starts=[0, 4])
    assert table == [[-1] * 4, [-1, 0, 1, -1]] and pos == [4, 5, 6, 7, 8, 9, -1] and slots == [0, 1, 2, 3, 4, 5, -1]
    assert free == [False, False, True, True, True, True]
