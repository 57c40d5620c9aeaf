"""The serving lines of the package's introduction, run as they stand there."""

import os

import pytest
import torch

import serving_oracle as S

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def lines(first, last):
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")).read()
    return text[text.index(first):text.index(last)]


@pytest.mark.parametrize("pages", [2000, 17])
def test_many_requests_behind_one_text(pages):
    """Eight requests behind a text of 100 tokens, some at the end of a page; in the small pool some of these wait, keep what they have and get no output."""
    import experiment_swa_kda_b200 as m
    torch.manual_seed(4)
    code = lines("# many requests behind one text", "# behind the reference's own boundary")
    assert code.count("pages=2000") == 1 and code.count("pool.plan(") == 1
    build, step = code.replace("pages=2000", f"pages={pages}").split("cu_seqlens, positions", 1)
    step = "cu_seqlens, positions" + step
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    names = {"torch": torch, "PagedCache": m.PagedCache, "PagedAttention": m.PagedAttention}
    exec(build, names)
    pool, prefix, own = names["pool"], 100, [4, 12, 28, 5, 60, 11, 12, 1]      # 100 + 12 and 100 + 28 fill their pages
    own = own if pages == 2000 else [4, 12, 28, 5, 12, 11, 12, 1]
    pool.k.normal_(), pool.v.normal_()
    names["starts"] = i32([prefix] * 8 + [0])
    pool.kv_lens.copy_(i32([prefix + x for x in own] + [prefix]))
    names["new_lens"] = pool.kv_lens.clone()
    pool.plan(names["new_lens"], max_tokens=4096, starts=names["starts"])      # the pages of what they have, written above
    held = pool.block_table.clone()
    before = pool.k.clone(), pool.v.clone()
    names["new_lens"] = i32([1] * 8 + [0])
    pool.kv_lens[:8] += 1
    want = S.plan_pages(held.tolist(), pool.kv_lens.tolist(), pool.page_free.tolist(), [1] * 8 + [0], 16, 8, [prefix] * 8 + [0])
    names["x"] = torch.randn(8, 384, device=DEV).bfloat16()
    exec(step, names)
    torch.cuda.synchronize()
    assert pool.kv_lens.tolist() == want[1] and names["cu_seqlens"].tolist() == want[3]
    served = [b - a for a, b in zip(want[3], want[3][1:])][:8]
    assert (sum(served) == 8) == (pages == 2000)
    for n in range(8):
        for c, now in zip(before, (pool.k, pool.v)):
            for col in range(prefix // 16, -(-(prefix + own[n]) // 16)):
                lo, hi = max(prefix - 16 * col, 0), min(prefix + own[n] - 16 * col, 16)
                assert torch.equal(now[held[n, col].long(), lo:hi], c[held[n, col].long(), lo:hi])
    y = names["y_t"][0]
    assert y.shape == (8, 384) and bool((y[sum(served):] == 0).all()) and bool((y[:sum(served)] != 0).any(-1).all())
    assert names["row"].tolist() == [n for n in range(8) if served[n]] + [8] * (8 - sum(served))
    names["full"](names["x"][:0].view(1, 0, 384), names["serve"], torch.zeros(9, dtype=torch.int32, device=DEV))      # nothing was reported
