"""What the serving operators do to the caller's arrays: nothing when they refuse, and the same when one array stands for two."""

import pytest
import torch

from test_plan_pages_gpu import DEV, i32

pytestmark = pytest.mark.gpu


def test_arrays_of_inference_mode_outside_of_it():
    """torch refuses to write them in place; so do the operators, and leave them as they were."""
    import experiment_swa_kda_b200 as m
    with torch.inference_mode():
        cache = m.PagedCache.pool(2, 32, 8, 4, 2, 32, DEV)
        cache.kv_lens.copy_(i32([5, 3]))
        new, q, k = i32([5, 3]), torch.randn(8, 4, 32, device=DEV).bfloat16(), torch.randn(8, 2, 32, device=DEV).bfloat16()
        cos = sin = torch.ones(32, 16, device=DEV)
    with pytest.raises(RuntimeError, match="InferenceMode"):
        cache.plan(new, 8)
    torch.cuda.synchronize()
    with torch.inference_mode():
        assert bool((cache.block_table == -1).all()) and bool(cache.page_free.all())
        cu, _, _ = cache.plan(new, 8)
        assert cu.tolist() == [0, 5, 8]
    cu = i32([0, 5, 8])
    with pytest.raises(RuntimeError, match="InferenceMode"):
        m.qk_norm_rope_append(q, k, k, cos, sin, cache.k, cache.v, cache.block_table, cache.kv_lens, cu)
    torch.cuda.synchronize()
    with torch.inference_mode():
        assert bool((cache.k == 0).all()) and bool((cache.v == 0).all())
        m.qk_norm_rope_append(q, k, k, cos, sin, cache.k, cache.v, cache.block_table, cache.kv_lens, cu)
        assert not bool((cache.v == 0).all())


@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("overtake", [False, True])
def test_one_array_for_lengths_and_new_tokens(rows, overtake):
    """A first step, in which all of a request is new: the lengths are the new tokens' counts themselves."""
    import experiment_swa_kda_b200 as m
    lens = [(7 * n) % 30 for n in range(rows)]
    outs = []
    for same in (False, True):
        table, free = torch.full((rows, 8), -1, dtype=torch.int32, device=DEV), torch.ones(rows * 3, dtype=torch.bool, device=DEV)
        kv = i32(lens)
        new = kv if same else i32(lens)
        outs.append([*m.plan_pages(table, kv, free, new, page_size=4, max_tokens=sum(lens) * 2 // 3, overtake=overtake), table, free, kv])
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and 0 < int(outs[0][-1].sum()) < sum(lens)
