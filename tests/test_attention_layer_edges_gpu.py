"""The attention layer at the edges of what its arguments allow."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_a_step_without_tokens(shared, packed):
    """No sequence has a new token: an empty result, and the cache as it was."""
    import experiment_swa_kda_b200 as m
    layer = m.PagedAttention(128, 4, 2, 32, max_positions=64).to(DEV)
    cache = m.PagedCache.zeros(3, 40, 8, 2, 32, DEV)
    cache.kv_lens.fill_(9)
    if shared:
        cache.prefix_table, cache.prefix_lens = cache.block_table[:1].clone(), torch.full((1,), 8, dtype=torch.int32, device=DEV)
    before = cache.k.normal_().clone()
    x = torch.zeros(1 if packed else 3, 0, 128, device=DEV, dtype=torch.bfloat16)
    y = layer(x, cache, torch.zeros(4, dtype=torch.int32, device=DEV) if packed else None)
    assert y.shape == x.shape and torch.equal(cache.k, before)
