"""KDA and attention layers serving together (examples/hybrid_serving.py): a prompt in chunks and token by token against one call,
and the attention layer against a float64 restatement."""

import os
import sys

import pytest
import torch

import attention_oracle as A

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))

pytestmark = pytest.mark.gpu


def test_pieces_of_a_prompt_match_the_whole():
    import hybrid_serving
    # four bf16 layers in series: the bound that the layer tests use for several bf16 products one after the other
    assert hybrid_serving.main() <= 3e-2


def test_attention_layer_of_a_packed_batch():
    import experiment_swa_kda_b200 as m
    torch.manual_seed(1)
    layer = m.PagedAttention(256, 4, 2, 64, window=40, max_positions=512).to("cuda:0")
    with torch.no_grad():
        layer.q_norm.mul_(1.3)
    cache = m.PagedCache.zeros(3, 200, 16, 2, 64, "cuda:0")
    steps = [[100, 7, 1], [1, 1, 1], [20, 90, 1], [1, 30, 64]]
    total = [0, 0, 0]
    for q_lens in steps:
        total = [a + b for a, b in zip(total, q_lens)]
        x = torch.randn(1, sum(q_lens), 256, device="cuda:0").bfloat16()
        cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32).to("cuda:0")
        cache.kv_lens.copy_(torch.tensor(total, dtype=torch.int32))
        y = layer(x, cache, cu, max_q_len=max(q_lens))
        # the layer's own projections in bf16, then float64 from there
        qkv = layer.qkv_proj(x).detach().reshape(-1, 8, 64).cpu()
        pos = torch.cat([torch.arange(n - a, n) for a, n in zip(q_lens, total)])
        q = A.norm_rope(qkv[:, :4], layer.cos.cpu()[pos], layer.sin.cpu()[pos], layer.q_norm.detach().cpu()).bfloat16()
        o, _, _ = A.paged_attention(q, cache.k.cpu(), cache.v.cpu(), cache.block_table.cpu(), total, q_lens, window=40)
        want = layer.o_proj(o.bfloat16().to("cuda:0").reshape(1, len(pos), -1)).double()
        assert (y.double() - want).norm() <= 1e-2 * want.norm()
