"""Attention behind a shared prefix: refusals and argument checks without a GPU."""

import pytest
import torch

import experiment_swa_kda_b200 as m


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def batch():
    q, c = torch.zeros(2, 4, 64), torch.zeros(3, 16, 2, 64)
    return [q, c, c.clone(), torch.zeros(2, 3, dtype=torch.int32), i32(20, 18), torch.zeros(1, 1, dtype=torch.int32), i32(16)]


def test_refusals_name_the_argument():
    with pytest.raises(RuntimeError, match="CPU"):
        m.shared_prefix_attention(*batch())
    for at, bad, match in ((0, torch.zeros(2, 64), "q must"), (3, torch.zeros(2, 3), "block_table"), (4, torch.zeros(2), "kv_lens")):
        args = batch()
        args[at] = bad
        with pytest.raises(ValueError, match=match):
            m.shared_prefix_attention(*args)


def test_a_sliding_window_layer_takes_no_prefix():
    layer = m.PagedAttention(32, 2, 1, 16, window=8, max_positions=32)
    cache = m.PagedCache.zeros(2, 16, 4, 1, 16, "cpu")
    cache.prefix_table, cache.prefix_lens = torch.zeros(1, 1, dtype=torch.int32), i32(4)
    with pytest.raises(ValueError, match="sliding-window"):
        layer(torch.zeros(2, 1, 32), cache)


def test_abi_checks_run_before_any_launch():
    from experiment_swa_kda_b200 import _lib
    lib = _lib.load()
    s = _lib.PagedShape(tokens=4, n_seq=2, q_heads=4, kv_heads=2, head_dim=64, io_dtype=1, n_pages=3, page_size=16, table_width=2, scale=1.0)
    p = _lib.PrefixShape(n_groups=1, table_width=1, table_stride=1)
    call = lambda: lib.kda_shared_prefix_attention(s, p, *([None] * 12), 0, None)
    assert call() == -5 and lib.kda_shared_prefix_attention_workspace_bytes(s, p) > 0
    p.n_groups = 3
    assert call() == -1
    p.n_groups, s.window = 1, 5
    assert call() == -1
    s.window, p.table_width = 0, 1 << 28
    assert call() == -1 and lib.kda_shared_prefix_attention_workspace_bytes(s, p) == 0
