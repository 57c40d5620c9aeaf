"""Refusals of the attention operators that need no GPU."""

import pytest
import torch

import experiment_swa_kda_b200 as m


def batch():
    q, c = torch.zeros(2, 4, 64), torch.zeros(3, 16, 2, 64)
    return [q, c, c.clone(), torch.zeros(1, 3, dtype=torch.int32), torch.tensor([2], dtype=torch.int32)]


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CPU"):
        m.paged_attention(*batch())
    q, k_cache, v_cache, table, lens = batch()
    cos = torch.zeros(8, 32)
    with pytest.raises(RuntimeError, match="CPU"):
        m.qk_norm_rope_append(q, q[:, :2], q[:, :2], cos, cos, k_cache, v_cache, table, lens)
    with pytest.raises(RuntimeError, match="CPU"):
        m.qk_norm_rope(q[None], q[None], cos, cos)


def test_shapes_are_named():
    q, k_cache, v_cache, table, lens = batch()
    for at, bad, match in ((0, q[0], "q must"), (1, k_cache[:2], "share shape"), (3, table.long(), "block_table"), (4, lens.long(), "kv_lens")):
        args = batch()
        args[at] = bad
        with pytest.raises(ValueError, match=match):
            m.paged_attention(*args)
    with pytest.raises(ValueError, match="divide"):
        m.paged_attention(q[:, :3], k_cache, v_cache, table, lens)
    with pytest.raises(ValueError, match="same number"):
        m.paged_attention(q, k_cache, v_cache, table.expand(3, 3), lens.expand(3))
    cos = torch.zeros(8, 40)
    with pytest.raises(ValueError, match="rotate more"):
        m.qk_norm_rope(q[None], q[None], cos, cos)


def test_abi_checks_run_before_any_launch():
    from experiment_swa_kda_b200 import _lib
    lib = _lib.load()
    s = _lib.PagedShape(tokens=4, n_seq=2, q_heads=4, kv_heads=2, head_dim=64, io_dtype=1, n_pages=3, page_size=16, table_width=2, scale=1.0)
    assert lib.kda_paged_attention(s, *([None] * 9), 0, None) == -5
    s.q_heads = 3
    assert lib.kda_paged_attention(s, *([None] * 9), 0, None) == -1
    s.q_heads, s.scale = 4, 0.0
    assert lib.kda_paged_attention(s, *([None] * 9), 0, None) == -1
    s.scale, s.io_dtype = 1.0, 7
    assert lib.kda_paged_attention(s, *([None] * 9), 0, None) == -2
    r = _lib.RotaryShape(tokens=2, seq_len=2, q_heads=2, kv_heads=1, head_dim=64, rotary_dim=64, table_len=8, io_dtype=0, eps=1e-6)
    assert lib.kda_norm_rope_fwd(r, *([None] * 10)) == -5
    r.rotary_dim = 66
    assert lib.kda_norm_rope_fwd(r, *([None] * 10)) == -1
    assert lib.kda_norm_rope_bwd_scratch_bytes(r) == 0
    assert b"block table" in lib.kda_error_string(-8) and b"position" in lib.kda_error_string(-9)
