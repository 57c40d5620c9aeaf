"""C entries of the serving operators: what they refuse before anything is launched.  Pointers here are never followed."""

import pytest

from experiment_swa_kda_b200 import _lib

NULL, BAD_SHAPE = -5, -1
SOME = 4096      # an address


def paged(**more):
    return _lib.PagedShape(**{**dict(tokens=4, n_seq=2, q_heads=4, kv_heads=2, head_dim=64, io_dtype=0, n_pages=3, page_size=16, table_width=2, table_stride=2, scale=1.0), **more})


@pytest.mark.parametrize("n_pages", [0, 3])
def test_a_table_that_would_be_read_has_to_be_there(n_pages):
    """Also where the cache has no page at all: the kernels look the pages up before they find that out."""
    lib, s = _lib.load(), paged(n_pages=n_pages)
    assert lib.kda_paged_attention(s, SOME, SOME, SOME, None, SOME, None, SOME, None, SOME, 1 << 40, None) == NULL
    r = _lib.RotaryShape(tokens=4, seq_len=1, q_heads=4, kv_heads=2, head_dim=64, rotary_dim=64, table_len=8, io_dtype=0, eps=1e-6)
    assert lib.kda_norm_rope_append(r, s, *[SOME] * 5, None, None, None, SOME, None, *[SOME] * 3, None) == NULL
    p = _lib.PrefixShape(n_groups=1, table_width=1, table_stride=1)
    for table, prefix_table in ((None, SOME), (SOME, None)):
        assert lib.kda_shared_prefix_attention(s, p, SOME, SOME, SOME, table, SOME, None, prefix_table, SOME, None, SOME, None, SOME, 1 << 40, None) == NULL
    if n_pages:
        assert lib.kda_paged_attention(s, SOME, None, SOME, SOME, SOME, None, SOME, None, SOME, 1 << 40, None) == NULL
