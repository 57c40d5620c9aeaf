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


def test_shapes_of_a_plan_that_lead_out_of_its_table():
    """Rows that overlap would be written by two blocks at once; columns are counted up to the next multiple of 128, in 32 bits."""
    lib = _lib.load()

    def call(**more):
        s = _lib.PlanShape(**{**dict(rows=2, width=4, page_size=4, n_pages=6, max_tokens=0, table_stride=4), **more})
        return lib.kda_plan_pages(s, SOME, None, SOME, SOME, None, SOME, None, None, None, 0, None), lib.kda_plan_pages_workspace_bytes(s)

    assert call()[0] == NULL and call(rows=1, table_stride=0)[0] == NULL      # as far as the missing lengths
    for bad in (dict(table_stride=3), dict(table_stride=0), dict(table_stride=-4), dict(rows=1, width=2 ** 31 - 1, page_size=1), dict(rows=1, width=2 ** 31 - 127, page_size=1)):
        assert call(**bad) == (BAD_SHAPE, 0)
