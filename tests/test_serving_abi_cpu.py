"""C entries of the serving operators: what they refuse before anything is launched.  Pointers here are never followed."""

import pytest

from experiment_swa_kda_b200 import _lib

NULL, BAD_SHAPE, WORKSPACE = -5, -1, -3
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


def strided(**more):
    h, hk, d, page = (more.get(n, x) for n, x in (("q_heads", 16), ("kv_heads", 4), ("head_dim", 128), ("page_size", 64)))
    return paged(**{**dict(q_heads=h, kv_heads=hk, head_dim=d, page_size=page, io_dtype=1, n_pages=4096, q_token_stride=h * d, q_head_stride=d,
                           k_page_stride=page * hk * d, k_row_stride=hk * d, k_head_stride=d, v_page_stride=page * hk * d, v_row_stride=hk * d, v_head_stride=d), **more})


def test_a_call_asks_for_the_workspace_of_the_way_it_takes():
    """Prompts that go through prefix and own keys in one pass have no sums to keep; what any call may need covers each of them."""
    lib = _lib.load()
    cases = [(strided(tokens=65536, n_seq=32, max_q_len=2048, table_width=80), 16), (strided(tokens=65536, n_seq=64, max_q_len=1024, kv_heads=16, table_width=80), 16)]
    for s, width in cases:
        p = _lib.PrefixShape(n_groups=1, table_width=width, table_stride=width)
        of_call = lambda *at: lib.kda_shared_prefix_attention_call_bytes(s, p, *at)
        assert of_call(SOME, SOME, SOME, SOME, SOME) <= 1 << 20
        assert of_call(SOME, SOME, SOME, None, SOME) <= 1 << 20
        assert lib.kda_shared_prefix_attention_workspace_bytes(s, p) >= of_call(SOME + 2, SOME, SOME, SOME, SOME) >= 2 * 65536 * 16 * 128 * 4      # the CUDA cores' two parts
    for s, width in cases + [(strided(tokens=n * q, n_seq=n, max_q_len=q, table_width=t, io_dtype=dtype, head_dim=d, page_size=page), w) for n, q in ((1, 1), (32, 1), (64, 5), (4, 512), (3, 0))
                             for t, w in ((3, 2), (64, 33), (1024, 1024)) for dtype, d, page in ((1, 128, 64), (1, 64, 16), (1, 200, 16), (0, 64, 16), (1, 128, 48))]:
        p = _lib.PrefixShape(n_groups=1, table_width=width, table_stride=width)
        most = lib.kda_shared_prefix_attention_workspace_bytes(s, p)
        for cu in (None, SOME):
            for at in (SOME, SOME + 2):
                need = lib.kda_shared_prefix_attention_call_bytes(s, p, SOME, at, SOME, cu, SOME)
                assert need <= most and need % 256 == 0
                if need:
                    call = lambda ws, n: lib.kda_shared_prefix_attention(s, p, SOME, at, SOME, SOME, SOME, cu, SOME, SOME, None, SOME, None, ws, n, None)
                    assert call(None, need) == call(SOME, need - 256) == call(SOME + 4, need) == WORKSPACE
