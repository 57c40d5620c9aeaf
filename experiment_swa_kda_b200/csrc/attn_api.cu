// C entries of the attention over a paged cache: argument checks, and which kernel takes a call.

#include "attn.cuh"

using namespace kda;
using namespace kda::attn;

namespace {

int check(const KdaPagedShape* s, bool packed) {
    if (!s) return KDA_ERR_NULL;
    if (s->tokens < 0 || s->n_seq <= 0 || s->q_heads <= 0 || s->kv_heads <= 0 || s->head_dim <= 0 || s->n_pages < 0 || s->page_size <= 0 ||
        s->table_width < 0 || s->window < 0 || s->max_q_len < 0)
        return KDA_ERR_BAD_SHAPE;
    if (s->head_dim > KDA_MAX_DIM || s->q_heads % s->kv_heads != 0 || s->kv_heads > 65535) return KDA_ERR_BAD_SHAPE;
    if (!packed && s->tokens % s->n_seq != 0) return KDA_ERR_BAD_SHAPE;
    if ((long long)s->tokens * s->q_heads >= 1ll << 31 || (long long)s->table_width * s->page_size >= 1ll << 31) return KDA_ERR_BAD_SHAPE;
    if (!(s->scale > 0.f)) return KDA_ERR_BAD_SHAPE;
    if (s->io_dtype != KDA_DTYPE_F32 && s->io_dtype != KDA_DTYPE_BF16) return KDA_ERR_UNSUPPORTED;
    return KDA_OK;
}

// Parts a row's keys may be cut into where its blocks alone leave SMs idle.  What a row sees is known on the device alone, so the
// bound is the table's.
int split_count(const KdaPagedShape& s, bool packed, int rows, int keys, int resident, int least) {      // a part has `least` key tiles
    int per_seq;
    const int group = s.q_heads / s.kv_heads;
    const int max_q = packed ? s.max_q_len : s.tokens / s.n_seq;
    const long long blocks = tile_slots(s.tokens, s.n_seq, max_q, group, rows, packed, per_seq) * s.kv_heads;
    long long reach = (long long)s.table_width * s.page_size;
    if (s.window > 0 && max_q > 0 && reach > (long long)s.window + max_q) reach = (long long)s.window + max_q;
    const long long tiles = (reach + keys - 1) / keys;
    long long n = resident / (blocks > 0 ? blocks : 1);
    if (n > tiles / least) n = tiles / least;
    return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
int general_splits(const KdaPagedShape& s, bool packed) { return split_count(s, packed, 64, 64, 2 * 148, 1); }
// The tensor-core kernel finds on the device how long a part should be, with a thread for each row tile; blocks without a part end at
// once, so there may be more of them than SMs.  Parts pay where the row tiles leave half of the SMs idle: 500 new tokens over 16,384
// 118 us without them, 76 with; 12 sequences of 128 row tiles 68 without, 76 with.
int tc_splits(const KdaPagedShape& s, bool packed) {
    int per_seq;
    const int max_q = packed ? s.max_q_len : s.tokens / s.n_seq;
    const long long slots = tile_slots(s.tokens, s.n_seq, max_q, s.q_heads / s.kv_heads, 256, packed, per_seq);
    return slots <= 384 && slots * s.kv_heads <= 148 / 2 ? split_count(s, packed, 256, 128, 3 * 148, 4) : 1;
}

}  // namespace

extern "C" size_t kda_paged_attention_workspace_bytes(const KdaPagedShape* s) {
    if (check(s, true)) return 0;
    const size_t rows = (size_t)s->tokens * s->q_heads;
    size_t most = 0;
    for (int packed = 0; packed < 2; ++packed) {      // whether the batch has cu_seqlens is not known here
        if (!packed && s->tokens % s->n_seq != 0) continue;
        const size_t n = (size_t)general_splits(*s, packed);
        size_t need = n > 1 ? align_up(rows * n * sizeof(float2), 256) + rows * n * s->head_dim * sizeof(float) : 0;
        if (need > most) most = need;
        int per_seq;
        const long long slots = tile_slots(s->tokens, s->n_seq, packed ? s->max_q_len : s->tokens / s->n_seq, s->q_heads / s->kv_heads, 256, packed, per_seq);
        need = tc_workspace(slots, s->kv_heads, tc_splits(*s, packed), s->head_dim);
        if (need > most) most = need;
    }
    const int each = s->tokens / s->n_seq, max_q = s->max_q_len > each ? s->max_q_len : each;
    const size_t few = decode_workspace(s->n_seq, s->kv_heads, s->table_width, s->page_size, s->window, max_q, s->head_dim);
    return align_up(most > few ? most : few, 256);
}

extern "C" int kda_paged_attention(const KdaPagedShape* s, const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                                   const int32_t* kv_lens, const int32_t* cu_seqlens, void* o, float* lse, void* workspace, size_t workspace_bytes,
                                   void* stream) {
    if (int rc = check(s, cu_seqlens != nullptr)) return rc;
    if (s->tokens == 0) return KDA_OK;
    if (!q || !kv_lens || !o) return KDA_ERR_NULL;
    const bool cached = s->n_pages > 0 && s->table_width > 0;
    if (cached && (!k_cache || !v_cache || !block_table)) return KDA_ERR_NULL;
    const size_t need = kda_paged_attention_workspace_bytes(s);
    if (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 || workspace_bytes < need)) return KDA_ERR_WORKSPACE;
    const bool packed = cu_seqlens != nullptr;
    const int q_len = packed ? 0 : s->tokens / s->n_seq;
    Call c;
    c.batch = Batch{block_table, kv_lens, cu_seqlens, status_mirror(), s->table_stride, s->n_seq, s->tokens, q_len, s->n_pages, s->page_size, s->table_width};
    c.heads = Heads{s->q_heads, s->kv_heads, s->q_heads / s->kv_heads, s->head_dim};
    c.strides = Strides{s->q_token_stride, s->q_head_stride, s->k_page_stride, s->k_row_stride, s->k_head_stride, s->v_page_stride, s->v_row_stride, s->v_head_stride};
    c.q = q; c.k = k_cache; c.v = v_cache; c.o = o; c.lse = lse;
    c.scale = s->scale;
    c.window = s->window;
    c.bf16 = s->io_dtype == KDA_DTYPE_BF16;
    c.max_q_len = packed ? s->max_q_len : q_len;
    c.workspace = workspace;
    if (decode_takes(c)) return decode(c, (cudaStream_t)stream);
    return tc_takes(c) ? tc(c, tc_splits(*s, packed), (cudaStream_t)stream) : general(c, general_splits(*s, packed), (cudaStream_t)stream);
}
