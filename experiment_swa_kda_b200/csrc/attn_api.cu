// C entries of the attention over a paged cache: argument checks, and which kernel takes a call.

#include <math.h>

#include <initializer_list>

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
    if (s->table_width > 0 && (!block_table || (s->n_pages > 0 && (!k_cache || !v_cache)))) return KDA_ERR_NULL;      // a table is read whether or not there are pages
    const size_t need = kda_paged_attention_workspace_bytes(s);
    if (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 || workspace_bytes < need)) return KDA_ERR_WORKSPACE;
    const bool packed = cu_seqlens != nullptr;
    const int q_len = packed ? 0 : s->tokens / s->n_seq;
    Call c;
    c.batch = GroupView{};
    static_cast<Batch&>(c.batch) =
        Batch{block_table, kv_lens, cu_seqlens, status_mirror(), s->table_stride, s->n_seq, s->tokens, q_len, s->n_pages, s->page_size, s->table_width, s->padded};
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

// ------------------------------------------------------------------------------------------------ behind a shared prefix

namespace {

int check_prefix(const KdaPagedShape* s, const KdaPrefixShape* p, bool packed, bool grouped) {
    if (int rc = check(s, packed)) return rc;
    if (!p) return KDA_ERR_NULL;
    if (p->n_groups <= 0 || p->n_groups > s->n_seq || p->table_width < 0 || s->window != 0) return KDA_ERR_BAD_SHAPE;
    if (!grouped && s->n_seq % p->n_groups != 0) return KDA_ERR_BAD_SHAPE;
    if ((long long)p->table_width * s->page_size >= 1ll << 31) return KDA_ERR_BAD_SHAPE;
    return KDA_OK;
}

GroupView groups_of(const KdaPagedShape& s, const KdaPrefixShape& p) {
    GroupView v = {};
    v.n_seq = s.n_seq;
    v.tokens = s.tokens;
    v.p.n = p.n_groups;
    return v;
}
// Parts of a prefix at most, where its row tiles leave SMs idle.
int prefix_split_count(const KdaPagedShape& s, const KdaPrefixShape& p, int rows, int keys, int resident) {
    int per;
    const long long blocks = group_slots(groups_of(s, p), s.q_heads / s.kv_heads, rows, per) * s.kv_heads;
    const long long tiles = ((long long)p.table_width * s.page_size + keys - 1) / keys;
    long long n = resident / (blocks > 0 ? blocks : 1);
    if (n > tiles) n = tiles;
    return (int)(n < 1 ? 1 : n > kPartTries ? kPartTries : n);
}
int tc_prefix_splits(const KdaPagedShape& s, const KdaPrefixShape& p) {
    int per;
    const int rows = prefix_rows(s.tokens, p.n_groups, s.q_heads / s.kv_heads);
    const long long slots = group_slots(groups_of(s, p), s.q_heads / s.kv_heads, rows, per);
    // a long prefix beside short ones may have more than its share of the blocks
    return slots * s.kv_heads <= kMaxListed ? prefix_split_count(s, p, rows, 128, p.n_groups > 1 ? 3 * kSms : kSms) : 1;
}
int general_prefix_splits(const KdaPagedShape& s, const KdaPrefixShape& p) { return prefix_split_count(s, p, 64, 64, 2 * 148); }

// What the tables' widths say of lengths: prefixes fill theirs, and sequences go on for up to what theirs have besides.
long long behind_of(const KdaPagedShape& s, const KdaPrefixShape& p) {
    return (long long)(s.table_width > p.table_width ? s.table_width - p.table_width : 0) * s.page_size;
}

// The best that the passes over prefixes and over own keys of few rows can do side by side, and the blocks of the first with which they do.
float side_by_side_us(const KdaPagedShape& s, const KdaPrefixShape& p, int splits, int max_q, long long own_tiles, int& blocks) {
    const int group = s.q_heads / s.kv_heads, rows = prefix_rows(s.tokens, p.n_groups, group);
    const long long tiles = ((long long)p.table_width * s.page_size + 127) / 128;
    const long long row_tiles = (((long long)s.tokens * group + p.n_groups - 1) / p.n_groups + rows - 1) / rows * p.n_groups * s.kv_heads;
    const float own_us = own_tiles_us(own_tiles, s.head_dim, max_q * group);
    blocks = 0;
    if (splits < 2 || tiles == 0) return (float)(10.0 + (double)row_tiles * tiles * 2 / kSms + own_us / kSms);
    float least = INFINITY;
    for (int tries = 1; tries <= splits && (tries == 1 || row_tiles * tries <= kSms); ++tries) {
        const int part = (int)((tiles + tries - 1) / tries), n = (int)(row_tiles * ((tiles + part - 1) / part));
        const float us = passes_us(part, n, rows, own_us);
        if (us < least) least = us, blocks = n;
    }
    return least;
}

// Token steps whose sequences have few keys all in all go through the prefix and their own keys one after the other: reading a short prefix again for
// each costs less than two passes and their join.  In tiles of 64 keys, us: 288 13 and 21, 768 15 and 19, 1,188 19 and 20; beyond, one pass goes on to grow with them
// and two hardly (1,536 21, 3,200 21).  The tiles are the table's, as nothing else is known here: a batch of 768 in a table of 4,096 tokens takes two, 21 us.
bool few_keys(const KdaPagedShape& s) {
    return ((long long)s.table_width * s.page_size + 63) / 64 * s.n_seq * s.kv_heads <= 1200;
}

// So do sequences of more rows where that is quicker, by estimates in microseconds.  One pass: blocks of a row tile of a sequence, 1.3 a key tile of 128
// (2 with more than 128 rows) and 8 besides.  Two: the prefix in whole row tiles, own keys in blocks as these or by the token steps' kernel, and the join.
// 16 sequences of 40 rows behind 2,000 tokens 31 and 44 us with 3 heads, 78 and 70 with 16; 30 of 400 behind 1,000 61 and 132; 64 of 20 behind 4,097 150 and 68.
bool takes_both(const KdaPagedShape& s, const KdaPrefixShape& p, long long max_q) {      // max_q: a bound on a sequence's new tokens, 0: unknown
    const int group = s.q_heads / s.kv_heads;
    const double rows = (double)s.tokens * group / s.n_seq;      // of a sequence and kv head
    const bool few = max_q > 0 && max_q * group <= 24;
    if (max_q > 0 && max_q * group <= 16) return false;
    const double each = rows <= 128 ? 1.3 : 2.0, tiles = (double)s.table_width * s.page_size / 128 + 1, own = behind_of(s, p) * 0.6 / 128 + 1;
    const double units = (double)s.n_seq * s.kv_heads * ceil(rows / 256);
    const double one = units <= kSms / 2 ? 12 + each * fmax(fmin(tiles, 8), tiles * units / kSms) : ceil(units / kSms) * (8 + each * tiles);
    const double join = 4 + (double)s.tokens * s.q_heads / 800;
    int blocks;
    if (few) return one < side_by_side_us(s, p, tc_prefix_splits(s, p), (int)max_q, (long long)(2 * own * s.n_seq * s.kv_heads), blocks) + 6 + join;
    const double row_tiles = ceil((double)s.tokens * group / 256) * s.kv_heads, prefix = (double)p.table_width * s.page_size / 128;
    const double two = 10 + fmax(row_tiles * prefix * 2 / kSms, row_tiles > kSms / 2 ? ceil(row_tiles / kSms) * prefix * 2 : 0) + ceil(units / kSms) * (10 + each * own) + join;
    return one < two;
}

// Blocks of the pass over own keys.  A block that finds no work costs 6 us where it starts late, once others have ended, so there are as many as
// find a place beside the prefixes, by what the tables' widths say: prefixes fill theirs, and sequences go on for 0.6 of what theirs have
// besides (an assumption, of lengths spread from little to all).  Where both are as wide, as rows of one pool's table are, that says nothing, and own keys may fill theirs as well: too many blocks cost
// 3 to 6 us, too few as often the pass as they are too few (256 sequences in a pool's table 90 us, 290 to 1,340 with blocks for own keys of half a page).
// How the work is cut is decided on the device, by the lengths.
int own_blocks(const KdaPagedShape& s, const KdaPrefixShape& p, bool packed, int splits) {
    const int group = s.q_heads / s.kv_heads;
    const long long behind = p.table_width < s.table_width ? behind_of(s, p) : (long long)s.table_width * s.page_size;
    const long long most = ((behind + 63) / 64 + 1) * s.n_seq * s.kv_heads / 2, own_tiles = (behind * 3 / 5 + 32) * s.n_seq * s.kv_heads / 64;
    int best = 0;
    const int max_q = packed ? s.max_q_len : s.tokens / s.n_seq;
    side_by_side_us(s, p, splits, max_q, own_tiles, best);
    const long long n = (long long)own_rows_per_sm(s.head_dim, max_q * group) * (best < kSms ? kSms - best : kSms);
    return (int)(most < 2 ? 2 : most < n ? most : n);
}

// The shares of a workspace on the tensor cores.
struct SharedSpace {
    size_t prefix, own;
};
SharedSpace shared_space(const KdaPagedShape& s, const KdaPrefixShape& p, bool packed, bool few) {
    SharedSpace w;
    int per;
    const int group = s.q_heads / s.kv_heads, max_q = packed ? s.max_q_len : s.tokens / s.n_seq;
    const int rows = prefix_rows(s.tokens, p.n_groups, group);
    w.prefix = align_up(tc_parts_bytes(group_slots(groups_of(s, p), group, rows, per), rows, s.kv_heads, tc_prefix_splits(s, p), s.head_dim), 256) +
               align_up((size_t)s.tokens * sizeof(int4), 256);
    w.own = few ? own_rows_workspace(s, max_q) : tc_parts_bytes(tile_slots(s.tokens, s.n_seq, max_q, group, 256, packed, per), 256, s.kv_heads, tc_splits(s, packed), s.head_dim);
    w.own = align_up(w.own, 256);
    return w;
}

// The ways a call can go, and the workspace of each.  Nothing is asked for but what the way taken needs: prompts in one pass need next to nothing, where the sums
// of two passes over 65,536 tokens of 16 heads are a gigabyte.
enum class Way { general, one_pass, one_list, two_passes };
Way way_of(const Call& c, const KdaPagedShape& s, const KdaPrefixShape& p) {
    if (!tc_takes(c)) return Way::general;
    if (takes_both(s, p, c.max_q_len)) return Way::one_pass;
    return few_keys(s) && decode_takes(c) ? Way::one_list : Way::two_passes;
}
size_t workspace_of(const Call& c, const KdaPagedShape& s, const KdaPrefixShape& p) {
    const bool packed = c.batch.cu != nullptr;
    int per_seq;
    switch (way_of(c, s, p)) {
        case Way::general:
            return general_shared_workspace((size_t)s.tokens * s.q_heads, general_prefix_splits(s, p) + general_splits(s, packed), s.head_dim);
        case Way::one_pass:
            return tc_workspace(tile_slots(s.tokens, s.n_seq, c.max_q_len, c.heads.group, 256, packed, per_seq), s.kv_heads, tc_splits(s, packed), s.head_dim);
        case Way::one_list:
            return decode_workspace(s.n_seq, s.kv_heads, s.table_width, s.page_size, 0, c.max_q_len, s.head_dim);
        case Way::two_passes: {
            const SharedSpace w = shared_space(s, p, packed, own_rows_take(c));
            return w.prefix + w.own;
        }
    }
    return 0;
}

Call call_of(const KdaPagedShape* s, const KdaPrefixShape* p, const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table, const int32_t* kv_lens,
             const int32_t* cu_seqlens, const int32_t* prefix_table, const int32_t* prefix_lens, const int32_t* cu_groups, void* o, float* lse, void* workspace) {
    const int q_len = cu_seqlens ? 0 : s->tokens / s->n_seq;
    Call c;
    c.batch = GroupView{};
    static_cast<Batch&>(c.batch) =
        Batch{block_table, kv_lens, cu_seqlens, nullptr, s->table_stride, s->n_seq, s->tokens, q_len, s->n_pages, s->page_size, s->table_width, s->padded};
    c.batch.p = Prefix{prefix_table, prefix_lens, cu_groups, p->table_stride, p->n_groups, p->table_width, s->n_seq / p->n_groups};
    c.heads = Heads{s->q_heads, s->kv_heads, s->q_heads / s->kv_heads, s->head_dim};
    c.strides = Strides{s->q_token_stride, s->q_head_stride, s->k_page_stride, s->k_row_stride, s->k_head_stride, s->v_page_stride, s->v_row_stride, s->v_head_stride};
    c.q = q; c.k = k_cache; c.v = v_cache; c.o = o; c.lse = lse;
    c.scale = s->scale;
    c.window = 0;
    c.bf16 = s->io_dtype == KDA_DTYPE_BF16;
    c.max_q_len = cu_seqlens ? s->max_q_len : q_len;
    c.workspace = workspace;
    return c;
}

}  // namespace

extern "C" size_t kda_shared_prefix_attention_call_bytes(const KdaPagedShape* s, const KdaPrefixShape* p, const void* q, const void* k_cache, const void* v_cache,
                                                         const int32_t* cu_seqlens, const void* o) {
    if (check_prefix(s, p, cu_seqlens != nullptr, true) || s->tokens == 0) return 0;
    return align_up(workspace_of(call_of(s, p, q, k_cache, v_cache, nullptr, nullptr, cu_seqlens, nullptr, nullptr, nullptr, const_cast<void*>(o), nullptr, nullptr), *s, *p), 256);
}

extern "C" size_t kda_shared_prefix_attention_workspace_bytes(const KdaPagedShape* s, const KdaPrefixShape* p) {
    if (check_prefix(s, p, true, true)) return 0;
    size_t most = 256;
    const int32_t any = 0;
    // whether the batch has cu_seqlens is not known here, nor where the arrays lie: on 16 bytes, or not
    for (const int32_t* cu : {&any, static_cast<const int32_t*>(nullptr)})
        for (uintptr_t at : {uintptr_t(256), uintptr_t(1)}) {
            const void* x = reinterpret_cast<const void*>(at);
            if (cu == nullptr && s->tokens % s->n_seq != 0) continue;
            const size_t need = kda_shared_prefix_attention_call_bytes(s, p, x, x, x, cu, x);
            if (need > most) most = need;
        }
    return most;
}

extern "C" int kda_shared_prefix_attention(const KdaPagedShape* s, const KdaPrefixShape* p, const void* q, const void* k_cache, const void* v_cache,
                                           const int32_t* block_table, const int32_t* kv_lens, const int32_t* cu_seqlens, const int32_t* prefix_table,
                                           const int32_t* prefix_lens, const int32_t* cu_groups, void* o, float* lse, void* workspace, size_t workspace_bytes,
                                           void* stream) {
    if (int rc = check_prefix(s, p, cu_seqlens != nullptr, cu_groups != nullptr)) return rc;
    if (s->tokens == 0) return KDA_OK;
    if (!q || !kv_lens || !o || !prefix_lens) return KDA_ERR_NULL;
    if ((s->table_width > 0 && !block_table) || (p->table_width > 0 && !prefix_table) || (s->n_pages > 0 && (!k_cache || !v_cache))) return KDA_ERR_NULL;
    Call c = call_of(s, p, q, k_cache, v_cache, block_table, kv_lens, cu_seqlens, prefix_table, prefix_lens, cu_groups, o, lse, workspace);
    const size_t need = workspace_of(c, *s, *p);
    if (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 || workspace_bytes < need)) return KDA_ERR_WORKSPACE;
    c.batch.mirror = status_mirror();
    const cudaStream_t st = (cudaStream_t)stream;
    const bool packed = cu_seqlens != nullptr;
    switch (way_of(c, *s, *p)) {
        case Way::general: return general_shared(c, general_prefix_splits(*s, *p), general_splits(*s, packed), st);
        case Way::one_pass: return tc_both(c, tc_splits(*s, packed), st);
        case Way::one_list: return decode_both(c, st);
        case Way::two_passes: break;
    }
    const bool few = own_rows_take(c);
    const int prefix_splits = tc_prefix_splits(*s, *p), own_splits = tc_splits(*s, packed);
    Call own = c;
    own.workspace = static_cast<char*>(workspace) + shared_space(*s, *p, packed, few).prefix;
    OwnRows rows;
    if (int rc = tc_prefix(c, prefix_splits, few, st)) return rc;
    if (int rc = few ? own_rows(own, prefix_splits, own_blocks(*s, *p, packed, prefix_splits), rows, st) : tc_own(own, own_splits, st)) return rc;
    return tc_shared_join(c, prefix_splits, own, own_splits, few ? &rows : nullptr, st);
}
