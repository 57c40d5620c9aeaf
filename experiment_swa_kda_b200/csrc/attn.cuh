// What the attention kernels share: the batch as the device sees it, and how a block finds its sequence in it.
#pragma once

#include "common.cuh"

namespace kda {
namespace attn {

// A load of what the caller's arrays hold: not one of constant memory, which the compiler may move ahead of a wait for the launch before.  The kernels behind a
// shared prefix start early: the first of a call waits for everything before it and lets the second start only then, which reads the batch without a wait.
template <class T>
__device__ __forceinline__ T ld_input(const T* p) {
    return *p;
}

// A batch of new tokens over a paged cache.  Every array is the caller's and read on the device, so nothing that is read
// there is trusted as an index before it has been clamped.
struct Batch {
    const int* table;
    const int* kv_lens;
    const int* cu;          // null: q_len new tokens each
    int* mirror;            // page-locked host word for errors found here, or null
    long long table_stride;
    int n_seq, tokens, q_len, n_pages, page_size, table_width;
    int padded;             // tokens behind the last sequence are expected

    // Said by every thread that finds it, as long as the call runs: these calls have no status word of their own in which a first teller could be
    // known (a captured call has nothing that tells one replay from the next).  The host therefore clears the word behind the stream's work.
    __device__ __forceinline__ void tell(int code) const {
        if (mirror != nullptr) *reinterpret_cast<volatile int*>(mirror) = code;
    }
    __device__ __forceinline__ int many() const { return n_seq; }
    // first new token of sequence n of a packed batch
    __device__ __forceinline__ int edge(int n) const { return min(max(ld_input(cu + n), 0), tokens); }
    // new tokens [first, first + count) of sequence n
    __device__ __forceinline__ void span(int n, int& first, int& count) const {
        if (cu == nullptr) {
            first = n * q_len;
            count = q_len;
            return;
        }
        const int a = ld_input(cu + n), b = ld_input(cu + n + 1);
        first = min(max(a, 0), tokens);
        count = min(max(b, first), tokens) - first;
    }
    // whether the table of new tokens is consistent at sequence n
    __device__ __forceinline__ bool span_ok(int n) const {
        if (cu == nullptr) return true;
        const int a = ld_input(cu + n), b = ld_input(cu + n + 1);
        return a >= 0 && a <= b && b <= tokens && (n > 0 || a == 0) && (n + 1 < n_seq || b == tokens || padded);
    }
    // tokens that are some sequence's; those from here on are padding
    __device__ __forceinline__ int end() const { return cu == nullptr ? tokens : edge(n_seq); }
    // tokens of sequence n that the table has room for
    __device__ __forceinline__ int kv_len(int n) const {
        const long long room = (long long)table_width * page_size;
        const int len = max(ld_input(kv_lens + n), 0);
        return (long long)len > room ? (int)room : len;
    }
    __device__ __forceinline__ bool kv_len_ok(int n) const {
        const int len = ld_input(kv_lens + n);
        return len >= 0 && (long long)len <= (long long)table_width * page_size;
    }
    // the page of column `col`, or -1 where the table names none
    __device__ __forceinline__ int page(int n, int col) const {
        const int p = ld_input(table + n * table_stride + col);
        return (unsigned)p < (unsigned)n_pages ? p : -1;
    }
    // sequence of token t: the last one that starts at or before it
    __device__ __forceinline__ int seq_of(int t) const {
        if (cu == nullptr) return t / q_len;
        int lo = 0, hi = n_seq;      // cu[lo] <= t < cu[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (ld_input(cu + mid) <= t) lo = mid;
            else hi = mid;
        }
        return lo;
    }
    // The same by LANES converged lanes (lane l of them, `mask` in the warp): the place where t would lie in a batch of equal
    // lengths is looked at first, then LANES places at a time.
    template <int LANES>
    __device__ __forceinline__ int seq_of(int t, int l, unsigned mask) const {
        if (cu == nullptr) return t / q_len;
        const int guess = (int)((long long)t * n_seq / tokens);
        if (ld_input(cu + guess) <= t && t < ld_input(cu + guess + 1)) return guess;
        int lo = 0, hi = n_seq;
        while (hi - lo > 1) {
            const int step = (hi - lo + LANES - 1) / LANES, at = lo + step * l;
            const unsigned below = __ballot_sync(mask, at < hi && ld_input(cu + at) <= t) & mask;
            lo += step * max(__popc(below) - 1, 0);
            hi = min(hi, lo + step);
        }
        return lo;
    }
};

// Sequences that start with the same text.  Sequences [groups[g], groups[g + 1]) are group g (null: `each` a group), whose text is lens[g]
// tokens in the pages of the table's row g.  A sequence shares it if all its new tokens lie behind it; it then has own keys from there on.
// One that does not - a place in the batch without a request, a shorter text - has all its keys to itself.
struct Prefix {
    const int* table;
    const int* lens;
    const int* groups;
    long long table_stride;
    int n, width, each;
};

// A batch of which every sequence sees its own keys only: those behind its prefix.
struct OwnView : Batch {
    Prefix p;
    __device__ __forceinline__ int group_edge(int g) const { return p.groups == nullptr ? g * p.each : min(max(ld_input(p.groups + g), 0), n_seq); }
    // the group of sequence n, or -1
    __device__ __forceinline__ int group_of(int n) const {
        if (p.groups == nullptr) return n / p.each;
        int lo = 0, hi = p.n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (group_edge(mid) <= n) lo = mid;
            else hi = mid;
        }
        return n >= group_edge(lo) && n < group_edge(lo + 1) ? lo : -1;
    }
    __device__ __forceinline__ int prefix_len(int g) const {
        const long long room = (long long)p.width * page_size;
        const int len = max(ld_input(p.lens + g), 0);
        return (long long)len > room ? (int)room : len;
    }
    // the prefix of sequence n's group, whether or not the sequence shares it
    __device__ __forceinline__ int prefix_of(int n) const {
        if (p.n == 1) {      // nothing here waits for anything else
            const int a = group_edge(0), b = group_edge(1), len = prefix_len(0);
            return n >= a && n < b ? len : 0;
        }
        const int g = group_of(n);
        return g < 0 ? 0 : prefix_len(g);
    }
    __device__ __forceinline__ bool groups_ok(int g) const {
        if (p.groups != nullptr) {
            const int a = ld_input(p.groups + g), b = ld_input(p.groups + g + 1);
            if (a < 0 || a > b || b > n_seq) return false;
        }
        return true;
    }
    // the page of column `col` of group g's prefix, or -1
    __device__ __forceinline__ int prefix_page(int g, int col) const {
        const int at = ld_input(p.table + g * p.table_stride + col);
        return (unsigned)at < (unsigned)n_pages ? at : -1;
    }
    __device__ __forceinline__ bool prefix_ok(int g) const {
        const int len = ld_input(p.lens + g);
        return len >= 0 && (long long)len <= (long long)p.width * page_size;
    }
};

// A batch of which every sequence sees the prefix it shares, and then its own keys.
struct BothView : OwnView {};

// The same batch with each group as one sequence: all new tokens of the group see the whole prefix, and nothing else.
struct GroupView : BothView {
    __device__ __forceinline__ int many() const { return p.n; }
    __device__ __forceinline__ int edge(int g) const {
        const int s = group_edge(g);
        return cu == nullptr ? s * q_len : min(max(ld_input(cu + s), 0), tokens);
    }
    __device__ __forceinline__ void span(int g, int& first, int& count) const {
        first = edge(g);
        count = max(edge(g + 1) - first, 0);
    }
    __device__ __forceinline__ int page(int g, int col) const { return prefix_page(g, col); }
};

// Tiles of `rows` packed rows (token-major, the query heads of one kv head beside each other) of all sequences.  With a bound
// on the tokens of a sequence every sequence has tiles_per_seq slots; without one sequence n starts at slot
// first * group / rows + n, which leaves room for its last, partial tile and needs no sum over the sequences before it.
struct Tiles {
    int rows, group, per_seq;
    template <class B>
    __device__ __forceinline__ int start(const B& b, int i) const {
        return per_seq > 0 ? i * per_seq : (int)((long long)b.edge(i) * group / rows) + i;
    }
    template <class B>
    __device__ __forceinline__ bool find(const B& b, int slot, int& n, int& tile) const {
        const int many = b.many();
        if (per_seq > 0) {
            n = slot / per_seq;
            tile = slot - n * per_seq;
            return n < many;
        }
        int lo = 0, hi = many;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start(b, mid) <= slot) lo = mid;
            else hi = mid;
        }
        n = lo;
        tile = slot - start(b, lo);
        return tile >= 0;
    }
};

// Host: slots that cover a batch, and the per_seq that goes with them.
inline long long tile_slots(int tokens, int n_seq, int max_q_len, int group, int rows, bool packed, int& per_seq) {
    const long long each = ((long long)max_q_len * group + rows - 1) / rows;
    const long long by_seq = each * n_seq, by_tokens = (long long)tokens * group / rows + n_seq;
    if (!packed || (max_q_len > 0 && by_seq <= by_tokens)) {
        per_seq = (int)each;
        return by_seq;
    }
    per_seq = 0;
    return by_tokens;
}

// Rows of a row tile in the tensor-core pass over prefixes.
inline int prefix_rows(int tokens, int n_groups, int group) { return (long long)tokens * group <= 128ll * n_groups ? 128 : 256; }
inline long long group_slots(const GroupView& b, int group, int rows, int& per_group) {
    per_group = 0;
    if (b.p.n > 1) return (long long)b.tokens * group / rows + b.p.n;
    per_group = (int)(((long long)b.tokens * group + rows - 1) / rows);
    return per_group;
}

// The first key that a token at `pos` sees; in this order nothing leaves 32 bits, however negative a padding token's position or wide the window.
__device__ __forceinline__ int first_key(int pos, int window) { return window > 0 && pos >= window ? pos - window + 1 : 0; }

// A block's share of one tile: which rows, and which keys any of them sees.
struct Unit {
    int n, first, count;       // sequence, its first new token and how many it has
    int row0, rows;            // packed rows [row0, row0 + rows) of the sequence
    int base;                  // position of its first new token (negative: padding)
    int lo, hi;                // keys in reach of the tile
    int from;                  // no row sees a key before this one
};
__device__ __forceinline__ bool make_unit(const GroupView& b, const Tiles& t, int slot, int, Unit& u) {
    int tile;
    if (!t.find(b, slot, u.n, tile)) return false;
    b.span(u.n, u.first, u.count);
    u.row0 = tile * t.rows;
    u.rows = min(t.rows, u.count * t.group - u.row0);
    if (u.rows <= 0) return false;
    u.base = 0;
    u.lo = u.from = 0;
    u.hi = b.prefix_len(u.n);
    return true;
}
__device__ __forceinline__ int own_from(const Batch&, const Unit&) { return 0; }
__device__ __forceinline__ int own_from(const OwnView& b, const Unit& u) {
    const int p = b.prefix_of(u.n);
    return u.base >= p ? p : 0;
}
template <class B>
__device__ __forceinline__ bool make_unit(const B& b, const Tiles& t, int slot, int window, Unit& u) {
    int tile;
    if (!t.find(b, slot, u.n, tile)) return false;
    b.span(u.n, u.first, u.count);
    u.row0 = tile * t.rows;
    u.rows = min(t.rows, u.count * t.group - u.row0);
    if (u.rows <= 0) return false;
    const int len = b.kv_len(u.n);
    u.base = len - u.count;
    const int i0 = u.row0 / t.group, i1 = (u.row0 + u.rows - 1) / t.group;
    u.hi = max(u.base + i1 + 1, 0);
    u.from = own_from(b, u);
    u.lo = max(first_key(u.base + i0, window), u.from);
    return true;
}
// What a batch got wrong is reported by the blocks of the first tile of each sequence.
__device__ __forceinline__ void check_group(const OwnView& b, int g) {
    if (!b.groups_ok(g)) b.tell(KDA_ERR_CU_SEQLENS);
    if (!b.prefix_ok(g)) b.tell(KDA_ERR_BLOCK_TABLE);
}
__device__ __forceinline__ void check_batch(const GroupView& b, const Tiles&, int g, int tile) {
    if (tile == 0) check_group(b, g);
}
__device__ __forceinline__ void check_batch(const Batch& b, const Tiles& t, int n, int tile) {
    if (tile != 0) return;
    if (!b.span_ok(n)) b.tell(KDA_ERR_CU_SEQLENS);
    if (!b.kv_len_ok(n)) b.tell(KDA_ERR_BLOCK_TABLE);
    if (t.per_seq > 0 && b.cu != nullptr) {
        int first, count;
        b.span(n, first, count);
        if ((long long)count * t.group > (long long)t.per_seq * t.rows) b.tell(KDA_ERR_CU_SEQLENS);
    }
}

struct Heads {
    int q_heads, kv_heads, group, dim;
};
struct Strides {
    long long q_token, q_head, k_page, k_row, k_head, v_page, v_row, v_head;
};

// Running softmax in powers of two.  A row that has seen no key has max -inf; one that has seen keys is never below the lowest
// finite value, so that a row of -inf scores ends as 0/0, as the formula says, and a row without keys as nothing.
constexpr float kLowest = -3.402823466e38f;
constexpr float kLn2 = 0.6931471805599453f;

// Own keys of sequence n in tiles of 64.
__device__ __forceinline__ int own_tiles_of(const OwnView& b, int n) {
    int first, count;
    b.Batch::span(n, first, count);
    const int len = b.kv_len(n), p = b.prefix_of(n);
    if (count <= 0) return 0;
    return (len + 63) / 64 - (len - count >= p ? p : 0) / 64;
}

// Attention behind a prefix is two passes side by side, one over the prefixes and one over own keys, and the SMs are dealt out so that both end
// together.  What a group's prefix is in work: tiles of 128 keys, and row tiles that go through them.
struct PrefixWork {
    int tiles, row_tiles;
};
__device__ __forceinline__ PrefixWork prefix_work(const GroupView& b, int g, int heads_of_group, int tile_rows) {
    int first, count;
    b.span(g, first, count);
    const int rows = count * heads_of_group;
    return PrefixWork{rows > 0 ? max((b.prefix_len(g) + 127) / 128, 1) : 0, (rows + tile_rows - 1) / tile_rows};
}
constexpr int kSms = 148, kPartTries = 128;
// Microseconds that both passes take where the one over prefixes has `blocks` SMs and parts of `part` key tiles: 0.95 a key tile with row tiles of 128 and 2
// with 256, all own keys `own_us` of an SM (own_tiles_us), and either pass 10 besides.  A model of whole calls, fitted to them: the loop itself takes 1.25 (64
// blocks) to 1.45 (120) a key tile of 128 rows and 1.7 to 1.9 of 256, but with 1.3 here 32 sequences behind 16,384 tokens take 28.8, not 27.5, and no case less.
__host__ __device__ __forceinline__ float passes_us(int part, int blocks, int tile_rows, float own_us) {
    const float prefix_us = 10.f + (float)part * (tile_rows == 128 ? 0.95f : 2.f);
    return own_us > 0.f && blocks < kSms ? fmaxf(prefix_us, 10.f + own_us / (float)(kSms - blocks)) : prefix_us + own_us / kSms;
}
// ... by tiles of 64, with so many rows a sequence and kv head
__host__ __device__ __forceinline__ float own_tiles_us(long long tiles, int dim, int rows) {
    return (float)tiles * (rows > 16 ? 1.5f : rows > 8 ? 1.2f : 0.8f) * (dim <= 64 ? 0.75f : 1.f);
}
// Key tiles of a part, and the blocks that gives: each of the first kPartTries threads tries one number of parts for the longest prefix.  Called by all
// `warps` warps; `work` is filled, `best` has two places a warp.
struct PartChoice {
    int part, blocks;
};
__device__ __forceinline__ PartChoice choose_parts(const PrefixWork* work, int groups, int tile_rows, int kv_heads, float own_us, int splits, unsigned* best, int warps) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int longest = 0, row_tiles = 0;
    for (int g = 0; g < groups; ++g) {
        longest = max(longest, work[g].tiles);
        row_tiles += work[g].row_tiles;
    }
    const int tries = tid + 1, part = (longest + tries - 1) / tries;
    int blocks = 0;
    if (longest > 0)
        for (int g = 0; g < groups; ++g) blocks += work[g].row_tiles * ((work[g].tiles + part - 1) / part);
    blocks *= kv_heads;
    const float us = passes_us(part, blocks, tile_rows, own_us);
    const bool fits = tid < kPartTries && tries <= splits && blocks <= max(kSms, row_tiles * kv_heads);
    const unsigned cost = fits ? __float_as_uint(us) : 0x7f800000u;
    unsigned least = __reduce_min_sync(0xffffffffu, cost);
    if (lane == 0) best[warp] = least;
    __syncthreads();
    least = __reduce_min_sync(0xffffffffu, lane < warps ? best[lane] : 0x7f800000u);
    const unsigned who = __reduce_min_sync(0xffffffffu, fits && cost == least ? (unsigned)tries : 0xffffu);
    if (lane == 0) best[warps + warp] = who;
    __syncthreads();
    const int parts = (int)__reduce_min_sync(0xffffffffu, lane < warps ? best[warps + lane] : 0xffffu);
    PartChoice c{max((longest + parts - 1) / parts, 1), 0};
    for (int g = 0; g < groups; ++g) c.blocks += work[g].row_tiles * ((work[g].tiles + c.part - 1) / c.part) * kv_heads;
    return c;
}
// Whether the pass over the prefixes is cut into parts: where its row tiles leave half of the SMs idle.
constexpr int kMaxListed = kSms / 2;

// Which keys a pass goes through.
enum Keys { kAllKeys, kPrefixKeys, kOwnKeys, kTurnKeys, kBothKeys };      // kTurnKeys: a prefix by row tiles of 128 (attn_tc.cu); kBothKeys: prefix, then own
template <int KEYS>
struct ViewOf {
    using type = Batch;
};
template <>
struct ViewOf<kPrefixKeys> {
    using type = GroupView;
};
template <>
struct ViewOf<kTurnKeys> {
    using type = GroupView;
};
template <>
struct ViewOf<kBothKeys> {
    using type = BothView;
};
template <>
struct ViewOf<kOwnKeys> {
    using type = OwnView;
};

struct Combine {
    int tokens, q_heads, dim, splits;
    const float* part_o;      // [splits][tokens * q_heads][dim], not divided by the sum
    const float2* part_ml;    // [splits][tokens * q_heads] (max, sum)
    void* o;
    float* lse;
    int bf16;
    int prefix_splits;        // of them parts of a prefix
    GroupView batch;
};

struct Call {
    GroupView batch;
    Heads heads;
    Strides strides;
    const void *q, *k, *v;
    void* o;
    float* lse;
    float scale;
    int window, bf16, max_q_len;
    void* workspace;
};
template <int KEYS>
__device__ __forceinline__ const typename ViewOf<KEYS>::type& view(const Call& c) {
    return c.batch;
}
int general(const Call& c, int splits, cudaStream_t st);
bool tc_takes(const Call& c);      // bf16, head width, page size and strides that the tensor-core kernel can load
int tc(const Call& c, int splits, cudaStream_t st);
size_t tc_workspace(long long slots, int kv_heads, int splits, int dim);
bool decode_takes(const Call& c);      // ... and at most 16 rows a sequence and kv head
size_t decode_workspace(int n_seq, int kv_heads, int table_width, int page_size, int window, int max_q, int dim);
int decode(const Call& c, cudaStream_t st);
int decode_both(const Call& c, cudaStream_t st);      // prefix and own keys one after the other, a finished result
// The passes of attention behind a shared prefix; their sums stay in the workspace, undivided, for a join.
int general_shared(const Call& c, int prefix_splits, int own_splits, cudaStream_t st);
size_t general_shared_workspace(size_t rows, int parts, int dim);
int tc_prefix(const Call& c, int splits, bool own_rows, cudaStream_t st);      // own_rows: the pass below runs beside it
int tc_own(const Call& c, int splits, cudaStream_t st);
int tc_both(const Call& c, int splits, cudaStream_t st);      // prefix and own keys one after the other, a finished result
size_t tc_parts_bytes(long long slots, int rows, int kv_heads, int splits, int dim);
// Own keys of few rows a sequence and kv head, where the token steps' kernel left them: rows of sequences that one stretch had to itself are
// whole; of the others stretch k has [2][rows][D] sums, place 1 of a sequence that begins in it, place 0 of one that goes on.
struct OwnRows {
    const float* part_o;
    const float2* part_ml;
    const float* row_o;
    const float2* row_ml;
    const int2* spans;      // [n_seq][kv_heads]: the first and the last stretch, or -1
    int rows, blocks;
};
bool own_rows_take(const Call& c);
int own_rows_per_sm(int dim, int rows);      // blocks an SM
size_t own_rows_workspace(const KdaPagedShape& s, int max_q);
int own_rows(const Call& c, int prefix_splits, int most_blocks, OwnRows& own, cudaStream_t st);
// The join: own keys as own_rows left them, or (null) as tc_own did in own.workspace.
int tc_shared_join(const Call& prefix, int prefix_splits, const Call& own, int own_splits, const OwnRows* rows, cudaStream_t st);

}  // namespace attn
}  // namespace kda
