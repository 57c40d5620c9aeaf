// What the attention kernels share: the batch as the device sees it, and how a block finds its sequence in it.
#pragma once

#include "common.cuh"

namespace kda {
namespace attn {

// A batch of new tokens over a paged cache.  Every array is the caller's and read on the device, so nothing that is read
// there is trusted as an index before it has been clamped.
struct Batch {
    const int* table;
    const int* kv_lens;
    const int* cu;          // null: q_len new tokens each
    int* mirror;            // page-locked host word for errors found here, or null
    long long table_stride;
    int n_seq, tokens, q_len, n_pages, page_size, table_width;

    // Said by every thread that finds it, as long as the call runs: these calls have no status word of their own in which a first teller could be
    // known (a captured call has nothing that tells one replay from the next).  The host therefore clears the word behind the stream's work.
    __device__ __forceinline__ void tell(int code) const {
        if (mirror != nullptr) *reinterpret_cast<volatile int*>(mirror) = code;
    }
    // new tokens [first, first + count) of sequence n
    __device__ __forceinline__ void span(int n, int& first, int& count) const {
        if (cu == nullptr) {
            first = n * q_len;
            count = q_len;
            return;
        }
        const int a = __ldg(cu + n), b = __ldg(cu + n + 1);
        first = min(max(a, 0), tokens);
        count = min(max(b, first), tokens) - first;
    }
    // whether the table of new tokens is consistent at sequence n
    __device__ __forceinline__ bool span_ok(int n) const {
        if (cu == nullptr) return true;
        const int a = __ldg(cu + n), b = __ldg(cu + n + 1);
        return a >= 0 && a <= b && b <= tokens && (n > 0 || a == 0) && (n + 1 < n_seq || b == tokens);
    }
    // tokens of sequence n that the table has room for
    __device__ __forceinline__ int kv_len(int n) const {
        const long long room = (long long)table_width * page_size;
        const int len = max(__ldg(kv_lens + n), 0);
        return (long long)len > room ? (int)room : len;
    }
    __device__ __forceinline__ bool kv_len_ok(int n) const {
        const int len = __ldg(kv_lens + n);
        return len >= 0 && (long long)len <= (long long)table_width * page_size;
    }
    // the page of column `col`, or -1 where the table names none
    __device__ __forceinline__ int page(int n, int col) const {
        const int p = __ldg(table + n * table_stride + col);
        return (unsigned)p < (unsigned)n_pages ? p : -1;
    }
    // sequence of token t: the last one that starts at or before it
    __device__ __forceinline__ int seq_of(int t) const {
        if (cu == nullptr) return t / q_len;
        int lo = 0, hi = n_seq;      // cu[lo] <= t < cu[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (__ldg(cu + mid) <= t) lo = mid;
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
        if (__ldg(cu + guess) <= t && t < __ldg(cu + guess + 1)) return guess;
        int lo = 0, hi = n_seq;
        while (hi - lo > 1) {
            const int step = (hi - lo + LANES - 1) / LANES, at = lo + step * l;
            const unsigned below = __ballot_sync(mask, at < hi && __ldg(cu + at) <= t) & mask;
            lo += step * max(__popc(below) - 1, 0);
            hi = min(hi, lo + step);
        }
        return lo;
    }
};

// Tiles of `rows` packed rows (token-major, the query heads of one kv head beside each other) of all sequences.  With a bound
// on the tokens of a sequence every sequence has tiles_per_seq slots; without one sequence n starts at slot
// first * group / rows + n, which leaves room for its last, partial tile and needs no sum over the sequences before it.
struct Tiles {
    int rows, group, per_seq;
    __device__ __forceinline__ bool find(const Batch& b, int slot, int& n, int& tile) const {
        if (per_seq > 0) {
            n = slot / per_seq;
            tile = slot - n * per_seq;
            return n < b.n_seq;
        }
        auto start = [&](int i) { return (int)((long long)min(max(__ldg(b.cu + i), 0), b.tokens) * group / rows) + i; };
        int lo = 0, hi = b.n_seq;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start(mid) <= slot) lo = mid;
            else hi = mid;
        }
        n = lo;
        tile = slot - start(lo);
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

// The first key that a token at `pos` sees; in this order nothing leaves 32 bits, however negative a padding token's position or wide the window.
__device__ __forceinline__ int first_key(int pos, int window) { return window > 0 && pos >= window ? pos - window + 1 : 0; }

// A block's share of one tile: which rows, and which keys any of them sees.
struct Unit {
    int n, first, count;       // sequence, its first new token and how many it has
    int row0, rows;            // packed rows [row0, row0 + rows) of the sequence
    int base;                  // position of its first new token (negative: padding)
    int lo, hi;                // keys in reach of the tile
};
__device__ __forceinline__ bool make_unit(const Batch& b, const Tiles& t, int slot, int window, Unit& u) {
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
    u.lo = first_key(u.base + i0, window);
    return true;
}
// What a batch got wrong is reported by the blocks of the first tile of each sequence.
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

struct Combine {
    int tokens, q_heads, dim, splits;
    const float* part_o;      // [splits][tokens * q_heads][dim], not divided by the sum
    const float2* part_ml;    // [splits][tokens * q_heads] (max, sum)
    void* o;
    float* lse;
    int bf16;
};
int combine(const Combine& c, cudaStream_t st);

struct Call {
    Batch batch;
    Heads heads;
    Strides strides;
    const void *q, *k, *v;
    void* o;
    float* lse;
    float scale;
    int window, bf16, max_q_len;
    void* workspace;
};
int general(const Call& c, int splits, cudaStream_t st);
bool tc_takes(const Call& c);      // bf16, head width, page size and strides that the tensor-core kernel can load
int tc(const Call& c, int splits, cudaStream_t st);
size_t tc_workspace(long long slots, int kv_heads, int splits, int dim);
bool decode_takes(const Call& c);      // ... and at most 16 rows a sequence and kv head
size_t decode_workspace(int n_seq, int kv_heads, int table_width, int page_size, int window, int max_q, int dim);
int decode(const Call& c, cudaStream_t st);

}  // namespace attn
}  // namespace kda
