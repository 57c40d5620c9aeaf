// Pages of a paged cache dealt out and the slots of new tokens mapped, from the lengths of a batch's requests.
//
// Row n is to hold the columns [floor(start_n / page), ceil(len_n / page)) of its table.  What it holds besides goes back; the
// entries it lacks take the free pages in ascending order, rows first, columns next, so the result depends on which pages are free
// and on nothing else (a call repeated on its own result changes nothing).  A row is served if the entries lacking up to and with it
// are at most the free pages, and the new tokens up to and with it at most max_tokens; one that is not goes without its new tokens.
//
// All of it is a handful of sums over rows and over pages, each of which the next step waits for: bound by latency, not by bytes
// (256 rows of 256 columns and 32,768 pages are 300 KB).  So it is one launch, a cluster of blocks that meet at its barriers:
//   1  entries outside of their row's columns go back; missing ones are counted, 128 columns a warp
//   2  free pages of each block's share are counted; every block sums up all rows for itself
//   3  who is served; the first free pages are listed in order
//   4  missing entries take theirs; rows that have to wait give back what their new tokens would have needed
//   5  position and slot of each new token
// A batch that one block can read at once takes a single block, whose barriers cost less.

#include "common.cuh"

namespace kda {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32, kBlocks = 8, kColumns = 128;
constexpr int kMaxRows = 16384;      // two numbers a row in shared memory

struct PlanArgs {
    int* table;
    int* kv_lens;
    unsigned char* free_;
    const int* new_lens;
    const int* starts;      // or null
    int *cu, *positions;
    long long* slots;
    int* missing;           // [rows][items of a row]
    int* dealt;             // [n_pages]: the free pages in order
    int* mirror;
    long long table_stride;
    int rows, width, page, n_pages, max_tokens, items;

    __device__ __forceinline__ void tell(int code) const {
        if (mirror != nullptr) *reinterpret_cast<volatile int*>(mirror) = code;
    }
};

// What a row asks for, made sound.
struct Ask {
    int len, add, start;
    bool bad_len, bad_new;
    __device__ __forceinline__ int first(int page) const { return start / page; }
    __device__ __forceinline__ int end(int page) const { return (int)(((long long)len + page - 1) / page); }
    __device__ __forceinline__ int end_without(int page) const { return (int)(((long long)len - add + page - 1) / page); }
};
__device__ __forceinline__ Ask ask_of(const PlanArgs& a, int n) {
    const int room = a.width * a.page;      // the host sees to it that this fits
    Ask r;
    r.len = a.kv_lens[n];
    r.add = a.new_lens[n];
    r.bad_len = r.len < 0 || r.len > room;
    r.len = max(r.len, 0);
    r.bad_new = !r.bad_len && (r.add < 0 || r.add > r.len);
    r.add = min(max(r.add, 0), r.len);
    if (r.len > room) {      // no room in the table: as if it had asked for nothing
        r.len = min(r.len - r.add, room);
        r.add = 0;
    }
    r.start = a.starts != nullptr ? min(max(a.starts[n], 0), r.len) : 0;
    return r;
}

// Exclusive sums over the block's threads, and the totals.
struct Pair {
    long long need, add;
};
__device__ __forceinline__ Pair block_scan(Pair mine, Pair* sums, Pair& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Pair upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto.need, o), y = __shfl_up_sync(0xffffffffu, upto.add, o);
        if (lane >= o) upto.need += x, upto.add += y;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    const Pair of = sums[lane];      // kWarps == 32
    Pair before = of;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, before.need, o), y = __shfl_up_sync(0xffffffffu, before.add, o);
        if (lane >= o) before.need += x, before.add += y;
    }
    total = Pair{__shfl_sync(0xffffffffu, before.need, 31), __shfl_sync(0xffffffffu, before.add, 31)};
    const Pair base = Pair{__shfl_sync(0xffffffffu, before.need - of.need, warp), __shfl_sync(0xffffffffu, before.add - of.add, warp)};
    __syncthreads();
    return Pair{base.need + upto.need - mine.need, base.add + upto.add - mine.add};
}
static_assert(kWarps == 32, "a warp sums up the warps");

// Pages 16 k .. 16 k + 15 of `pages` flags: which are free.  Flags may begin at any address; `wide`: they lie on 16 bytes.
__device__ __forceinline__ unsigned free_bits(const unsigned char* flags, int at, int end, bool wide) {
    unsigned bits = 0;
    if (wide && at + 16 <= end) {
        const uint4 x = *reinterpret_cast<const uint4*>(flags + at);
        const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) bits |= ((w[i] >> (8 * j) & 0xffu) != 0 ? 1u : 0u) << (4 * i + j);
    } else {
        for (int i = 0; i < 16 && at + i < end; ++i) bits |= (flags[at + i] != 0 ? 1u : 0u) << i;
    }
    return bits;
}

__global__ void __launch_bounds__(kThreads, 1) plan_pages_kernel(const __grid_constant__ PlanArgs a) {
    extern __shared__ int rows_sm[];
    int *base_of = rows_sm, *cu = rows_sm + a.rows;      // entries lacking before a row (-1: it is not served); [rows + 1]
    __shared__ Pair sums[kWarps];
    __shared__ int counts[kBlocks];                      // free pages of each block's share
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int blocks = gridDim.x, rank = blockIdx.x;     // the grid is one cluster
    auto meet = [&]() {
        if (blocks > 1) cluster_sync();
        else __syncthreads();
    };

    // ------------------------------------------------------------------ 1: what rows hold, and lack
    const int all = a.rows * a.items;
    for (int i = rank * kWarps + warp; i < all; i += blocks * kWarps) {
        const int n = i / a.items, c0 = (i - n * a.items) * kColumns + lane;
        const Ask r = ask_of(a, n);
        if (lane == 0 && i == n * a.items) {
            if (r.bad_len) a.tell(KDA_ERR_BLOCK_TABLE);
            if (r.bad_new) a.tell(KDA_ERR_CU_SEQLENS);
        }
        const int first = r.first(a.page), end = r.end(a.page);
        int* row = a.table + n * a.table_stride;
        int entry[kColumns / 32], lacks = 0;
#pragma unroll
        for (int k = 0; k < kColumns / 32; ++k) entry[k] = c0 + 32 * k < a.width ? row[c0 + 32 * k] : -1;
#pragma unroll
        for (int k = 0; k < kColumns / 32; ++k) {
            const int c = c0 + 32 * k;
            const bool names = (unsigned)entry[k] < (unsigned)a.n_pages, held = c >= first && c < end;
            if (entry[k] >= a.n_pages) a.tell(KDA_ERR_BLOCK_TABLE);
            if (held && !names) ++lacks;
            if (!held && c < a.width && entry[k] != -1) {
                if (names) a.free_[entry[k]] = 1;
                row[c] = -1;
            }
        }
        lacks = __reduce_add_sync(0xffffffffu, lacks);
        if (lane == 0) a.missing[i] = lacks;
    }
    meet();

    // ------------------------------------------------------------------ 2: free pages of this block's share; sums over all rows
    const int share = ((a.n_pages + blocks - 1) / blocks + 15) / 16 * 16, p0 = min(rank * share, a.n_pages), p1 = min(p0 + share, a.n_pages);
    const int each_page = ((share + kThreads - 1) / kThreads + 15) / 16 * 16, my_p0 = min(p0 + tid * each_page, p1), my_p1 = min(my_p0 + each_page, p1);
    const bool wide = reinterpret_cast<uintptr_t>(a.free_) % 16 == 0;
    int my_free = 0;
    for (int p = my_p0; p < my_p1; p += 16) my_free += __popc(free_bits(a.free_, p, my_p1, wide));
    const int each = (a.rows + kThreads - 1) / kThreads, n0 = min(tid * each, a.rows), n1 = min(n0 + each, a.rows);
    Pair mine{0, 0}, total;
    for (int n = n0; n < n1; ++n) {
        int need = 0;
        for (int i = 0; i < a.items; ++i) need += a.missing[n * a.items + i];
        base_of[n] = need;
        mine.need += need;
        mine.add += ask_of(a, n).add;
    }
    Pair before = block_scan(mine, sums, total);
    Pair shares;
    const int free_before = (int)block_scan(Pair{my_free, 0}, sums, shares).need;
    if (blocks > 1) {
        if (tid < blocks) {
            uint32_t at;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(counts + rank)), "r"(tid));
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"((int)shares.need) : "memory");
        }
    } else if (tid == 0) {
        counts[0] = (int)shares.need;
    }
    meet();

    // ------------------------------------------------------------------ 3: who is served; the free pages they take, in order
    int free_all = 0, free_base = 0;
    for (int b = 0; b < blocks; ++b) {
        if (b < rank) free_base += counts[b];
        free_all += counts[b];
    }
    mine = Pair{0, 0};
    for (int n = n0; n < n1; ++n) {
        const int need = base_of[n], add = ask_of(a, n).add;
        const long long upto = before.need + need, tokens = before.add + add;
        const bool served = (upto <= free_all && tokens <= a.max_tokens) || (need == 0 && add == 0);
        base_of[n] = served ? (int)before.need : -1;
        cu[n] = served ? add : 0;
        if (served) mine.need += need, mine.add += add;
        before = Pair{upto, tokens};
    }
    Pair given = block_scan(mine, sums, total);
    const int dealt = (int)total.need;
    int at = (int)given.add;
    for (int n = n0; n < n1; ++n) {
        const int add = cu[n];
        cu[n] = at;
        if (n % blocks == rank) a.cu[n] = at;
        at += add;
    }
    if (tid == 0) {
        cu[a.rows] = (int)total.add;
        if (rank == 0) a.cu[a.rows] = (int)total.add;
    }
    if (dealt > 0) {
        int k = free_base + free_before;
        for (int p = my_p0; p < my_p1 && k < dealt; p += 16) {
            unsigned bits = free_bits(a.free_, p, my_p1, wide);
            while (bits != 0 && k < dealt) {
                const int page = p + __ffs(bits) - 1;
                bits &= bits - 1;
                a.dealt[k++] = page;
                a.free_[page] = 0;
            }
        }
    }
    meet();

    // ------------------------------------------------------------------ 4: entries that were missing
    for (int i = rank * kWarps + warp; i < all; i += blocks * kWarps) {
        const int n = i / a.items, item = i - n * a.items, c0 = item * kColumns + lane, base = base_of[n];
        if (base >= 0 && a.missing[i] == 0) continue;
        const Ask r = ask_of(a, n);
        int* row = a.table + n * a.table_stride;
        if (base < 0) {      // it waits: its columns end where they did
            const int end = r.end_without(a.page);
            for (int k = 0; k < kColumns / 32; ++k) {
                const int c = c0 + 32 * k;
                if (c >= a.width || c < end) continue;
                const int entry = row[c];
                if (entry == -1) continue;
                if ((unsigned)entry < (unsigned)a.n_pages) a.free_[entry] = 1;
                row[c] = -1;
            }
            continue;
        }
        const int first = r.first(a.page), end = r.end(a.page);
        int k0 = base;
        for (int j = 0; j < item; ++j) k0 += a.missing[n * a.items + j];
#pragma unroll 1
        for (int k = 0; k < kColumns / 32; ++k) {
            const int c = c0 + 32 * k;
            const bool lacks = c >= first && c < end && (unsigned)row[c] >= (unsigned)a.n_pages;
            const unsigned who = __ballot_sync(0xffffffffu, lacks);
            if (lacks) row[c] = a.dealt[k0 + __popc(who & ((1u << lane) - 1))];
            k0 += __popc(who);
        }
    }
    meet();

    // ------------------------------------------------------------------ 5: where the new tokens go
    for (int n = rank * kThreads + tid; n < a.rows; n += blocks * kThreads) {
        const Ask r = ask_of(a, n);
        const int len = base_of[n] < 0 ? r.len - r.add : r.len;
        if (base_of[n] < 0 || r.bad_len) a.kv_lens[n] = len;      // rows without tokens below
    }
    const int tokens = cu[a.rows];
    for (int t = rank * kThreads + tid; t < a.max_tokens; t += blocks * kThreads) {
        int pos = -1;
        long long slot = -1;
        if (t < tokens) {
            int lo = 0, hi = a.rows;      // cu[lo] <= t < cu[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= t) lo = mid;
                else hi = mid;
            }
            pos = a.kv_lens[lo] - (cu[lo + 1] - cu[lo]) + (t - cu[lo]);
            const int col = pos / a.page;
            slot = (long long)a.table[lo * a.table_stride + col] * a.page + (pos - col * a.page);
        }
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
}

int check(const KdaPlanShape* s) {
    if (!s) return KDA_ERR_NULL;
    if (s->rows <= 0 || s->width <= 0 || s->page_size <= 0 || s->n_pages < 0 || s->max_tokens < 0) return KDA_ERR_BAD_SHAPE;
    if (s->rows > kMaxRows) return KDA_ERR_UNSUPPORTED;
    if ((long long)s->width * s->page_size >= 1ll << 31 || (long long)s->rows * s->width >= 1ll << 31 || s->n_pages > (1 << 30) || s->max_tokens > (1 << 30))
        return KDA_ERR_BAD_SHAPE;
    return KDA_OK;
}
int items_of(const KdaPlanShape& s) { return ceil_div(s.width, kColumns); }

}  // namespace
}  // namespace kda

using namespace kda;

extern "C" size_t kda_plan_pages_workspace_bytes(const KdaPlanShape* s) {
    if (check(s)) return 0;
    return align_up((size_t)s->rows * items_of(*s) * sizeof(int), 256) + align_up((size_t)(s->n_pages + 1) * sizeof(int), 256);
}

extern "C" int kda_plan_pages(const KdaPlanShape* s, int32_t* block_table, int32_t* kv_lens, uint8_t* page_free, const int32_t* new_lens, const int32_t* starts,
                              int32_t* cu_seqlens, int32_t* positions, int64_t* slots, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check(s)) return rc;
    if (!block_table || !kv_lens || !new_lens || !cu_seqlens || (s->n_pages > 0 && !page_free) || (s->max_tokens > 0 && (!positions || !slots))) return KDA_ERR_NULL;
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 || workspace_bytes < kda_plan_pages_workspace_bytes(s)) return KDA_ERR_WORKSPACE;
    PlanArgs a;
    a.table = block_table; a.kv_lens = kv_lens; a.free_ = page_free; a.new_lens = new_lens; a.starts = starts;
    a.cu = cu_seqlens; a.positions = positions; a.slots = reinterpret_cast<long long*>(slots);
    a.rows = s->rows; a.width = s->width; a.page = s->page_size; a.n_pages = s->n_pages; a.max_tokens = s->max_tokens;
    a.items = items_of(*s);
    a.missing = static_cast<int*>(workspace);
    a.dealt = reinterpret_cast<int*>(static_cast<char*>(workspace) + align_up((size_t)a.rows * a.items * sizeof(int), 256));
    a.mirror = status_mirror();
    a.table_stride = s->table_stride;
    const size_t smem = (2 * (size_t)a.rows + 1) * sizeof(int);
    if (int rc = set_smem_limit(plan_pages_kernel, smem)) return rc;
    // what one block reads in a few loads a thread
    const bool small = a.rows * a.items <= 2 * kWarps && a.n_pages <= 16 * kThreads && a.max_tokens <= 2 * kThreads;
    const int blocks = small ? 1 : kBlocks;
    cudaError_t e = cudaSuccess;
    KDA_LAUNCH("plan_pages_kernel", (cudaStream_t)stream,
               e = launch_early(plan_pages_kernel, dim3(blocks), kThreads, smem, (cudaStream_t)stream, false, blocks, a));
    return e == cudaSuccess ? launch_status() : KDA_ERR_CUDA;
}
