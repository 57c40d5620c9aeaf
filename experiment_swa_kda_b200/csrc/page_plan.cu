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
constexpr int kMaxRows = 16384;      // three numbers a row in shared memory

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

// Entries lacking, new tokens and free pages.  The host sees to it that the first and the last fit in 32 bits; new tokens stop at kFull, which is
// more than any step takes.
struct Sums {
    int need, add, free_;
};
constexpr int kMostTokens = 1 << 30, kFull = kMostTokens + 1;
__device__ __forceinline__ int add_tokens(int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)kFull); }
__device__ __forceinline__ Sums operator+(Sums a, Sums b) { return Sums{a.need + b.need, add_tokens(a.add, b.add), a.free_ + b.free_}; }
// Sums over the block's threads up to, and without, this one; `total` over all.  `sums` has a place a warp and is written anew by each call.
__device__ __forceinline__ Sums block_scan(Sums mine, Sums* sums, Sums& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto scan = [&](Sums x) {
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const Sums y{__shfl_up_sync(0xffffffffu, x.need, o), __shfl_up_sync(0xffffffffu, x.add, o), __shfl_up_sync(0xffffffffu, x.free_, o)};
            if (lane >= o) x = x + y;
        }
        return x;
    };
    auto from = [&](Sums x, int l) { return Sums{__shfl_sync(0xffffffffu, x.need, l), __shfl_sync(0xffffffffu, x.add, l), __shfl_sync(0xffffffffu, x.free_, l)}; };
    const Sums upto = scan(mine);
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    const Sums warps = scan(sums[lane]);      // kWarps == 32
    total = from(warps, 31);
    Sums base = from(warps, max(warp - 1, 0)), before{__shfl_up_sync(0xffffffffu, upto.need, 1), __shfl_up_sync(0xffffffffu, upto.add, 1), __shfl_up_sync(0xffffffffu, upto.free_, 1)};
    if (warp == 0) base = Sums{0, 0, 0};
    if (lane == 0) before = Sums{0, 0, 0};
    return base + before;
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

// The items (a row, 128 of its columns) of a table are dealt out to the warps in runs of at most 32; lane l of a warp has what the row of
// the run's l-th item asks for.
struct Run {
    int first, many;      // items
    int row, col0, col1, col1_without;      // of this lane's item: its row, the columns that shall be held, and their end without the new tokens
};

__global__ void __launch_bounds__(kThreads, 1) plan_pages_kernel(const __grid_constant__ PlanArgs a) {
    extern __shared__ int rows_sm[];
    // of each row: entries lacking before it (-1: it is not served); new tokens, then the sum before it; its length.   With one block entries missing follow, [items]
    int *base_of = rows_sm, *cu = base_of + a.rows, *len_of = cu + a.rows + 1;
    __shared__ Sums sums[2][kWarps];
    __shared__ int counts[kBlocks];                      // free pages of each block's share
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int blocks = gridDim.x, rank = blockIdx.x;     // the grid is one cluster
    int* missing = blocks > 1 ? a.missing : len_of + a.rows;
    auto meet = [&]() {
        if (blocks > 1) cluster_sync();
        else __syncthreads();
    };
    const int all = a.rows * a.items, warps = blocks * kWarps, run = min((all + warps - 1) / warps, 32);
    auto run_at = [&](int i0) {
        Run r{i0, min(run, all - i0), 0, 0, 0, 0};
        if (lane < r.many) {
            r.row = (i0 + lane) / a.items;
            const Ask ask = ask_of(a, r.row);
            r.col0 = ask.first(a.page);
            r.col1 = ask.end(a.page);
            r.col1_without = ask.end_without(a.page);
        }
        return r;
    };

    // ------------------------------------------------------------------ 1: what rows hold, and lack
    constexpr int kAtOnce = 4, kEach = kColumns / 32;
    for (int i0 = (rank * kWarps + warp) * run; i0 < all; i0 += warps * run) {
        const Run r = run_at(i0);
        int lacks = 0;
        for (int x = 0; x < r.many; x += kAtOnce) {
            int entry[kAtOnce][kEach];
#pragma unroll
            for (int y = 0; y < kAtOnce; ++y) {
                const int n = __shfl_sync(0xffffffffu, r.row, min(x + y, r.many - 1)), c0 = (i0 + x + y - n * a.items) * kColumns + lane;
#pragma unroll
                for (int k = 0; k < kEach; ++k) entry[y][k] = x + y < r.many && c0 + 32 * k < a.width ? a.table[n * a.table_stride + c0 + 32 * k] : -1;
            }
#pragma unroll
            for (int y = 0; y < kAtOnce; ++y) {
                const int l = min(x + y, r.many - 1), n = __shfl_sync(0xffffffffu, r.row, l), c0 = (i0 + l - n * a.items) * kColumns + lane;
                const int first = __shfl_sync(0xffffffffu, r.col0, l), end = __shfl_sync(0xffffffffu, r.col1, l);
                if (x + y >= r.many) break;
                int here = 0;
#pragma unroll
                for (int k = 0; k < kEach; ++k) {
                    const int c = c0 + 32 * k, e = entry[y][k];
                    const bool names = (unsigned)e < (unsigned)a.n_pages, held = c >= first && c < end;
                    if (e >= a.n_pages) a.tell(KDA_ERR_BLOCK_TABLE);
                    if (held && !names) ++here;
                    if (!held && e != -1) {
                        if (names) a.free_[e] = 1;
                        a.table[n * a.table_stride + c] = -1;
                    }
                }
                here = __reduce_add_sync(0xffffffffu, here);
                if (lane == l) lacks = here;
            }
        }
        if (lane < r.many) missing[i0 + lane] = lacks;
    }
    meet();

    // ------------------------------------------------------------------ 2: free pages of this block's share; sums over all rows
    const int share = ((a.n_pages + blocks - 1) / blocks + 15) / 16 * 16, p0 = min(rank * share, a.n_pages), p1 = min(p0 + share, a.n_pages);
    const int each_page = ((share + kThreads - 1) / kThreads + 15) / 16 * 16, my_p0 = min(p0 + tid * each_page, p1), my_p1 = min(my_p0 + each_page, p1);
    const bool wide = reinterpret_cast<uintptr_t>(a.free_) % 16 == 0;
    int my_free = 0;
    for (int p = my_p0; p < my_p1; p += 16) my_free += __popc(free_bits(a.free_, p, my_p1, wide));
    const int each = (a.rows + kThreads - 1) / kThreads, n0 = min(tid * each, a.rows), n1 = min(n0 + each, a.rows);
    Sums mine{0, 0, my_free}, total;
#pragma unroll 4
    for (int n = n0; n < n1; ++n) {
        int need = 0;
        for (int i = 0; i < a.items; ++i) need += missing[n * a.items + i];
        const Ask r = ask_of(a, n);
        if (n % blocks == rank) {
            if (r.bad_len) a.tell(KDA_ERR_BLOCK_TABLE);
            if (r.bad_new) a.tell(KDA_ERR_CU_SEQLENS);
        }
        base_of[n] = need;
        cu[n] = r.add;
        len_of[n] = r.len;
        mine = mine + Sums{need, r.add, 0};
    }
    const Sums before = block_scan(mine, sums[0], total);
    if (blocks > 1) {
        if (tid < blocks) {
            uint32_t at;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(counts + rank)), "r"(tid));
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(total.free_) : "memory");
        }
    } else if (tid == 0) {
        counts[0] = total.free_;
    }
    meet();

    // ------------------------------------------------------------------ 3: who is served; the free pages they take, in order
    int free_all = 0, free_base = 0;
    for (int b = 0; b < blocks; ++b) {
        if (b < rank) free_base += counts[b];
        free_all += counts[b];
    }
    Sums upto = before;
    bool all_served = true;
    mine = Sums{0, 0, 0};
    for (int n = n0; n < n1; ++n) {
        const Sums row{base_of[n], cu[n], 0};
        upto = upto + row;
        const bool served = (upto.need <= free_all && upto.add <= a.max_tokens) || (row.need == 0 && row.add == 0);
        if (served) {
            base_of[n] = upto.need - row.need;
            mine = mine + row;
        } else {
            base_of[n] = -1;
            cu[n] = 0;
            len_of[n] -= row.add;
            all_served = false;
        }
    }
    // Rows that lack pages and are served are the first of those that lack any, so the sums of all rows hold for what they lack, and for
    // the tokens too if nobody waits.
    int at = before.add;
    if (!__syncthreads_and(all_served)) at = block_scan(mine, sums[1], total).add;
    const int dealt = total.need;
    for (int n = n0; n < n1; ++n) {
        const int add = cu[n];
        cu[n] = at;
        if (n % blocks == rank) a.cu[n] = at;
        at += add;
    }
    if (tid == 0) {
        cu[a.rows] = total.add;
        if (rank == 0) a.cu[a.rows] = total.add;
    }
    if (dealt > 0) {
        int k = free_base + before.free_;
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
    for (int i0 = (rank * kWarps + warp) * run; i0 < all; i0 += warps * run) {
        const Run r = run_at(i0);
        int lacks = 0, base = 0, from = 0;
        if (lane < r.many) {
            lacks = missing[i0 + lane];
            base = from = base_of[r.row];
            if (base >= 0 && lacks > 0)
                for (int i = r.row * a.items; i < i0 + lane; ++i) from += missing[i];
        }
        for (unsigned todo = __ballot_sync(0xffffffffu, base < 0 || lacks > 0); todo != 0; todo &= todo - 1) {
            const int l = __ffs(todo) - 1, n = __shfl_sync(0xffffffffu, r.row, l), c0 = (i0 + l - n * a.items) * kColumns + lane;
            const bool waits = __shfl_sync(0xffffffffu, base, l) < 0;
            const int first = __shfl_sync(0xffffffffu, r.col0, l), end = __shfl_sync(0xffffffffu, waits ? r.col1_without : r.col1, l);
            int k0 = __shfl_sync(0xffffffffu, from, l), entry[kEach];
            int* row = a.table + n * a.table_stride;
#pragma unroll
            for (int k = 0; k < kEach; ++k) entry[k] = c0 + 32 * k < a.width ? row[c0 + 32 * k] : -1;
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                const int c = c0 + 32 * k;
                if (waits) {      // its columns end where they did
                    if (c < end || entry[k] == -1) continue;
                    if ((unsigned)entry[k] < (unsigned)a.n_pages) a.free_[entry[k]] = 1;
                    row[c] = -1;
                } else {
                    const bool is = c >= first && c < end && (unsigned)entry[k] >= (unsigned)a.n_pages;
                    const unsigned who = __ballot_sync(0xffffffffu, is);
                    if (is) row[c] = a.dealt[k0 + __popc(who & ((1u << lane) - 1))];
                    k0 += __popc(who);
                }
            }
        }
    }
    meet();

    // ------------------------------------------------------------------ 5: where the new tokens go
    for (int n = rank * kThreads + tid; n < a.rows; n += blocks * kThreads)
        if (a.kv_lens[n] != len_of[n]) a.kv_lens[n] = len_of[n];
    const int tokens = cu[a.rows], stride = blocks * kThreads;
    for (int t0 = rank * kThreads + tid; t0 < a.max_tokens; t0 += kAtOnce * stride) {
        int pos[kAtOnce], col[kAtOnce], entry[kAtOnce];
#pragma unroll
        for (int y = 0; y < kAtOnce; ++y) {
            const int t = t0 + y * stride;
            pos[y] = -1;
            if (t >= tokens) continue;
            int lo = 0, hi = a.rows;      // cu[lo] <= t < cu[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= t) lo = mid;
                else hi = mid;
            }
            pos[y] = len_of[lo] - (cu[lo + 1] - t);
            col[y] = pos[y] / a.page;
            entry[y] = a.table[lo * a.table_stride + col[y]];
        }
#pragma unroll
        for (int y = 0; y < kAtOnce; ++y) {
            const int t = t0 + y * stride;
            if (t >= a.max_tokens) break;
            a.positions[t] = pos[y];
            a.slots[t] = pos[y] < 0 ? -1ll : (long long)entry[y] * a.page + (pos[y] - col[y] * a.page);
        }
    }
}

int check(const KdaPlanShape* s) {
    if (!s) return KDA_ERR_NULL;
    if (s->rows <= 0 || s->width <= 0 || s->page_size <= 0 || s->n_pages < 0 || s->max_tokens < 0) return KDA_ERR_BAD_SHAPE;
    if (s->rows > kMaxRows) return KDA_ERR_UNSUPPORTED;
    if ((long long)s->width * s->page_size >= 1ll << 31 || (long long)s->rows * s->width >= 1ll << 31 || s->n_pages > (1 << 30) || s->max_tokens > kMostTokens)
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
    // what one block reads in a few loads a thread
    const bool small = a.rows * a.items <= 2 * kWarps && a.n_pages <= 16 * kThreads && a.max_tokens <= 2 * kThreads;
    const int blocks = small ? 1 : kBlocks;
    const size_t smem = (3 * (size_t)a.rows + 1 + (small ? a.rows * a.items : 0)) * sizeof(int);
    if (int rc = set_smem_limit(plan_pages_kernel, smem)) return rc;
    cudaError_t e = cudaSuccess;
    KDA_LAUNCH("plan_pages_kernel", (cudaStream_t)stream,
               e = launch_early(plan_pages_kernel, dim3(blocks), kThreads, smem, (cudaStream_t)stream, false, blocks, a));
    return e == cudaSuccess ? launch_status() : KDA_ERR_CUDA;
}
