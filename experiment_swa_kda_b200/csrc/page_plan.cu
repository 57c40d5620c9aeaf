// Pages of a paged cache dealt out and the slots of new tokens mapped, from the lengths of a batch's requests.
//
// Row n is to hold the columns [floor(start_n / page), ceil(len_n / page)) of its table.  What it holds besides goes back; the
// entries it lacks take the free pages in ascending order, rows first, columns next, so the result depends on which pages are free
// and on nothing else (a call repeated on its own result changes nothing).  A row is served if the entries lacking up to and with it
// are at most the free pages, and the new tokens up to and with it at most max_tokens; one that is not goes without its new tokens.
//
// All of it is a handful of sums over rows and over pages, each of which the next step waits for: up to some hundred rows bound by latency, not by bytes
// (256 rows of 256 columns and 32,768 pages are 300 KB).  So it is one launch, a cluster of blocks that meet at its barriers (0.5 us each); thousands of rows
// are bound by what its eight SMs get through:
//   1  entries outside of their row's columns go back; missing ones are counted, 128 columns a warp
//   2  every block sums up all rows and all free pages for itself, which costs less than meeting once more
//   3  who is served: the first rows that fit, or (overtake) all that still fit; the first free pages are listed in order
//   4  missing entries take theirs; rows that have to wait give back what their new tokens would have needed
//   5  position and slot of each new token
// A block has a range of the rows from 1 to 5.  A batch that one block can read at once takes a single block, which keeps its lists to itself.
//
// One conversation 5.6 us from first to last instruction (6 a call), 256 rows 9 to 14, 4,096 rows of 128 columns with 262,144 pages 33, of
// which 10 are phase 1 (16 rows a warp, four on their way) and 13 are 4 and 5.  Measured and left out: one barrier more to count free pages by shares also in small
// pools (0.6 us), pages listed by the threads that counted them (4,096 rows 37 -> 50), scans of 64-bit sums (0.5 each).

#include <limits.h>

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
    int rows, width, page, n_pages, max_tokens, items, overtake;
    int split, slice;       // blocks count free pages by shares of `slice`, a multiple of 512
    int thread_pages;       // pages whose flags a thread counts: a power of two, 16 at least

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

__global__ void __launch_bounds__(kThreads, 1) plan_pages_kernel(const __grid_constant__ PlanArgs a) {
    extern __shared__ int rows_sm[];
    // of each row: entries lacking before it (-1: it is not served); new tokens, then the sum before it; its length.  One block alone also has
    // the entries lacking of each item and the pages dealt out here.
    int *base_of = rows_sm, *cu = base_of + a.rows, *len_of = cu + a.rows + 1;
    __shared__ Sums sums[2][kWarps];
    __shared__ int free_before[kThreads], counts[kBlocks];      // free pages before each thread's; of each block's share
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int blocks = gridDim.x, rank = blockIdx.x;     // the grid is one cluster
    const bool alone = blocks == 1;
    dependency_wait();      // launched early: two calls one behind the other 17 us, not 13, without
    int *missing = alone ? len_of + a.rows : a.missing, *dealt = alone ? missing + a.rows * a.items : a.dealt;
    auto meet = [&]() {
        if (alone) __syncthreads();
        else cluster_sync();
    };
    // this block's rows, in items of 128 columns; a warp takes a run of at most 32 of them, lane l the l-th one's row
    auto first_row = [&](int b) { return alone ? b * a.rows : a.rows * b / kBlocks; };
    const int r0 = first_row(rank), r1 = first_row(rank + 1);
    const int item0 = r0 * a.items, item1 = r1 * a.items, run = min((item1 - item0 + kWarps - 1) / kWarps, 32);
    struct Run {
        int many, row, col0, col1, col1_without;      // the columns that the row shall hold, and their end without its new tokens
    };
    auto run_at = [&](int i0) {
        Run r{min(run, item1 - i0), 0, 0, 0, 0};
        if (lane < r.many) {
            r.row = (i0 + lane) / a.items;
            const Ask ask = ask_of(a, r.row);
            r.col0 = ask.first(a.page);
            r.col1 = ask.end(a.page);
            r.col1_without = ask.end_without(a.page);
        }
        return r;
    };

    // all rows, for the sums: a thread has a few beside each other
    const int each = (a.rows + kThreads - 1) / kThreads, n0 = min(tid * each, a.rows), n1 = min(n0 + each, a.rows);
    for (int n = n0; n < n1; ++n) {
        const Ask r = ask_of(a, n);
        if (n >= r0 && n < r1) {
            if (r.bad_len) a.tell(KDA_ERR_BLOCK_TABLE);
            if (r.bad_new) a.tell(KDA_ERR_CU_SEQLENS);
        }
        cu[n] = r.add;
        len_of[n] = r.len;
    }

    // ------------------------------------------------------------------ 1: what rows hold, and lack
    constexpr int kAtOnce = 4, kEach = kColumns / 32;
    const bool wide_rows = (reinterpret_cast<uintptr_t>(a.table) | (uintptr_t)a.table_stride * 4) % 16 == 0;
    for (int i0 = item0 + warp * run; i0 < item1; i0 += kWarps * run) {
        const Run r = run_at(i0);
        int lacks = 0;
        for (int x = 0; x < r.many; x += kAtOnce) {
            int entry[kAtOnce][kEach];      // of columns 4 lane .. 4 lane + 3 of an item
#pragma unroll
            for (int y = 0; y < kAtOnce; ++y) {
                const int l = min(x + y, r.many - 1), n = __shfl_sync(0xffffffffu, r.row, l), c0 = (i0 + l - n * a.items) * kColumns + kEach * lane;
                const int* at = a.table + n * a.table_stride + c0;
                if (wide_rows && c0 + kEach <= a.width) {
                    const int4 v = *reinterpret_cast<const int4*>(at);
                    entry[y][0] = v.x, entry[y][1] = v.y, entry[y][2] = v.z, entry[y][3] = v.w;
                } else {
#pragma unroll
                    for (int k = 0; k < kEach; ++k) entry[y][k] = c0 + k < a.width ? at[k] : -1;
                }
            }
#pragma unroll
            for (int y = 0; y < kAtOnce; ++y) {
                const int l = min(x + y, r.many - 1), n = __shfl_sync(0xffffffffu, r.row, l), c0 = (i0 + l - n * a.items) * kColumns + kEach * lane;
                const int first = __shfl_sync(0xffffffffu, r.col0, l), held = max(__shfl_sync(0xffffffffu, r.col1, l) - first, 0);
                int here = 0;
                bool other = false;      // an entry to give back
#pragma unroll
                for (int k = 0; k < kEach; ++k) {
                    const bool hold = (unsigned)(c0 + k - first) < (unsigned)held;
                    here += hold && (unsigned)entry[y][k] >= (unsigned)a.n_pages;
                    other |= hold ? entry[y][k] >= a.n_pages : entry[y][k] != -1;
                }
                if (x + y >= r.many) break;
                if (other) {
#pragma unroll
                    for (int k = 0; k < kEach; ++k) {
                        const int e = entry[y][k];
                        if (e >= a.n_pages) a.tell(KDA_ERR_BLOCK_TABLE);
                        if ((unsigned)(c0 + k - first) < (unsigned)held || e == -1) continue;
                        if ((unsigned)e < (unsigned)a.n_pages) a.free_[e] = 1;
                        a.table[n * a.table_stride + c0 + k] = -1;
                    }
                }
                here = __reduce_add_sync(0xffffffffu, here);
                if (lane == l) lacks = here;
            }
        }
        if (lane < r.many) missing[i0 + lane] = lacks;
    }
    meet();

    // ------------------------------------------------------------------ 2: sums over all rows, and over free pages
    // of a large pool each block counts its share, and they tell each other
    const int s0 = a.split ? rank * a.slice : 0, s1 = a.split ? min(s0 + a.slice, a.n_pages) : a.n_pages;
    const int each_page = a.thread_pages, p0 = (int)min((long long)s0 + (long long)tid * each_page, (long long)s1), p1 = min(p0 + each_page, s1);
    const bool wide = reinterpret_cast<uintptr_t>(a.free_) % 16 == 0;
    Sums mine{0, 0, 0}, total;
#pragma unroll 4
    for (int p = p0; p < p1; p += 16) mine.free_ += __popc(free_bits(a.free_, p, p1, wide));
    for (int n = n0; n < n1; ++n) {
        int need = 0;
        for (int i = 0; i < a.items; ++i) need += missing[n * a.items + i];
        base_of[n] = need;
        mine = mine + Sums{need, cu[n], 0};
    }
    const Sums before = block_scan(mine, sums[0], total);
    free_before[tid] = before.free_;
    int free_all = total.free_, free_base = 0;
    if (a.split) {
        if (tid < blocks) {
            uint32_t at;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(counts + rank)), "r"(tid));
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(total.free_) : "memory");
        }
        cluster_sync();
        free_all = 0;
        for (int b = 0; b < blocks; ++b) {
            if (b < rank) free_base += counts[b];
            free_all += counts[b];
        }
    }

    // ------------------------------------------------------------------ 3: who is served; the free pages they take, in order
    const bool enough = total.need <= free_all && total.add <= a.max_tokens;      // for everybody
    if (!enough && a.overtake) {
        // Who is served depends on all before, so a warp goes through the rows, 32 at a time.  What is more than is left never fits again and drops out at once;
        // of the others those up to the first that fits no more are served.  Needs are at most what is left, and all of them fit in 32 bits.
        // 16,384 rows none of which fits take 52 us more than without (144), 4,096 13, 256 1; one row after the other took 1,020, 255 and 16.
        if (warp == 0) {
            int left = free_all, tokens = 0;
            for (int m0 = 0; m0 < a.rows; m0 += 32) {
                const int n = min(m0 + lane, a.rows - 1), need = m0 + lane < a.rows ? base_of[n] : 0, add = m0 + lane < a.rows ? cu[n] : 0;
                bool open = need > 0 || add > 0, served = !open;      // open: not known yet
                for (;;) {
                    open = open && need <= left && add <= a.max_tokens - tokens;
                    if (!__any_sync(0xffffffffu, open)) break;
                    Sums upto{open ? need : 0, open ? add : 0, 0};
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const Sums x{__shfl_up_sync(0xffffffffu, upto.need, o), __shfl_up_sync(0xffffffffu, upto.add, o), 0};
                        if (lane >= o) upto = upto + x;
                    }
                    const unsigned over = __ballot_sync(0xffffffffu, open && (upto.need > left || upto.add > a.max_tokens - tokens));
                    const int first = over != 0 ? __ffs(over) - 1 : 32;      // not lane 0's: an open row fits by itself
                    served |= open && lane < first;
                    open = open && lane > first;
                    left -= __shfl_sync(0xffffffffu, upto.need, first - 1);
                    tokens += __shfl_sync(0xffffffffu, upto.add, first - 1);
                    if (over == 0) break;
                }
                if (!served) base_of[n] = -1;
            }
        }
        __syncthreads();
    }
    Sums upto = before, at = before;
    mine = Sums{0, 0, 0};
    for (int n = n0; n < n1; ++n) {
        const Sums row{base_of[n], cu[n], 0};
        upto = upto + row;
        if (enough || (a.overtake ? row.need >= 0 : (upto.need <= free_all && upto.add <= a.max_tokens) || (row.need == 0 && row.add == 0))) {
            mine = mine + row;
        } else {
            base_of[n] = -1;
            cu[n] = 0;
            len_of[n] -= row.add;
        }
    }
    __syncthreads();
    if (!enough) at = block_scan(mine, sums[1], total);      // of the rows served
    const int taken = total.need;
    for (int n = n0; n < n1; ++n) {
        const int need = base_of[n], add = cu[n];
        if (need >= 0) {
            base_of[n] = at.need;
            at.need += need;
        }
        cu[n] = at.add;
        if (n >= r0 && n < r1) a.cu[n] = at.add;
        at.add += add;
    }
    if (tid == 0) {
        cu[a.rows] = total.add;
        if (rank == 0) a.cu[a.rows] = total.add;
    }
    // A warp lists those of 512 pages at a time, 16 a lane.  The flags change once nobody counts any more.
    const int unit = max(512, each_page), u_warp = a.split ? warp : rank * kWarps + warp, u_warps = a.split ? kWarps : blocks * kWarps;
    for (int u0 = u_warp * unit; s0 + u0 < s1; u0 += u_warps * unit) {
        int k = free_base + free_before[u0 / each_page];
        for (int q = s0 + u0; q < min(s0 + u0 + unit, s1) && k < taken; q += 512) {
            unsigned bits = q + 16 * lane < s1 ? free_bits(a.free_, q + 16 * lane, s1, wide) : 0;
            int upto_lane = __popc(bits);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto_lane, o);
                if (lane >= o) upto_lane += x;
            }
            for (int i = k + upto_lane - __popc(bits); bits != 0 && i < taken; bits &= bits - 1) dealt[i++] = q + 16 * lane + __ffs(bits) - 1;
            k += __shfl_sync(0xffffffffu, upto_lane, 31);
        }
    }
    meet();

    // ------------------------------------------------------------------ 4: entries that were missing
    for (int k = rank * kThreads + tid; k < taken; k += blocks * kThreads) a.free_[dealt[k]] = 0;
    for (int i0 = item0 + warp * run; i0 < item1; i0 += kWarps * run) {
        const Run r = run_at(i0);
        int lacks = 0, base = 0, from = 0;
        if (lane < r.many) {
            lacks = missing[i0 + lane];
            base = from = base_of[r.row];
            if (base >= 0 && lacks > 0)
                for (int i = r.row * a.items; i < i0 + lane; ++i) from += missing[i];
        }
        for (unsigned todo = __ballot_sync(0xffffffffu, base < 0 || lacks > 0); todo != 0;) {
            int of[kAtOnce], entry[kAtOnce][kEach];      // the next items, of columns lane, 32 + lane, ...
#pragma unroll
            for (int y = 0; y < kAtOnce; ++y) {
                of[y] = __ffs(todo) - 1;
                todo &= todo - 1;
                const int l = max(of[y], 0), n = __shfl_sync(0xffffffffu, r.row, l), c0 = (i0 + l - n * a.items) * kColumns + lane;
#pragma unroll
                for (int k = 0; k < kEach; ++k) entry[y][k] = of[y] >= 0 && c0 + 32 * k < a.width ? a.table[n * a.table_stride + c0 + 32 * k] : -1;
            }
#pragma unroll
            for (int y = 0; y < kAtOnce; ++y) {
                if (of[y] < 0) break;
                const int l = of[y], n = __shfl_sync(0xffffffffu, r.row, l), c0 = (i0 + l - n * a.items) * kColumns + lane;
                const bool waits = __shfl_sync(0xffffffffu, base, l) < 0;
                const int first = __shfl_sync(0xffffffffu, r.col0, l), end = __shfl_sync(0xffffffffu, waits ? r.col1_without : r.col1, l);
                int k0 = __shfl_sync(0xffffffffu, from, l);
                int* row = a.table + n * a.table_stride;
#pragma unroll
                for (int k = 0; k < kEach; ++k) {
                    const int c = c0 + 32 * k, e = entry[y][k];
                    if (waits) {      // its columns end where they did
                        if (c < end || e == -1) continue;
                        if ((unsigned)e < (unsigned)a.n_pages) a.free_[e] = 1;
                        row[c] = -1;
                    } else {
                        const bool is = c >= first && c < end && (unsigned)e >= (unsigned)a.n_pages;
                        const unsigned who = __ballot_sync(0xffffffffu, is);
                        if (is) row[c] = dealt[k0 + __popc(who & ((1u << lane) - 1))];
                        k0 += __popc(who);
                    }
                }
            }
        }
    }
    // A block's rows are its own, and so are their tokens, unless one block has so many that all of them share.
    const int tokens = cu[a.rows];
    bool share = false;
    if (!alone && tokens > 8 * kThreads)
        for (int b = 0; b < blocks; ++b) share |= cu[first_row(b + 1)] - cu[first_row(b)] > 8 * kThreads;
    if (share) cluster_sync();
    else __syncthreads();

    // ------------------------------------------------------------------ 5: where the new tokens go
    for (int n = r0 + tid; n < r1; n += kThreads)
        if (a.kv_lens[n] != len_of[n]) a.kv_lens[n] = len_of[n];
    const int stride = share ? blocks * kThreads : kThreads, t_begin = share ? rank * kThreads : cu[r0], t_end = share ? tokens : cu[r1];
    const int n_begin = share ? 0 : r0, n_end = share ? a.rows : r1;
    for (int t0 = t_begin + tid; t0 < t_end; t0 += kAtOnce * stride) {
        int pos[kAtOnce], col[kAtOnce], entry[kAtOnce];
#pragma unroll
        for (int y = 0; y < kAtOnce; ++y) {
            const int t = t0 + y * stride;
            if (t >= t_end) continue;
            int lo = n_begin, hi = n_end;      // cu[lo] <= t < cu[hi]
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
            if (t >= t_end) break;
            a.positions[t] = pos[y];
            a.slots[t] = (long long)entry[y] * a.page + (pos[y] - col[y] * a.page);
        }
    }
    for (int t = tokens + rank * kThreads + tid; t < a.max_tokens; t += blocks * kThreads) {
        a.positions[t] = -1;
        a.slots[t] = -1;
    }
}

int check(const KdaPlanShape* s) {
    if (!s) return KDA_ERR_NULL;
    if (s->rows <= 0 || s->width <= 0 || s->page_size <= 0 || s->n_pages < 0 || s->max_tokens < 0) return KDA_ERR_BAD_SHAPE;
    if (s->rows > kMaxRows) return KDA_ERR_UNSUPPORTED;
    if ((long long)s->width * s->page_size >= 1ll << 31 || (long long)s->rows * s->width >= 1ll << 31 || s->n_pages > (1 << 30) || s->max_tokens > kMostTokens)
        return KDA_ERR_BAD_SHAPE;
    // columns are counted in whole items, in 32 bits; rows are written, each by its own block
    if (s->width > INT_MAX - kColumns || (s->rows > 1 && s->table_stride < s->width)) return KDA_ERR_BAD_SHAPE;
    return KDA_OK;
}
int items_of(const KdaPlanShape& s) { return ceil_div(s.width, kColumns); }
// What one block reads in a few loads a thread, and keeps in shared memory.
bool alone(const KdaPlanShape& s) { return (long long)s.rows * items_of(s) <= 2 * kWarps && s.n_pages <= 16 * kThreads && s.max_tokens <= 2 * kThreads; }

}  // namespace
}  // namespace kda

using namespace kda;

extern "C" size_t kda_plan_pages_workspace_bytes(const KdaPlanShape* s) {
    if (check(s) || alone(*s)) return 0;
    return align_up((size_t)s->rows * items_of(*s) * sizeof(int), 256) + align_up((size_t)(s->n_pages + 1) * sizeof(int), 256);
}

extern "C" int kda_plan_pages(const KdaPlanShape* s, int32_t* block_table, int32_t* kv_lens, uint8_t* page_free, const int32_t* new_lens, const int32_t* starts,
                              int32_t* cu_seqlens, int32_t* positions, int64_t* slots, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check(s)) return rc;
    if (!block_table || !kv_lens || !new_lens || !cu_seqlens || (s->n_pages > 0 && !page_free) || (s->max_tokens > 0 && (!positions || !slots))) return KDA_ERR_NULL;
    const size_t need = kda_plan_pages_workspace_bytes(s);
    if (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 || workspace_bytes < need)) return KDA_ERR_WORKSPACE;
    PlanArgs a;
    a.table = block_table; a.kv_lens = kv_lens; a.free_ = page_free; a.new_lens = new_lens; a.starts = starts;
    a.cu = cu_seqlens; a.positions = positions; a.slots = reinterpret_cast<long long*>(slots);
    a.rows = s->rows; a.width = s->width; a.page = s->page_size; a.n_pages = s->n_pages; a.max_tokens = s->max_tokens; a.overtake = s->overtake;
    a.items = items_of(*s);
    // every block for itself: 2 us for 262,144 pages, where meeting once more costs 0.6
    a.split = a.n_pages > 64 * kThreads;
    a.slice = ceil_div(ceil_div(a.n_pages, kBlocks), 512) * 512;
    for (a.thread_pages = 16; (long long)a.thread_pages * kThreads < (a.split ? a.slice : a.n_pages);) a.thread_pages *= 2;
    a.missing = a.dealt = nullptr;
    if (need > 0) {
        a.missing = static_cast<int*>(workspace);
        a.dealt = reinterpret_cast<int*>(static_cast<char*>(workspace) + align_up((size_t)a.rows * a.items * sizeof(int), 256));
    }
    a.mirror = status_mirror();
    a.table_stride = s->table_stride;
    const int blocks = need > 0 ? kBlocks : 1;
    const size_t smem = (3 * (size_t)a.rows + 1 + (need > 0 ? 0 : a.rows * a.items + a.n_pages)) * sizeof(int);
    if (int rc = set_smem_limit(plan_pages_kernel, smem)) return rc;
    cudaError_t e = cudaSuccess;
    KDA_LAUNCH("plan_pages_kernel", (cudaStream_t)stream,
               e = launch_early(plan_pages_kernel, dim3(blocks), kThreads, smem, (cudaStream_t)stream, true, blocks, a));
    return e == cudaSuccess ? launch_status() : KDA_ERR_CUDA;
}
