// Attention over a paged cache for few rows a sequence (bf16, heads up to 128 wide, at most 16 rows: new tokens x query heads of
// one kv head): the token step of serving.
//
//   o_i = sum_j 2^(c s_ij - c m_i) v_j / sum_j 2^(c s_ij - c m_i),   s = q k^T,  c = scale / ln 2
//
// Bound by the cache's bytes: a key costs 4 D bytes and at most 64 D operations.  All that counts is that every SM has its share of the
// keys and enough copies in flight.  16 heads on 4: 32 conversations of up to 16,384 tokens 106 to 111 us (0.87 to 0.91 of the copy rate), 128 of
// them 0.99 to 1.0; 256 with windows of 512 59 us (0.68: 9 tiles a sequence and head, so that start, ends and join count); one of
// 3 heads and 4,097 tokens 12 to 14 us, two launches of a handful of dependent reads each.
//
// - The tiles (64 keys of one sequence and kv head) of the whole batch are one list, sequence after sequence, and each block
//   takes an equal stretch of it, whatever the sequences' lengths are.  The list is known on the device alone: every block adds up the
//   lengths itself.  Where a stretch ends inside a sequence its part of the softmax goes to the workspace, and
//   attn_decode_join_kernel puts the parts together.
// - A warp takes 16 keys of a tile through a ring of its own (K and V by TMA, 128-byte swizzle), so that warps meet only where a
//   sequence or the stretch ends.  The ring runs ahead across those places.  (Warps with stretches of their own, which never meet, left
//   four times the parts to join and took longer: 32 x 16 heads 118 us, one conversation 22.)
// - Products are mma.sync m16n8k16 with the keys as their 16 rows and the query rows as their 8 columns: S^T = K Q^T and O^T = V^T P^T
//   (P^T comes from S^T's registers by movmatrix).  Up to 8 rows take half the products that rows of queries would.  The weights
//   go as two bf16 terms, p = hi + lo to 2^-16, which leaves the output with the error of its own rounding.
// - What runs once a sequence (its queries, the join of the warps' sums) is kept short in code: unrolled it was fetched anew every time
//   and took 5 us.

#include "attn.cuh"
#include "tc_common.cuh"

namespace kda {
namespace tc {
int make_map_paged(CUtensorMap* m, const void* ptr, uint64_t dim, uint64_t rows, uint64_t heads, uint64_t pages, int64_t row_ld, int64_t head_ld, int64_t page_ld,
                   uint32_t box_rows);
}
namespace attn {
namespace {

using namespace tc;

constexpr int kMaxRows = 16, kTile = 64, kWarps = 4, kThreads = 128, kStages = 3;
constexpr int kPerSm = 2;             // blocks an SM: 102 KB each, 106 with more than 8 rows
// Up to so many tiles a sequence and kv head stay together: they take about as long as two of them and the join, which is a launch less (3
// conversations of 40 tokens 14.5 us in parts, 8.4 whole; 16 of 100 12.5 and 10.4).  Six where there are sequences for every SM (200 of up
// to 380 36 and 33), four where parts would have some to themselves (one of 300 12.4 and 13.2 with six).
constexpr int kWholeTiles = 4, kWholeTilesOfMany = 6;
constexpr int kMinTiles = 2;          // a stretch has at least these many tiles
constexpr float kLazy = 8.f;          // as in the kernel for long chunks: sums are rescaled when a maximum grew by 2^8
constexpr int kStatusWait = 121;

template <int DP, int NR>
struct Layout {
    static constexpr int kHalf = 16 * 128;                            // 16 keys of 64 values
    static constexpr int kStage = 2 * (DP / 64) * kHalf;              // K and V of 16 keys
    static constexpr int kRowsOf = 8 * NR;
    static constexpr int kQ = kWarps * kStages * kStage;              // two sequences' queries
    static constexpr int kBars = kQ + 2 * kRowsOf * DP * 2;
    static constexpr int kBytes = kBars + 1024 + 1024;      // barriers and what the warps tell each other; slack to align the tiles
};

struct Args {
    Call c;
    int blocks, box_rows;
    int whole;            // stretches begin and end with a sequence and kv head: no parts
    float* part_o;        // [blocks][2][rows][D]
    float2* part_ml;      // [blocks][2][rows]
};

// One sequence's tiles and rows.
struct Seq {
    int first, count, base, lo, hi, t0, t1;
};
// what a sequence is read from: the ends of its new tokens and its length, as they stand in memory
struct Raw {
    int a, b, len;
};
__device__ __forceinline__ Raw raw_at(const Batch& b, int n) {
    if (n >= b.n_seq) return Raw{0, 0, 0};
    return b.cu != nullptr ? Raw{__ldg(b.cu + n), __ldg(b.cu + n + 1), __ldg(b.kv_lens + n)} : Raw{n * b.q_len, (n + 1) * b.q_len, __ldg(b.kv_lens + n)};
}
__device__ __forceinline__ Seq seq_of_raw(const Batch& b, const Raw& r, int window) {
    Seq s;
    s.first = min(max(r.a, 0), b.tokens);
    s.count = min(max(r.b, s.first), b.tokens) - s.first;
    const long long room = (long long)b.table_width * b.page_size;
    const int len = max(r.len, 0) > room ? (int)room : max(r.len, 0);
    s.base = len - s.count;
    s.hi = s.count > 0 ? len : 0;
    s.lo = min(first_key(s.base, window), s.hi);
    s.t0 = s.lo / kTile;
    s.t1 = (s.hi + kTile - 1) / kTile;
    return s;
}
__device__ __forceinline__ Seq seq_at(const Batch& b, int n, int window) { return seq_of_raw(b, raw_at(b, n), window); }

// How the list is cut: the first `longer` stretches have `each` + 1 tiles, the others `each`.
struct Cut {
    int total, each, longer, used;
    __device__ __forceinline__ int begin(int id) const { return id >= used ? total : id * each + min(id, longer); }
};
struct Start {
    Seq s;                // where a stretch begins
    Raw after;
    int n, hk, tile;
    int begin, end;       // the stretch, of the list, where it is whole
};
// The cut, and where stretch `id` begins.  Called by all THREADS of a block; `sums` has a place for each warp.  The host takes
// care that the list has less than 2^31 tiles.
template <int THREADS, bool whole>
__device__ __forceinline__ Cut find_start(const Batch& b, int kv_heads, int window, int blocks, int id, Start* start, int* sums) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int each = (b.n_seq + THREADS - 1) / THREADS, n0 = min(tid * each, b.n_seq), n1 = min(n0 + each, b.n_seq);
    int mine = 0;
    for (int n = n0; n < n1; ++n) {
        const Seq s = seq_at(b, n, window);
        mine += (s.t1 - s.t0) * kv_heads;
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    Cut cut;
    cut.total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) upto += sums[w];
        cut.total += sums[w];
    }
    cut.used = min(blocks, max(whole ? cut.total : cut.total / kMinTiles, 1));
    cut.each = cut.total / cut.used;
    cut.longer = cut.total - cut.each * cut.used;
    if (whole) {
        if (tid == 0) {
            start->begin = cut.begin(id);
            start->end = cut.begin(id + 1);
        }
        __syncthreads();
    }
#pragma unroll
    for (int side = 0; side <= (whole ? 1 : 0); ++side) {      // whole: both ends move on to the next beginning of a sequence and kv head
        const int place = cut.begin(id + side);
        int at = upto - mine;
        if (place < at || place >= upto) continue;
        for (int n = n0; n < n1; ++n) {
            Seq s = seq_at(b, n, window);
            int nt = s.t1 - s.t0;
            const int here = nt * kv_heads;
            if (place < at + here) {
                const int rest = place - at;
                int hk = rest / nt, tile = s.t0 + rest - hk * nt;
                const int on = whole && tile > s.t0 ? s.t1 - tile : 0;
                if (side == 1) {
                    start->end = place + on;
                    break;
                }
                if (on > 0) {
                    start->begin = place + on;
                    if (++hk == kv_heads) {
                        hk = 0;
                        do {
                            if (++n >= b.n_seq) break;
                            s = seq_at(b, n, window);
                        } while (s.t1 <= s.t0);
                    }
                    tile = s.t0;
                }
                start->s = s;
                start->after = raw_at(b, n + 1);
                start->n = n;
                start->hk = hk;
                start->tile = tile;
                break;
            }
            at += here;
        }
    }
    __syncthreads();
    return cut;
}

// A place in the list.
struct Walk {
    Seq s;
    Raw after;      // of the next sequence, read when this one is entered: nothing waits for it
    int n, hk, tile;
    __device__ __forceinline__ void set(const Start& at) {
        s = at.s;
        after = at.after;
        n = at.n;
        hk = at.hk;
        tile = at.tile;
    }
    __device__ __forceinline__ void next(const Batch& b, int kv_heads, int window) {
        if (++tile < s.t1) return;
        if (++hk == kv_heads) {
            hk = 0;
            do {
                if (++n >= b.n_seq) return;      // behind the end of the list: not used
                s = seq_of_raw(b, after, window);
                after = raw_at(b, n + 1);
            } while (s.t1 <= s.t0);
        }
        tile = s.t0;
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t turned(uint32_t x) {      // an 8 x 8 tile of 16-bit values, transposed
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <int DP, int NR>
__global__ void __launch_bounds__(kThreads, kPerSm) attn_decode_kernel(const __grid_constant__ CUtensorMap mK, const __grid_constant__ CUtensorMap mV,
                                                                       const __grid_constant__ Args a) {
    using L = Layout<DP, NR>;
    constexpr int kHalves = DP / 64, kSteps = DP / 16, kRows = 8 * NR;
    extern __shared__ uint8_t raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::kBars);
    Start& start = *reinterpret_cast<Start*>(bars + kWarps * kStages);
    int* sums = reinterpret_cast<int*>(&start + 1);
    volatile int* flags = reinterpret_cast<volatile int*>(sums + kWarps);      // [0] an expired wait, [1], [2] values that are not finite (of sequences in turn)
    float2* row_ml = reinterpret_cast<float2*>(bars + 64);                     // [warps][rows]
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, c4 = lane & 3, r8 = lane >> 2;
    const Batch& b = a.c.batch;
    const int g = a.c.heads.group, D = a.c.heads.dim, Hk = a.c.heads.kv_heads, Hq = a.c.heads.q_heads, window = a.c.window;

    uint64_t* bar = bars + warp * kStages;
    dependents_go();
    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(bar + s, 1);
        mbar_fence_init();
    }
    if (tid == 0) flags[0] = flags[1] = flags[2] = 0;
    const Cut cut = a.whole ? find_start<kThreads, true>(b, Hk, window, a.blocks, blockIdx.x, &start, sums)
                            : find_start<kThreads, false>(b, Hk, window, a.blocks, blockIdx.x, &start, sums);
    const int tiles = a.whole ? start.end - start.begin : cut.begin(blockIdx.x + 1) - cut.begin(blockIdx.x);

    uint8_t* ring = sm + warp * kStages * L::kStage;
    Walk ahead = {}, w = {};
    auto in_reach = [&](const Walk& x) {
        const int k0 = x.tile * kTile + 16 * warp;
        return k0 < x.s.hi && k0 + 16 > x.s.lo;
    };
    // a box a lane: K or V, half of the head, rows of one page
    const int boxes = 16 / a.box_rows, l_kv = lane / (kHalves * boxes), l_half = lane / boxes % kHalves, l_box = lane % boxes;
    int row = 0, page = -1;
    auto look = [&]() {
        const int key = ahead.tile * kTile + 16 * warp + l_box * a.box_rows;
        page = -1;
        if (l_kv < 2 && ahead.n < b.n_seq && key < ahead.s.hi && key + a.box_rows > ahead.s.lo) {
            const int col = key / b.page_size;
            row = key - col * b.page_size;
            page = b.page(ahead.n, col);
            if (page < 0) b.tell(KDA_ERR_BLOCK_TABLE);
        }
    };
    auto load = [&](int i) {      // the tile `ahead` is at, into the ring's place i; then on to the next one
        const int s = i % kStages;
        if (in_reach(ahead)) {
            const int loads = __popc(__ballot_sync(0xffffffffu, page >= 0));
            if (lane == 0) mbar_expect_tx(bar + s, loads * a.box_rows * 128);
            __syncwarp();
            if (page >= 0)
                asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
                                 smem_u32(ring + s * L::kStage + (l_kv * kHalves + l_half) * L::kHalf + l_box * a.box_rows * 128)),
                             "l"(l_kv ? &mV : &mK), "r"(smem_u32(bar + s)), "r"(l_half * 64), "r"(row), "r"(ahead.hk), "r"(page)
                             : "memory");
        }
        ahead.next(b, Hk, window);
        look();
    };
    // queries of one sequence and kv head: a piece of eight values a thread and 8 rows, first to registers, then to shared memory
    uint4 piece[NR];
    auto fetch_q = [&](const Walk& x) {
        const int rows = min(x.s.count * g, kRows);
#pragma unroll
        for (int y = 0; y < NR; ++y) {
            const int e = tid + y * kThreads, r = e / (DP / 8), d = 8 * (e % (DP / 8));
            piece[y] = make_uint4(0, 0, 0, 0);
            if (r < rows && d < D) {
                const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.c.q) + (x.s.first + r / g) * a.c.strides.q_token + (x.hk * g + r % g) * a.c.strides.q_head + d;
                piece[y] = __ldg(reinterpret_cast<const uint4*>(src));
            }
        }
    };
    auto q_at = [&](int buffer, int r, int chunk) { return sm + L::kQ + buffer * kRows * DP * 2 + r * DP * 2 + ((chunk ^ (r & 7)) << 4); };
    auto put_q = [&](int buffer) {
#pragma unroll
        for (int y = 0; y < NR; ++y) {
            const int e = tid + y * kThreads;
            if (e < kRows * DP / 8) *reinterpret_cast<uint4*>(q_at(buffer, e / (DP / 8), e % (DP / 8))) = piece[y];
        }
    };

    int issued = 0;
    if (tiles > 0) {
        ahead.set(start);
        w = ahead;
        look();
        fetch_q(w);
        for (; issued < kStages - 1 && issued < tiles; ++issued) load(issued);
    }
    // sequences without a key in reach have no tile: their rows are nothing
    for (int n = blockIdx.x; n < b.n_seq; n += gridDim.x) {
        const Seq s = seq_at(b, n, window);
        if (tid == 0) {
            if (!b.span_ok(n) || s.count * g > kRows) b.tell(KDA_ERR_CU_SEQLENS);
            if (!b.kv_len_ok(n)) b.tell(KDA_ERR_BLOCK_TABLE);
        }
        if (s.t1 > s.t0) continue;
        const size_t r0 = (size_t)s.first * Hq;
        for (long long e = tid; e < (long long)s.count * Hq * D; e += kThreads) static_cast<__nv_bfloat16*>(a.c.o)[r0 * D + e] = __float2bfloat16(0.f);
        if (a.c.lse != nullptr)
            for (int e = tid; e < s.count * Hq; e += kThreads) a.c.lse[r0 + e] = -INFINITY;
    }
    if (tiles <= 0) return;
    put_q(0);
    __syncthreads();

    const float c = a.c.scale * 1.4426950408889634f, lazy = kLazy / c;
    uint32_t q[NR][kSteps][2];
    float acc[NR][kSteps][4], m[NR][2], l[NR][2];      // O^T: values r8, r8 + 8 of each 16, rows 2 c4, 2 c4 + 1 of each 8
    int last[NR][2], first[NR][2], rows = 0, all_lo = 0, all_hi = 0, unit_begin = 0, q_buffer = 0;
    bool fresh = true;
    uint32_t phases = 0;      // of the ring's barriers: a tile out of this warp's reach leaves its place as it is
    const int mi = lane >> 3, mr = lane & 7;

    for (int i = 0; i < tiles; ++i) {
        if (issued < tiles) {
            __syncwarp();
            load(issued++);
        }
        if (fresh) {
            fresh = false;
            Walk then = w;      // the queries that come next, on their way while these work
            then.tile = w.s.t1 - 1;
            then.next(b, Hk, window);
            if (tiles - i > w.s.t1 - w.tile) fetch_q(then);
            rows = min(w.s.count * g, kRows);
            unit_begin = w.tile;
            all_lo = first_key(w.s.base + (rows - 1) / g, window);
            all_hi = w.s.base + 1;
#pragma unroll
            for (int y = 0; y < NR; ++y) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int r = 8 * y + 2 * c4 + x;
                    last[y][x] = r < rows ? w.s.base + r / g : -1;
                    first[y][x] = first_key(last[y][x], window);
                    m[y][x] = -INFINITY;
                    l[y][x] = 0.f;
                }
#pragma unroll
                for (int t = 0; t < kSteps; ++t)
#pragma unroll
                    for (int x = 0; x < 4; ++x) acc[y][t][x] = 0.f;
#pragma unroll
                for (int k = 0; k < kSteps; k += 2) {
                    uint32_t f[4];
                    ldm4(f, smem_u32(q_at(q_buffer, 8 * y + mr, 2 * k + mi)));
                    q[y][k][0] = f[0]; q[y][k][1] = f[1]; q[y][k + 1][0] = f[2]; q[y][k + 1][1] = f[3];
                }
            }
        }
        if (in_reach(w)) {
            const int s = i % kStages, k0 = w.tile * kTile + 16 * warp;
            if (!flags[0] && !mbar_poll(bar + s, (phases >> s) & 1u, kSpinLimit)) {      // carries on: the warps meet further down
                flags[0] = 1;
                b.tell(kStatusWait);
            }
            __syncwarp();
            phases ^= 1u << s;
            uint8_t* kv = ring + s * L::kStage;
            const uint32_t sk = smem_u32(kv), sv = sk + kHalves * L::kHalf;
            const bool partial = k0 < all_lo || k0 + 16 > all_hi;
            if (partial) {
                // keys that no row sees hold anything: their values are blanked, and so are values that are not finite at keys
                // only some rows see (added at the end by those that do)
#pragma unroll 1
                for (int e = lane; e < 16 * kHalves * 8; e += 32) {
                    const int r = e & 15, ch = e >> 4, key = k0 + r;
                    if (key >= all_lo && key < all_hi) continue;
                    uint4* at = reinterpret_cast<uint4*>(kv + (kHalves + (ch >> 3)) * L::kHalf + sw128_off(r, ch & 7));
                    if (key < w.s.lo || key >= w.s.hi) {
                        *at = make_uint4(0, 0, 0, 0);
                        continue;
                    }
                    uint4 x = *at;
                    uint32_t* y = reinterpret_cast<uint32_t*>(&x);
                    bool odd = false;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if ((y[k] & 0x7f80u) == 0x7f80u) y[k] &= 0xffff0000u, odd = true;
                        if ((y[k] & 0x7f800000u) == 0x7f800000u) y[k] &= 0xffffu, odd = true;
                    }
                    if (odd) {
                        *at = x;
                        flags[1 + q_buffer] = 1;
                    }
                }
                fence_async_smem();
                __syncwarp();
            }
            float s2[2][NR][4] = {};      // S^T: keys r8, r8 + 8, rows 2 c4, 2 c4 + 1; two chains
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t kf[4];
                ldm4(kf, sk + (k >> 2) * L::kHalf + sw128_off((mi & 1) * 8 + mr, 2 * (k & 3) + (mi >> 1)));
#pragma unroll
                for (int y = 0; y < NR; ++y) mma(s2[k & 1][y], kf, q[y][k][0], q[y][k][1]);
            }
            float sc[NR][4];
            bool grow = false;
            float top[NR][2];
#pragma unroll
            for (int y = 0; y < NR; ++y) {
#pragma unroll
                for (int x = 0; x < 4; ++x) sc[y][x] = s2[0][y][x] + s2[1][y][x];
#pragma unroll
                for (int x = 0; x < 2; ++x) top[y][x] = kLowest;
                if (partial) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int key = k0 + r8 + 8 * (x >> 1);
                        if (key < first[y][x & 1] || key > last[y][x & 1]) sc[y][x] = -INFINITY;
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        if (last[y][x] < k0 || first[y][x] >= k0 + 16) top[y][x] = -INFINITY;
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    top[y][x] = max_nan(top[y][x], max_nan(sc[y][x], sc[y][x + 2]));
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) top[y][x] = max_nan(top[y][x], __shfl_xor_sync(0xffffffffu, top[y][x], o));
                    grow |= !(top[y][x] <= m[y][x] + lazy) && !(top[y][x] == -INFINITY);
                }
            }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int y = 0; y < NR; ++y) {
                    float f[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float next = max_nan(m[y][x], top[y][x]);
                        f[x] = m[y][x] == -INFINITY ? 0.f : ex2((m[y][x] - next) * c);
                        m[y][x] = next;
                        l[y][x] *= f[x];
                    }
#pragma unroll
                    for (int t = 0; t < kSteps; ++t)
#pragma unroll
                        for (int x = 0; x < 4; ++x) acc[y][t][x] *= f[x & 1];
                }
            }
            uint32_t hi[NR][2], lo[NR][2];      // P^T: keys 0 .. 7, 8 .. 15
#pragma unroll
            for (int y = 0; y < NR; ++y) {
                float mc[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) mc[x] = m[y][x] == -INFINITY ? 0.f : max_nan(m[y][x] * c, kLowest);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const float p0 = ex2(fmaf(sc[y][2 * t], c, -mc[0])), p1 = ex2(fmaf(sc[y][2 * t + 1], c, -mc[1]));
                    l[y][0] += p0;
                    l[y][1] += p1;
                    // hi cut, not rounded, and lo at least 2^-20 of the weight: both of one sign, neither 0, or their sum with an infinite value were NaN
                    const uint32_t h = __byte_perm(__float_as_uint(p0), __float_as_uint(p1), 0x7632);
                    hi[y][t] = turned(h);
                    lo[y][t] = turned(pack_bf16(fmaxf(p0 - __uint_as_float(h << 16), p0 * 0x1p-20f), fmaxf(p1 - __uint_as_float(h & 0xffff0000u), p1 * 0x1p-20f)));
                }
            }
#pragma unroll
            for (int t = 0; t < kSteps; ++t) {
                uint32_t vf[4];
                ldm4t(vf, sv + (t >> 2) * L::kHalf + sw128_off((mi >> 1) * 8 + mr, 2 * (t & 3) + (mi & 1)));
#pragma unroll
                for (int y = 0; y < NR; ++y) {
                    mma(acc[y][t], vf, hi[y][0], hi[y][1]);
                    mma(acc[y][t], vf, lo[y][0], lo[y][1]);
                }
            }
        }
        const bool ends = w.tile + 1 == w.s.t1;
        Walk then = w;
        then.next(b, Hk, window);
        if (ends || i + 1 == tiles) {
            // ------------------------------------------------------------------ the warps' sums become one
            fresh = true;
            // through the ring's places of this tile, which are free until the next but one; [row][value], pieces of eight values
            // exchanged so that the lanes' rows lie in different banks
            static_assert(L::kStage >= kRows * DP * 4, "a warp's sums fit a place of the ring");
            const int place = i % kStages * L::kStage;
            float* mine = reinterpret_cast<float*>(ring + place);
#pragma unroll
            for (int y = 0; y < NR; ++y)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int r = 8 * y + 2 * c4 + x;
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) l[y][x] += __shfl_xor_sync(0xffffffffu, l[y][x], o);
                    if (r8 == 0) row_ml[warp * kRows + r] = make_float2(m[y][x], l[y][x]);
#pragma unroll
                    for (int t = 0; t < kSteps; ++t) {
                        mine[r * DP + ((16 * t + r8) ^ (c4 << 3))] = acc[y][t][x];
                        mine[r * DP + ((16 * t + r8 + 8) ^ (c4 << 3))] = acc[y][t][x + 2];
                    }
                }
            __syncthreads();
            const bool begins = unit_begin == w.s.t0, whole = begins && ends;
            // a stretch's part: place 0 goes on from the block before, place 1 begins here
            const size_t part = ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * kRows;
#pragma unroll 1
            for (int e = tid; e < rows * (D / 4); e += kThreads) {
                const int r = e / (D / 4), d = 4 * (e - r * (D / 4));
                float2 ml[kWarps];
                float M = -INFINITY, sum = 0.f;
                f2 o0 = f2_all(0.f), o1 = f2_all(0.f);
#pragma unroll
                for (int k = 0; k < kWarps; ++k) {
                    ml[k] = row_ml[k * kRows + r];
                    M = max_nan(M, ml[k].x);
                }
#pragma unroll
                for (int k = 0; k < kWarps; ++k) {
                    if (ml[k].x == -INFINITY) continue;      // its sums are 0
                    const float f = ex2((ml[k].x - M) * c);
                    sum = fmaf(ml[k].y, f, sum);
                    const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm + k * kStages * L::kStage + place) + r * DP + (d ^ (((r >> 1) & 3) << 3)));
                    o0 = f2_fma(f2_make(x.x, x.y), f2_all(f), o0);
                    o1 = f2_fma(f2_make(x.z, x.w), f2_all(f), o1);
                }
                float2 oa = f2_get(o0), ob = f2_get(o1);
                float o[4] = {oa.x, oa.y, ob.x, ob.y};
                if (M == kLowest) sum = 0.f;      // nothing but -inf: 0 / 0
                if (flags[1 + q_buffer]) {
                    const int to = w.s.base + r / g, from = first_key(to, window);
#pragma unroll 1
                    for (int key = max(from, unit_begin * kTile); key <= min(to, (w.tile + 1) * kTile - 1); ++key) {
                        if (key >= all_lo && key < all_hi) continue;
                        const int pg = b.page(w.n, key / b.page_size);
                        if (pg < 0) continue;
                        const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.c.v) + pg * a.c.strides.v_page + (key % b.page_size) * a.c.strides.v_row +
                                                 w.hk * a.c.strides.v_head + d;
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float val = __bfloat162float(v[x]);
                            if (!isfinite(val)) o[x] += val;
                        }
                    }
                }
                if (!whole) {
                    if (d == 0) a.part_ml[part + r] = make_float2(M == -INFINITY ? M : max_nan(M * c, kLowest), sum);
                    *reinterpret_cast<float4*>(a.part_o + (part + r) * D + d) = make_float4(o[0], o[1], o[2], o[3]);
                    continue;
                }
                const size_t out = (size_t)(w.s.first + r / g) * Hq + w.hk * g + r % g;
                const float inv = M == -INFINITY ? 0.f : 1.f / sum;
                if (d == 0 && a.c.lse != nullptr) a.c.lse[out] = M == -INFINITY ? -INFINITY : (M * c + log2f(sum)) * kLn2;
                *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.c.o) + out * D + d) = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
            }
            q_buffer ^= 1;
            if (tid == 0) flags[1 + q_buffer] = 0;
            if (i + 1 < tiles) put_q(q_buffer);
            fence_async_smem();
            __syncthreads();
        }
        w = then;
    }
    if (flags[0])      // no copy may be in flight when the block ends
        for (int s = 0; s < kStages; ++s) mbar_poll(bar + s, (phases >> s) & 1u, kSpinLimit / 8);
}

// Joins the parts of a sequence's kv head that more than one stretch has worked on.  Block i looks at the place where stretch i + 1
// begins; the first such place inside a sequence takes all its parts.  Four values a thread; with few rows several threads share the
// parts of one place and add up through shared memory.
constexpr int kJoinThreads = 512, kMaxBlocks = 148 * kPerSm;
template <int NR>
__global__ void __launch_bounds__(kJoinThreads) attn_decode_join_kernel(const __grid_constant__ Args a) {
    constexpr int kRows = 8 * NR;
    __shared__ Start start;
    __shared__ int sums[kJoinThreads / 32];
    __shared__ float weight[kMaxBlocks * kRows], row_l[kRows], row_m[kRows];
    __shared__ float4 acc[kJoinThreads];
    const Batch& b = a.c.batch;
    const int g = a.c.heads.group, D = a.c.heads.dim, Hk = a.c.heads.kv_heads, Hq = a.c.heads.q_heads, window = a.c.window, id = blockIdx.x + 1;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Cut cut = find_start<kJoinThreads, false>(b, Hk, window, a.blocks, id, &start, sums);
    // No block ends before the stretches have: whoever is launched behind this kernel takes that for the end of both.
    if (id >= cut.used) {
        dependency_wait();
        return;
    }
    const Seq s = start.s;
    const int unit = cut.begin(id) - (start.tile - s.t0), unit_end = unit + (s.t1 - s.t0);      // of the list
    if (unit == cut.begin(id) || cut.begin(id - 1) > unit) {
        dependency_wait();
        return;
    }
    int parts = 1;      // stretches id - 1 .. id - 1 + parts
    while (id + parts < cut.used && cut.begin(id + parts) < unit_end) ++parts;
    const int rows = min(s.count * g, kRows);
    auto place = [&](int k, int r) { return ((size_t)(id - 1 + k) * 2 + (k == 0 ? 1 : 0)) * kRows + r; };
    dependency_wait();
    for (int r = warp; r < rows; r += kJoinThreads / 32) {      // a warp a row: 2^(m_k - m) of each part
        float m = -INFINITY, l = 0.f;
        for (int k = lane; k <= parts; k += 32) m = max_nan(m, ld_after_f32(&a.part_ml[place(k, r)].x));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        for (int k = lane; k <= parts; k += 32) {
            const uint2 x = ld_after8(a.part_ml + place(k, r));
            const float f = __uint_as_float(x.x) == -INFINITY ? 0.f : ex2(__uint_as_float(x.x) - m);
            l = fmaf(__uint_as_float(x.y), f, l);
            weight[k * kRows + r] = f;
        }
        l = warp_sum(l);
        if (lane == 0) {
            row_m[r] = m;
            row_l[r] = l;
        }
    }
    __syncthreads();
    const int items = rows * (D / 4), share = max(kJoinThreads / items, 1), at = tid % min(items, kJoinThreads), of = tid / min(items, kJoinThreads);
    if (of < share) {
        const int r = at / (D / 4), d = 4 * (at - r * (D / 4));
        float o[4] = {};
#pragma unroll 8
        for (int k = of; k <= parts; k += share) {
            const uint4 v = ld_after16(a.part_o + place(k, r) * D + d);
            const float f = weight[k * kRows + r];
            o[0] = fmaf(__uint_as_float(v.x), f, o[0]);
            o[1] = fmaf(__uint_as_float(v.y), f, o[1]);
            o[2] = fmaf(__uint_as_float(v.z), f, o[2]);
            o[3] = fmaf(__uint_as_float(v.w), f, o[3]);
        }
        acc[tid] = make_float4(o[0], o[1], o[2], o[3]);
    }
    __syncthreads();
    if (of != 0) return;
    {
        const int r = at / (D / 4), d = 4 * (at - r * (D / 4));
        float4 o = acc[at];
        for (int k = 1; k < share; ++k) {
            const float4 x = acc[k * items + at];
            o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
        }
        const size_t out = (size_t)(s.first + r / g) * Hq + start.hk * g + r % g;
        const float m = row_m[r], l = row_l[r], inv = m == -INFINITY ? 0.f : 1.f / l;
        if (d == 0 && a.c.lse != nullptr) a.c.lse[out] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * kLn2;
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.c.o) + out * D + d) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
    }
}

template <int DP, int NR>
int launch(const CUtensorMap& mK, const CUtensorMap& mV, const Args& a, cudaStream_t st) {
    constexpr int kBytes = Layout<DP, NR>::kBytes;
    if (int rc = set_smem_limit(attn_decode_kernel<DP, NR>, kBytes)) return rc;
    KDA_LAUNCH("attn_decode_kernel", st, attn_decode_kernel<DP, NR><<<a.blocks, kThreads, kBytes, st>>>(mK, mV, a));
    if (int rc = launch_status()) return rc;
    if (a.blocks == 1 || a.whole) return KDA_OK;
    cudaError_t e = cudaSuccess;
    KDA_LAUNCH("attn_decode_join_kernel", st, e = launch_early(attn_decode_join_kernel<NR>, dim3(a.blocks - 1), kJoinThreads, 0, st, true, 1, a));
    return e == cudaSuccess ? launch_status() : KDA_ERR_CUDA;
}

bool keeps_whole(int n_seq, int kv_heads, long long reach) {
    return reach <= ((long long)n_seq * kv_heads >= 148 ? kWholeTilesOfMany : kWholeTiles) * kTile;
}
// Stretches: as many as the machine holds, or as the longest batch that fits the table could use.
int stretches(int n_seq, int kv_heads, long long reach) {
    const long long tiles = ((reach + kTile - 1) / kTile + 1) * n_seq * kv_heads, n = keeps_whole(n_seq, kv_heads, reach) ? tiles : tiles / kMinTiles;
    return (int)(n < 1 ? 1 : n < kMaxBlocks ? n : kMaxBlocks);
}
long long reach_of(int table_width, int page_size, int window, int max_q) {
    long long reach = (long long)table_width * page_size;
    if (window > 0 && reach > (long long)window + max_q) reach = (long long)window + max_q;
    return reach;
}

}  // namespace

bool decode_takes(const Call& c) {
    const long long tiles = (long long)c.batch.n_seq * c.heads.kv_heads * ((long long)c.batch.table_width * c.batch.page_size / kTile + 2);
    return c.max_q_len > 0 && (long long)c.max_q_len * c.heads.group <= kMaxRows && tiles < 1ll << 31 && tc_takes(c);
}

size_t decode_workspace(int n_seq, int kv_heads, int table_width, int page_size, int window, int max_q, int dim) {
    const size_t rows = (size_t)stretches(n_seq, kv_heads, reach_of(table_width, page_size, window, max_q)) * 2 * kMaxRows;
    return align_up(rows * sizeof(float2), 256) + rows * dim * sizeof(float);
}

int decode(const Call& c, cudaStream_t st) {
    Args a;
    a.c = c;
    a.blocks = stretches(c.batch.n_seq, c.heads.kv_heads, reach_of(c.batch.table_width, c.batch.page_size, c.window, c.max_q_len));
    a.box_rows = c.batch.page_size < 16 ? c.batch.page_size : 16;
    a.whole = keeps_whole(c.batch.n_seq, c.heads.kv_heads, reach_of(c.batch.table_width, c.batch.page_size, c.window, c.max_q_len));
    a.part_ml = static_cast<float2*>(c.workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(c.workspace) + align_up((size_t)a.blocks * 2 * kMaxRows * sizeof(float2), 256));
    CUtensorMap mK, mV;
    const Strides& s = c.strides;
    int rc = make_map_paged(&mK, c.k, c.heads.dim, c.batch.page_size, c.heads.kv_heads, c.batch.n_pages, s.k_row, s.k_head, s.k_page, a.box_rows);
    if (!rc) rc = make_map_paged(&mV, c.v, c.heads.dim, c.batch.page_size, c.heads.kv_heads, c.batch.n_pages, s.v_row, s.v_head, s.v_page, a.box_rows);
    if (rc) return rc;
    const bool few = c.max_q_len * c.heads.group <= 8;
    if (c.heads.dim <= 64) return few ? launch<64, 1>(mK, mV, a, st) : launch<64, 2>(mK, mV, a, st);
    return few ? launch<128, 1>(mK, mV, a, st) : launch<128, 2>(mK, mV, a, st);
}

}  // namespace attn
}  // namespace kda
