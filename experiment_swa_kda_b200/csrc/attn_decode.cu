// Attention over a paged cache for few rows a sequence (bf16, heads up to 128 wide, at most 16 rows: new tokens x query heads of
// one kv head): the token step of serving.
//
//   o_i = sum_j 2^(c s_ij - c m_i) v_j / sum_j 2^(c s_ij - c m_i),   s = q k^T,  c = scale / ln 2
//
// Bound by the cache's bytes: a key costs 4 D bytes and at most 64 D operations.  All that counts is that every SM has its share of the
// keys and enough copies in flight.
//
// - The tiles (64 keys of one sequence and kv head) of the whole batch are one list, sequence after sequence, and each block
//   takes an equal stretch of it, whatever the sequences' lengths are.  The list is known on the device alone: every block adds up the
//   lengths itself.  Where a stretch ends inside a sequence its part of the softmax goes to the workspace, and
//   attn_decode_join_kernel puts the parts together.
// - A warp takes 16 keys of a tile through a ring of its own (K and V by TMA, 128-byte swizzle), so that warps meet only where a
//   sequence or the stretch ends.  The ring runs ahead across those places.
// - Products are mma.sync m16n8k16: 16 rows are its height, and at 23 bytes a cycle and SM its rate is not felt.  The weights go as
//   two bf16 terms, p = hi + lo, which costs products that nothing waits for and leaves the output with the error of its own rounding.

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

constexpr int kRows = 16, kTile = 64, kWarps = 4, kThreads = 128, kStages = 3;
constexpr int kPerSm = 2;             // blocks an SM: 98 KB each
constexpr int kMinTiles = 2;          // a stretch has at least these many tiles
constexpr float kLazy = 8.f;          // as in the kernel for long chunks: sums are rescaled when a maximum grew by 2^8
constexpr int kStatusWait = 121;

template <int DP>
struct Layout {
    static constexpr int kHalf = 16 * 128;                            // 16 keys of 64 values
    static constexpr int kStage = 2 * (DP / 64) * kHalf;              // K and V of 16 keys
    static constexpr int kBars = kWarps * kStages * kStage;
    static constexpr int kBytes = kBars + 1024 + 1024;
};

struct Args {
    Call c;
    int blocks, box_rows, q4;
    float* part_o;        // [blocks][2][16][D]
    float2* part_ml;      // [blocks][2][16]
};

// One sequence's tiles and rows.
struct Seq {
    int first, count, base, lo, hi, t0, t1;
};
__device__ __forceinline__ Seq seq_at(const Batch& b, int n, int window) {
    Seq s;
    b.span(n, s.first, s.count);
    const int len = b.kv_len(n);
    s.base = len - s.count;
    s.hi = s.count > 0 ? len : 0;
    s.lo = window > 0 ? min(max(s.base - window + 1, 0), s.hi) : 0;
    s.t0 = s.lo / kTile;
    s.t1 = (s.hi + kTile - 1) / kTile;
    return s;
}

struct Start {
    long long total, begin, end;      // tiles of the batch; this stretch
    int blocks;                       // stretches in use
    int n, hk, tile;                  // where it begins
};
// The stretch of block `id`; called by all threads of a block of kThreads.
__device__ __forceinline__ void find_start(const Batch& b, int kv_heads, int window, int blocks, int id, Start* shared, long long* sums) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int each = (b.n_seq + kThreads - 1) / kThreads, n0 = min(tid * each, b.n_seq), n1 = min(n0 + each, b.n_seq);
    long long mine = 0;
    for (int n = n0; n < n1; ++n) {
        const Seq s = seq_at(b, n, window);
        mine += (long long)(s.t1 - s.t0) * kv_heads;
    }
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) upto += sums[w];
        total += sums[w];
    }
    const long long used = min((long long)blocks, max(total / kMinTiles, 1ll));
    const long long begin = id < used ? total * id / used : total, end = id < used ? total * (id + 1) / used : total;
    long long at = upto - mine;
    if (begin < end && begin >= at && begin < upto) {
        for (int n = n0; n < n1; ++n) {
            const Seq s = seq_at(b, n, window);
            const long long here = (long long)(s.t1 - s.t0) * kv_heads;
            if (begin < at + here) {
                const int rest = (int)(begin - at), nt = s.t1 - s.t0;
                shared->n = n;
                shared->hk = rest / nt;
                shared->tile = s.t0 + rest % nt;
                break;
            }
            at += here;
        }
    }
    if (tid == 0) {
        shared->total = total;
        shared->begin = begin;
        shared->end = end;
        shared->blocks = (int)used;
    }
    __syncthreads();
}

// A place in the list.
struct Walk {
    Seq s;
    int n, hk, tile;
    __device__ __forceinline__ void set(const Batch& b, const Start& at, int window) {
        n = at.n;
        hk = at.hk;
        tile = at.tile;
        s = seq_at(b, n, window);
    }
    __device__ __forceinline__ void next(const Batch& b, int kv_heads, int window) {
        if (++tile < s.t1) return;
        if (++hk == kv_heads) {
            hk = 0;
            do {
                if (++n >= b.n_seq) return;      // behind the end of the list: not used
                s = seq_at(b, n, window);
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

template <int DP>
__global__ void __launch_bounds__(kThreads, kPerSm) attn_decode_kernel(const __grid_constant__ CUtensorMap mK, const __grid_constant__ CUtensorMap mV,
                                                                       const __grid_constant__ Args a) {
    using L = Layout<DP>;
    constexpr int kHalves = DP / 64, kNt = DP / 8;
    extern __shared__ uint8_t raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::kBars);
    Start& start = *reinterpret_cast<Start*>(bars + kWarps * kStages);
    long long* sums = reinterpret_cast<long long*>(&start + 1);
    volatile int* flags = reinterpret_cast<volatile int*>(sums + kWarps);      // [0] an expired wait, [1] values that are not finite
    float2* row_ml = reinterpret_cast<float2*>(sums + kWarps + 2);             // [warps][16]
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, c4 = lane & 3, r8 = lane >> 2;
    const Batch& b = a.c.batch;
    const int g = a.c.heads.group, D = a.c.heads.dim, Hk = a.c.heads.kv_heads, Hq = a.c.heads.q_heads, window = a.c.window;

    uint64_t* bar = bars + warp * kStages;
    dependents_go();
    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(bar + s, 1);
        mbar_fence_init();
    }
    if (tid == 0) flags[0] = flags[1] = 0;
    find_start(b, Hk, window, a.blocks, blockIdx.x, &start, sums);

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
    const long long tiles = start.end - start.begin;
    if (tiles <= 0) return;

    uint8_t* ring = sm + warp * kStages * L::kStage;
    Walk ahead, w;
    ahead.set(b, start, window);
    w.set(b, start, window);
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
    auto load = [&](long long i) {      // the tile `ahead` is at, into the ring's place i; then on to the next one
        const int s = (int)(i % kStages);
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
    look();
    long long issued = 0;
    for (; issued < kStages - 1 && issued < tiles; ++issued) load(issued);

    const float c = a.c.scale * 1.4426950408889634f, lazy = kLazy / c;
    uint32_t q[kHalves * 4][4];
    float acc[kNt][4], m[2], l[2];
    int last[2], first[2], all_lo = 0, all_hi = 0, unit_begin = 0;
    bool fresh = true;
    uint32_t phases = 0;      // of the ring's barriers: a tile out of this warp's reach leaves its place as it is
    const int mi = lane >> 3, mr = lane & 7;

    for (long long i = 0; i < tiles; ++i) {
        if (issued < tiles) {
            __syncwarp();
            load(issued++);
        }
        const int rows = w.s.count * g < kRows ? w.s.count * g : kRows;
        auto global_row = [&](int r) { return (size_t)(w.s.first + r / g) * Hq + w.hk * g + r % g; };
        if (fresh) {
            fresh = false;
            unit_begin = w.tile;
            all_lo = window > 0 ? max(w.s.base + (rows - 1) / g - window + 1, 0) : 0;
            all_hi = w.s.base + 1;
            const __nv_bfloat16* src[2];
            bool is[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int r = r8 + 8 * x;
                is[x] = r < rows;
                last[x] = is[x] ? w.s.base + r / g : -1;
                first[x] = window > 0 ? last[x] - window + 1 : 0;
                src[x] = static_cast<const __nv_bfloat16*>(a.c.q) + (w.s.first + r / g) * a.c.strides.q_token + (w.hk * g + r % g) * a.c.strides.q_head;
                m[x] = -INFINITY;
                l[x] = 0.f;
            }
#pragma unroll
            for (int k = 0; k < kHalves * 4; ++k)
#pragma unroll
                for (int x = 0; x < 4; ++x) {      // rows r8, r8 + 8; values 2 c4, 2 c4 + 8 of step k
                    const int d = 16 * k + 2 * c4 + 8 * (x >> 1);
                    uint32_t v = 0;
                    if (is[x & 1] && d < D) {
                        if (a.q4) {
                            v = __ldg(reinterpret_cast<const uint32_t*>(src[x & 1] + d));
                        } else {
                            const unsigned short* s = reinterpret_cast<const unsigned short*>(src[x & 1] + d);
                            v = s[0] | (uint32_t)s[1] << 16;
                        }
                    }
                    q[k][x] = v;
                }
#pragma unroll
            for (int t = 0; t < kNt; ++t)
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[t][x] = 0.f;
        }
        if (in_reach(w)) {
            const int s = (int)(i % kStages), k0 = w.tile * kTile + 16 * warp;
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
                        flags[1] = 1;
                    }
                }
                fence_async_smem();
                __syncwarp();
            }
            float s2[2][2][4] = {};      // scores of keys 0 .. 7, 8 .. 15; two chains each
#pragma unroll
            for (int k = 0; k < kHalves * 4; ++k) {
                uint32_t kf[4];
                ldm4(kf, sk + (k >> 2) * L::kHalf + sw128_off((mi >> 1) * 8 + mr, 2 * (k & 3) + (mi & 1)));
                mma(s2[k & 1][0], q[k], kf[0], kf[1]);
                mma(s2[k & 1][1], q[k], kf[2], kf[3]);
            }
            float sc[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int x = 0; x < 4; ++x) sc[t][x] = s2[0][t][x] + s2[1][t][x];
            float top[2] = {kLowest, kLowest};
            if (partial) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int key = k0 + 8 * t + 2 * c4 + (x & 1);
                        if (key < first[x >> 1] || key > last[x >> 1]) sc[t][x] = -INFINITY;
                    }
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    if (last[x] < k0 || first[x] >= k0 + 16) top[x] = -INFINITY;
            }
            bool grow = false;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                top[x] = max_nan(top[x], max_nan(max_nan(sc[0][2 * x], sc[0][2 * x + 1]), max_nan(sc[1][2 * x], sc[1][2 * x + 1])));
                top[x] = max_nan(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
                top[x] = max_nan(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
                grow |= !(top[x] <= m[x] + lazy) && !(top[x] == -INFINITY);
            }
            if (__any_sync(0xffffffffu, grow)) {
                float f[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float next = max_nan(m[x], top[x]);
                    f[x] = m[x] == -INFINITY ? 0.f : ex2((m[x] - next) * c);
                    m[x] = next;
                    l[x] *= f[x];
                }
#pragma unroll
                for (int t = 0; t < kNt; ++t)
#pragma unroll
                    for (int x = 0; x < 4; ++x) acc[t][x] *= f[x >> 1];
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float mc = m[x] == -INFINITY ? 0.f : max_nan(m[x] * c, kLowest);
                    const float p0 = ex2(fmaf(sc[t][2 * x], c, -mc)), p1 = ex2(fmaf(sc[t][2 * x + 1], c, -mc));
                    l[x] += p0 + p1;
                    const uint32_t h = pack_bf16(p0, p1);
                    hi[2 * t + x] = h;
                    lo[2 * t + x] = pack_bf16(p0 - __uint_as_float(h << 16), p1 - __uint_as_float(h & 0xffff0000u));
                }
#pragma unroll
            for (int t = 0; t < kNt / 2; ++t) {
                uint32_t vf[4];
                ldm4t(vf, sv + (t >> 2) * L::kHalf + sw128_off((mi & 1) * 8 + mr, 2 * (t & 3) + (mi >> 1)));
                mma(acc[2 * t], hi, vf[0], vf[1]);
                mma(acc[2 * t + 1], hi, vf[2], vf[3]);
                mma(acc[2 * t], lo, vf[0], vf[1]);
                mma(acc[2 * t + 1], lo, vf[2], vf[3]);
            }
        }
        const bool ends = w.tile + 1 == w.s.t1;
        if (ends || i + 1 == tiles) {
            // ------------------------------------------------------------------ the warps' sums become one
            fresh = true;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
                l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
                if (c4 == 0) row_ml[warp * kRows + r8 + 8 * x] = make_float2(m[x], l[x]);
            }
            __syncthreads();
            float M[2], Lsum[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float2 o[kWarps];
                M[x] = -INFINITY;
#pragma unroll
                for (int k = 0; k < kWarps; ++k) {
                    o[k] = row_ml[k * kRows + r8 + 8 * x];
                    M[x] = max_nan(M[x], o[k].x);
                }
                Lsum[x] = 0.f;
#pragma unroll
                for (int k = 0; k < kWarps; ++k) Lsum[x] += o[k].x == -INFINITY ? 0.f : o[k].y * ex2((o[k].x - M[x]) * c);
                const float f = m[x] == -INFINITY ? 0.f : ex2((m[x] - M[x]) * c);
#pragma unroll
                for (int t = 0; t < kNt; ++t) {
                    acc[t][2 * x] *= f;
                    acc[t][2 * x + 1] *= f;
                }
            }
            // through the ring's places of this tile, which are free until the next but one
            static_assert(L::kStage == kRows * DP * 4, "a warp's sums fill a place of the ring");
#pragma unroll
            for (int half = kWarps / 2; half > 0; half >>= 1) {
                if (warp >= half && warp < 2 * half) {
                    float4* join = reinterpret_cast<float4*>(ring + (int)(i % kStages) * L::kStage);
#pragma unroll
                    for (int t = 0; t < kNt; ++t) join[t * 32 + lane] = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
                }
                __syncthreads();
                if (warp < half) {
                    const float4* join = reinterpret_cast<const float4*>(sm + ((warp + half) * kStages + (int)(i % kStages)) * L::kStage);
#pragma unroll
                    for (int t = 0; t < kNt; ++t) {
                        const float4 o = join[t * 32 + lane];
                        acc[t][0] += o.x; acc[t][1] += o.y; acc[t][2] += o.z; acc[t][3] += o.w;
                    }
                }
            }
            fence_async_smem();
            if (warp == 0) {
                const bool begins = unit_begin == w.s.t0, whole = begins && ends;
                if (flags[1]) {
                    for (int key = max(w.s.lo, unit_begin * kTile); key < min(w.s.hi, (w.tile + 1) * kTile); ++key) {
                        if (key >= all_lo && key < all_hi) continue;
                        const int pg = b.page(w.n, key / b.page_size);
                        if (pg < 0) continue;
                        const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.c.v) + pg * a.c.strides.v_page + (key % b.page_size) * a.c.strides.v_row +
                                                 w.hk * a.c.strides.v_head;
#pragma unroll
                        for (int t = 0; t < kNt; ++t)
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const int d = 8 * t + 2 * c4 + (x & 1);
                                if (d >= D || key < first[x >> 1] || key > last[x >> 1]) continue;
                                const float val = __bfloat162float(v[d]);
                                if (!isfinite(val)) acc[t][x] += val;
                            }
                    }
                    __syncwarp();
                    if (lane == 0) flags[1] = 0;
                }
                // a stretch's part: place 0 goes on from the block before, place 1 begins here
                const size_t part = ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * kRows;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int r = r8 + 8 * x;
                    if (r >= rows) continue;
                    if (M[x] == kLowest) Lsum[x] = 0.f;      // nothing but -inf: 0 / 0
                    if (!whole) {
                        if (c4 == 0) a.part_ml[part + r] = make_float2(M[x] * c, Lsum[x]);
#pragma unroll
                        for (int t = 0; t < kNt; ++t)
                            if (8 * t < D) *reinterpret_cast<float2*>(a.part_o + (part + r) * D + 8 * t + 2 * c4) = make_float2(acc[t][2 * x], acc[t][2 * x + 1]);
                        continue;
                    }
                    const size_t out = global_row(r);
                    const float inv = M[x] == -INFINITY ? 0.f : 1.f / Lsum[x];
                    if (c4 == 0 && a.c.lse != nullptr) a.c.lse[out] = M[x] == -INFINITY ? -INFINITY : (M[x] * c + log2f(Lsum[x])) * kLn2;
#pragma unroll
                    for (int t = 0; t < kNt; ++t)
                        if (8 * t < D)
                            *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.c.o) + out * D + 8 * t + 2 * c4) =
                                pack_bf16(acc[t][2 * x] * inv, acc[t][2 * x + 1] * inv);
                }
            }
            __syncthreads();
        }
        w.next(b, Hk, window);
    }
    if (flags[0])      // no copy may be in flight when the block ends
        for (int s = 0; s < kStages; ++s) mbar_poll(bar + s, (phases >> s) & 1u, kSpinLimit / 8);
}

// Joins the parts of a sequence's kv head that more than one stretch has worked on.  Block i looks at the place where stretch i + 1
// begins; the first such place inside a sequence takes all its parts.
__global__ void __launch_bounds__(kThreads) attn_decode_join_kernel(const __grid_constant__ Args a) {
    __shared__ Start start;
    __shared__ long long sums[kWarps];
    const Batch& b = a.c.batch;
    const int g = a.c.heads.group, D = a.c.heads.dim, Hk = a.c.heads.kv_heads, Hq = a.c.heads.q_heads, window = a.c.window, id = blockIdx.x + 1;
    find_start(b, Hk, window, a.blocks, id, &start, sums);
    if (start.begin >= start.end) return;
    const Seq s = seq_at(b, start.n, window);
    const long long unit = start.begin - (start.tile - s.t0), unit_end = unit + (s.t1 - s.t0);      // of the list
    if (unit == start.begin || start.total * (id - 1) / start.blocks > unit) return;
    int parts = 1;      // stretches id - 1 .. id - 1 + parts
    while (id + parts < start.blocks && start.total * (id + parts) / start.blocks < unit_end) ++parts;
    dependency_wait();
    const int rows = min(s.count * g, kRows);
    for (int e = threadIdx.x; e < rows * (D / 4); e += kThreads) {
        const int r = e / (D / 4), d = 4 * (e - r * (D / 4));
        auto place = [&](int k) { return ((size_t)(id - 1 + k) * 2 + (k == 0 ? 1 : 0)) * kRows + r; };
        auto ml = [&](int k) {
            const uint2 x = ld_after8(a.part_ml + place(k));
            return make_float2(__uint_as_float(x.x), __uint_as_float(x.y));
        };
        float m = -INFINITY, l = 0.f, o[4] = {};
#pragma unroll 4
        for (int k = 0; k <= parts; ++k) m = max_nan(m, ml(k).x);
#pragma unroll 4
        for (int k = 0; k <= parts; ++k) {
            const float2 x = ml(k);
            const uint4 v = ld_after16(a.part_o + place(k) * D + d);
            const float f = x.x == -INFINITY ? 0.f : ex2(x.x - m);
            l = fmaf(x.y, f, l);
            if (x.x == -INFINITY) continue;      // its sums are 0
            o[0] = fmaf(__uint_as_float(v.x), f, o[0]);
            o[1] = fmaf(__uint_as_float(v.y), f, o[1]);
            o[2] = fmaf(__uint_as_float(v.z), f, o[2]);
            o[3] = fmaf(__uint_as_float(v.w), f, o[3]);
        }
        const size_t out = (size_t)(s.first + r / g) * Hq + start.hk * g + r % g;
        const float inv = m == -INFINITY ? 0.f : 1.f / l;
        if (d == 0 && a.c.lse != nullptr) a.c.lse[out] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * kLn2;
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.c.o) + out * D + d) = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
    }
}

template <int DP>
int launch(const CUtensorMap& mK, const CUtensorMap& mV, const Args& a, cudaStream_t st) {
    if (int rc = set_smem_limit(attn_decode_kernel<DP>, Layout<DP>::kBytes)) return rc;
    KDA_LAUNCH("attn_decode_kernel", st, attn_decode_kernel<DP><<<a.blocks, kThreads, Layout<DP>::kBytes, st>>>(mK, mV, a));
    if (int rc = launch_status()) return rc;
    if (a.blocks == 1) return KDA_OK;
    cudaError_t e = cudaSuccess;
    KDA_LAUNCH("attn_decode_join_kernel", st, e = launch_early(attn_decode_join_kernel, dim3(a.blocks - 1), kThreads, 0, st, true, 1, a));
    return e == cudaSuccess ? launch_status() : KDA_ERR_CUDA;
}

// Stretches: as many as the machine holds, or as the longest batch that fits the table could use.
int stretches(int n_seq, int kv_heads, long long reach) {
    const long long tiles = ((reach + kTile - 1) / kTile + 1) * n_seq * kv_heads, n = tiles / kMinTiles;
    return (int)(n < 1 ? 1 : n < 148 * kPerSm ? n : 148 * kPerSm);
}
long long reach_of(int table_width, int page_size, int window, int max_q) {
    long long reach = (long long)table_width * page_size;
    if (window > 0 && reach > (long long)window + max_q) reach = (long long)window + max_q;
    return reach;
}

}  // namespace

bool decode_takes(const Call& c) { return c.max_q_len > 0 && (long long)c.max_q_len * c.heads.group <= kRows && tc_takes(c); }

size_t decode_workspace(int n_seq, int kv_heads, int table_width, int page_size, int window, int max_q, int dim) {
    const size_t rows = (size_t)stretches(n_seq, kv_heads, reach_of(table_width, page_size, window, max_q)) * 2 * kRows;
    return align_up(rows * sizeof(float2), 256) + rows * dim * sizeof(float);
}

int decode(const Call& c, cudaStream_t st) {
    Args a;
    a.c = c;
    a.blocks = stretches(c.batch.n_seq, c.heads.kv_heads, reach_of(c.batch.table_width, c.batch.page_size, c.window, c.max_q_len));
    a.box_rows = c.batch.page_size < 16 ? c.batch.page_size : 16;
    a.q4 = reinterpret_cast<uintptr_t>(c.q) % 4 == 0 && c.strides.q_token % 2 == 0 && c.strides.q_head % 2 == 0;
    a.part_ml = static_cast<float2*>(c.workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(c.workspace) + align_up((size_t)a.blocks * 2 * kRows * sizeof(float2), 256));
    CUtensorMap mK, mV;
    const Strides& s = c.strides;
    int rc = make_map_paged(&mK, c.k, c.heads.dim, c.batch.page_size, c.heads.kv_heads, c.batch.n_pages, s.k_row, s.k_head, s.k_page, a.box_rows);
    if (!rc) rc = make_map_paged(&mV, c.v, c.heads.dim, c.batch.page_size, c.heads.kv_heads, c.batch.n_pages, s.v_row, s.v_head, s.v_page, a.box_rows);
    if (rc) return rc;
    return c.heads.dim <= 64 ? launch<64>(mK, mV, a, st) : launch<128>(mK, mV, a, st);
}

}  // namespace attn
}  // namespace kda
