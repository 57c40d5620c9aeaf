// Attention over a paged cache on the tensor cores (bf16, heads up to 128 wide).
//
//   S = Q K^T,  p_ij = 2^(c s_ij - c m_i),  o_i = sum_j p_ij v_j / sum_j p_ij,   c = scale / ln 2
//
// in one pass over the keys.  A block has 256 rows - token-major, the query heads of one kv head side by side, so that every
// key tile serves all of them and a chunk of few tokens still fills the tile - as two tiles of 128, and walks through the keys
// 128 at a time.  Per key tile and row tile the tensor pipe does S (M128 N128 K = head) and O += P V (M128 N = head K128); the
// two row tiles take turns: while one's scores are turned into weights by its four warps, the other's products run.  S and O
// live in tensor memory, P (bf16) takes S's place there and is the A operand of its product, so nothing but K and V goes through
// shared memory.  A thread owns a row: maximum and sum need no exchange.  (Two threads a row, with twice the warps to cover each other's
// waits, took as long: what the exchange of "a maximum has grown" costs is what they gain.)
//
// O is rescaled only when a row's maximum has grown by more than 2^kLazy since the last time (the weights are then at most
// 2^kLazy, which costs bf16 nothing: its rounding is relative); after a few tiles that no longer happens.
// P is rounded to bf16 because the product takes one type and V is bf16; sums and statistics are float32.
//
// 8,191 tokens of 16 heads on 4, calls one behind the other: 268 to 271 us (1,020 TFLOP/s, 0.74 of the measured sustained rate of a library
// product, 0.62 of its burst rate), under the power cap; 235 in runs too short for it.  The tensor pipe is busy for 55 % of them.  A pair of row tiles
// takes 2,900 to 3,350 cycles a key tile, of which its products need 2,048 and the special function unit 1,536: a row tile's softmax,
// 2,000 cycles of two warps a scheduler, and the products behind it, 1,300, follow one another, and the other tile covers most of
// that, not all.  Measured and left out (short runs, where this took 232 to 241): the exponentials of the two tiles in turns (270 us), maxima only
// where sums ask for them (261), two threads a row (265), P in columns of its own for 64-wide heads (196 -> 248).  A block costs 12,000 to 16,000 cycles besides its tiles - its rows,
// the first keys, the output -, which shows in windows: four times 2,048 tokens with windows of 1,024 take 107 us, 0.37 of the burst rate.
//
// K and V come page by page by TMA into one ring (K 0, V 0, K 1, V 1, ...).  A tile that some row sees only in part is masked
// in registers, to weights of exactly 0; in its V tile the keys that no row sees are blanked, since 0 times what lies in an unused slot may be NaN, and
// so are values that are not finite at keys only some rows see: these are added by the rows that see them at the end.

#include "attn.cuh"
#include "tc_common.cuh"

namespace kda {
namespace tc {
int make_map_paged(CUtensorMap* m, const void* ptr, uint64_t dim, uint64_t rows, uint64_t heads, uint64_t pages, int64_t row_ld, int64_t head_ld, int64_t page_ld,
                   uint32_t box_rows);
int make_map_packed(CUtensorMap* m, const void* ptr, uint64_t dim, uint64_t heads, uint64_t tokens, int64_t head_ld, int64_t token_ld, uint32_t box_heads,
                    uint32_t box_tokens);
}
namespace attn {
namespace {

using namespace tc;

constexpr int kKeys = 128, kRows = 256;
constexpr int kSoftmaxWarps = 8, kMmaWarp = 8, kLoadWarp = 9, kFixWarp = 10, kThreads = 384;
// Registers a thread: a row of scores is 128, and the loop over them needs room to overlap its steps.  384 x 168 in all.
#define KDA_SOFTMAX_REGS "216"
#define KDA_OTHER_REGS "72"
constexpr int kPolyOf = 4;            // one pair of weights of so many is made by ex2_pair (8,191 tokens: none 252 us, 1/4 246, 1/2 263; 64-wide heads 229, 206, 231)
constexpr int kMinPart = 8;           // key tiles of a part at least
constexpr float kLazy = 8.f;
constexpr int kStatusWait = 120;      // device status of an expired wait

template <int DP>
struct Layout {
    static constexpr int kTile = DP / 64 * 16384;             // 128 rows of Q, K or V: one or two blocks of 64 columns
    static constexpr int kStages = DP == 128 ? 5 : 10;
    static constexpr int kRing = 2 * kTile;
    static constexpr int kBars = kRing + kStages * kTile;
    static constexpr int kBytes = kBars + 512 + 1024;         // barriers; slack to align the tiles
};

struct Args {
    Call c;
    Tiles tiles;
    int slots, splits, box_rows, q_boxes;
    // Where rows are cut into parts: how many each block's have, [slots][kv heads]; of each part, [splits][slots][kv heads], a row's maximum
    // and sum [256] and its sums [2 row tiles][2 halves of the columns][128][DP / 2], pieces of 16 bytes exchanged within a row as
    // part_off() says.
    int* parts;
    float2* part_ml;
    float* part_o;
};
// byte offset of 16-byte piece c of row r in half a row tile's sums
template <int DP>
__device__ __forceinline__ int part_off(int r, int c) {
    return r * DP * 2 + ((c ^ (r & 7)) << 4);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// a maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// 2^x of a pair on the multiply-add pipes: x = n + f with |f| <= 1/2, 2^f by the polynomial of degree 4 with 2^0 = 1 whose largest relative
// error is least there (2.8e-6; degree 3 leaves 7.5e-5, which the sums of few weights show), n added to the exponent.  -127 and all below it, the -inf of a
// hidden key too, give f = 0 and n = -127: no bit is left, so a hidden key weighs nothing whatever its value is.  The special function unit gives 16
// values a cycle and SM, the tensor pipe wants 128 x 128 of them every 1,024 cycles, so part of them is made here.
__device__ __forceinline__ f2 ex2_pair(f2 x) {
    const float2 v = f2_get(x);
    x = f2_make(fmaxf(v.x, -127.f), fmaxf(v.y, -127.f));
    const f2 magic = f2_all(12582912.f);      // 1.5 x 2^23: the sum's low bits are n
    const f2 t = f2_add(x, magic), f = f2_add(x, f2_fma(t, f2_all(-1.f), magic));
    f2 p = f2_fma(f2_all(0.0095828531f), f, f2_all(0.0559064248f));
    p = f2_fma(p, f, f2_all(0.2402409864f));
    p = f2_fma(p, f, f2_all(0.6931241928f));
    p = f2_fma(p, f, f2_all(1.f));
    const float2 r = f2_get(p), n = f2_get(t);
    return f2_make(__uint_as_float(__float_as_uint(r.x) + (__float_as_uint(n.x) << 23)), __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(n.y) << 23)));
}
// The key tiles a row tile goes through, of those of its block.
struct Range {
    int begin, end;
};

template <int DP>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const __grid_constant__ CUtensorMap mK, const __grid_constant__ CUtensorMap mV,
                                                              const __grid_constant__ CUtensorMap mQ, const __grid_constant__ CUtensorMap mO,
                                                              const __grid_constant__ Args a) {
    using L = Layout<DP>;
    extern __shared__ uint8_t raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bar = reinterpret_cast<uint64_t*>(sm + L::kBars);
    uint64_t *bar_q = bar, *bar_s = bar + 1, *bar_p = bar + 3, *bar_o = bar + 7, *bar_end = bar + 9, *bar_full = bar + 10, *bar_free = bar_full + L::kStages,
             *bar_part = bar_free + L::kStages;
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(bar + 60);
    volatile int& abort_flag = *reinterpret_cast<volatile int*>(bar + 61);
    volatile int& odd_values = *reinterpret_cast<volatile int*>(bar + 62);

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const Batch& b = a.c.batch;
    const int g = a.c.heads.group, D = a.c.heads.dim, hk = blockIdx.y, z = blockIdx.z, window = a.c.window;
    // a sequence's last rows see the most keys: they start first
    const int slot = a.slots - 1 - (int)blockIdx.x;
    Unit u;
    const bool some = make_unit(b, a.tiles, slot, window, u);
    if (hk == 0 && z == 0 && tid == 0) {
        int n, tile;
        if (a.tiles.find(b, slot, n, tile)) check_batch(b, a.tiles, n, tile);
    }
    if (!some) return;

    // keys any row of the block sees: [u.lo, u.hi); keys all of them see: [all_lo, all_hi)
    const int first_pos = u.base + u.row0 / g, last_pos = u.base + (u.row0 + u.rows - 1) / g;
    const int all_lo = first_key(last_pos, window), all_hi = first_pos + 1;
    // Key tiles start at the first box in reach, not at multiples of their size: a window of 1,024 keys and 64 rows is 9 tiles, not 10.
    const int key0 = u.lo / a.box_rows * a.box_rows, nt = max((u.hi - key0 + kKeys - 1) / kKeys, 0);
    int t_begin = 0, t_end = nt;
    bool split = false;
    if (a.splits > 1) {
        // The shortest parts with which all blocks run side by side, looked for by one length a warp, twice; none where they would be
        // little shorter than the longest row tile's keys (a part costs some 5 tiles of its own, and the join).  The host sees to it
        // that a thread has a slot.
        constexpr int kTries = kThreads / 32;
        int *tiles_of = reinterpret_cast<int*>(sm), *blocks_of = tiles_of + kThreads;      // nothing else is there yet
        int tiles = 0;
        Unit v;
        if (tid < a.slots && make_unit(b, a.tiles, tid, window, v)) tiles = max((v.hi - v.lo / a.box_rows * a.box_rows + kKeys - 1) / kKeys, 1);
        tiles_of[tid] = tiles;
        __syncthreads();
        int longest = 0;
        for (int i = lane; i < a.slots; i += 32) longest = max(longest, tiles_of[i]);
        longest = __reduce_max_sync(0xffffffffu, longest);
        int lo = min(kMinPart, longest), hi = longest;      // hi is long enough, or nothing is
#pragma unroll
        for (int round = 0; round < 2; ++round) {
            const int step = (hi - lo) / kTries + 1, mine = min(lo + warp * step, hi);
            int sum = 0;
            for (int i = lane; i < a.slots; i += 32) sum += (tiles_of[i] + mine - 1) / mine;
            sum = __reduce_add_sync(0xffffffffu, sum);
            if (lane == 0) blocks_of[round * kTries + warp] = sum;
            __syncthreads();
            int first = 0;
            while (first < kTries - 1 && blocks_of[round * kTries + first] * a.c.heads.kv_heads > 148) ++first;
            hi = min(lo + first * step, hi);
            lo = first > 0 ? min(lo + (first - 1) * step + 1, hi) : hi;
        }
        const int part = 4 * hi > 3 * longest ? longest : hi, parts = min(max((nt + part - 1) / part, 1), a.splits);
        if (z >= parts) return;
        fence_async_smem();      // the list's place is written by copies next
        split = parts > 1;
        t_begin = nt * z / parts;
        t_end = nt * (z + 1) / parts;
        if (z == 0 && tid == 0) a.parts[slot * a.c.heads.kv_heads + hk] = parts;
    }
    auto range_of = [&](int t) {      // key tiles of row tile t
        const int r0 = u.row0 + 128 * t, r1 = min(r0 + 128, u.row0 + u.rows) - 1;
        if (r0 > r1) return Range{0, 0};
        const int hi = u.base + r1 / g + 1, lo = first_key(u.base + r0 / g, window);
        Range r{max(t_begin, (lo - key0) / kKeys), min(t_end, (max(hi - key0, 0) + kKeys - 1) / kKeys)};
        if (r.end < r.begin) r.end = r.begin;
        return r;
    };
    const Range range[2] = {range_of(0), range_of(1)};
    // the tiles some row sees only in part
    auto partial = [&](int j) { return key0 + j * kKeys < all_lo || key0 + (j + 1) * kKeys > all_hi; };

    if (warp == 0 && elect_one()) {
        mbar_init(bar_q, a.q_boxes ? 1 : kSoftmaxWarps);
        mbar_init(bar_end, 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(bar_s + t, 1);
            mbar_init(bar_p + 2 * t, 4);      // P of keys [0, 64) and [64, 128)
            mbar_init(bar_p + 2 * t + 1, 4);
            mbar_init(bar_o + t, 1);
        }
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(bar_full + s, 1);
            mbar_init(bar_free + s, 1);
            mbar_init(bar_part + s, 1);
        }
        mbar_fence_init();
        abort_flag = 0;
        odd_values = 0;
    }
    if (warp == kMmaWarp) tmem_alloc(&tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    constexpr uint32_t cS = 0, cO = 256;      // S (then P) of the two row tiles: 128 columns each; O: DP each
    auto wait = [&](uint64_t* w, uint32_t parity) {
        if (mbar_poll(w, parity, kSpinLimit)) return true;
        abort_flag = 1;
        b.tell(kStatusWait);
        return false;
    };
    // The same for a warp that goes on together: a limit that runs out in some lanes and not in others is every lane's, or those left would
    // wait in the warp's next collective for lanes that are gone.
    auto warp_wait = [&](uint64_t* w, uint32_t parity) { return __all_sync(0xffffffffu, wait(w, parity)) != 0; };
    // stage and phase of the ring's i-th tile
    auto stage = [](int i) { return i % L::kStages; };
    auto turn = [](int i) { return (uint32_t)(i / L::kStages) & 1u; };

    if (warp < kSoftmaxWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 " KDA_SOFTMAX_REGS ";");
        const int t = warp >> 2;
        // ------------------------------------------------------------------ Q into shared memory, where it does not come by TMA
        if (!a.q_boxes) {
            // DP / 8 lanes a row; all of a thread's copies are in flight together
            constexpr int kChunks = DP / 8, kStep = 128 / kChunks;      // rows a pass
            const int x = tid & 127, c = x % kChunks;
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.c.q) + 8 * c;
            int r = x / kChunks, pr = u.row0 + 128 * t + r, tok = pr / g, head = pr - tok * g;
#pragma unroll 1
            for (; r < 128; r += kStep) {
                const bool is = 128 * t + r < u.rows && 8 * c < D;
                const __nv_bfloat16* src = is ? q + (u.first + tok) * a.c.strides.q_token + (hk * g + head) * a.c.strides.q_head : q;
                const uint32_t dst = smem_u32(sm + t * L::kTile + (c >> 3) * 16384 + sw128_off(r, c & 7));
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(is ? 16 : 0) : "memory");
                for (head += kStep; head >= g; head -= g) ++tok;
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_async_smem();
            warp_arrive(bar_q, lane);
        }
        // ------------------------------------------------------------------ softmax of row tile t, a row a thread
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + lanes + cS + 128 * t, tO = tmem + lanes + cO + DP * t;
        const int row = 128 * t + (tid & 127), prow = u.row0 + row;
        const int last = row < u.rows ? u.base + prow / g : last_pos;      // rows behind the last one compute along, unseen
        const int first = first_key(last, window);
        // keys all rows of the warp see
        const int w_lo = __reduce_max_sync(0xffffffffu, first), w_hi = __reduce_min_sync(0xffffffffu, last) + 1;
        const float c = a.c.scale * 1.4426950408889634f, lazy = kLazy / c;
        const Range r = t ? range[1] : range[0];
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = r.begin; j < r.end; ++j) {
            const int i = j - r.begin;
            ok = warp_wait(bar_s + t, i & 1);
            if (!ok) break;
            tc_fence_after();
            uint32_t s[4][32];
#pragma unroll
            for (int q = 0; q < 4; ++q) tmem_ld32(tS + 32 * q, s[q]);
            tmem_ld_wait();
            float top = kLowest;
            const int k0 = key0 + j * kKeys;
            if (k0 < w_lo || k0 + kKeys > w_hi) {
                const int from = first - k0, to = last - k0;      // of the tile's keys the row sees [from, to]
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int lo = min(max(from - 32 * q, 0), 32), hi = min(max(to - 32 * q + 1, 0), 32);
                    const uint32_t seen = (uint32_t)((1ull << hi) - 1) & ~(uint32_t)((1ull << lo) - 1);
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!(seen & 1u << e)) s[q][e] = 0xff800000u;
                }
                if (to < 0 || from >= kKeys) top = -INFINITY;
            }
            {
                float x[4] = {top, top, top, top};
#pragma unroll
                for (int e = 0; e < 32; e += 2)
#pragma unroll
                    for (int q = 0; q < 4; ++q) x[q] = max_nan(x[q], __uint_as_float(s[q][e]), __uint_as_float(s[q][e + 1]));
                top = max_nan(max_nan(x[0], x[1], x[2]), x[3]);
            }
            const bool grow = !(top <= m + lazy) && !(top == -INFINITY);      // a NaN too
            if (__any_sync(0xffffffffu, grow)) {
                const float next = max_nan(m, top);
                const float f = grow ? (m == -INFINITY ? 0.f : ex2((m - next) * c)) : 1.f;
                if (grow) m = next;
                l *= f;
                if (i > 0) {      // the sums so far are complete once the product before has ended
                    ok = warp_wait(bar_o + t, (i - 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int q = 0; q < DP / 32; ++q) {
                        uint32_t o[32];
                        tmem_ld32(tO + 32 * q, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st32(tO + 32 * q, o);
                    }
                }
            }
            const float mc = m == -INFINITY ? 0.f : max_nan(m * c, kLowest);
            const f2 c2 = f2_all(c), n2 = f2_all(-mc);
            f2 sum[2] = {f2_all(0.f), f2_all(0.f)};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t p[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const int q = 2 * h + (e >> 4), at = 2 * (e & 15);
                    const f2 x = f2_fma(f2_make(__uint_as_float(s[q][at]), __uint_as_float(s[q][at + 1])), c2, n2);
                    f2 y;
                    if (e % kPolyOf == 0) {
                        y = ex2_pair(x);
                    } else {
                        const float2 z = f2_get(x);
                        y = f2_make(ex2(z.x), ex2(z.y));
                    }
                    sum[e & 1] = f2_add(sum[e & 1], y);
                    p[e] = f2_to_bf16(y);
                }
                tmem_st32(tS + 32 * h, p);
                tmem_st_wait();
                tc_fence_before();
                warp_arrive(bar_p + 2 * t + h, lane);      // its product starts
            }
            const float2 both = f2_get(f2_add(sum[0], sum[1]));
            l += both.x + both.y;
        }
        // ------------------------------------------------------------------ O / l
        const int n = r.end - r.begin;
        const bool full = !split && a.q_boxes && 128 * (t + 1) <= u.rows;      // the same for the row tile's warps
        // The output goes through the queries' place.  With a key, what is read there has been read when the last product ends; without one (a
        // row tile of padding, or a part behind its keys) its queries may still be on their way there, if anything fetched them.
        if (ok && n > 0) {
            ok = warp_wait(bar_o + t, (n - 1) & 1);
        } else if (ok && (!a.q_boxes || t_begin < t_end)) {
            ok = warp_wait(bar_q, 0);
        }
        if (ok && 128 * t + 32 * (warp & 3) < u.rows) {
            tc_fence_after();
            const bool mine = row < u.rows;
            if (!(m < INFINITY)) l = __int_as_float(0x7fffffff);      // a NaN or +inf among the scores, which ex2_pair does not pass on
            const int tok = u.first + prow / g, head = hk * g + prow % g;
            const size_t out = (size_t)tok * a.c.heads.q_heads + head;
            const size_t part = ((size_t)z * a.slots + slot) * a.c.heads.kv_heads + hk;
            const float inv = split ? 1.f : m == -INFINITY ? 0.f : 1.f / l;
            if (mine && split) a.part_ml[part * kRows + row] = make_float2(m == -INFINITY ? m : m < INFINITY ? max_nan(m * c, kLowest) : __int_as_float(0x7fffffff), l);
            if (mine && !split && a.c.lse != nullptr) a.c.lse[out] = m == -INFINITY ? -INFINITY : (m * c + log2f(l)) * kLn2;
            uint8_t* stage_out = sm + t * L::kTile;      // Q has been read; rows as TMA lays them out
            const int x0 = 32 * (warp & 3);
#pragma unroll 1
            for (int q = 0; q < DP / 64; ++q) {
                uint32_t o[2][32];
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    if (n > 0) tmem_ld32(tO + 64 * q + 32 * y, o[y]);
                    else
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[y][e] = 0;
                }
                tmem_ld_wait();
                if (odd_values && n > 0) {
                    // keys that only some rows of the block see: [u.lo, all_lo) and [all_hi, u.hi)
#pragma unroll 1
                    for (int key = max(first, key0 + r.begin * kKeys); key <= min(last, key0 + r.end * kKeys - 1); ++key) {
                        if (key >= all_lo && key < all_hi) {
                            key = all_hi - 1;
                            continue;
                        }
                        const int page = b.page(u.n, key / b.page_size);
                        if (page < 0) continue;
                        const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.c.v) + page * a.c.strides.v_page + (key % b.page_size) * a.c.strides.v_row +
                                                 hk * a.c.strides.v_head + 64 * q;
#pragma unroll
                        for (int e = 0; e < 64; ++e)
                            if (64 * q + e < D) {
                                const float x = __bfloat162float(v[e]);
                                if (!isfinite(x)) o[e >> 5][e & 31] = __float_as_uint(__uint_as_float(o[e >> 5][e & 31]) + x);
                            }
                    }
                }
                if (split) {
                    // a warp's rows, half of the columns at a time (64-wide heads: both halves here), as they lie in the workspace
#pragma unroll
                    for (int h = 0; h < 128 / DP; ++h) {
                        constexpr int kCols = DP / 2;
                        uint8_t* at = stage_out + x0 * DP * 2;
                        if (q + h > 0) {      // the copy before has read its place
                            tma_store_wait_read();
                            __syncwarp();
                        }
#pragma unroll
                        for (int x = 0; x < kCols / 4; ++x) {
                            const int e = kCols * h + 4 * x;
                            *reinterpret_cast<uint4*>(at + part_off<DP>(lane, x)) = make_uint4(o[e >> 5][e & 31], o[e >> 5][(e & 31) + 1], o[e >> 5][(e & 31) + 2], o[e >> 5][(e & 31) + 3]);
                        }
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            const float* dst = a.part_o + ((part * 2 + t) * 2 + q + h) * (128 * kCols) + x0 * kCols;
                            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(at)), "r"(32 * kCols * 4) : "memory");
                            tma_store_commit();
                        }
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = pack_bf16(__uint_as_float(o[x >> 2][8 * (x & 3) + 2 * e]) * inv, __uint_as_float(o[x >> 2][8 * (x & 3) + 2 * e + 1]) * inv);
                        *reinterpret_cast<uint4*>(stage_out + q * 16384 + sw128_off(x0 + lane, x)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            if (split) {
                tma_store_wait_read();
            } else if (!full) {
                __syncwarp();
                constexpr int kLanes = DP / 8;      // lanes that hold a row
                __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.c.o);
                const int chunk = lane % kLanes;
                int x = lane / kLanes, pr = u.row0 + 128 * t + x0 + x, tk = pr / g, hd = pr - tk * g;
#pragma unroll 2
                for (; x < 32; x += 32 / kLanes) {
                    const uint4 v = *reinterpret_cast<const uint4*>(stage_out + (chunk >> 3) * 16384 + sw128_off(x0 + x, chunk & 7));
                    if (128 * t + x0 + x < u.rows && 8 * chunk < D)
                        *reinterpret_cast<uint4*>(o + ((size_t)(u.first + tk) * a.c.heads.q_heads + hk * g + hd) * D + 8 * chunk) = v;
                    for (hd += 32 / kLanes; hd >= g; hd -= g) ++tk;
                }
            }
        }
        if (full) {
            // a full tile leaves by TMA, as Q came; its warps meet whatever their waits said
            fence_async_smem();
            asm volatile("bar.sync %0, 128;" ::"r"(2 + t) : "memory");
            if ((warp & 3) == 0 && !abort_flag && elect_one()) {
                for (int h = 0; h < DP / 64; ++h)
                    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(&mO),
                                 "r"(smem_u32(sm + t * L::kTile + h * 16384)), "r"(h * 64), "r"(hk * g), "r"(u.first + (u.row0 + 128 * t) / g)
                                 : "memory");
                tma_store_commit();
                tma_store_wait_read();
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 " KDA_OTHER_REGS ";");
        if (warp == kMmaWarp) {
            // -------------------------------------------------------------- products
            if (t_begin < t_end && elect_one()) {
                const uint32_t s0 = smem_u32(sm);
                constexpr uint32_t idS = umma_idesc_bf16(128, 128, kMajorK, kMajorK), idO = umma_idesc_bf16(128, DP, kMajorK, kMajorMN);
                bool ok = wait(bar_q, 0);
                auto in = [&](int t, int j) { return j >= range[t].begin && j < range[t].end; };
                auto scores = [&](int t, int j, int i) {      // S_t = Q_t K_j^T
                    const UmmaDesc q = umma_smem_desc_sw128(s0 + t * L::kTile, 16, 1024), k = umma_smem_desc_sw128(s0 + L::kRing + stage(i) * L::kTile, 16, 1024);
#pragma unroll
                    for (int x = 0; x < DP / 16; ++x) {
                        const uint32_t off = (x >> 2) * 16384 + (x & 3) * 32;
                        umma_bf16_ss(tmem + cS + 128 * t, q + off, k + off, idS, x > 0);
                    }
                    umma_commit(bar_s + t);
                };
                if (ok) ok = wait(bar_full + stage(0), turn(0));
                if (ok) {
                    tc_fence_after();
                    for (int t = 0; t < 2; ++t)
                        if (in(t, t_begin)) scores(t, t_begin, 0);
                    umma_commit(bar_free + stage(0));
                }
                for (int j = t_begin; j < t_end && ok; ++j) {
                    const int iv = 2 * (j - t_begin) + 1, ik = iv + 1;      // places of V_j and K_j+1 in the ring
                    ok = wait(bar_full + stage(iv), turn(iv));
                    if (ok && j + 1 < t_end) ok = wait(bar_full + stage(ik), turn(ik));
                    for (int t = 0; t < 2 && ok; ++t) {
                        if (in(t, j)) {
                            const int i = j - range[t].begin;
                            const UmmaDesc v = umma_smem_desc_sw128(s0 + L::kRing + stage(iv) * L::kTile, 16384, 1024);
                            for (int h = 0; h < 2 && ok; ++h) {      // O_t += P_t V_j, half of the keys as soon as their weights are there
                                ok = wait(bar_p + 2 * t + h, i & 1);
                                if (!ok) break;
                                tc_fence_after();
#pragma unroll
                                for (int x = 0; x < 4; ++x)
                                    umma_bf16_ts(tmem + cO + DP * t, tmem + cS + 128 * t + 32 * h + 8 * x, v + (h * 8192 + x * 2048), idO, i > 0 || h > 0 || x > 0);
                            }
                            if (!ok) break;
                            umma_commit(bar_o + t);
                        }
                        if (j + 1 < t_end && in(t, j + 1)) scores(t, j + 1, ik);
                    }
                    if (ok) {
                        umma_commit(bar_free + stage(iv));
                        if (j + 1 < t_end) umma_commit(bar_free + stage(ik));
                    }
                }
                // no product may be in flight when the block ends
                umma_commit(bar_end);
                wait(bar_end, 0);
            }
        } else if (warp == kLoadWarp) {
            // -------------------------------------------------------------- K and V, a box a lane
            constexpr int kHalves = DP / 64;
            const int boxes = kKeys / a.box_rows, box = lane / kHalves, half = lane - box * kHalves;
            const uint32_t box_bytes = (uint32_t)a.box_rows * 128;
            bool ok = true;
            const int total = 2 * (t_end - t_begin);
            auto look = [&](int j, int& row) {      // page of this lane's box, -1: nothing to load
                const int key = key0 + j * kKeys + box * a.box_rows;
                if (box >= boxes || j >= t_end || key >= u.hi || key + a.box_rows <= u.lo) return -1;
                const int col = key / b.page_size;
                row = key - col * b.page_size;
                const int page = b.page(u.n, col);
                if (page < 0) b.tell(KDA_ERR_BLOCK_TABLE);
                return page;
            };
            int row = 0, next_row = 0, page = look(t_begin, row), next_page = -1, i = 0;
            if (a.q_boxes && t_begin < t_end) {
                // 128 rows are whole tokens of g heads.  Rows behind the sequence's last one come along, and stay by themselves.
                const int tiles = u.rows > 128 ? 2 : 1;
                if (lane == 0) mbar_expect_tx(bar_q, tiles * L::kTile);
                __syncwarp();
                const int t = lane / kHalves, h = lane - t * kHalves;
                if (t < tiles)
                    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                                     smem_u32(sm + t * L::kTile + h * 16384)),
                                 "l"(&mQ), "r"(smem_u32(bar_q)), "r"(h * 64), "r"(hk * g), "r"(u.first + (u.row0 + 128 * t) / g)
                                 : "memory");
            }
            for (; i < total; ++i) {
                const int j = t_begin + (i >> 1), s = stage(i);
                const bool isv = i & 1;
                if (i >= L::kStages) ok = warp_wait(bar_free + s, turn(i - L::kStages));
                if (!ok) break;
                if (!isv) next_page = look(j + 1, next_row);
                uint64_t* f = isv && partial(j) ? bar_part + s : bar_full + s;
                const int loads = __popc(__ballot_sync(0xffffffffu, page >= 0));
                if (lane == 0) mbar_expect_tx(f, loads * box_bytes);
                __syncwarp();
                if (page >= 0) {
                    const CUtensorMap* map = isv ? &mV : &mK;
                    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
                                     smem_u32(sm + L::kRing + s * L::kTile + half * 16384 + box * box_bytes)),
                                 "l"(map), "r"(smem_u32(f)), "r"(half * 64), "r"(row), "r"(hk), "r"(page)
                                 : "memory");
                }
                if (isv) {
                    page = next_page;
                    row = next_row;
                }
            }
            // no copy may be in flight when the block ends
            if (!ok && a.q_boxes && lane == 0) mbar_poll(bar_q, 0, kSpinLimit / 8);
            if (!ok && lane == 0)
                for (int x = i > L::kStages ? i - L::kStages : 0; x < i; ++x)
                    mbar_poll((x & 1) && partial(t_begin + (x >> 1)) ? bar_part + stage(x) : bar_full + stage(x), turn(x), kSpinLimit / 8);
        } else {
            // -------------------------------------------------------------- V tiles that some row sees only in part
            uint32_t phase = 0;      // of each stage's barrier
            bool odd = false;
            for (int j = t_begin; j < t_end; ++j) {
                if (!partial(j)) continue;
                const int i = 2 * (j - t_begin) + 1, s = stage(i);
                const bool ok = warp_wait(bar_part + s, (phase >> s) & 1u);
                phase ^= 1u << s;
                uint8_t* v = sm + L::kRing + s * L::kTile;
                // Keys [0, head) and [tail, 128) of the tile, a piece of eight values a thread, DP / 8 threads a row: those outside of
                // [u.lo, u.hi) are blanked, the others looked through.  The product of the tile waits for this.
                constexpr int kChunks = DP / 8, kStep = 64 / kChunks;
                const int k0 = key0 + j * kKeys, head = min(max(all_lo - k0, 0), kKeys), tail = max(min(max(all_hi - k0, 0), kKeys), head);
                const int x = tid - kFixWarp * 32, ch = x % kChunks, y0 = x / kChunks;
                auto place = [&](int r) { return reinterpret_cast<uint4*>(v + (ch >> 3) * 16384 + sw128_off(r, ch & 7)); };
                auto through = [&](int from, int to) {
                    constexpr int kAhead = 8;
                    for (int r = from + y0; r < to; r += kAhead * kStep) {
                        uint4 w[kAhead];
#pragma unroll
                        for (int k = 0; k < kAhead; ++k) w[k] = *place(min(r + k * kStep, kKeys - 1));
#pragma unroll
                        for (int k = 0; k < kAhead; ++k) {
                            // an exponent of ones and one more is the sign's bit
                            auto ones = [](uint32_t z) { return ((z & 0x7f807f80u) + 0x00800080u) & 0x80008000u; };
                            if (r + k * kStep >= to || (ones(w[k].x) | ones(w[k].y) | ones(w[k].z) | ones(w[k].w)) == 0) continue;
                            odd = true;
                            uint32_t* p = reinterpret_cast<uint32_t*>(&w[k]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if ((p[i] & 0x7f80u) == 0x7f80u) p[i] &= 0xffff0000u;
                                if ((p[i] & 0x7f800000u) == 0x7f800000u) p[i] &= 0xffffu;
                            }
                            *place(r + k * kStep) = w[k];
                        }
                    }
                };
                auto blank = [&](int from, int to) {
                    for (int r = from + y0; r < to; r += kStep) *place(r) = make_uint4(0, 0, 0, 0);
                };
                const int lo = min(max(u.lo - k0, 0), kKeys), hi = min(max(u.hi - k0, 0), kKeys);      // keys in reach
                if (ok) {
                    blank(0, min(lo, head));
                    through(min(lo, head), min(head, hi));
                    blank(hi, head);
                    blank(tail, lo);
                    through(max(tail, lo), hi);
                    blank(max(tail, hi), kKeys);
                }
                if (odd) odd_values = 1;
                __threadfence_block();
                fence_async_smem();
                asm volatile("bar.sync 1, 64;" ::: "memory");      // the two warps meet whatever their waits said
                if (tid == kFixWarp * 32 && !abort_flag) mbar_arrive(bar_full + s);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// Joins the parts of 32 rows: a warp four of them, eight lanes a row.
template <int DP>
__global__ void __launch_bounds__(256) attn_tc_join_kernel(const __grid_constant__ Args a) {
    const Batch& b = a.c.batch;
    const int slot = blockIdx.x >> 3, hk = blockIdx.y, g = a.c.heads.group, D = a.c.heads.dim, Hk = a.c.heads.kv_heads;
    const int lane = threadIdx.x & 31, l8 = lane & 7, row = 32 * (blockIdx.x & 7) + 4 * (threadIdx.x >> 5) + (lane >> 3);
    Unit u;
    if (!make_unit(b, a.tiles, slot, a.c.window, u) || 32 * (int)(blockIdx.x & 7) >= u.rows) return;
    const int parts = a.parts[slot * Hk + hk];
    if (parts < 2) return;
    const size_t step = (size_t)a.slots * Hk, unit = (size_t)slot * Hk + hk;
    float m = -INFINITY, l = 0.f;
    for (int z = l8; z < parts; z += 8) m = max_nan(m, a.part_ml[(unit + z * step) * kRows + row].x);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    constexpr int kPieces = DP / 32, kAhead = 4;      // pieces of four values a lane: l8, l8 + 8, ... of the row's; parts on their way
    f2 acc[kPieces][2];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) acc[i][0] = acc[i][1] = f2_all(0.f);
    const int r = row & 127;
    for (int z0 = 0; z0 < parts; z0 += kAhead) {
        float2 ml[kAhead];
        float4 v[kAhead][kPieces];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const size_t part = unit + min(z0 + k, parts - 1) * step;
            ml[k] = a.part_ml[part * kRows + row];
            const char* src = reinterpret_cast<const char*>(a.part_o + (part * 2 + (row >> 7)) * (128 * DP));
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int piece = l8 + 8 * i, half = piece / (DP / 8), c = piece % (DP / 8);
                v[k][i] = *reinterpret_cast<const float4*>(src + half * (128 * DP * 2) + part_off<DP>(r, c));
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (z0 + k >= parts || ml[k].x == -INFINITY) continue;      // without a key its sums are 0
            const float f = ex2(ml[k].x - m);
            l = fmaf(ml[k].y, f, l);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                acc[i][0] = f2_fma(f2_make(v[k][i].x, v[k][i].y), f2_all(f), acc[i][0]);
                acc[i][1] = f2_fma(f2_make(v[k][i].z, v[k][i].w), f2_all(f), acc[i][1]);
            }
        }
    }
    if (row >= u.rows) return;
    const int pr = u.row0 + row, tok = pr / g;
    const size_t out = (size_t)(u.first + tok) * a.c.heads.q_heads + hk * g + pr - tok * g;
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
    if (l8 == 0 && a.c.lse != nullptr) a.c.lse[out] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * kLn2;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int d = 4 * (l8 + 8 * i);
        if (d < D)
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.c.o) + out * D + d) = make_uint2(f2_to_bf16(f2_mul(acc[i][0], f2_all(inv))), f2_to_bf16(f2_mul(acc[i][1], f2_all(inv))));
    }
}

template <int DP>
int launch(const Call& c, const CUtensorMap& mK, const CUtensorMap& mV, const CUtensorMap& mQ, const CUtensorMap& mO, const Args& a, cudaStream_t st) {
    if (int rc = set_smem_limit(attn_tc_kernel<DP>, Layout<DP>::kBytes)) return rc;
    const dim3 grid((unsigned)a.slots, (unsigned)c.heads.kv_heads, (unsigned)a.splits);
    KDA_LAUNCH("attn_tc_kernel", st, attn_tc_kernel<DP><<<grid, kThreads, Layout<DP>::kBytes, st>>>(mK, mV, mQ, mO, a));
    if (int rc = launch_status()) return rc;
    if (a.splits == 1) return KDA_OK;
    const dim3 joins((unsigned)a.slots * 8, (unsigned)c.heads.kv_heads);
    KDA_LAUNCH("attn_tc_join_kernel", st, attn_tc_join_kernel<DP><<<joins, 256, 0, st>>>(a));
    return launch_status();
}

}  // namespace



bool tc_takes(const Call& c) {
    const Strides& s = c.strides;
    const int page = c.batch.page_size;
    if (!c.bf16 || c.heads.dim > 128 || c.heads.dim % 8 != 0 || !(page % kKeys == 0 || (kKeys % page == 0 && page >= 8))) return false;
    if (c.batch.n_pages == 0 || c.batch.table_width == 0) return false;
    const long long all = s.q_token | s.q_head | s.k_page | s.k_row | s.k_head | s.v_page | s.v_row | s.v_head;
    if (all % 8 != 0 || reinterpret_cast<uintptr_t>(c.q) % 16 != 0 || reinterpret_cast<uintptr_t>(c.k) % 16 != 0 || reinterpret_cast<uintptr_t>(c.v) % 16 != 0 || reinterpret_cast<uintptr_t>(c.o) % 16 != 0)
        return false;
    for (long long x : {s.k_page, s.k_row, s.k_head, s.v_page, s.v_row, s.v_head})
        if (x <= 0 || x >= 1ll << 39) return false;
    return true;
}

int tc(const Call& c, int splits, cudaStream_t st) {
    Args a;
    a.c = c;
    a.tiles = Tiles{kRows, c.heads.group, 0};
    a.slots = (int)tile_slots(c.batch.tokens, c.batch.n_seq, c.max_q_len, c.heads.group, kRows, c.batch.cu != nullptr, a.tiles.per_seq);
    a.splits = splits;
    a.box_rows = c.batch.page_size < kKeys ? c.batch.page_size : kKeys;
    a.parts = nullptr;
    a.part_ml = nullptr;
    a.part_o = nullptr;
    if (splits > 1) {
        const size_t units = (size_t)a.slots * c.heads.kv_heads;
        char* ws = static_cast<char*>(c.workspace);
        a.parts = reinterpret_cast<int*>(ws);
        a.part_ml = reinterpret_cast<float2*>(ws + align_up(units * sizeof(int), 256));
        a.part_o = reinterpret_cast<float*>(a.part_ml + units * splits * kRows);
    }
    CUtensorMap mK, mV, mQ, mO;
    const Strides& s = c.strides;
    int rc = make_map_paged(&mK, c.k, c.heads.dim, c.batch.page_size, c.heads.kv_heads, c.batch.n_pages, s.k_row, s.k_head, s.k_page, a.box_rows);
    if (!rc) rc = make_map_paged(&mV, c.v, c.heads.dim, c.batch.page_size, c.heads.kv_heads, c.batch.n_pages, s.v_row, s.v_head, s.v_page, a.box_rows);
    mQ = mO = mK;
    a.q_boxes = 128 % c.heads.group == 0 && s.q_head > 0 && s.q_token > 0 && s.q_head < 1ll << 39 && s.q_token < 1ll << 39;
    if (!rc && a.q_boxes) rc = make_map_packed(&mQ, c.q, c.heads.dim, c.heads.q_heads, c.batch.tokens, s.q_head, s.q_token, c.heads.group, 128 / c.heads.group);
    if (!rc && a.q_boxes)
        rc = make_map_packed(&mO, c.o, c.heads.dim, c.heads.q_heads, c.batch.tokens, c.heads.dim, (int64_t)c.heads.q_heads * c.heads.dim, c.heads.group, 128 / c.heads.group);
    if (!rc) rc = c.heads.dim <= 64 ? launch<64>(c, mK, mV, mQ, mO, a, st) : launch<128>(c, mK, mV, mQ, mO, a, st);
    return rc;
}

// of a call whose rows are cut into `splits` parts at most
size_t tc_workspace(long long slots, int kv_heads, int splits, int dim) {
    if (splits < 2) return 0;
    const size_t units = (size_t)slots * kv_heads, width = dim <= 64 ? 64 : 128;
    return align_up(units * sizeof(int), 256) + units * splits * kRows * (sizeof(float2) + width * sizeof(float));
}

}  // namespace attn
}  // namespace kda
