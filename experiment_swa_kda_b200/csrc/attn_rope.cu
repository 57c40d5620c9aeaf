// Per-head RMS norm of queries and keys with the rotation by position in the same pass, forward and backward, and the form
// that puts a serving batch's keys and values into their pages.
//
//   u = x r w, r = (mean x^2 + eps)^-1/2;   y_a = u_a c - u_b s, y_b = u_b c + u_a s for a pair (a, b)
//   backward: du_a = dy_a c + dy_b s, du_b = dy_b c - dy_a s;  dw = sum over rows of du x r;
//             dx = r (w du - x r^2 mean(w du x))
//
// Everything is float32 between the load and the one rounding of the store.  r is formed again in the backward: it costs a sum
// over values that are in registers anyway, a saved one would be read.
//
// Bound by memory, and close behind it by issue: 65,536 tokens of 16 + 4 heads take 122 us forward (5.5 TB/s, 0.84 of the copy
// rate) and 225 backward (4.5 TB/s, 63 % of the issue slots); 8,191 tokens into the cache 29.  Two forms each way: norm_rope_rows_* for widths, strides and addresses that allow wide accesses, and
// norm_rope_kernel / norm_rope_bwd_kernel for all others.

#include <initializer_list>

#include "attn.cuh"

namespace kda {
namespace attn {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBlocks = 2;      // blocks an SM of the kernels that go by rows (three: 80 registers, spilled, 640 us where two take 336)

struct Rope {
    KdaRotaryShape s;
    const void *q, *k, *v;
    const float *cos, *sin, *q_weight, *k_weight;
    const void* positions;
    void *q_out, *k_out;            // forward: q', k' (append: k cache); backward: dq, dk
    void* v_out;                    // append: v cache
    const void *d_q, *d_k;          // backward: cotangents of q', k'
    float* part;                    // backward: [blocks][2][head_dim] partial sums of the weights' gradients
    Batch batch;                    // append
    Strides cache;
    int* mirror;
    int run;                        // norm_rope_rows_*: pieces of a token or of the next that a group of lanes takes one after the other
};

// Where a token goes: its position, and the cache rows of its key and value (append).
struct Place {
    int pos;                        // negative: padding
    long long k_at, v_at;           // element offsets of the page's row, or -1: no page
};

template <bool APPEND, int LANES = 1>
__device__ __forceinline__ Place place_of(const Rope& p, int t, int l = 0, unsigned mask = 0) {
    Place r;
    if (APPEND) {
        const Batch& b = p.batch;
        const int n = LANES > 1 ? b.seq_of<LANES>(t, l, mask) : b.seq_of(t);
        int first, count;
        b.span(n, first, count);
        r.pos = b.kv_len(n) - count + (t - first);
        r.k_at = r.v_at = -1;
        if (t < first || t >= first + count) r.pos = -1;      // a token of no sequence
        if (r.pos >= 0) {
            const int page = b.page(n, r.pos / b.page_size), row = r.pos % b.page_size;
            if (page >= 0) {
                r.k_at = page * p.cache.k_page + row * p.cache.k_row;
                r.v_at = page * p.cache.v_page + row * p.cache.v_row;
            } else {
                b.tell(KDA_ERR_BLOCK_TABLE);
            }
        }
        if (t == first || t == 0) {
            if (!b.kv_len_ok(n)) b.tell(KDA_ERR_BLOCK_TABLE);
            if (!b.span_ok(n)) b.tell(KDA_ERR_CU_SEQLENS);
        }
    } else {
        r.k_at = r.v_at = 0;
        long long pos = p.positions == nullptr ? t % p.s.seq_len
                        : p.s.positions_64     ? static_cast<const long long*>(p.positions)[t]
                                               : static_cast<const int*>(p.positions)[t];
        r.pos = pos < 0 ? 0 : pos > INT_MAX ? INT_MAX : (int)pos;
        if (pos < 0 && p.mirror != nullptr) *reinterpret_cast<volatile int*>(p.mirror) = KDA_ERR_POSITION;
    }
    if (r.pos >= p.s.table_len) {
        r.pos = p.s.table_len - 1;
        if (p.mirror != nullptr) *reinterpret_cast<volatile int*>(p.mirror) = KDA_ERR_POSITION;
    }
    return r;
}

// The other member of value e's pair, the pair's number, and the sign of the sine in y_e; e < rotary_dim.
__device__ __forceinline__ void pair_of(int e, int rot, int interleaved, int& other, int& i, float& sign) {
    if (interleaved) {
        other = e ^ 1;
        i = e >> 1;
        sign = (e & 1) ? 1.f : -1.f;
    } else {
        const int half = rot >> 1;
        other = e < half ? e + half : e - half;
        i = e < half ? e : e - half;
        sign = e < half ? -1.f : 1.f;
    }
}

// ---------------------------------------------------------------------------------------------- any width, any address
// A warp a row, lane i holds values i, i + 32, ...; the partner of a value is read again.
template <bool APPEND>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(Rope p) {
    const int lane = threadIdx.x & 31, D = p.s.head_dim, R = p.s.rotary_dim, bf16 = p.s.io_dtype == KDA_DTYPE_BF16;
    const int heads = p.s.q_heads + p.s.kv_heads, all = heads + (APPEND ? p.s.kv_heads : 0);
    const long long rows = (long long)p.s.tokens * all;
    for (long long row = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); row < rows; row += (long long)gridDim.x * kWarps) {
        const int t = (int)(row / all), h = (int)(row - (long long)t * all);
        const Place at = place_of<APPEND>(p, t);
        const bool isq = h < p.s.q_heads;
        const int hk = isq ? 0 : h < heads ? h - p.s.q_heads : h - heads;
        void* out = isq ? p.q_out : p.k_out;
        long long dst = isq ? ((long long)t * p.s.q_heads + h) * D : ((long long)t * p.s.kv_heads + hk) * D;
        if (APPEND && !isq) {
            if (at.pos < 0 || at.k_at < 0) continue;
            if (h >= heads) {      // a value row goes as it is
                const long long src = t * p.s.v_token_stride + hk * p.s.v_head_stride;
                for (int e = lane; e < D; e += 32) st_io(p.v_out, at.v_at + hk * p.cache.v_head + e, bf16, ld_io(p.v, src + e, bf16));
                continue;
            }
            dst = at.k_at + hk * p.cache.k_head;
        }
        if (APPEND && at.pos < 0) {
            for (int e = lane; e < D; e += 32) st_io(out, dst + e, bf16, 0.f);
            continue;
        }
        const void* src = isq ? p.q : p.k;
        const long long from = isq ? t * p.s.q_token_stride + h * p.s.q_head_stride : t * p.s.k_token_stride + hk * p.s.k_head_stride;
        const float* w = isq ? p.q_weight : p.k_weight;
        float x[8], ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = lane + 32 * j;
            x[j] = e < D ? ld_io(src, from + e, bf16) : 0.f;
            ss = fmaf(x[j], x[j], ss);
        }
        const float r = rsqrtf(warp_sum(ss) / D + p.s.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = lane + 32 * j;
            if (e >= D) break;
            float y = x[j] * r * (w ? w[e] : 1.f);
            if (e < R) {
                int o, i;
                float sign;
                pair_of(e, R, p.s.interleaved, o, i, sign);
                const float other = ld_io(src, from + o, bf16) * r * (w ? w[o] : 1.f);
                const size_t c = (size_t)at.pos * (R / 2) + i;
                y = fmaf(y, p.cos[c], sign * other * p.sin[c]);
            }
            st_io(out, dst + e, bf16, y);
        }
    }
}

__global__ void __launch_bounds__(kThreads) norm_rope_bwd_kernel(Rope p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = p.s.head_dim, R = p.s.rotary_dim, bf16 = p.s.io_dtype == KDA_DTYPE_BF16;
    float dw[2][8] = {};
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const int H = which ? p.s.kv_heads : p.s.q_heads;
        const void *src = which ? p.k : p.q, *dy = which ? p.d_k : p.d_q;
        void* dst = which ? p.k_out : p.q_out;
        const float* w = which ? p.k_weight : p.q_weight;
        const long long ts = which ? p.s.k_token_stride : p.s.q_token_stride, hs = which ? p.s.k_head_stride : p.s.q_head_stride;
        const long long rows = (long long)p.s.tokens * H;
        for (long long row = (long long)blockIdx.x * kWarps + warp; row < rows; row += (long long)gridDim.x * kWarps) {
            const int t = (int)(row / H), h = (int)(row - (long long)t * H);
            const Place at = place_of<false>(p, t);
            const long long from = t * ts + h * hs, to = row * D;
            float x[8], du[8], ss = 0.f, dot = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = lane + 32 * j;
                x[j] = du[j] = 0.f;
                if (e < D) {
                    x[j] = ld_io(src, from + e, bf16);
                    du[j] = ld_io(dy, to + e, bf16);
                    if (e < R) {
                        int o, i;
                        float sign;
                        pair_of(e, R, p.s.interleaved, o, i, sign);
                        const size_t c = (size_t)at.pos * (R / 2) + i;
                        du[j] = fmaf(du[j], p.cos[c], -sign * ld_io(dy, to + o, bf16) * p.sin[c]);
                    }
                }
                ss = fmaf(x[j], x[j], ss);
            }
            const float r = rsqrtf(warp_sum(ss) / D + p.s.eps);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = lane + 32 * j;
                dw[which][j] = fmaf(du[j] * x[j], r, dw[which][j]);
                if (w && e < D) du[j] *= w[e];
                dot = fmaf(du[j], x[j], dot);
            }
            const float f = warp_sum(dot) / D * r * r;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = lane + 32 * j;
                if (e < D) st_io(dst, to + e, bf16, r * (du[j] - x[j] * f));
            }
        }
    }
    if (p.part == nullptr) return;
    __shared__ float sum[kWarps][2][KDA_MAX_DIM];
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[warp][which][lane + 32 * j] = dw[which][j];
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * D; e += kThreads) {
        const int which = e / D, d = e - which * D;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) s += sum[k][which][d];
        p.part[(size_t)blockIdx.x * 2 * D + e] = s;
    }
}

// ---------------------------------------------------------------------------------------------- eight values a lane
// LANES lanes a row, and both members of a pair in one lane: two pieces of four adjacent values, half the rotated width apart in the
// split order.  What bounds such a loop after memory is issue and the shuffles of the rows' sums, so rows go four at a time (backward
// two, with two sums each) and their four sums are reduced together: 5 shuffles, not 16, and 4 that hand them out.
//
// Such a piece of rows - of one token, and of q, k or (append) v - is what a group of lanes works on at a time, and it takes runs of
// them, so that a token's place, its cosines and sines and the weights are read once for all of them.  Each lane copies its own
// values through a ring in shared memory that runs ahead by kStages - 1 pieces: rows held in registers would be waited for
// by all of a piece's arithmetic, and with 16 to 24 warps an SM too few were on their way (65,536 tokens of 20 heads, forward and
// backward: 397 us).

// values [0..3], [4..7] of a lane: 8 or 16 bytes each
template <bool BF16>
struct Vec8 {
    static constexpr int kBytes = BF16 ? 8 : 16;
    static constexpr int kValue = BF16 ? 2 : 4;
    static __device__ __forceinline__ void copy(uint32_t dst, const char* src) {
        if (BF16) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
        else asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    }
    static __device__ __forceinline__ void get(const char* p, f2& a, f2& b) {
        if (BF16) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            a = f2_from_bf16(v.x);
            b = f2_from_bf16(v.y);
        } else {
            const float4 v = *reinterpret_cast<const float4*>(p);
            a = f2_make(v.x, v.y);
            b = f2_make(v.z, v.w);
        }
    }
    static __device__ __forceinline__ void store(char* p, f2 a, f2 b) {
        if (BF16) {
            *reinterpret_cast<uint2*>(p) = make_uint2(f2_to_bf16(a), f2_to_bf16(b));
        } else {
            const float2 x = f2_get(a), y = f2_get(b);
            *reinterpret_cast<float4*>(p) = make_float4(x.x, x.y, y.x, y.y);
        }
    }
};
// The ring: [stage][8 values' worth of pieces of four][thread].
template <bool BF16>
struct Ring {
    static constexpr int kStages = BF16 ? 4 : 2, kPiece = kThreads * Vec8<BF16>::kBytes, kStage = 8 * kPiece, kBytes = kStages * kStage;
    char* mine;                 // this thread's place of the first piece
    uint32_t address;
    int in = 0, out = 0;        // stages to fill and to empty, as offsets
    __device__ __forceinline__ explicit Ring(char* smem) : mine(smem + threadIdx.x * Vec8<BF16>::kBytes), address((uint32_t)__cvta_generic_to_shared(mine)) {}
    __device__ __forceinline__ uint32_t to(int piece) const { return address + in + piece * kPiece; }
    __device__ __forceinline__ const char* from(int piece) const { return mine + out + piece * kPiece; }
    static __device__ __forceinline__ int after(int stage) { return stage + kStage == kBytes ? 0 : stage + kStage; }
    static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory"); }      // the oldest is there
};

// The pieces of a token: ROWS rows each of q's heads, then k's, then v's.  A group goes through runs of `run` pieces, the next one
// `stride` pieces behind the one before; counted, since a division a piece costs as much as its rows.
template <int ROWS>
struct Pieces {
    int each, of_q, of_k;       // pieces of a token, of q and k
    int at, all, left;          // this piece of all the batch's; pieces left of the run
    int t, n, which, h, rows;   // token, piece of the token; q, k or v; first head, heads

    __device__ __forceinline__ Pieces(const KdaRotaryShape& s, bool values, int first, int run) {
        of_q = (s.q_heads + ROWS - 1) / ROWS;
        of_k = (s.kv_heads + ROWS - 1) / ROWS;
        each = of_q + of_k + (values ? of_k : 0);
        all = s.tokens * each;
        set(s, first, run);
    }
    __device__ __forceinline__ bool more() const { return at < all; }
    __device__ __forceinline__ void set(const KdaRotaryShape& s, int i, int run) {
        at = i;
        left = run;
        t = i / each;
        n = i - t * each;
        place(s);
    }
    __device__ __forceinline__ void place(const KdaRotaryShape& s) {
        which = n < of_q ? 0 : n < of_q + of_k ? 1 : 2;
        h = ROWS * (n - (which == 0 ? 0 : which == 1 ? of_q : of_q + of_k));
        rows = min(ROWS, (which ? s.kv_heads : s.q_heads) - h);
    }
    __device__ __forceinline__ void next(const KdaRotaryShape& s, int run, int stride) {
        if (--left > 0) {
            ++at;
            if (++n == each) {
                n = 0;
                ++t;
            }
            place(s);
        } else {
            const long long to = (long long)at + 1 + stride - run;
            if (to < all) set(s, (int)to, run);
            else at = all;
        }
    }
};

// The sums of four values over the lanes of a group; lane l ends with that of value l & 3.
template <int LANES>
__device__ __forceinline__ float sum4(float a0, float a1, float a2, float a3, int l, unsigned mask) {
    const bool b0 = l & 1, b1 = l & 2;
    float x = b0 ? a1 : a0, y = b0 ? a3 : a2;
    x += __shfl_xor_sync(mask, b0 ? a0 : a1, 1);
    y += __shfl_xor_sync(mask, b0 ? a2 : a3, 1);
    float z = b1 ? y : x;
    z += __shfl_xor_sync(mask, b1 ? x : y, 2);
#pragma unroll
    for (int o = 4; o < LANES; o <<= 1) z += __shfl_xor_sync(mask, z, o);
    return z;
}

__device__ __forceinline__ f2 swapped(f2 a) {
    const float2 x = f2_get(a);
    return f2_make(x.y, x.x);
}
__device__ __forceinline__ float f2_dot(const f2 (&x)[4], const f2 (&y)[4]) {
    const float2 t = f2_get(f2_fma(x[0], y[0], f2_fma(x[1], y[1], f2_fma(x[2], y[2], f2_mul(x[3], y[3])))));
    return t.x + t.y;
}

// A lane's share of a row.
template <int LANES, bool INTER>
struct Lane {
    int l, d0, d1;                  // lane of the group, its first value of each piece
    bool on, turned;                // the row has these values; they are rotated
    unsigned mask;

    __device__ __forceinline__ Lane(const KdaRotaryShape& s) {
        const int lane = threadIdx.x & 31;
        l = lane & (LANES - 1);
        mask = LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1u) << (lane & ~(LANES - 1));
        on = 8 * l < s.head_dim;
        turned = 8 * l < s.rotary_dim;
        d0 = 8 * l;
        d1 = d0 + 4;
        if (!INTER && turned) {
            d0 = 4 * l;
            d1 = s.rotary_dim / 2 + 4 * l;
        }
    }
    // y_e = x_e c_e + x_other s_e for the lane's values; 1 and 0 where they are not rotated
    __device__ __forceinline__ void angles(const Rope& p, int pos, f2 (&c)[4], f2 (&s)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c[i] = f2_all(1.f);
            s[i] = f2_all(0.f);
        }
        if (!turned) return;
        const size_t at = (size_t)pos * (p.s.rotary_dim / 2) + 4 * l;
        const float4 cc = __ldg(reinterpret_cast<const float4*>(p.cos + at)), ss = __ldg(reinterpret_cast<const float4*>(p.sin + at));
        if (INTER) {
            c[0] = f2_all(cc.x); c[1] = f2_all(cc.y); c[2] = f2_all(cc.z); c[3] = f2_all(cc.w);
            s[0] = f2_make(-ss.x, ss.x); s[1] = f2_make(-ss.y, ss.y); s[2] = f2_make(-ss.z, ss.z); s[3] = f2_make(-ss.w, ss.w);
        } else {
            c[0] = c[2] = f2_make(cc.x, cc.y);
            c[1] = c[3] = f2_make(cc.z, cc.w);
            s[0] = f2_make(-ss.x, -ss.y);
            s[1] = f2_make(-ss.z, -ss.w);
            s[2] = f2_make(ss.x, ss.y);
            s[3] = f2_make(ss.z, ss.w);
        }
    }
    __device__ __forceinline__ void weights(const float* w, f2 (&x)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = f2_all(1.f);
        if (w == nullptr || !on) return;
        const float4 a = __ldg(reinterpret_cast<const float4*>(w + d0)), b = __ldg(reinterpret_cast<const float4*>(w + d1));
        x[0] = f2_make(a.x, a.y); x[1] = f2_make(a.z, a.w); x[2] = f2_make(b.x, b.y); x[3] = f2_make(b.z, b.w);
    }
    // the partners of a lane's values.  A lane that is not rotated has none: 0, since 0 times an infinite value would be NaN.
    __device__ __forceinline__ void other(const f2 (&x)[4], f2 (&o)[4], bool all_turned) const {
        if (INTER) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = swapped(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = x[i ^ 2];
        }
        if (!all_turned && !turned)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = f2_all(0.f);
    }
};

template <int LANES, bool BF16, bool INTER, bool APPEND>
__global__ void __launch_bounds__(kThreads, kBlocks) norm_rope_rows_kernel(Rope p) {
    extern __shared__ __align__(16) char smem[];
    using V = Vec8<BF16>;
    using R = Ring<BF16>;
    R ring(smem);
    constexpr int kGroups = kThreads / LANES;
    const Lane<LANES, INTER> ln(p.s);
    const int Hq = p.s.q_heads, Hk = p.s.kv_heads, D = p.s.head_dim, piece_gap = (ln.d1 - ln.d0) * V::kValue;
    const bool all_turned = p.s.rotary_dim == D;
    const float inv = 1.f / D;
    const int stride = gridDim.x * kGroups * p.run;
    Pieces<4> ahead(p.s, APPEND, (blockIdx.x * kGroups + threadIdx.x / LANES) * p.run, p.run);
    Pieces<4> w = ahead;
    auto copy = [&]() {
        if (ahead.more()) {
            const void* src = ahead.which == 0 ? p.q : ahead.which == 1 ? p.k : p.v;
            const long long ts = ahead.which == 0 ? p.s.q_token_stride : ahead.which == 1 ? p.s.k_token_stride : p.s.v_token_stride;
            const long long hs = ahead.which == 0 ? p.s.q_head_stride : ahead.which == 1 ? p.s.k_head_stride : p.s.v_head_stride;
            const char* from = static_cast<const char*>(src) + (ahead.t * ts + ahead.h * hs + ln.d0) * V::kValue;
            const long long step = hs * V::kValue;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (ln.on && i < ahead.rows) {
                    V::copy(ring.to(2 * i), from + i * step);
                    V::copy(ring.to(2 * i + 1), from + i * step + piece_gap);
                }
            ahead.next(p.s, p.run, stride);
        }
        R::commit();
        ring.in = R::after(ring.in);
    };
#pragma unroll
    for (int i = 0; i < R::kStages - 1; ++i) copy();
    Place at = {};
    f2 c[4], s[4], a[4], b[4];
    int token = -1, kind = -1;
    for (; w.more(); w.next(p.s, p.run, stride)) {
        copy();
        if (w.t != token) {
            token = w.t;
            kind = -1;
            at = place_of<APPEND, LANES>(p, token, ln.l, ln.mask);
            ln.angles(p, max(at.pos, 0), c, s);
        }
        if (w.which != kind && w.which < 2) {
            kind = w.which;
            f2 own[4];      // u_e c + u_other s with u = x r w: a = w_e c, b = w_other s
            ln.weights(kind ? p.k_weight : p.q_weight, own);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = f2_mul(own[i], c[i]);
                b[i] = f2_mul(INTER ? swapped(own[i]) : own[i ^ 2], s[i]);
            }
        }
        R::wait();
        f2 x[4][4];
        float ss[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            V::get(ring.from(2 * i), x[i][0], x[i][1]);
            V::get(ring.from(2 * i + 1), x[i][2], x[i][3]);
            ss[i] = ln.on ? f2_dot(x[i], x[i]) : 0.f;
        }
        ring.out = R::after(ring.out);
        void* dst = w.which == 0 ? p.q_out : w.which == 1 ? p.k_out : p.v_out;
        long long to = ((long long)w.t * (w.which ? Hk : Hq) + w.h) * D, hs = D;
        if (APPEND && w.which) {
            if (at.pos < 0 || at.k_at < 0) continue;
            hs = w.which == 1 ? p.cache.k_head : p.cache.v_head;
            to = (w.which == 1 ? at.k_at : at.v_at) + w.h * hs;
        }
        char* into = static_cast<char*>(dst) + (to + ln.d0) * V::kValue;
        const long long step = hs * V::kValue;
        const float r = rsqrtf(fmaf(sum4<LANES>(ss[0], ss[1], ss[2], ss[3], ln.l, ln.mask), inv, p.s.eps));
        const bool none = APPEND && at.pos < 0;      // padding
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f2 r2 = f2_all(__shfl_sync(ln.mask, r, i, LANES));
            f2 y[4];
            if (APPEND && w.which == 2) {      // values go as they are
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = x[i][k];
            } else {
                f2 o[4];
                ln.other(x[i], o, all_turned);
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = none ? f2_all(0.f) : f2_mul(f2_fma(x[i][k], a[k], f2_mul(o[k], b[k])), r2);
            }
            if (ln.on && i < w.rows) {
                V::store(into + i * step, y[0], y[1]);
                V::store(into + i * step + piece_gap, y[2], y[3]);
            }
        }
    }
}

// The same rows backward; each lane sums its weights' gradients over all rows it meets, a block over its lanes, and
// norm_rope_dw_kernel over the blocks, all in a fixed order.
template <int LANES, bool BF16, bool INTER>
__global__ void __launch_bounds__(kThreads, kBlocks) norm_rope_rows_bwd_kernel(Rope p) {
    extern __shared__ __align__(16) char smem[];
    using V = Vec8<BF16>;
    using R = Ring<BF16>;
    R ring(smem);
    constexpr int kGroups = kThreads / LANES;
    dependents_go();
    const Lane<LANES, INTER> ln(p.s);
    const int Hq = p.s.q_heads, Hk = p.s.kv_heads, D = p.s.head_dim, piece_gap = (ln.d1 - ln.d0) * V::kValue;
    const bool all_turned = p.s.rotary_dim == D;
    const float inv = 1.f / D;
    const int stride = gridDim.x * kGroups * p.run;
    Pieces<2> ahead(p.s, false, (blockIdx.x * kGroups + threadIdx.x / LANES) * p.run, p.run);
    Pieces<2> w = ahead;
    auto copy = [&]() {
        if (ahead.more()) {
            const void *src = ahead.which ? p.k : p.q, *grad = ahead.which ? p.d_k : p.d_q;
            const long long hs = ahead.which ? p.s.k_head_stride : p.s.q_head_stride;
            const char* from = static_cast<const char*>(src) + (ahead.t * (ahead.which ? p.s.k_token_stride : p.s.q_token_stride) + ahead.h * hs + ln.d0) * V::kValue;
            const char* to = static_cast<const char*>(grad) + ((long long)(ahead.t * (ahead.which ? Hk : Hq) + ahead.h) * D + ln.d0) * V::kValue;
            const long long step = hs * V::kValue;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (ln.on && i < ahead.rows) {
                    V::copy(ring.to(4 * i), from + i * step);
                    V::copy(ring.to(4 * i + 1), from + i * step + piece_gap);
                    V::copy(ring.to(4 * i + 2), to + i * D * V::kValue);
                    V::copy(ring.to(4 * i + 3), to + i * D * V::kValue + piece_gap);
                }
            ahead.next(p.s, p.run, stride);
        }
        R::commit();
        ring.in = R::after(ring.in);
    };
#pragma unroll
    for (int i = 0; i < R::kStages - 1; ++i) copy();
    f2 dw[2][4], c[4], s[4], own[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[0][i] = dw[1][i] = f2_all(0.f);
    int token = -1, kind = -1;
    for (; w.more(); w.next(p.s, p.run, stride)) {
        copy();
        if (w.t != token) {
            token = w.t;
            const Place at = place_of<false>(p, token);
            ln.angles(p, at.pos, c, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = f2_mul(s[i], f2_all(-1.f));      // the transposed rotation
        }
        if (w.which != kind) {
            kind = w.which;
            ln.weights(kind ? p.k_weight : p.q_weight, own);
        }
        R::wait();
        f2 x[2][4], du[2][4];
        float ss[2], dot[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f2 g[4], o[4], sum = f2_all(0.f);
            V::get(ring.from(4 * i), x[i][0], x[i][1]);
            V::get(ring.from(4 * i + 1), x[i][2], x[i][3]);
            V::get(ring.from(4 * i + 2), g[0], g[1]);
            V::get(ring.from(4 * i + 3), g[2], g[3]);
            ln.other(g, o, all_turned);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                du[i][k] = f2_fma(o[k], s[k], f2_mul(g[k], c[k]));
                sum = f2_fma(f2_mul(du[i][k], own[k]), x[i][k], sum);
            }
            const float2 t2 = f2_get(sum);
            ss[i] = ln.on ? f2_dot(x[i], x[i]) : 0.f;
            dot[i] = ln.on ? t2.x + t2.y : 0.f;
        }
        ring.out = R::after(ring.out);
        char* into = static_cast<char*>(w.which ? p.k_out : p.q_out) + ((long long)(w.t * (w.which ? Hk : Hq) + w.h) * D + ln.d0) * V::kValue;
        const float mean = sum4<LANES>(ss[0], ss[1], dot[0], dot[1], ln.l, ln.mask) * inv;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float r = rsqrtf(__shfl_sync(ln.mask, mean, i, LANES) + p.s.eps), f = -r * r * __shfl_sync(ln.mask, mean, 2 + i, LANES);
            if (!ln.on || i >= w.rows) continue;
            const f2 r2 = f2_all(r), g2 = f2_all(f);
            f2 y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const f2 t = f2_mul(f2_mul(du[i][k], x[i][k]), r2);
                if (w.which) dw[1][k] = f2_add(dw[1][k], t);
                else dw[0][k] = f2_add(dw[0][k], t);
                y[k] = f2_mul(f2_fma(x[i][k], g2, f2_mul(du[i][k], own[k])), r2);
            }
            V::store(into + i * D * V::kValue, y[0], y[1]);
            V::store(into + i * D * V::kValue + piece_gap, y[2], y[3]);
        }
    }
    if (p.part == nullptr) return;
    asm volatile("cp.async.wait_all;" ::: "memory");
    float* sum = reinterpret_cast<float*>(smem);      // [groups][8 LANES]
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k)
            *reinterpret_cast<float2*>(sum + threadIdx.x / LANES * 8 * LANES + (k < 2 ? ln.d0 : ln.d1 - 4) + 2 * k) = f2_get(dw[which][k]);
        __syncthreads();
        for (int d = threadIdx.x; d < D; d += kThreads) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < kGroups; ++k) v += sum[k * 8 * LANES + d];
            p.part[((size_t)blockIdx.x * 2 + which) * D + d] = v;
        }
    }
}

// Sums of the blocks' parts: 32 columns a block, each warp a share of the parts in their order, then the warps in theirs.
__global__ void __launch_bounds__(1024) norm_rope_dw_kernel(int blocks, int D, const float* part, float* dq_weight, float* dk_weight) {
    __shared__ float sum[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
    dependency_wait();
    float s = 0.f;
    if (e < 2 * D)
#pragma unroll 8
        for (int i = warp; i < blocks; i += 32) s += ld_after_f32(part + (size_t)i * 2 * D + e);
    sum[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && e < 2 * D) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += sum[i][lane];
        float* out = e < D ? dq_weight : dk_weight;
        if (out != nullptr) out[e < D ? e : e - D] = s;
    }
}

int check(const KdaRotaryShape* s) {
    if (!s) return KDA_ERR_NULL;
    if (s->tokens < 0 || s->q_heads <= 0 || s->kv_heads <= 0 || s->head_dim <= 0 || s->rotary_dim < 0 || s->table_len <= 0) return KDA_ERR_BAD_SHAPE;
    if (s->head_dim > KDA_MAX_DIM || s->rotary_dim > s->head_dim || s->rotary_dim % 2 != 0) return KDA_ERR_BAD_SHAPE;
    if ((long long)s->tokens * (s->q_heads + 2ll * s->kv_heads) >= 1ll << 31) return KDA_ERR_BAD_SHAPE;
    if (s->io_dtype != KDA_DTYPE_F32 && s->io_dtype != KDA_DTYPE_BF16) return KDA_ERR_UNSUPPORTED;
    return KDA_OK;
}

int blocks_for(long long units, int per_block, int per_sm) {
    const long long most = 148ll * per_sm, want = (units + per_block - 1) / per_block;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

bool on16(std::initializer_list<const void*> ps) {
    uintptr_t a = 0;
    for (const void* p : ps) a |= reinterpret_cast<uintptr_t>(p);
    return a % 16 == 0;
}
// Whether rows can be taken in pieces of eight values: the width, what is rotated, and every address and stride.
bool rows8(const Rope& p, std::initializer_list<long long> strides) {
    const KdaRotaryShape& s = p.s;
    const int unit = s.io_dtype == KDA_DTYPE_BF16 ? 8 : 4;      // elements in 16 bytes
    long long all = 0;
    for (long long x : strides) all |= x;
    return s.head_dim % 8 == 0 && s.rotary_dim % 8 == 0 && all % unit == 0 &&
           on16({p.q, p.k, p.v, p.cos, p.sin, p.q_weight, p.k_weight, p.q_out, p.k_out, p.v_out, p.d_q, p.d_k});
}
int lanes_for(int dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }
// How many pieces a group takes in a row, and the blocks: a token's while the machine is full all the same, one where it is not.
int runs_for(Rope& p, int each, int lanes) {
    const long long pieces = (long long)p.s.tokens * each, groups = 148ll * kBlocks * (kThreads / lanes);
    p.run = (int)(pieces >= groups * each ? each : pieces > groups ? pieces / groups : 1);
    const long long runs = (pieces + p.run - 1) / p.run, blocks = (runs + kThreads / lanes - 1) / (kThreads / lanes);
    return (int)(blocks < 1 ? 1 : blocks < 148 * kBlocks ? blocks : 148 * kBlocks);
}
int pieces_of(int heads, int rows) { return (heads + rows - 1) / rows; }
template <class K>
int run_rows(K kern, bool bf16, const Rope& p, int blocks, cudaStream_t st) {
    const size_t bytes = bf16 ? Ring<true>::kBytes : Ring<false>::kBytes;
    if (int rc = set_smem_limit(kern, bytes)) return rc;
    kern<<<blocks, kThreads, bytes, st>>>(p);
    return KDA_OK;
}
template <template <int, bool, bool> class K>
int by_shape(const Rope& p, int blocks, cudaStream_t st) {
    const bool bf = p.s.io_dtype == KDA_DTYPE_BF16, in = p.s.interleaved != 0;
    const int lanes = lanes_for(p.s.head_dim);
#define KDA_ROPE_CASE(L)                                                                                                                            \
    if (lanes == L)                                                                                                                                 \
        return bf ? (in ? run_rows(K<L, true, true>::kernel(), true, p, blocks, st) : run_rows(K<L, true, false>::kernel(), true, p, blocks, st))   \
                  : (in ? run_rows(K<L, false, true>::kernel(), false, p, blocks, st) : run_rows(K<L, false, false>::kernel(), false, p, blocks, st));
    KDA_ROPE_CASE(8) KDA_ROPE_CASE(16) KDA_ROPE_CASE(32)
#undef KDA_ROPE_CASE
    return KDA_ERR_UNSUPPORTED;
}
template <int L, bool B, bool I>
struct Forward {
    static auto kernel() { return norm_rope_rows_kernel<L, B, I, false>; }
};
template <int L, bool B, bool I>
struct Append {
    static auto kernel() { return norm_rope_rows_kernel<L, B, I, true>; }
};
template <int L, bool B, bool I>
struct Backward {
    static auto kernel() { return norm_rope_rows_bwd_kernel<L, B, I>; }
};

Rope fill(const KdaRotaryShape& s, const void* q, const void* k, const float* cos, const float* sin, const void* positions, const float* qw, const float* kw) {
    Rope p = {};
    p.s = s;
    p.q = q; p.k = k; p.cos = cos; p.sin = sin; p.positions = positions; p.q_weight = qw; p.k_weight = kw;
    p.mirror = status_mirror();
    return p;
}

}  // namespace
}  // namespace attn
}  // namespace kda

using namespace kda;
using namespace kda::attn;

extern "C" int kda_norm_rope_fwd(const KdaRotaryShape* s, const void* q, const void* k, const float* cos, const float* sin, const void* positions,
                                 const float* q_weight, const float* k_weight, void* q_out, void* k_out, void* stream) {
    if (int rc = check(s)) return rc;
    if (s->tokens == 0) return KDA_OK;
    if (!positions && s->seq_len <= 0) return KDA_ERR_BAD_SHAPE;
    if (!q || !k || !q_out || !k_out || (s->rotary_dim > 0 && (!cos || !sin))) return KDA_ERR_NULL;
    Rope p = fill(*s, q, k, cos, sin, positions, q_weight, k_weight);
    p.q_out = q_out; p.k_out = k_out;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows8(p, {s->q_token_stride, s->q_head_stride, s->k_token_stride, s->k_head_stride})) {
        const int blocks = runs_for(p, pieces_of(s->q_heads, 4) + pieces_of(s->kv_heads, 4), lanes_for(s->head_dim));
        int rc = KDA_OK;
        KDA_LAUNCH("norm_rope_rows_kernel", st, rc = by_shape<Forward>(p, blocks, st));
        return rc ? rc : launch_status();
    }
    const int blocks = blocks_for((long long)s->tokens * (s->q_heads + s->kv_heads), kWarps, 8);
    KDA_LAUNCH("norm_rope_kernel", st, norm_rope_kernel<false><<<blocks, kThreads, 0, st>>>(p));
    return launch_status();
}

extern "C" size_t kda_norm_rope_bwd_scratch_bytes(const KdaRotaryShape* s) {
    if (check(s)) return 0;
    return align_up((size_t)blocks_for((long long)s->tokens * (s->q_heads + s->kv_heads), 1, kBlocks) * 2 * s->head_dim * sizeof(float), 256);
}

extern "C" int kda_norm_rope_bwd(const KdaRotaryShape* s, const void* q, const void* k, const float* cos, const float* sin, const void* positions,
                                 const float* q_weight, const float* k_weight, const void* d_q_out, const void* d_k_out, void* dq, void* dk,
                                 float* dq_weight, float* dk_weight, void* scratch, size_t scratch_bytes, void* stream) {
    if (int rc = check(s)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (s->tokens > 0) {
        if (!positions && s->seq_len <= 0) return KDA_ERR_BAD_SHAPE;
        if (!q || !k || !d_q_out || !d_k_out || !dq || !dk || (s->rotary_dim > 0 && (!cos || !sin))) return KDA_ERR_NULL;
    }
    const bool sums = dq_weight != nullptr || dk_weight != nullptr;
    if (sums && (!scratch || reinterpret_cast<uintptr_t>(scratch) % 256 != 0 || scratch_bytes < kda_norm_rope_bwd_scratch_bytes(s))) return KDA_ERR_WORKSPACE;
    Rope p = fill(*s, q, k, cos, sin, positions, q_weight, k_weight);
    p.q_out = dq; p.k_out = dk; p.d_q = d_q_out; p.d_k = d_k_out;
    p.part = sums ? static_cast<float*>(scratch) : nullptr;
    int blocks;
    if (rows8(p, {s->q_token_stride, s->q_head_stride, s->k_token_stride, s->k_head_stride})) {
        blocks = runs_for(p, pieces_of(s->q_heads, 2) + pieces_of(s->kv_heads, 2), lanes_for(s->head_dim));
        int rc = KDA_OK;
        KDA_LAUNCH("norm_rope_rows_bwd_kernel", st, rc = by_shape<Backward>(p, blocks, st));
        if (rc) return rc;
    } else {
        blocks = blocks_for((long long)s->tokens * (s->q_heads + s->kv_heads), kWarps, kBlocks);
        KDA_LAUNCH("norm_rope_bwd_kernel", st, norm_rope_bwd_kernel<<<blocks, kThreads, 0, st>>>(p));
    }
    if (int rc = launch_status()) return rc;
    if (!sums) return KDA_OK;
    cudaError_t e = cudaSuccess;
    KDA_LAUNCH("norm_rope_dw_kernel", st,
               e = launch_early(norm_rope_dw_kernel, dim3((2 * s->head_dim + 31) / 32), 1024, 0, st, true, 1, blocks, s->head_dim, p.part, dq_weight, dk_weight));
    return e == cudaSuccess ? launch_status() : KDA_ERR_CUDA;
}

extern "C" int kda_norm_rope_append(const KdaRotaryShape* s, const KdaPagedShape* g, const void* q, const void* k, const void* v, const float* cos,
                                    const float* sin, const float* q_weight, const float* k_weight, const int32_t* block_table, const int32_t* kv_lens,
                                    const int32_t* cu_seqlens, void* q_out, void* k_cache, void* v_cache, void* stream) {
    if (int rc = check(s)) return rc;
    if (!g) return KDA_ERR_NULL;
    if (g->tokens != s->tokens || g->q_heads != s->q_heads || g->kv_heads != s->kv_heads || g->head_dim != s->head_dim || g->io_dtype != s->io_dtype ||
        g->n_seq <= 0 || g->n_pages < 0 || g->page_size <= 0 || g->table_width < 0 || (long long)g->table_width * g->page_size >= 1ll << 31)
        return KDA_ERR_BAD_SHAPE;
    if (!cu_seqlens && g->tokens % g->n_seq != 0) return KDA_ERR_BAD_SHAPE;
    if (s->tokens == 0) return KDA_OK;
    if (!q || !k || !v || !kv_lens || !q_out || (s->rotary_dim > 0 && (!cos || !sin))) return KDA_ERR_NULL;
    if (g->table_width > 0 && (!block_table || (g->n_pages > 0 && (!k_cache || !v_cache)))) return KDA_ERR_NULL;
    Rope p = fill(*s, q, k, cos, sin, nullptr, q_weight, k_weight);
    p.v = v; p.q_out = q_out; p.k_out = k_cache; p.v_out = v_cache;
    p.batch = Batch{block_table, kv_lens, cu_seqlens, p.mirror, g->table_stride, g->n_seq, g->tokens, cu_seqlens ? 0 : g->tokens / g->n_seq,
                    g->n_pages, g->page_size, g->table_width, g->padded};
    p.cache = Strides{0, 0, g->k_page_stride, g->k_row_stride, g->k_head_stride, g->v_page_stride, g->v_row_stride, g->v_head_stride};
    cudaStream_t st = (cudaStream_t)stream;
    if (rows8(p, {s->q_token_stride, s->q_head_stride, s->k_token_stride, s->k_head_stride, s->v_token_stride, s->v_head_stride, g->k_page_stride, g->k_row_stride,
                  g->k_head_stride, g->v_page_stride, g->v_row_stride, g->v_head_stride})) {
        const int blocks = runs_for(p, pieces_of(s->q_heads, 4) + 2 * pieces_of(s->kv_heads, 4), lanes_for(s->head_dim));
        int rc = KDA_OK;
        KDA_LAUNCH("norm_rope_append_rows_kernel", st, rc = by_shape<Append>(p, blocks, st));
        return rc ? rc : launch_status();
    }
    const int blocks = blocks_for((long long)s->tokens * (s->q_heads + 2 * s->kv_heads), kWarps, 8);
    KDA_LAUNCH("norm_rope_append_kernel", st, norm_rope_kernel<true><<<blocks, kThreads, 0, st>>>(p));
    return launch_status();
}
