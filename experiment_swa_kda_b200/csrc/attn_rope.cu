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
// Bound by memory.  Two forms each way: norm_rope_rows_* for widths, strides and addresses that allow wide accesses, and
// norm_rope_kernel / norm_rope_bwd_kernel for all others.

#include <initializer_list>

#include "attn.cuh"

namespace kda {
namespace attn {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
#ifndef V_BG
#define V_BG 2
#define V_FG 3
#endif
constexpr int kFwdBlocks = V_FG;
constexpr int kBwdBlocks = V_BG;      // blocks an SM of the backward: each leaves one part of the weights' gradients

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
    int slice, slices;              // norm_rope_rows_*: heads of a token a group of lanes takes, and groups a token has
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

#ifndef V_FB
#define V_FB 3
#define V_BB 2
#endif
// ---------------------------------------------------------------------------------------------- eight values a lane
// LANES lanes a row, and both members of a pair in one lane: two pieces of four adjacent values, half the rotated width apart in the
// split order.  A group of lanes takes a token's heads one after the other - all of them, or a slice where there are too few
// tokens to fill the machine -, so that the token's place, its cosines and sines and the weights are read once for all of them.
// What bounds such a loop after memory is issue and the shuffles of the rows' sums, so rows go four at a time (backward two, with
// two sums each) and their four sums are reduced together: 5 shuffles, not 16, and 4 that hand them out.

// values [0..3], [4..7] of a lane
template <bool BF16>
struct Vec8;
template <>
struct Vec8<true> {
    uint2 a, b;
    __device__ __forceinline__ void load(const void* p, long long at0, long long at1) {
        a = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + at0));
        b = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + at1));
    }
    __device__ __forceinline__ void zero() { a = b = make_uint2(0, 0); }
    __device__ __forceinline__ void get(f2 (&x)[4]) const {
        x[0] = f2_from_bf16(a.x); x[1] = f2_from_bf16(a.y); x[2] = f2_from_bf16(b.x); x[3] = f2_from_bf16(b.y);
    }
    static __device__ __forceinline__ void store(void* p, long long at0, long long at1, const f2 (&x)[4]) {
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p) + at0) = make_uint2(f2_to_bf16(x[0]), f2_to_bf16(x[1]));
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p) + at1) = make_uint2(f2_to_bf16(x[2]), f2_to_bf16(x[3]));
    }
};
template <>
struct Vec8<false> {
    float4 a, b;
    __device__ __forceinline__ void load(const void* p, long long at0, long long at1) {
        a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + at0));
        b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + at1));
    }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void get(f2 (&x)[4]) const {
        x[0] = f2_make(a.x, a.y); x[1] = f2_make(a.z, a.w); x[2] = f2_make(b.x, b.y); x[3] = f2_make(b.z, b.w);
    }
    static __device__ __forceinline__ void store(void* p, long long at0, long long at1, const f2 (&x)[4]) {
        const float2 a = f2_get(x[0]), b = f2_get(x[1]), c = f2_get(x[2]), e = f2_get(x[3]);
        *reinterpret_cast<float4*>(static_cast<float*>(p) + at0) = make_float4(a.x, a.y, b.x, b.y);
        *reinterpret_cast<float4*>(static_cast<float*>(p) + at1) = make_float4(c.x, c.y, e.x, e.y);
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

// `heads` rows of one token from `from` on, from_stride apart, to `to`, to_stride apart: y = r (x a + x_other b)
template <int LANES, bool BF16, bool INTER>
__device__ __forceinline__ void turn_rows(const Lane<LANES, INTER>& ln, const KdaRotaryShape& sh, const void* src, long long from, long long from_stride, void* dst,
                                          long long to, long long to_stride, int heads, const f2 (&a)[4], const f2 (&b)[4]) {
    const bool all_turned = sh.rotary_dim == sh.head_dim;
    const float inv = 1.f / sh.head_dim;
    for (int h = 0; h < heads; h += 4) {
        Vec8<BF16> v[4];
        f2 x[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i].zero();
            if (ln.on && h + i < heads) v[i].load(src, from + (h + i) * from_stride + ln.d0, from + (h + i) * from_stride + ln.d1);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i].get(x[i]);
        const float r = rsqrtf(fmaf(sum4<LANES>(f2_dot(x[0], x[0]), f2_dot(x[1], x[1]), f2_dot(x[2], x[2]), f2_dot(x[3], x[3]), ln.l, ln.mask), inv, sh.eps));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f2 r2 = f2_all(__shfl_sync(ln.mask, r, i, LANES));
            f2 o[4], y[4];
            ln.other(x[i], o, all_turned);
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = f2_mul(f2_fma(x[i][k], a[k], f2_mul(o[k], b[k])), r2);
            if (ln.on && h + i < heads) Vec8<BF16>::store(dst, to + (h + i) * to_stride + ln.d0, to + (h + i) * to_stride + ln.d1, y);
        }
    }
}

template <int LANES, bool BF16, bool INTER, bool APPEND>
__global__ void __launch_bounds__(kThreads, V_FB) norm_rope_rows_kernel(Rope p) {
    constexpr int kGroups = kThreads / LANES;
    const Lane<LANES, INTER> ln(p.s);
    const int Hq = p.s.q_heads, Hk = p.s.kv_heads, all = Hq + Hk + (APPEND ? Hk : 0), D = p.s.head_dim;
    const long long units = (long long)p.s.tokens * p.slices;
    for (long long unit = (long long)blockIdx.x * kGroups + threadIdx.x / LANES; unit < units; unit += (long long)gridDim.x * kGroups) {
        const int t = (int)(unit / p.slices), h0 = (int)(unit - (long long)t * p.slices) * p.slice, h1 = min(h0 + p.slice, all);
        const Place at = place_of<APPEND, LANES>(p, t, ln.l, ln.mask);
        f2 c[4], s[4];
        ln.angles(p, max(at.pos, 0), c, s);
        // u_e c + u_other s with u = x r w: a = w_e c, b = w_other s
        auto coefficients = [&](const float* w, f2 (&a)[4], f2 (&b)[4]) {
            f2 own[4];
            ln.weights(w, own);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = f2_mul(own[i], c[i]);
                b[i] = f2_mul(INTER ? swapped(own[i]) : own[i ^ 2], s[i]);
            }
        };
        f2 a[4], b[4];
        if (h0 < Hq) {
            const int n = min(h1, Hq) - h0;
            const long long to = ((long long)t * Hq + h0) * D;
            if (APPEND && at.pos < 0) {
                const f2 none[4] = {f2_all(0.f), f2_all(0.f), f2_all(0.f), f2_all(0.f)};
                for (int h = 0; h < n; ++h)
                    if (ln.on) Vec8<BF16>::store(p.q_out, to + (long long)h * D + ln.d0, to + (long long)h * D + ln.d1, none);
            } else {
                coefficients(p.q_weight, a, b);
                turn_rows<LANES, BF16>(ln, p.s, p.q, t * p.s.q_token_stride + h0 * p.s.q_head_stride, p.s.q_head_stride, p.q_out, to, D, n, a, b);
            }
        }
        if (APPEND && (at.pos < 0 || at.k_at < 0)) continue;
        const int k0 = max(h0 - Hq, 0), k1 = min(h1 - Hq, Hk);
        if (k0 < k1) {
            coefficients(p.k_weight, a, b);
            turn_rows<LANES, BF16>(ln, p.s, p.k, t * p.s.k_token_stride + k0 * p.s.k_head_stride, p.s.k_head_stride, p.k_out,
                                   APPEND ? at.k_at + k0 * p.cache.k_head : ((long long)t * Hk + k0) * D, APPEND ? p.cache.k_head : D, k1 - k0, a, b);
        }
        if (APPEND && ln.on) {      // values go as they are
            for (int v = max(h0 - Hq - Hk, 0); v < h1 - Hq - Hk; ++v) {
                Vec8<BF16> x;
                f2 y[4];
                x.load(p.v, t * p.s.v_token_stride + v * p.s.v_head_stride + ln.d0, t * p.s.v_token_stride + v * p.s.v_head_stride + ln.d1);
                x.get(y);
                Vec8<BF16>::store(p.v_out, at.v_at + v * p.cache.v_head + ln.d0, at.v_at + v * p.cache.v_head + ln.d1, y);
            }
        }
    }
}

// The same rows backward; each lane sums its weights' gradients over all rows it meets, a block over its lanes, and
// norm_rope_dw_kernel over the blocks, all in a fixed order.
template <int LANES, bool BF16, bool INTER>
__global__ void __launch_bounds__(kThreads, V_BB) norm_rope_rows_bwd_kernel(Rope p) {
    constexpr int kGroups = kThreads / LANES;
    dependents_go();
    const Lane<LANES, INTER> ln(p.s);
    const int Hq = p.s.q_heads, Hk = p.s.kv_heads, all = Hq + Hk, D = p.s.head_dim;
    const bool all_turned = p.s.rotary_dim == D;
    const float inv = 1.f / D;
    const long long units = (long long)p.s.tokens * p.slices;
    f2 dw[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[0][i] = dw[1][i] = f2_all(0.f);
    for (long long unit = (long long)blockIdx.x * kGroups + threadIdx.x / LANES; unit < units; unit += (long long)gridDim.x * kGroups) {
        const int t = (int)(unit / p.slices), h0 = (int)(unit - (long long)t * p.slices) * p.slice, h1 = min(h0 + p.slice, all);
        const Place at = place_of<false>(p, t);
        f2 c[4], s[4];
        ln.angles(p, at.pos, c, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = f2_mul(s[i], f2_all(-1.f));      // the transposed rotation
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const int H = which ? Hk : Hq, a0 = which ? max(h0 - Hq, 0) : h0, a1 = which ? h1 - Hq : min(h1, Hq);
            if (a0 >= a1) continue;
            const long long hs = which ? p.s.k_head_stride : p.s.q_head_stride;
            const long long from = t * (which ? p.s.k_token_stride : p.s.q_token_stride), to = (long long)t * H * D;
            const void *src = which ? p.k : p.q, *grad = which ? p.d_k : p.d_q;
            void* dst = which ? p.k_out : p.q_out;
            f2 own[4];
            ln.weights(which ? p.k_weight : p.q_weight, own);
            for (int h = a0; h < a1; h += 2) {
                Vec8<BF16> xv[2], gv[2];
                f2 x[2][4], du[2][4];
                float ss[2], dot[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    xv[i].zero();
                    gv[i].zero();
                    if (ln.on && h + i < a1) {
                        xv[i].load(src, from + (h + i) * hs + ln.d0, from + (h + i) * hs + ln.d1);
                        gv[i].load(grad, to + (long long)(h + i) * D + ln.d0, to + (long long)(h + i) * D + ln.d1);
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    f2 o[4];
                    xv[i].get(x[i]);
                    gv[i].get(du[i]);
                    ln.other(du[i], o, all_turned);
                    ss[i] = f2_dot(x[i], x[i]);
                    f2 sum = f2_all(0.f);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const f2 d = f2_fma(o[k], s[k], f2_mul(du[i][k], c[k]));
                        sum = f2_fma(f2_mul(d, own[k]), x[i][k], sum);
                        du[i][k] = d;
                    }
                    const float2 t2 = f2_get(sum);
                    dot[i] = t2.x + t2.y;
                }
                const float mean = sum4<LANES>(ss[0], ss[1], dot[0], dot[1], ln.l, ln.mask) * inv;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float r = rsqrtf(__shfl_sync(ln.mask, mean, i, LANES) + p.s.eps), f = -r * r * __shfl_sync(ln.mask, mean, 2 + i, LANES);
                    const f2 r2 = f2_all(r), g2 = f2_all(f);
                    f2 y[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        dw[which][k] = f2_fma(f2_mul(du[i][k], x[i][k]), r2, dw[which][k]);
                        y[k] = f2_mul(f2_fma(x[i][k], g2, f2_mul(du[i][k], own[k])), r2);
                    }
                    if (ln.on && h + i < a1) Vec8<BF16>::store(dst, to + (long long)(h + i) * D + ln.d0, to + (long long)(h + i) * D + ln.d1, y);
                }
            }
        }
    }
    if (p.part == nullptr) return;
    __shared__ float sum[kGroups][8 * LANES];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) *reinterpret_cast<float2*>(&sum[threadIdx.x / LANES][(k < 2 ? ln.d0 : ln.d1 - 4) + 2 * k]) = f2_get(dw[which][k]);
        __syncthreads();
        for (int d = threadIdx.x; d < D; d += kThreads) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < kGroups; ++k) v += sum[k][d];
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
// Heads of a token a group takes: all of them while that still gives every SM its threads, a part otherwise.
void slice_heads(Rope& p, int heads, int lanes) {
    const long long groups = 148ll * 2048 / lanes;
    long long n = groups / (p.s.tokens > 0 ? p.s.tokens : 1);
    if (n < 1) n = 1;
    if (n > heads) n = heads;
    p.slice = (int)((heads + n - 1) / n);
    p.slices = (heads + p.slice - 1) / p.slice;
}
template <template <int, bool, bool> class K>
void by_shape(const Rope& p, int blocks, cudaStream_t st) {
    const bool bf = p.s.io_dtype == KDA_DTYPE_BF16, in = p.s.interleaved != 0;
    const int lanes = lanes_for(p.s.head_dim);
#define KDA_ROPE_CASE(L)                                                                                             \
    if (lanes == L) {                                                                                                \
        if (bf) in ? K<L, true, true>::run(p, blocks, st) : K<L, true, false>::run(p, blocks, st);                   \
        else in ? K<L, false, true>::run(p, blocks, st) : K<L, false, false>::run(p, blocks, st);                    \
    }
    KDA_ROPE_CASE(8) KDA_ROPE_CASE(16) KDA_ROPE_CASE(32)
#undef KDA_ROPE_CASE

}
template <int L, bool B, bool I>
struct RunForward {
    static void run(const Rope& p, int blocks, cudaStream_t st) { norm_rope_rows_kernel<L, B, I, false><<<blocks, kThreads, 0, st>>>(p); }
};
template <int L, bool B, bool I>
struct RunAppend {
    static void run(const Rope& p, int blocks, cudaStream_t st) { norm_rope_rows_kernel<L, B, I, true><<<blocks, kThreads, 0, st>>>(p); }
};
template <int L, bool B, bool I>
struct RunBackward {
    static void run(const Rope& p, int blocks, cudaStream_t st) { norm_rope_rows_bwd_kernel<L, B, I><<<blocks, kThreads, 0, st>>>(p); }
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
        const int lanes = lanes_for(s->head_dim);
        slice_heads(p, s->q_heads + s->kv_heads, lanes);
        const int blocks = blocks_for((long long)s->tokens * p.slices, kThreads / lanes, kFwdBlocks);
        KDA_LAUNCH("norm_rope_rows_kernel", st, by_shape<RunForward>(p, blocks, st));
        return launch_status();
    }
    const int blocks = blocks_for((long long)s->tokens * (s->q_heads + s->kv_heads), kWarps, 8);
    KDA_LAUNCH("norm_rope_kernel", st, norm_rope_kernel<false><<<blocks, kThreads, 0, st>>>(p));
    return launch_status();
}

extern "C" size_t kda_norm_rope_bwd_scratch_bytes(const KdaRotaryShape* s) {
    if (check(s)) return 0;
    return align_up((size_t)blocks_for((long long)s->tokens * (s->q_heads + s->kv_heads), 1, kBwdBlocks) * 2 * s->head_dim * sizeof(float), 256);
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
        const int lanes = lanes_for(s->head_dim);
        slice_heads(p, s->q_heads + s->kv_heads, lanes);
        blocks = blocks_for((long long)s->tokens * p.slices, kThreads / lanes, kBwdBlocks);
        KDA_LAUNCH("norm_rope_rows_bwd_kernel", st, by_shape<RunBackward>(p, blocks, st));
    } else {
        blocks = blocks_for((long long)s->tokens * (s->q_heads + s->kv_heads), kWarps, kBwdBlocks);
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
    if (g->n_pages > 0 && g->table_width > 0 && (!block_table || !k_cache || !v_cache)) return KDA_ERR_NULL;
    Rope p = fill(*s, q, k, cos, sin, nullptr, q_weight, k_weight);
    p.v = v; p.q_out = q_out; p.k_out = k_cache; p.v_out = v_cache;
    p.batch = Batch{block_table, kv_lens, cu_seqlens, p.mirror, g->table_stride, g->n_seq, g->tokens, cu_seqlens ? 0 : g->tokens / g->n_seq,
                    g->n_pages, g->page_size, g->table_width};
    p.cache = Strides{0, 0, g->k_page_stride, g->k_row_stride, g->k_head_stride, g->v_page_stride, g->v_row_stride, g->v_head_stride};
    cudaStream_t st = (cudaStream_t)stream;
    if (rows8(p, {s->q_token_stride, s->q_head_stride, s->k_token_stride, s->k_head_stride, s->v_token_stride, s->v_head_stride, g->k_page_stride, g->k_row_stride,
                  g->k_head_stride, g->v_page_stride, g->v_row_stride, g->v_head_stride})) {
        const int lanes = lanes_for(s->head_dim);
        slice_heads(p, s->q_heads + 2 * s->kv_heads, lanes);
        const int blocks = blocks_for((long long)s->tokens * p.slices, kThreads / lanes, kFwdBlocks);
        KDA_LAUNCH("norm_rope_append_rows_kernel", st, by_shape<RunAppend>(p, blocks, st));
        return launch_status();
    }
    const int blocks = blocks_for((long long)s->tokens * (s->q_heads + 2 * s->kv_heads), kWarps, 8);
    KDA_LAUNCH("norm_rope_append_kernel", st, norm_rope_kernel<true><<<blocks, kThreads, 0, st>>>(p));
    return launch_status();
}
