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
// Bound by memory.  Two forms each way: norm_rope_rows_* for widths, strides and addresses that allow 16-byte accesses, and
// norm_rope_kernel / norm_rope_bwd_kernel for all others.

#include <initializer_list>

#include "attn.cuh"

namespace kda {
namespace attn {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBwdBlocks = 4;      // blocks an SM of the backward: each leaves one part of the weights' gradients

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

// ---------------------------------------------------------------------------------------------- 16-byte accesses
// Eight adjacent values a lane, LANES lanes a row.  A group of lanes takes a token's heads one after the other - all of them, or a
// slice where there are too few tokens to fill the machine -, so that the token's place, its cosines and sines and the
// weights are read once for all of them.  In the split order a pair's members lie in two lanes and change places by shuffle, as
// they were loaded: bf16 pairs in one word.

template <bool BF16>
struct Vec8 {
    uint4 a, b;      // b: float32 only
};
template <bool BF16>
__device__ __forceinline__ Vec8<BF16> ld8(const void* p, long long at) {
    Vec8<BF16> r;
    if (BF16) {
        r.a = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + at));
    } else {
        const uint4* s = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + at);
        r.a = __ldg(s);
        r.b = __ldg(s + 1);
    }
    return r;
}
template <bool BF16>
__device__ __forceinline__ void unpack(const Vec8<BF16>& v, f2 (&x)[4]) {
    if (BF16) {
        x[0] = f2_from_bf16(v.a.x); x[1] = f2_from_bf16(v.a.y); x[2] = f2_from_bf16(v.a.z); x[3] = f2_from_bf16(v.a.w);
    } else {
        x[0] = f2_make(__uint_as_float(v.a.x), __uint_as_float(v.a.y));
        x[1] = f2_make(__uint_as_float(v.a.z), __uint_as_float(v.a.w));
        x[2] = f2_make(__uint_as_float(v.b.x), __uint_as_float(v.b.y));
        x[3] = f2_make(__uint_as_float(v.b.z), __uint_as_float(v.b.w));
    }
}
template <bool BF16>
__device__ __forceinline__ void st8(void* p, long long at, const f2 (&x)[4]) {
    if (BF16) {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p) + at) = make_uint4(f2_to_bf16(x[0]), f2_to_bf16(x[1]), f2_to_bf16(x[2]), f2_to_bf16(x[3]));
    } else {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
        const float2 a = f2_get(x[0]), b = f2_get(x[1]), c = f2_get(x[2]), e = f2_get(x[3]);
        d[0] = make_float4(a.x, a.y, b.x, b.y);
        d[1] = make_float4(c.x, c.y, e.x, e.y);
    }
}
template <bool BF16>
__device__ __forceinline__ Vec8<BF16> shuffle(const Vec8<BF16>& v, int src, int lanes, unsigned mask) {
    Vec8<BF16> r;
    r.a = make_uint4(__shfl_sync(mask, v.a.x, src, lanes), __shfl_sync(mask, v.a.y, src, lanes), __shfl_sync(mask, v.a.z, src, lanes),
                     __shfl_sync(mask, v.a.w, src, lanes));
    if (!BF16)
        r.b = make_uint4(__shfl_sync(mask, v.b.x, src, lanes), __shfl_sync(mask, v.b.y, src, lanes), __shfl_sync(mask, v.b.z, src, lanes),
                         __shfl_sync(mask, v.b.w, src, lanes));
    return r;
}
template <int LANES>
__device__ __forceinline__ float group_sum(float x, unsigned mask) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) x += __shfl_xor_sync(mask, x, o);
    return x;
}

// A lane's share of a row: its values, where their partners are, their weights and the partners'.
template <int LANES, bool INTER>
struct Lane {
    int l, d, src;                  // lane of the group, its first value, lane that holds the partners
    bool on, turned;                // the row has these values; they are rotated
    unsigned mask;
    int at;                         // first of its cosines
    float sign;                     // of the sine in y (split order)

    __device__ __forceinline__ Lane(const KdaRotaryShape& s) {
        const int lane = threadIdx.x & 31;
        l = lane & (LANES - 1);
        mask = LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1u) << (lane & ~(LANES - 1));
        d = 8 * l;
        on = d < s.head_dim;
        turned = d < s.rotary_dim;
        src = l;
        at = INTER ? d / 2 : 0;
        sign = 0.f;
        if (!INTER && turned) {
            const int half = s.rotary_dim / 2;
            src = d < half ? l + half / 8 : l - half / 8;
            at = d < half ? d : d - half;
            sign = d < half ? -1.f : 1.f;
        }
    }
    // y_e = u_e c_e + u_other s_e for the lane's values
    __device__ __forceinline__ void angles(const Rope& p, int pos, f2 (&c)[4], f2 (&s)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c[i] = f2_all(1.f);
            s[i] = f2_all(0.f);
        }
        if (!turned) return;
        const float* pc = p.cos + (size_t)pos * (p.s.rotary_dim / 2) + at;
        const float* ps = p.sin + (size_t)pos * (p.s.rotary_dim / 2) + at;
        const float4 c0 = __ldg(reinterpret_cast<const float4*>(pc)), s0 = __ldg(reinterpret_cast<const float4*>(ps));
        if (INTER) {
            c[0] = f2_all(c0.x); c[1] = f2_all(c0.y); c[2] = f2_all(c0.z); c[3] = f2_all(c0.w);
            s[0] = f2_make(-s0.x, s0.x); s[1] = f2_make(-s0.y, s0.y); s[2] = f2_make(-s0.z, s0.z); s[3] = f2_make(-s0.w, s0.w);
        } else {
            const float4 c1 = __ldg(reinterpret_cast<const float4*>(pc) + 1), s1 = __ldg(reinterpret_cast<const float4*>(ps) + 1);
            c[0] = f2_make(c0.x, c0.y); c[1] = f2_make(c0.z, c0.w); c[2] = f2_make(c1.x, c1.y); c[3] = f2_make(c1.z, c1.w);
            s[0] = f2_make(sign * s0.x, sign * s0.y); s[1] = f2_make(sign * s0.z, sign * s0.w);
            s[2] = f2_make(sign * s1.x, sign * s1.y); s[3] = f2_make(sign * s1.z, sign * s1.w);
        }
    }
    // the weights of values d .. d + 7, 1 without weights
    __device__ __forceinline__ void weights(const float* w, int d0, f2 (&x)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = f2_all(1.f);
        if (w == nullptr || !on) return;
        const float4 a = __ldg(reinterpret_cast<const float4*>(w + d0)), b = __ldg(reinterpret_cast<const float4*>(w + d0) + 1);
        x[0] = f2_make(a.x, a.y); x[1] = f2_make(a.z, a.w); x[2] = f2_make(b.x, b.y); x[3] = f2_make(b.z, b.w);
    }
    // the partners of a lane's values
    template <bool BF16>
    __device__ __forceinline__ void other(const Vec8<BF16>& v, const f2 (&x)[4], f2 (&o)[4]) const {
        if (INTER) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 t = f2_get(x[i]);
                o[i] = f2_make(t.y, t.x);
            }
        } else {
            unpack<BF16>(shuffle<BF16>(v, src, LANES, mask), o);
        }
    }
};

__device__ __forceinline__ float f2_sum(const f2 (&x)[4], const f2 (&y)[4]) {
    const float2 t = f2_get(f2_fma(x[0], y[0], f2_fma(x[1], y[1], f2_fma(x[2], y[2], f2_mul(x[3], y[3])))));
    return t.x + t.y;
}

constexpr int kAhead = 4;      // rows whose loads are in flight together

// `heads` rows of one token from `from` on, head_stride apart, to `to`, to_stride apart
template <int LANES, bool BF16, bool INTER>
__device__ __forceinline__ void turn_rows(const Lane<LANES, INTER>& ln, const KdaRotaryShape& sh, const void* src, long long from, long long from_stride, void* dst,
                                          long long to, long long to_stride, int heads, const f2 (&a)[4], const f2 (&b)[4]) {
    for (int h = 0; h < heads; h += kAhead) {
        Vec8<BF16> v[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            v[i].a = v[i].b = make_uint4(0, 0, 0, 0);
            if (ln.on && h + i < heads) v[i] = ld8<BF16>(src, from + (h + i) * from_stride + ln.d);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (h + i >= heads) break;      // the same for all lanes of the group
            f2 x[4], o[4];
            unpack<BF16>(v[i], x);
            ln.template other<BF16>(v[i], x, o);
            const float r = rsqrtf(group_sum<LANES>(f2_sum(x, x), ln.mask) / sh.head_dim + sh.eps);
            const f2 r2 = f2_all(r);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = f2_mul(f2_fma(x[k], a[k], f2_mul(o[k], b[k])), r2);
            if (ln.on) st8<BF16>(dst, to + (h + i) * to_stride + ln.d, x);
        }
    }
}

template <int LANES, bool BF16, bool INTER, bool APPEND>
__global__ void __launch_bounds__(kThreads) norm_rope_rows_kernel(Rope p) {
    constexpr int kGroups = kThreads / LANES;
    const Lane<LANES, INTER> ln(p.s);
    const int Hq = p.s.q_heads, Hk = p.s.kv_heads, all = Hq + Hk + (APPEND ? Hk : 0), D = p.s.head_dim;
    const long long units = (long long)p.s.tokens * p.slices;
    for (long long unit = (long long)blockIdx.x * kGroups + threadIdx.x / LANES; unit < units; unit += (long long)gridDim.x * kGroups) {
        const int t = (int)(unit / p.slices), h0 = (int)(unit - (long long)t * p.slices) * p.slice, h1 = min(h0 + p.slice, all);
        const Place at = place_of<APPEND, LANES>(p, t, ln.l, ln.mask);
        f2 c[4], s[4];
        ln.angles(p, max(at.pos, 0), c, s);
        // y = r (x (w c) + x_other (w_other s))
        auto coefficients = [&](const float* w, f2 (&a)[4], f2 (&b)[4]) {
            f2 own[4], other[4];
            ln.weights(w, ln.d, own);
            if (INTER) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 x = f2_get(own[i]);
                    other[i] = f2_make(x.y, x.x);
                }
            } else {
                ln.weights(w, 8 * ln.src, other);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = f2_mul(own[i], c[i]);
                b[i] = f2_mul(other[i], s[i]);
            }
        };
        f2 a[4], b[4];
        if (h0 < Hq) {
            const int n = min(h1, Hq) - h0;
            const long long to = ((long long)t * Hq + h0) * D;
            if (APPEND && at.pos < 0) {
                const f2 none[4] = {f2_all(0.f), f2_all(0.f), f2_all(0.f), f2_all(0.f)};
                for (int h = 0; h < n; ++h)
                    if (ln.on) st8<BF16>(p.q_out, to + (long long)h * D + ln.d, none);
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
                f2 x[4];
                unpack<BF16>(ld8<BF16>(p.v, t * p.s.v_token_stride + v * p.s.v_head_stride + ln.d), x);
                st8<BF16>(p.v_out, at.v_at + v * p.cache.v_head + ln.d, x);
            }
        }
    }
}

// The same rows backward; each lane sums its weights' gradients over all rows it meets, a block over its lanes, and
// norm_rope_dw_kernel over the blocks, all in a fixed order.
template <int LANES, bool BF16, bool INTER>
__global__ void __launch_bounds__(kThreads) norm_rope_rows_bwd_kernel(Rope p) {
    constexpr int kGroups = kThreads / LANES, kRowsAhead = BF16 ? 2 : 1;
    dependents_go();
    const Lane<LANES, INTER> ln(p.s);
    const int Hq = p.s.q_heads, Hk = p.s.kv_heads, all = Hq + Hk, D = p.s.head_dim;
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
            const long long ts = which ? p.s.k_token_stride : p.s.q_token_stride, hs = which ? p.s.k_head_stride : p.s.q_head_stride;
            const void *src = which ? p.k : p.q, *grad = which ? p.d_k : p.d_q;
            void* dst = which ? p.k_out : p.q_out;
            const float* w = which ? p.k_weight : p.q_weight;
            f2 own[4];
            ln.weights(w, ln.d, own);
            for (int h = a0; h < a1; h += kRowsAhead) {
                Vec8<BF16> xv[kRowsAhead], gv[kRowsAhead];
#pragma unroll
                for (int i = 0; i < kRowsAhead; ++i) {
                    xv[i].a = xv[i].b = gv[i].a = gv[i].b = make_uint4(0, 0, 0, 0);
                    if (ln.on && h + i < a1) {
                        xv[i] = ld8<BF16>(src, t * ts + (h + i) * hs + ln.d);
                        gv[i] = ld8<BF16>(grad, ((long long)t * H + h + i) * D + ln.d);
                    }
                }
#pragma unroll
                for (int i = 0; i < kRowsAhead; ++i) {
                    if (h + i >= a1) break;
                    f2 x[4], du[4], o[4];
                    unpack<BF16>(xv[i], x);
                    unpack<BF16>(gv[i], du);
                    ln.template other<BF16>(gv[i], du, o);
#pragma unroll
                    for (int k = 0; k < 4; ++k) du[k] = f2_fma(du[k], c[k], f2_mul(o[k], s[k]));
                    const float ss = group_sum<LANES>(f2_sum(x, x), ln.mask);
                    const float r = rsqrtf(ss / D + p.s.eps);
                    const f2 r2 = f2_all(r);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        dw[which][k] = f2_fma(f2_mul(du[k], x[k]), r2, dw[which][k]);
                        du[k] = f2_mul(du[k], own[k]);
                    }
                    const f2 f = f2_all(-r * r * group_sum<LANES>(f2_sum(du, x), ln.mask) / D);
#pragma unroll
                    for (int k = 0; k < 4; ++k) du[k] = f2_mul(f2_fma(x[k], f, du[k]), r2);
                    if (ln.on) st8<BF16>(dst, ((long long)t * H + h + i) * D + ln.d, du);
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
        for (int k = 0; k < 4; ++k) *reinterpret_cast<float2*>(&sum[threadIdx.x / LANES][ln.d + 2 * k]) = f2_get(dw[which][k]);
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
    return s.head_dim % 8 == 0 && s.rotary_dim % (s.interleaved ? 8 : 16) == 0 && all % unit == 0 &&
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
        const int blocks = blocks_for((long long)s->tokens * p.slices, kThreads / lanes, 16);
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
        const int blocks = blocks_for((long long)s->tokens * p.slices, kThreads / lanes, 16);
        KDA_LAUNCH("norm_rope_append_rows_kernel", st, by_shape<RunAppend>(p, blocks, st));
        return launch_status();
    }
    const int blocks = blocks_for((long long)s->tokens * (s->q_heads + 2 * s->kv_heads), kWarps, 8);
    KDA_LAUNCH("norm_rope_append_kernel", st, norm_rope_kernel<true><<<blocks, kThreads, 0, st>>>(p));
    return launch_status();
}
