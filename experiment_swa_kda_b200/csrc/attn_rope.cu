// Per-head RMS norm of queries and keys with the rotation by position in the same pass, forward and backward, and the form
// that puts a serving batch's keys and values into their pages.
//
//   u = x r w, r = (mean x^2 + eps)^-1/2;   y_a = u_a c - u_b s, y_b = u_b c + u_a s for a pair (a, b)
//   backward: du_a = dy_a c + dy_b s, du_b = dy_b c - dy_a s;  dw = sum over rows of du x r;
//             dx = r (w du - x r^2 mean(w du x))
//
// Everything is float32 between the load and the one rounding of the store.  r is formed again in the backward: it costs a sum
// over values that are in registers anyway, a saved one would be read.

#include "attn.cuh"

namespace kda {
namespace attn {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

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
};

// Where a token goes: its position, and the cache rows of its key and value (append).
struct Place {
    int pos;                        // negative: padding
    long long k_at, v_at;           // element offsets of the page's row, or -1: no page
};

template <bool APPEND>
__device__ __forceinline__ Place place_of(const Rope& p, int t) {
    Place r;
    if (APPEND) {
        const Batch& b = p.batch;
        const int n = b.seq_of(t);
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

// Sums of the blocks' parts, in their order: a warp a column.
__global__ void __launch_bounds__(kThreads) norm_rope_dw_kernel(int blocks, int D, const float* part, float* dq_weight, float* dk_weight) {
    const int e = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (e >= 2 * D) return;
    float s = 0.f;
    for (int i = lane; i < blocks; i += 32) s += part[(size_t)i * 2 * D + e];
    s = warp_sum(s);
    float* out = e < D ? dq_weight : dk_weight;
    if (lane == 0 && out != nullptr) out[e < D ? e : e - D] = s;
}

int check(const KdaRotaryShape* s) {
    if (!s) return KDA_ERR_NULL;
    if (s->tokens < 0 || s->q_heads <= 0 || s->kv_heads <= 0 || s->head_dim <= 0 || s->rotary_dim < 0 || s->table_len <= 0) return KDA_ERR_BAD_SHAPE;
    if (s->head_dim > KDA_MAX_DIM || s->rotary_dim > s->head_dim || s->rotary_dim % 2 != 0) return KDA_ERR_BAD_SHAPE;
    if ((long long)s->tokens * (s->q_heads + 2ll * s->kv_heads) >= 1ll << 31) return KDA_ERR_BAD_SHAPE;
    if (s->io_dtype != KDA_DTYPE_F32 && s->io_dtype != KDA_DTYPE_BF16) return KDA_ERR_UNSUPPORTED;
    return KDA_OK;
}

int blocks_for(long long rows) {
    const long long most = 148 * 8, want = (rows + kWarps - 1) / kWarps;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

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
    const int blocks = blocks_for((long long)s->tokens * (s->q_heads + s->kv_heads));
    KDA_LAUNCH("norm_rope_kernel", st, norm_rope_kernel<false><<<blocks, kThreads, 0, st>>>(p));
    return launch_status();
}

extern "C" size_t kda_norm_rope_bwd_scratch_bytes(const KdaRotaryShape* s) {
    if (check(s)) return 0;
    return align_up((size_t)blocks_for((long long)s->tokens * (s->q_heads + s->kv_heads)) * 2 * s->head_dim * sizeof(float), 256);
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
    const int blocks = blocks_for((long long)s->tokens * (s->q_heads + s->kv_heads));
    KDA_LAUNCH("norm_rope_bwd_kernel", st, norm_rope_bwd_kernel<<<blocks, kThreads, 0, st>>>(p));
    if (int rc = launch_status()) return rc;
    if (!sums) return KDA_OK;
    KDA_LAUNCH("norm_rope_dw_kernel", st,
               norm_rope_dw_kernel<<<(2 * s->head_dim + kWarps - 1) / kWarps, kThreads, 0, st>>>(blocks, s->head_dim, p.part, dq_weight, dk_weight));
    return launch_status();
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
    const int blocks = blocks_for((long long)s->tokens * (s->q_heads + 2 * s->kv_heads));
    KDA_LAUNCH("norm_rope_append_kernel", st, norm_rope_kernel<true><<<blocks, kThreads, 0, st>>>(p));
    return launch_status();
}
