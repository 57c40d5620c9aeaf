// Attention over a paged cache for any head width up to 256, any page size and both types: float32 arithmetic on the CUDA
// cores.  o_i = sum_j 2^(s_ij - m_i) v_j / sum_j 2^(s_ij - m_i), s in units of log 2, in one pass over the keys with the
// running maximum m and sum.
//
// A block holds 64 rows (token-major, the query heads of one kv head side by side, so that a key tile serves them all) and
// goes through its keys in tiles of 64.  Both products are 4 x 4 outputs a thread from 16-byte shared-memory reads: bound by
// the multiply-add pipes once there is work for every SM, by the way to memory before that.  Four threads fetch a row, one look at the
// table each, in 16-byte pieces where the addresses allow it.  Two times 257 tokens over 515, float32, 4 heads of 64 on 2: 27 us
// (288 blocks of one or two tiles, each the latency of its fetches and of 8,192 cycles of products at two warps a scheduler); tiles fetched
// ahead into registers took as long.  bf16 batches that the tensor-core kernels do not take come here too, and cost what these products cost: 2,048
// new tokens of 16 heads on 4 697 us in pages of 48 and 1,279 with heads of 256, where pages of 64 and heads of 128 take 37 there; a token of
// 32 conversations of up to 4,096 528 and 940, where 37.

#include "attn.cuh"

namespace kda {
namespace attn {
namespace {

constexpr int kRows = 64, kKeys = 64, kThreads = 256;

template <int DP>
struct Smem {
    float q[kRows][DP + 4];
    float k[kKeys][DP + 4];
    float v[kKeys][DP + 4];
    float p[kRows][kKeys + 4];
    int bad;      // a value in the tile is not finite
};

// A quarter of a row of `width` values from src[at] on to shared memory, as float32 and with zeros behind it; false if a value is
// not finite.  VEC: pieces of 16 bytes.
template <int DP, bool VEC>
__device__ __forceinline__ bool fetch(float* dst, const void* src, long long at, int width, int part, int bf16) {
    bool fine = true;
    if (!VEC) {
        for (int d = part; d < DP; d += 4) {
            const float x = d < width ? ld_io(src, (size_t)(at + d), bf16) : 0.f;
            fine &= isfinite(x);
            dst[d] = x;
        }
    } else if (bf16) {
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
            const int d = 8 * part + 32 * i;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (d < width) x = ld_input(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(src) + at + d));
            const float2 f0 = f2_get(f2_from_bf16(x.x)), f1 = f2_get(f2_from_bf16(x.y)), f2_ = f2_get(f2_from_bf16(x.z)), f3 = f2_get(f2_from_bf16(x.w));
            fine &= isfinite(f0.x) && isfinite(f0.y) && isfinite(f1.x) && isfinite(f1.y) && isfinite(f2_.x) && isfinite(f2_.y) && isfinite(f3.x) && isfinite(f3.y);
            *reinterpret_cast<float4*>(dst + d) = make_float4(f0.x, f0.y, f1.x, f1.y);
            *reinterpret_cast<float4*>(dst + d + 4) = make_float4(f2_.x, f2_.y, f3.x, f3.y);
        }
    } else {
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const int d = 4 * part + 16 * i;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (d < width) x = ld_input(reinterpret_cast<const float4*>(static_cast<const float*>(src) + at + d));
            fine &= isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w);
            *reinterpret_cast<float4*>(dst + d) = x;
        }
    }
    return fine;
}

template <int DP, bool VEC, int KEYS>
__global__ void __launch_bounds__(kThreads) attn_general_kernel(Call c, Tiles tiles, int splits, float* part_o, float2* part_ml) {
    extern __shared__ float4 raw[];
    Smem<DP>& sm = *reinterpret_cast<Smem<DP>*>(raw);
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int hk = blockIdx.y, z = blockIdx.z, g = c.heads.group, D = c.heads.dim;
    const auto& b = view<KEYS>(c);
    if (KEYS == kPrefixKeys) dependency_wait();      // launched early; what is launched early behind it may take all before it for done
    dependents_go();
    if (KEYS == kAllKeys && splits == 1 && hk == 0) {      // padding behind the last sequence; elsewhere the join does this
        const long long from = (long long)b.end() * c.heads.q_heads, to = (long long)b.tokens * c.heads.q_heads, step = (long long)gridDim.x * kThreads;
        for (long long e = from * D + (long long)blockIdx.x * kThreads + tid; e < to * D; e += step) st_io(c.o, e, c.bf16, 0.f);
        if (c.lse != nullptr)
            for (long long e = from + (long long)blockIdx.x * kThreads + tid; e < to; e += step) c.lse[e] = -INFINITY;
    }
    Unit u;
    if (!make_unit(b, tiles, blockIdx.x, c.window, u)) {
        int n, tile;
        if (hk == 0 && z == 0 && tid == 0 && tiles.find(b, blockIdx.x, n, tile)) check_batch(b, tiles, n, tile);
        if (KEYS == kOwnKeys) dependency_wait();      // the end of this kernel stands for that of the one before too
        return;
    }
    if (hk == 0 && z == 0 && tid == 0) check_batch(b, tiles, u.n, u.row0 / kRows);
    const int t0 = u.lo / kKeys, nt = max((u.hi + kKeys - 1) / kKeys - t0, 0);
    const int t_begin = t0 + (int)((long long)nt * z / splits), t_end = t0 + (int)((long long)nt * (z + 1) / splits);

    auto token_of = [&](int r) { return u.first + (u.row0 + r) / g; };
    auto head_of = [&](int r) { return hk * g + (u.row0 + r) % g; };
    const int f_row = tid >> 2, f_part = tid & 3;      // the row this thread fetches, and its part
    {
        const bool is = f_row < u.rows;
        const long long at = is ? token_of(f_row) * c.strides.q_token + head_of(f_row) * c.strides.q_head : 0;
        fetch<DP, VEC>(sm.q[f_row], c.q, at, is ? D : 0, f_part, c.bf16);
    }
    // the keys each of this thread's rows sees
    int last[4], first[4];
    float m[4], l[4], acc[4][DP / 64][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty + 16 * i;
        last[i] = r >= u.rows ? -1 : KEYS == kPrefixKeys ? u.hi - 1 : u.base + (u.row0 + r) / g;
        first[i] = KEYS == kAllKeys ? first_key(last[i], c.window) : u.from;
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int x = 0; x < DP / 64; ++x)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][x][j] = 0.f;
    }
    const float scale = c.scale * 1.4426950408889634f;

    for (int t = t_begin; t < t_end; ++t) {
        __syncthreads();
        if (tid == 0) sm.bad = 0;
        __syncthreads();
        const int key = t * kKeys + f_row;
        long long k_at = 0, v_at = 0;
        int width = 0;
        if (key >= u.lo && key < u.hi) {
            const int page = b.page(u.n, key / b.page_size), row = key % b.page_size;
            if (page >= 0) {
                width = D;
                k_at = page * c.strides.k_page + row * c.strides.k_row + hk * c.strides.k_head;
                v_at = page * c.strides.v_page + row * c.strides.v_row + hk * c.strides.v_head;
            } else if (f_part == 0) {
                b.tell(KDA_ERR_BLOCK_TABLE);
            }
        }
        fetch<DP, VEC>(sm.k[f_row], c.k, k_at, width, f_part, c.bf16);
        const bool bad = !fetch<DP, VEC>(sm.v[f_row], c.v, v_at, width, f_part, c.bf16);
        if (bad) sm.bad = 1;
        __syncthreads();

        float s[4][4] = {};
#pragma unroll 4
        for (int d = 0; d < DP; d += 4) {
            float4 a[4], k[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(&sm.q[ty + 16 * i][d]);
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4*>(&sm.k[tx + 16 * j][d]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][j] = fmaf(a[i].x, k[j].x, s[i][j]);
                    s[i][j] = fmaf(a[i].y, k[j].y, s[i][j]);
                    s[i][j] = fmaf(a[i].z, k[j].z, s[i][j]);
                    s[i][j] = fmaf(a[i].w, k[j].w, s[i][j]);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = -INFINITY;
            bool seen[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = t * kKeys + tx + 16 * j;
                seen[j] = key <= last[i] && key >= first[i];
                s[i][j] *= scale;
                if (seen[j]) top = fmaxf(top, fmaxf(s[i][j], kLowest));
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float next = fmaxf(m[i], top);
            const float keep = m[i] == -INFINITY ? 0.f : exp2f(m[i] - next);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = seen[j] ? exp2f(s[i][j] - next) : 0.f;
                sum += p;
                sm.p[ty + 16 * i][tx + 16 * j] = p;
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l[i] = l[i] * keep + sum;
            m[i] = next;
#pragma unroll
            for (int x = 0; x < DP / 64; ++x)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][x][j] *= keep;
        }
        __syncthreads();
        if (!sm.bad) {
#pragma unroll 2
            for (int j = 0; j < kKeys; j += 4) {
                float4 p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(&sm.p[ty + 16 * i][j]);
#pragma unroll
                for (int x = 0; x < DP / 64; ++x)
#pragma unroll
                    for (int jj = 0; jj < 4; ++jj) {
                        const float4 v = *reinterpret_cast<const float4*>(&sm.v[j + jj][4 * tx + 64 * x]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float w = jj == 0 ? p[i].x : jj == 1 ? p[i].y : jj == 2 ? p[i].z : p[i].w;
                            acc[i][x][0] = fmaf(w, v.x, acc[i][x][0]);
                            acc[i][x][1] = fmaf(w, v.y, acc[i][x][1]);
                            acc[i][x][2] = fmaf(w, v.z, acc[i][x][2]);
                            acc[i][x][3] = fmaf(w, v.w, acc[i][x][3]);
                        }
                    }
            }
        } else {
            // 0 times a value that is not finite is NaN: keys that a row does not see are left out of its sum
            for (int j = 0; j < kKeys; ++j) {
                const int key = t * kKeys + j;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (key <= last[i] && key >= first[i]) {
                        const float w = sm.p[ty + 16 * i][j];
#pragma unroll
                        for (int x = 0; x < DP / 64; ++x)
#pragma unroll
                            for (int q = 0; q < 4; ++q) acc[i][x][q] = fmaf(w, sm.v[j][4 * tx + 64 * x + q], acc[i][x][q]);
                    }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty + 16 * i;
        if (r >= u.rows) continue;
        const size_t row = (size_t)token_of(r) * c.heads.q_heads + head_of(r);
        if (splits > 1 || KEYS != kAllKeys) {
            const size_t at = (size_t)z * b.tokens * c.heads.q_heads + row;
            if (tx == 0) part_ml[at] = make_float2(m[i], l[i]);
#pragma unroll
            for (int x = 0; x < DP / 64; ++x)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int d = 4 * tx + 64 * x + j;
                    if (d < D) part_o[at * D + d] = acc[i][x][j];
                }
            continue;
        }
        const float inv = m[i] == -INFINITY ? 0.f : 1.f / l[i];
        if (tx == 0 && c.lse != nullptr) c.lse[row] = m[i] == -INFINITY ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
#pragma unroll
        for (int x = 0; x < DP / 64; ++x)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int d = 4 * tx + 64 * x + j;
                if (d < D) st_io(c.o, row * D + d, c.bf16, acc[i][x][j] * inv);
            }
    }
    if (KEYS == kOwnKeys) dependency_wait();
}

// Joins the parts of a row: a warp a row.  SHARED: those of the prefix, which come first, only where the row's sequence shares it.
template <bool SHARED>
__global__ void __launch_bounds__(128) attn_combine_kernel(Combine c) {
    const long long rows = (long long)c.tokens * c.q_heads;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    dependency_wait();      // in every block: the end of this kernel stands for that of the one before too
    if (row >= rows) return;
    int z_first = 0, z_end = c.splits;
    if (row / c.q_heads >= c.batch.Batch::end()) {      // padding behind the last sequence has no parts
        z_end = 0;
    } else if (SHARED) {
        const int n = c.batch.seq_of<32>((int)(row / c.q_heads), lane, 0xffffffffu);
        int first, count;
        c.batch.OwnView::span(n, first, count);
        const int prefix = c.batch.prefix_of(n);
        if (prefix == 0 || c.batch.kv_len(n) - count < prefix) z_first = c.prefix_splits;
    }
    float m = -INFINITY;
    for (int z = z_first + lane; z < z_end; z += 32) m = fmaxf(m, ld_after_f32(&c.part_ml[z * rows + row].x));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float acc[8] = {}, l = 0.f;
    constexpr int kAhead = 4;
    for (int z0 = z_first; z0 < z_end; z0 += kAhead) {
        uint2 ml[kAhead];
        float v[kAhead][8];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const long long at = (long long)min(z0 + k, c.splits - 1) * rows + row;
            ml[k] = ld_after8(c.part_ml + at);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = lane + 32 * i < c.dim ? ld_after_f32(c.part_o + at * c.dim + lane + 32 * i) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const float x = __uint_as_float(ml[k].x);
            if (z0 + k >= c.splits || x == -INFINITY) continue;      // without a key its sums are 0
            const float w = exp2f(x - m);
            l += __uint_as_float(ml[k].y) * w;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, v[k][i], acc[i]);
        }
    }
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
    if (lane == 0 && c.lse != nullptr) c.lse[row] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * kLn2;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        const int d = lane + 32 * x;
        if (d < c.dim) st_io(c.o, row * c.dim + d, c.bf16, acc[x] * inv);
    }
}

template <int DP, int KEYS>
int launch(const Call& c, const Tiles& t, dim3 grid, int splits, float* part_o, float2* part_ml, cudaStream_t st) {
    const size_t smem = sizeof(Smem<DP>);
    const Strides& s = c.strides;
    const int unit = c.bf16 ? 8 : 4;      // values in 16 bytes
    const long long all = s.q_token | s.q_head | s.k_page | s.k_row | s.k_head | s.v_page | s.v_row | s.v_head | c.heads.dim;
    const bool vec = all % unit == 0 && (reinterpret_cast<uintptr_t>(c.q) | reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) % 16 == 0;
    auto kern = vec ? attn_general_kernel<DP, true, KEYS> : attn_general_kernel<DP, false, KEYS>;
    if (int rc = set_smem_limit(kern, smem)) return rc;
    cudaError_t e = cudaSuccess;      // of own keys: beside the pass over the prefix
    KDA_LAUNCH("attn_general_kernel", st, e = launch_early(kern, grid, kThreads, smem, st, KEYS != kAllKeys, 1, c, t, splits, part_o, part_ml));
    return e == cudaSuccess ? launch_status() : KDA_ERR_CUDA;
}

template <int KEYS>
int pass(const Call& c, int splits, float* part_o, float2* part_ml, cudaStream_t st) {
    Tiles t{kRows, c.heads.group, 0};
    const long long slots = KEYS == kPrefixKeys ? group_slots(c.batch, t.group, kRows, t.per_seq)
                                                : tile_slots(c.batch.tokens, c.batch.n_seq, c.max_q_len, t.group, kRows, c.batch.cu != nullptr, t.per_seq);
    const dim3 grid((unsigned)slots, (unsigned)c.heads.kv_heads, (unsigned)splits);
    if (c.heads.dim <= 64) return launch<64, KEYS>(c, t, grid, splits, part_o, part_ml, st);
    if (c.heads.dim <= 128) return launch<128, KEYS>(c, t, grid, splits, part_o, part_ml, st);
    return launch<256, KEYS>(c, t, grid, splits, part_o, part_ml, st);
}
int combine(const Combine& c, bool shared, cudaStream_t st) {
    const long long rows = (long long)c.tokens * c.q_heads;
    cudaError_t e = cudaSuccess;
    KDA_LAUNCH("attn_combine_kernel", st,
               e = launch_early(shared ? attn_combine_kernel<true> : attn_combine_kernel<false>, dim3((unsigned)((rows + 3) / 4)), 128, 0, st, true, 1, c));
    return e == cudaSuccess ? launch_status() : KDA_ERR_CUDA;
}

}  // namespace

int general(const Call& c, int splits, cudaStream_t st) {
    const size_t rows = (size_t)c.batch.tokens * c.heads.q_heads;
    float2* part_ml = static_cast<float2*>(c.workspace);
    float* part_o = reinterpret_cast<float*>(static_cast<char*>(c.workspace) + align_up(rows * splits * sizeof(float2), 256));
    const int rc = pass<kAllKeys>(c, splits, part_o, part_ml, st);
    if (rc || splits == 1) return rc;
    return combine(Combine{c.batch.tokens, c.heads.q_heads, c.heads.dim, splits, part_o, part_ml, c.o, c.lse, c.bf16, 0, c.batch}, false, st);
}

size_t general_shared_workspace(size_t rows, int parts, int dim) {
    return align_up(rows * parts * sizeof(float2), 256) + align_up(rows * parts * dim * sizeof(float), 256);
}
int general_shared(const Call& c, int prefix_splits, int own_splits, cudaStream_t st) {
    const size_t rows = (size_t)c.batch.tokens * c.heads.q_heads;
    const int parts = prefix_splits + own_splits;
    float2* part_ml = static_cast<float2*>(c.workspace);
    float* part_o = reinterpret_cast<float*>(static_cast<char*>(c.workspace) + align_up(rows * parts * sizeof(float2), 256));
    if (int rc = pass<kPrefixKeys>(c, prefix_splits, part_o, part_ml, st)) return rc;
    if (int rc = pass<kOwnKeys>(c, own_splits, part_o + rows * prefix_splits * c.heads.dim, part_ml + rows * prefix_splits, st)) return rc;
    return combine(Combine{c.batch.tokens, c.heads.q_heads, c.heads.dim, parts, part_o, part_ml, c.o, c.lse, c.bf16, prefix_splits, c.batch}, true, st);
}

}  // namespace attn
}  // namespace kda
