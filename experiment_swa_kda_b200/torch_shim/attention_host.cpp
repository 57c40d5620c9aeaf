// The native host path of attention.py: checks, allocations, launches and the autograd node of one operator in one call
// from Python.  As in kda_host.cpp an entry answers None, with nothing done, when its inputs are not the plain valid case;
// attention.py then runs its checks, which name the mistake.

#include <torch/extension.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <tuple>

#include "host_node.h"

namespace kda_host {
namespace {

constexpr int64_t kInt = INT_MAX;

// cos, sin [P, R/2] float32 beside q
bool tables_ok(const Tensor& cos, const Tensor& sin, const Tensor& q, int64_t D) {
    return cos.dim() == 2 && sin.sizes() == cos.sizes() && cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && on(cos, q) && on(sin, q) &&
           !cos.requires_grad() && !sin.requires_grad() && cos.size(0) > 0 && cos.size(0) <= kInt && 2 * cos.size(1) <= D;
}
bool weight_ok(const OptTensor& w, const Tensor& q, int64_t D) { return !has(w) || (w->dim() == 1 && w->numel() == D && w->is_floating_point() && on(*w, q)); }
const float* fptr(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
Tensor weight32(const OptTensor& w) { return has(w) ? dense_as(*w, at::kFloat) : Tensor(); }

// Rows of [B, T, H, D] with one stride from token to token across the batch; a copy where the strides are none of that kind.
Tensor rows_of(const Tensor& t) {
    const bool inner = t.size(3) == 1 || t.stride(3) == 1;
    const bool outer = t.size(0) == 1 || t.size(1) == 1 || t.stride(0) == t.size(1) * t.stride(1);
    return inner && outer ? t : t.contiguous();
}
int64_t token_stride(const Tensor& t) { return t.size(1) == 1 ? t.stride(0) : t.stride(1); }

KdaRotaryShape rotary_shape(int64_t tokens, int64_t seq_len, int64_t hq, int64_t hk, int64_t D, const Tensor& cos, int io, double eps, bool interleaved) {
    KdaRotaryShape s = {};
    s.tokens = (int32_t)tokens;
    s.seq_len = (int32_t)seq_len;
    s.q_heads = (int32_t)hq;
    s.kv_heads = (int32_t)hk;
    s.head_dim = (int32_t)D;
    s.rotary_dim = (int32_t)(2 * cos.size(1));
    s.table_len = (int32_t)cos.size(0);
    s.io_dtype = io;
    s.interleaved = interleaved ? 1 : 0;
    s.eps = (float)eps;
    return s;
}

struct NormRopeNode : public HostNode {
    KdaRotaryShape sh;
    bool has_qw = false, has_kw = false, has_pos = false;
    at::ScalarType qw_type = at::kFloat, kw_type = at::kFloat;
    std::vector<int64_t> q_sizes, k_sizes;
    c10::Device device = c10::Device(c10::kCUDA, 0);
    std::string name() const override { return "QKNormRopeBackward"; }
    // A saved tensor.  A saved-tensor hook may hand it back at other strides (one that offloads to the host makes slices dense), so none are
    // taken from the forward; of another shape, type or device it would be read out of range.
    Tensor back(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type) const {
        TORCH_CHECK(t.defined() && t.sizes() == sizes && t.scalar_type() == type && t.device() == device,
                    "a saved-tensor hook handed a tensor of another shape, type or device back to qk_norm_rope");
        return t;
    }
    variable_list apply(variable_list&& grads) override {
        std::vector<Tensor> t;
        {
            std::lock_guard<std::mutex> lk(mutex_);
            for (size_t i = 0; i < saved.size(); ++i) t.push_back(get(i));
        }
        at::AutoDispatchBelowADInplaceOrView below;
        c10::cuda::CUDAGuard guard(device);
        watch_status(device.index());
        const at::ScalarType io = sh.io_dtype == KDA_DTYPE_BF16 ? at::kBFloat16 : at::kFloat;
        const int64_t table[2] = {sh.table_len, sh.rotary_dim / 2}, place[2] = {q_sizes[0], q_sizes[1]}, width[1] = {sh.head_dim};
        const Tensor q = rows_of(back(t[0], q_sizes, io)), k = rows_of(back(t[1], k_sizes, io));
        const Tensor cos = dense(back(t[2], {table, 2}, at::kFloat)), sin = dense(back(t[3], {table, 2}, at::kFloat));
        size_t at_ = 4;
        const Tensor pos = has_pos ? dense(back(t[at_++], {place, 2}, sh.positions_64 ? at::kLong : at::kInt)) : Tensor();
        const Tensor qw = has_qw ? dense(back(t[at_++], {width, 1}, at::kFloat)) : Tensor(), kw = has_kw ? dense(back(t[at_++], {width, 1}, at::kFloat)) : Tensor();
        KdaRotaryShape s = sh;
        s.q_token_stride = token_stride(q), s.q_head_stride = q.stride(2);
        s.k_token_stride = token_stride(k), s.k_head_stride = k.stride(2);
        const Tensor dqo = grads[0].defined() ? dense_as(grads[0], q.scalar_type()) : at::zeros(q_sizes, q.options());
        const Tensor dko = grads[1].defined() ? dense_as(grads[1], k.scalar_type()) : at::zeros(k_sizes, k.options());
        Tensor dq = empty(q_sizes, q.scalar_type(), q), dk = empty(k_sizes, k.scalar_type(), k), dqw, dkw, scr;
        if (has_qw && task_should_compute_output(2)) dqw = empty({sh.head_dim}, at::kFloat, q);
        if (has_kw && task_should_compute_output(3)) dkw = empty({sh.head_dim}, at::kFloat, q);
        if (dqw.defined() || dkw.defined()) scr = bytes(kda_norm_rope_bwd_scratch_bytes(&s), q);
        must(kda_norm_rope_bwd(&s, q.const_data_ptr(), k.const_data_ptr(), fptr(cos), fptr(sin), has_pos ? pos.const_data_ptr() : nullptr, fptr(qw), fptr(kw),
                               dqo.const_data_ptr(), dko.const_data_ptr(), dq.data_ptr(), dk.data_ptr(), dqw.defined() ? dqw.data_ptr<float>() : nullptr,
                               dkw.defined() ? dkw.data_ptr<float>() : nullptr, scr.defined() ? scr.data_ptr() : nullptr,
                               scr.defined() ? (size_t)scr.numel() : 0, stream_of(q)),
             "kda_norm_rope_bwd");
        return {dq, dk, dqw.defined() && qw_type != at::kFloat ? dqw.to(qw_type) : dqw, dkw.defined() && kw_type != at::kFloat ? dkw.to(kw_type) : dkw};
    }
};

using TensorPair = c10::optional<std::tuple<Tensor, Tensor>>;

TensorPair norm_rope(const Tensor& q_, const Tensor& k_, const Tensor& cos_, const Tensor& sin_, const OptTensor& pos_, const OptTensor& qw_, const OptTensor& kw_,
                     double eps, bool interleaved) {
    if (tracing() || q_.dim() != 4 || k_.dim() != 4 || !q_.is_cuda() || !on(k_, q_) || !is_io(q_) || k_.scalar_type() != q_.scalar_type()) return c10::nullopt;
    const int64_t B = q_.size(0), T = q_.size(1), hq = q_.size(2), hk = k_.size(2), D = q_.size(3);
    if (k_.size(0) != B || k_.size(1) != T || k_.size(3) != D || hq < 1 || hk < 1 || D < 1 || D > KDA_MAX_DIM || B * T * (hq + 2 * hk) > kInt) return c10::nullopt;
    if (!tables_ok(cos_, sin_, q_, D) || !weight_ok(qw_, q_, D) || !weight_ok(kw_, q_, D)) return c10::nullopt;
    if (has(pos_)) {
        if (!on(*pos_, q_) || (pos_->scalar_type() != at::kInt && pos_->scalar_type() != at::kLong)) return c10::nullopt;
        if (pos_->dim() != 2 || pos_->size(0) != B || pos_->size(1) != T) return c10::nullopt;
    } else if (T > cos_.size(0)) {
        return c10::nullopt;
    }
    refuse_tangents(q_, k_, qw_, kw_);
    const Tensor none;
    const bool tracked = torch::autograd::compute_requires_grad(q_, k_, has(qw_) ? *qw_ : none, has(kw_) ? *kw_ : none);
    c10::cuda::CUDAGuard guard(q_.device());
    watch_status(q_.device().index());
    Tensor q, k, cos, sin, pos, qw, kw, qo, ko;
    KdaRotaryShape sh;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        q = rows_of(q_), k = rows_of(k_), cos = dense(cos_), sin = dense(sin_), qw = weight32(qw_), kw = weight32(kw_);
        if (has(pos_)) pos = dense(*pos_);
        qo = empty(q_.sizes(), q.scalar_type(), q);
        ko = empty(k_.sizes(), k.scalar_type(), k);
        sh = rotary_shape(B * T, T, hq, hk, D, cos, dt(q), eps, interleaved);
        sh.positions_64 = pos.defined() && pos.scalar_type() == at::kLong;
        sh.q_token_stride = token_stride(q), sh.q_head_stride = q.stride(2);
        sh.k_token_stride = token_stride(k), sh.k_head_stride = k.stride(2);
    }
    must(kda_norm_rope_fwd(&sh, q.const_data_ptr(), k.const_data_ptr(), fptr(cos), fptr(sin), pos.defined() ? pos.const_data_ptr() : nullptr, fptr(qw), fptr(kw),
                           qo.data_ptr(), ko.data_ptr(), stream_of(q)),
         "kda_norm_rope_fwd");
    if (tracked) {
        auto node = make_node<NormRopeNode>();
        node->set_next_edges(torch::autograd::collect_next_edges(q_, k_, has(qw_) ? *qw_ : none, has(kw_) ? *kw_ : none));
        node->sh = sh;
        node->device = q.device();
        node->has_pos = pos.defined(), node->has_qw = qw.defined(), node->has_kw = kw.defined();
        if (has(qw_)) node->qw_type = qw_->scalar_type();
        if (has(kw_)) node->kw_type = kw_->scalar_type();
        node->q_sizes = q_.sizes().vec(), node->k_sizes = k_.sizes().vec();
        for (const Tensor* t : {&q, &k, &cos, &sin}) node->keep(*t);
        for (const Tensor* t : {&pos, &qw, &kw})
            if (t->defined()) node->keep(*t);
        torch::autograd::set_history(qo, node);
        torch::autograd::set_history(ko, node);
    }
    return std::make_tuple(qo, ko);
}

// ------------------------------------------------------------------------------------------------ paged cache

// q [tokens, heads, D] with adjacent values beside a cache [pages, page, kv heads, D] and the batch's device arrays
bool paged_shape(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& table, const Tensor& lens, const OptTensor& cu, int64_t max_q, int64_t window,
                 KdaPagedShape& s) {
    if (q.dim() != 3 || kc.dim() != 4 || vc.sizes() != kc.sizes() || !q.is_cuda() || !is_io(q)) return false;
    if (kc.scalar_type() != q.scalar_type() || vc.scalar_type() != q.scalar_type() || !on(kc, q) || !on(vc, q)) return false;
    const int64_t T = q.size(0), H = q.size(1), D = q.size(2), pages = kc.size(0), page = kc.size(1), hk = kc.size(2);
    if (kc.size(3) != D || D < 1 || D > KDA_MAX_DIM || hk < 1 || hk > 65535 || H < 1 || H % hk != 0 || page < 1 || pages > kInt || T * H > kInt) return false;
    if (D > 1 && (q.stride(2) != 1 || kc.stride(3) != 1 || vc.stride(3) != 1)) return false;
    if (table.dim() != 2 || table.scalar_type() != at::kInt || !on(table, q) || table.size(0) < 1) return false;
    const int64_t N = table.size(0), width = table.size(1);
    if (width > 1 && table.stride(1) != 1) return false;
    if (lens.dim() != 1 || lens.numel() != N || lens.scalar_type() != at::kInt || !on(lens, q) || !lens.is_contiguous() || width * page > kInt || N > kInt)
        return false;
    if (has(cu)) {
        if (cu->dim() != 1 || cu->numel() != N + 1 || cu->scalar_type() != at::kInt || !on(*cu, q) || !cu->is_contiguous()) return false;
    } else if (T % N != 0) {
        return false;
    }
    if (max_q < 0 || max_q > kInt || window < 0) return false;
    s = {};
    s.tokens = (int32_t)T, s.n_seq = (int32_t)N, s.max_q_len = (int32_t)max_q;
    s.q_heads = (int32_t)H, s.kv_heads = (int32_t)hk, s.head_dim = (int32_t)D;
    s.io_dtype = dt(q);
    s.n_pages = (int32_t)pages, s.page_size = (int32_t)page, s.table_width = (int32_t)width;
    s.window = (int32_t)std::min(window, kInt);      // no sequence is longer
    s.scale = 1.f;
    s.table_stride = table.stride(0);
    s.q_token_stride = q.stride(0), s.q_head_stride = q.stride(1);
    s.k_page_stride = kc.stride(0), s.k_row_stride = kc.stride(1), s.k_head_stride = kc.stride(2);
    s.v_page_stride = vc.stride(0), s.v_row_stride = vc.stride(1), s.v_head_stride = vc.stride(2);
    return true;
}
const int32_t* iptr(const OptTensor& t) { return has(t) ? t->const_data_ptr<int32_t>() : nullptr; }

OptTensor append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos_, const Tensor& sin_, const Tensor& kc, const Tensor& vc, const Tensor& table,
                 const Tensor& lens, const OptTensor& cu, const OptTensor& qw_, const OptTensor& kw_, double eps, bool interleaved) {
    KdaPagedShape pg;
    if (tracing() || !paged_shape(q, kc, vc, table, lens, cu, 0, 0, pg)) return c10::nullopt;
    const int64_t T = q.size(0), D = q.size(2), hk = kc.size(2);
    const int64_t want[3] = {T, hk, D};
    if (k.sizes() != at::IntArrayRef(want, 3) || v.sizes() != k.sizes() || !on(k, q) || !on(v, q) || k.scalar_type() != q.scalar_type() ||
        v.scalar_type() != q.scalar_type() || (D > 1 && (k.stride(2) != 1 || v.stride(2) != 1)) || T * (q.size(1) + 2 * hk) > kInt)
        return c10::nullopt;
    if (!tables_ok(cos_, sin_, q, D) || !weight_ok(qw_, q, D) || !weight_ok(kw_, q, D)) return c10::nullopt;
    if (at::GradMode::is_enabled()) {
        for (const Tensor* t : {&q, &k, &v, &kc, &vc})
            if (t->requires_grad()) return c10::nullopt;
        if ((has(qw_) && qw_->requires_grad()) || (has(kw_) && kw_->requires_grad())) return c10::nullopt;
    }
    refuse_tangents(q, k, v, qw_, kw_);
    c10::cuda::CUDAGuard guard(q.device());
    watch_status(q.device().index());
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor cos = dense(cos_), sin = dense(sin_), qw = weight32(qw_), kw = weight32(kw_);
    Tensor out = empty(q.sizes(), q.scalar_type(), q);
    KdaRotaryShape sh = rotary_shape(T, 1, q.size(1), hk, D, cos, dt(q), eps, interleaved);
    sh.q_token_stride = q.stride(0), sh.q_head_stride = q.stride(1);
    sh.k_token_stride = k.stride(0), sh.k_head_stride = k.stride(1);
    sh.v_token_stride = v.stride(0), sh.v_head_stride = v.stride(1);
    must(kda_norm_rope_append(&sh, &pg, q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), fptr(cos), fptr(sin), fptr(qw), fptr(kw),
                              table.const_data_ptr<int32_t>(), lens.const_data_ptr<int32_t>(), iptr(cu), out.data_ptr(), kc.mutable_data_ptr(),
                              vc.mutable_data_ptr(), stream_of(q)),
         "kda_norm_rope_append");
    kc.unsafeGetTensorImpl()->bump_version();
    vc.unsafeGetTensorImpl()->bump_version();
    return out;
}

using AttentionOut = c10::optional<std::tuple<Tensor, OptTensor>>;

// q itself, or a copy where its address or strides would keep it from the kernels for wide accesses
Tensor wide(const Tensor& q) {
    const int64_t unit = q.scalar_type() == at::kBFloat16 ? 8 : 4;
    return reinterpret_cast<uintptr_t>(q.const_data_ptr()) % 16 == 0 && q.stride(0) % unit == 0 && q.stride(1) % unit == 0 ? q : q.clone(at::MemoryFormat::Contiguous);
}

AttentionOut attention(const Tensor& q_, const Tensor& kc, const Tensor& vc, const Tensor& table, const Tensor& lens, const OptTensor& cu, int64_t max_q,
                       int64_t window, c10::optional<double> scale, bool want_lse) {
    KdaPagedShape pg;
    if (tracing() || !paged_shape(q_, kc, vc, table, lens, cu, max_q, window, pg)) return c10::nullopt;
    if (at::GradMode::is_enabled() && (q_.requires_grad() || kc.requires_grad() || vc.requires_grad())) return c10::nullopt;
    pg.scale = scale.has_value() ? (float)*scale : (float)(1.0 / std::sqrt((double)pg.head_dim));
    if (!(pg.scale > 0.f) || !std::isfinite(pg.scale)) return c10::nullopt;
    refuse_tangents(q_, kc, vc);
    c10::cuda::CUDAGuard guard(q_.device());
    watch_status(q_.device().index());
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor q = wide(q_);
    pg.q_token_stride = q.stride(0), pg.q_head_stride = q.stride(1);
    Tensor o = empty(q.sizes(), q.scalar_type(), q), ws;
    OptTensor lse;
    if (want_lse) lse = empty({q.size(0), q.size(1)}, at::kFloat, q);
    const size_t need = kda_paged_attention_workspace_bytes(&pg);
    if (need > 0) ws = bytes(need, q);
    must(kda_paged_attention(&pg, q.const_data_ptr(), kc.const_data_ptr(), vc.const_data_ptr(), table.const_data_ptr<int32_t>(), lens.const_data_ptr<int32_t>(),
                             iptr(cu), o.data_ptr(), want_lse ? lse->data_ptr<float>() : nullptr, need > 0 ? ws.data_ptr() : nullptr, need, stream_of(q)),
         "kda_paged_attention");
    return std::make_tuple(o, lse);
}

}  // namespace

void bind_attention(pybind11::module_& m) {
    namespace py = pybind11;
    using nogil = py::call_guard<py::gil_scoped_release>;
    m.def("norm_rope", &norm_rope, nogil());
    m.def("append", &append, nogil());
    m.def("attention", &attention, nogil());
}

}  // namespace kda_host
