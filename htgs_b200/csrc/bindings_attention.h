// The torch layer of rotary positions and attention, part of the extension module `_C` (included by bindings.cpp): the checks, outputs and gradients of htgs_b200/sequence.py.
#pragma once

#include "bindings_sequence.h"

namespace sequence {

using OptInt = c10::optional<int64_t>;
using OptDouble = c10::optional<double>;

// `t` as [rows, heads, width]; a copy only where a head's values are not dense, rows or heads lie on one another, or 16-bit heads that could begin on 16 bytes do not.
Tensor heads_of(const Tensor& t) {
    Tensor m = t;
    if (m.dim() != 3) {
        int64_t rows = 1;
        for (int64_t i = 0; i + 2 < t.dim(); ++i) rows *= t.size(i);
        m = t.reshape({rows, t.size(-2), t.size(-1)});
    }
    const int64_t rows = m.size(0), heads = m.size(1), width = m.size(2);
    bool fits = (width == 1 || m.stride(2) == 1) && (heads == 1 || m.stride(1) >= 1) && (rows == 1 || m.stride(0) >= 1);
    if (fits && m.element_size() == 2 && width % 8 == 0)
        fits = reinterpret_cast<uintptr_t>(m.data_ptr()) % 16 == 0 && (heads == 1 || m.stride(1) % 8 == 0) && (rows == 1 || m.stride(0) % 8 == 0);
    return fits ? m : m.clone(at::MemoryFormat::Contiguous);
}
bool same_rows(const Tensor& a, const Tensor& b) {            // all dimensions but the heads
    return a.dim() == b.dim() && a.sizes().slice(0, a.dim() - 2) == b.sizes().slice(0, b.dim() - 2) && a.size(-1) == b.size(-1);
}

// ---- rotary positions -----------------------------------------------------------------------------------------------------------

struct Turning { Tensor positions; std::vector<int64_t> sections; double base; bool interleaved; };

variable_list turn(const variable_list& given, const Turning& by, bool inverse) {
    variable_list out;
    HtgsRotary r{};
    Tensor held[2];
    for (size_t i = 0; i < given.size(); ++i) {
        out.push_back(make(given[i], given[i].sizes()));
        const Tensor& x = held[i] = heads_of(given[i]);
        r.x[i] = x.data_ptr(); r.y[i] = out[i].data_ptr(); r.x_stride[i] = x.stride(0); r.x_head_stride[i] = x.stride(1); r.heads[i] = int32_t(x.size(1));
    }
    for (size_t i = 0; i < by.sections.size(); ++i) r.sections[i] = int32_t(by.sections[i]);
    r.positions = by.positions.data_ptr(); r.positions_stride = by.positions.stride(0); r.rows = held[0].size(0); r.base = by.base;
    r.axes = int32_t(by.sections.size()); r.positions_type = by.positions.scalar_type() == torch::kInt32; r.width = int32_t(held[0].size(2));
    r.type = type_of(held[0].scalar_type()); r.interleaved = by.interleaved; r.inverse = inverse;
    check(htgs_rotary(&r, stream_of(held[0])));
    return out;
}

struct Rotary : torch::autograd::Function<Rotary> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& positions, const std::vector<int64_t>& sections, double base, bool interleaved) {
        const c10::cuda::CUDAGuard guard(q.device());
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({positions});
        ctx->saved_data["sections"] = sections;
        ctx->saved_data["base"] = base;
        ctx->saved_data["interleaved"] = interleaved;
        return turn(k ? variable_list{q, *k} : variable_list{q}, {positions, sections, base, interleaved}, false);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return first_derivative([&] { return first_backward(ctx, grads); });
    }
    static variable_list first_backward(AutogradContext* ctx, const variable_list& grads) {
        variable_list there, out(6);
        for (const Tensor& g : grads)
            if (g.defined()) there.push_back(g);
        if (there.empty()) return out;
        const c10::cuda::CUDAGuard guard(there[0].device());
        const variable_list turned = turn(there, {ctx->get_saved_variables()[0], ctx->saved_data["sections"].toIntVector(), ctx->saved_data["base"].toDouble(),
                                                  ctx->saved_data["interleaved"].toBool()}, true);
        size_t at = 0;
        for (size_t i = 0; i < grads.size(); ++i)
            if (grads[i].defined()) out[i] = turned[at++];
        return out;
    }
};

std::tuple<Tensor, OptTensor> rotary(const Tensor& q, const OptTensor& k, const Tensor& positions, const c10::optional<std::vector<int64_t>>& given_sections, double base,
                                     bool interleaved) {
    check_value(q, "q");
    TORCH_CHECK_VALUE(q.dim() >= 3 && q.size(-1) % 2 == 0 && q.size(-1) >= 2 && q.size(-1) <= 256 && q.size(-2) >= 1, "q must have shape [..., rows, heads, width], width even and 2 to 256");
    if (k) {
        check_like(*k, "k", q.scalar_type(), q.device());
        TORCH_CHECK_VALUE(same_rows(q, *k) && k->size(-2) >= 1, "k must have the rows and width of q, ", q.sizes(), ", got ", k->sizes());
    }
    check_like(positions, "positions", positions.defined() && positions.scalar_type() == torch::kInt32 ? torch::kInt32 : torch::kFloat32, q.device());
    TORCH_CHECK_VALUE(positions.dim() == q.dim() - 1 && positions.sizes().slice(0, positions.dim() - 1) == q.sizes().slice(0, q.dim() - 2) && positions.size(-1) >= 1 && positions.size(-1) <= 4,
                      "positions must have shape [..., rows, axes], the rows of q and 1 to 4 axes");
    const int64_t axes = positions.size(-1), pairs = q.size(-1) / 2;
    std::vector<int64_t> sections;
    if (given_sections) {
        int64_t total = 0, least = 0;
        sections = *given_sections;
        for (const int64_t n : sections) { total += n; least = std::min(least, n); }
        TORCH_CHECK_VALUE(int64_t(sections.size()) == axes && least >= 0 && total == pairs, "sections must hold the pairs of each of ", axes, " axes, ", pairs, " in all");
    } else
        for (int64_t a = 0; a < axes; ++a) sections.push_back(pairs / axes + (a < pairs % axes));
    TORCH_CHECK_VALUE(base > 0.0 && std::isfinite(base), "base must be positive and finite");
    no_tangent(q); no_tangent(k); no_tangent(positions);
    TORCH_CHECK(!(c10::GradMode::is_enabled() && positions.requires_grad()), "rotary has no gradient with respect to positions: detach them");
    const Tensor rows = rows_of(positions);
    if (c10::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k))) {
        const variable_list out = Rotary::apply(q, k, rows, sections, base, interleaved);
        return {out[0], k ? OptTensor(out[1]) : OptTensor()};
    }
    const c10::cuda::CUDAGuard guard(q.device());
    const variable_list out = turn(k ? variable_list{q, *k} : variable_list{q}, {rows, sections, base, interleaved}, false);
    return {out[0], k ? OptTensor(out[1]) : OptTensor()};
}

// ---- attention ---------------------------------------------------------------------------------------------------------------------

struct Attending { int64_t sequences; bool causal; int64_t window; double scale; };

int64_t window_of(const OptInt& window) {
    TORCH_CHECK_VALUE(!window || *window >= 0, "window must not be negative");
    return window ? std::min<int64_t>(*window, 0x7fffffff) : -1;
}
double scale_of(const OptDouble& given, int64_t width) {
    const double scale = given ? *given : 1.0 / std::sqrt(double(width));
    TORCH_CHECK_VALUE(scale > 0.0 && std::isfinite(scale), "scale must be positive and finite");
    return scale;
}
HtgsAttention attention_of(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets, const Attending& how) {
    return {q.data_ptr(), k.data_ptr(), v.data_ptr(), offsets.defined() ? offsets.data_ptr<int32_t>() : nullptr, q.stride(0), k.stride(0), v.stride(0), q.stride(1), k.stride(1), v.stride(1),
            q.size(0), int32_t(q.size(1)), int32_t(k.size(1)), int32_t(q.size(2)), int32_t(how.sequences), type_of(q.scalar_type()), how.causal ? 1 : 0, int32_t(how.window), float(how.scale)};
}

struct Attention : torch::autograd::Function<Attention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& given_offsets, int64_t sequences, bool causal, int64_t window, double scale) {
        const c10::cuda::CUDAGuard guard(q.device());
        const Tensor qh = heads_of(q), kh = heads_of(k), vh = heads_of(v), offsets = given_offsets ? *given_offsets : Tensor();
        Tensor out = make(q, q.sizes()), sums = floats(q, {qh.size(1), qh.size(0)}), rest;
        if (q.element_size() == 2) rest = make(q, q.sizes());
        const HtgsAttention a = attention_of(qh, kh, vh, offsets, {sequences, causal, window, scale});
        check(htgs_attention(&a, out.data_ptr(), rest.defined() ? rest.data_ptr() : nullptr, sums.data_ptr<float>(), stream_of(q)));
        ctx->save_for_backward({qh, kh, vh, out, sums, offsets, rest});
        ctx->saved_data["sequences"] = sequences;
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["window"] = window;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["keys"] = k.sizes().vec();
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return first_derivative([&] { return first_backward(ctx, grads); });
    }
    static variable_list first_backward(AutogradContext* ctx, const variable_list& grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &sums = saved[4], &offsets = saved[5], &rest = saved[6];
        const c10::cuda::CUDAGuard guard(q.device());
        const Tensor grad = heads_of(grads[0]);
        const auto keys = ctx->saved_data["keys"].toIntVector();
        const HtgsAttention a = attention_of(q, k, v, offsets, {ctx->saved_data["sequences"].toInt(), ctx->saved_data["causal"].toBool(), ctx->saved_data["window"].toInt(),
                                                                ctx->saved_data["scale"].toDouble()});
        Tensor grad_q = make(q, grads[0].sizes()), grad_k = make(k, keys), grad_v = make(v, keys);
        const size_t size = htgs_attention_backward_workspace_bytes(&a);
        Tensor workspace = bytes(q, size);
        check(htgs_attention_backward(&a, out.data_ptr(), rest.defined() ? rest.data_ptr() : nullptr, sums.data_ptr<float>(), grad.data_ptr(), grad.stride(0), grad.stride(1), grad_q.data_ptr(), grad_k.data_ptr(), grad_v.data_ptr(),
                                      workspace.data_ptr(), size, stream_of(q)));
        return {grad_q, grad_k, grad_v, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& offsets, bool causal, OptInt given_window, OptDouble given_scale) {
    check_value(q, "q");
    check_like(k, "k", q.scalar_type(), q.device());
    check_like(v, "v", q.scalar_type(), q.device());
    TORCH_CHECK_VALUE((q.dim() == 3 || q.dim() == 4) && q.size(-1) >= 1 && q.size(-1) <= 128 && q.size(-2) >= 1,
                      "q must have shape [rows, heads, width] or [batch, rows, heads, width], width 1 to 128");
    TORCH_CHECK_VALUE(k.sizes() == v.sizes() && same_rows(q, k) && k.size(-2) >= 1 && q.size(-2) % k.size(-2) == 0, "k and v must have one shape, the rows and width of q, ", q.sizes(),
                      ", and a number of heads that divides q's");
    Tensor off;
    if (offsets) {
        check_like(*offsets, "offsets", torch::kInt32, q.device());
        TORCH_CHECK_VALUE(q.dim() == 3 && offsets->dim() == 1 && offsets->numel() >= 2, "offsets must hold sequences + 1 row numbers, for q of shape [rows, heads, width]");
        off = offsets->contiguous();
    }
    const int64_t sequences = q.dim() == 4 ? q.size(0) : off.defined() ? off.numel() - 1 : 1, window = window_of(given_window);
    const double scale = scale_of(given_scale, q.size(-1));
    no_tangent(q); no_tangent(k); no_tangent(v);
    if (q.numel() == 0) return q.add(k.sum().add(v.sum()));               // nothing, and yet of all three
    if (c10::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(v)))
        return Attention::apply(q, k, v, off.defined() ? OptTensor(off) : OptTensor(), sequences, causal, window, scale);
    const c10::cuda::CUDAGuard guard(q.device());
    const Tensor qh = heads_of(q), kh = heads_of(k), vh = heads_of(v);
    Tensor out = make(q, q.sizes());
    const HtgsAttention a = attention_of(qh, kh, vh, off, {sequences, causal, window, scale});
    check(htgs_attention(&a, out.data_ptr(), nullptr, nullptr, stream_of(q)));
    return out;
}

void check_cache(const Tensor& t, const char* name, at::IntArrayRef shape) {
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape [batch, capacity, key_heads, width], ", shape, ", got ", t.sizes());
    std::vector<std::pair<int64_t, int64_t>> dims;
    for (int64_t i = 0; i < 4; ++i)
        if (t.size(i) > 1) dims.push_back({t.stride(i), t.size(i)});
    std::sort(dims.begin(), dims.end());
    int64_t extent = 0;
    for (const auto& [stride, size] : dims) {
        TORCH_CHECK_VALUE(stride > extent, name, " must not have places that are one in memory: it is updated in place");
        extent += stride * (size - 1);
    }
    TORCH_CHECK_VALUE(t.stride(3) == 1 || t.size(3) == 1, name, " must have dense heads: it is updated in place");
}

Tensor attention_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& keys, const Tensor& values, const Tensor& lengths, OptInt given_window, OptDouble given_scale) {
    check_value(q, "q");
    check_like(k, "k", q.scalar_type(), q.device());
    check_like(v, "v", q.scalar_type(), q.device());
    check_like(keys, "keys", q.scalar_type(), q.device());
    check_like(values, "values", q.scalar_type(), q.device());
    check_like(lengths, "lengths", torch::kInt32, q.device());
    TORCH_CHECK_VALUE(q.dim() == 3 && q.size(2) >= 1 && q.size(2) <= 128 && q.size(1) >= 1, "q must have shape [batch, heads, width], width 1 to 128");
    TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.dim() == 3 && k.size(0) == q.size(0) && k.size(2) == q.size(2) && k.size(1) >= 1 && q.size(1) % k.size(1) == 0,
                      "k and v must have one shape, the batch and width of q, ", q.sizes(), ", and a number of heads that divides q's");
    TORCH_CHECK_VALUE(keys.dim() == 4, "keys must have shape [batch, capacity, key_heads, width]");
    const int64_t shape[4] = {k.size(0), keys.size(1), k.size(1), k.size(2)};
    check_cache(keys, "keys", shape);
    check_cache(values, "values", shape);
    TORCH_CHECK_VALUE(keys.numel() == 0 || keys.data_ptr() != values.data_ptr(), "keys and values must not be one tensor");
    TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == q.size(0), "lengths must have shape (", q.size(0), ",), got ", lengths.sizes());
    const int64_t window = window_of(given_window);
    const double scale = scale_of(given_scale, q.size(2));
    for (const Tensor* t : {&q, &k, &v, &keys, &values}) no_tangent(*t);
    TORCH_CHECK(!(c10::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(v) || wants_grad(keys) || wants_grad(values))),
                "attention_step has no gradient: use attention in training, or torch.no_grad()");
    const c10::cuda::CUDAGuard guard(q.device());
    Tensor out = make(q, q.sizes());
    if (q.size(0) == 0) return out;
    const Tensor qh = heads_of(q), kh = heads_of(k), vh = heads_of(v), n = lengths.contiguous();
    const HtgsAttentionStep step{qh.data_ptr(), kh.data_ptr(), vh.data_ptr(), keys.data_ptr(), values.data_ptr(), n.data_ptr<int32_t>(), qh.stride(0), kh.stride(0), vh.stride(0),
                                 qh.stride(1), kh.stride(1), vh.stride(1), keys.stride(0), values.stride(0), keys.stride(1), values.stride(1), keys.stride(2), values.stride(2), keys.size(1),
                                 int32_t(q.size(0)), int32_t(q.size(1)), int32_t(k.size(1)), int32_t(q.size(2)), type_of(q.scalar_type()), int32_t(window), float(scale)};
    const size_t size = htgs_attention_step_workspace_bytes(&step);
    Tensor workspace;
    if (size) workspace = bytes(q, size);
    check(htgs_attention_step(&step, out.data_ptr(), size ? workspace.data_ptr() : nullptr, size, stream_of(q)));
    for (const Tensor* t : {&keys, &values})
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    return out;
}

void define_attention(pybind11::module_& m) {
    m.def("rotary", &rotary);
    m.def("attention", &attention);
    m.def("attention_step", &attention_step);
}

}  // namespace sequence
