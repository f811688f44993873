// The torch layer of the sequence operators, part of the extension module `_C` (included by bindings.cpp): the checks, outputs and gradients of
// htgs_b200/sequence.py for the calls that are not worth Python's time.  sequence.py does the same over ctypes where the module has not been built.
// (Time of a call over ctypes and over this module, one row of 1024 in bf16: norm into 8 bits and back 41 and 11.7 us, product by 2048 rows 42 and 5.8 us.)
#pragma once

namespace sequence {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kBlock = 128;

int type_of(c10::ScalarType t) {
    return t == torch::kFloat32 ? HTGS_FLOAT32 : t == torch::kFloat16 ? HTGS_FLOAT16 : t == torch::kBFloat16 ? HTGS_BFLOAT16 : -1;
}
void check_value(const Tensor& t, const char* name) {
    TORCH_CHECK_TYPE(t.defined(), name, " must be a torch.Tensor");
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must live on a CUDA device");
    TORCH_CHECK_TYPE(type_of(t.scalar_type()) >= 0, name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
}
void check_like(const Tensor& t, const char* name, c10::ScalarType type, const c10::Device& device) {
    TORCH_CHECK_TYPE(t.defined(), name, " must be a torch.Tensor");
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must live on a CUDA device");
    TORCH_CHECK_VALUE(t.device() == device, name, " is on ", t.device(), ", expected ", device);
    TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t && t->requires_grad(); }
// A tangent would be dropped without a word: a dual tensor need not want a gradient.
void no_tangent(const Tensor& t) {
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "the sequence operators have no forward-mode derivative: unpack dual tensors first");
}
void no_tangent(const OptTensor& t) { if (t) no_tangent(*t); }

// `t` as a matrix of its last dimension's rows; a copy only where its rows are not evenly spaced or not dense.
Tensor rows_of(const Tensor& t) {
    Tensor m = t;
    if (m.dim() != 2) {
        int64_t rows = 1;
        for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
        m = t.reshape({rows, t.size(-1)});
    }
    if ((m.stride(1) != 1 && m.size(1) != 1) || (m.stride(0) < m.size(1) && m.size(0) > 1)) m = m.contiguous();
    return m;
}
std::vector<int64_t> with_last(const Tensor& t, int64_t last) {
    std::vector<int64_t> sizes(t.sizes().begin(), t.sizes().end());
    sizes.back() = last;
    return sizes;
}
cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
// Straight from the allocator: through the dispatcher each took a microsecond more.
Tensor make(const Tensor& like, at::IntArrayRef sizes, c10::ScalarType type) { return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt); }
Tensor make(const Tensor& like, at::IntArrayRef sizes) { return make(like, sizes, like.scalar_type()); }
Tensor bytes(const Tensor& like, size_t count) { return make(like, {int64_t(count)}, torch::kByte); }
Tensor floats(const Tensor& like, at::IntArrayRef sizes) { return make(like, sizes, torch::kFloat32); }
// Runs a backward pass.  Where its graph is created, the gradients hang on a node that raises: a second derivative is an error where one is taken, and only there.
template <typename F> variable_list first_derivative(F&& backward) {
    variable_list grads;
    {
        const c10::AutoGradMode off(false);
        grads = backward();
    }
    if (!c10::GradMode::is_enabled()) return grads;
    for (Tensor& grad : grads)
        if (grad.defined()) grad = grad.detach().set_requires_grad(true);
    const auto refusal = std::make_shared<torch::autograd::DelayedError>("the sequence operators have no second derivative", int64_t(grads.size()));
    return (*refusal)(std::move(grads));
}

// ---- norm ---------------------------------------------------------------------------------------------------------------------

void check_norm(const Tensor& x, const Tensor& weight, const OptTensor& residual) {
    check_value(x, "x");
    check_like(weight, "weight", x.scalar_type(), x.device());
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 8192, "x must have a last dimension of 1 to 8192 values");
    TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == x.size(-1), "weight must have shape (", x.size(-1), ",), got ", weight.sizes());
    if (residual) {
        check_like(*residual, "residual", x.scalar_type(), x.device());
        TORCH_CHECK_VALUE(residual->sizes() == x.sizes(), "residual must have the shape of x, ", x.sizes(), ", got ", residual->sizes());
    }
    no_tangent(x); no_tangent(weight); no_tangent(residual);
}

// y or codes and scales; sum where there is a residual.
void norm_into(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps, Tensor* y, Tensor* sum, Tensor* rstd, Tensor* codes, Tensor* scales) {
    const Tensor w = weight.contiguous();
    const int64_t width = x.size(1);
    check(htgs_add_rms_norm(x.data_ptr(), x.stride(0), residual.defined() ? residual.data_ptr() : nullptr, residual.defined() ? residual.stride(0) : 0, w.data_ptr(),
                            type_of(x.scalar_type()), x.size(0), int32_t(width), float(eps), y ? y->data_ptr() : nullptr, width, sum ? sum->data_ptr() : nullptr, width,
                            rstd ? rstd->data_ptr<float>() : nullptr, codes ? static_cast<uint8_t*>(codes->data_ptr()) : nullptr, codes ? codes->stride(0) : 0,
                            scales ? static_cast<uint8_t*>(scales->data_ptr()) : nullptr, scales ? scales->stride(0) : 0, stream_of(x)));
}

struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& given, double eps) {
        const Tensor residual = given ? *given : Tensor();
        const c10::cuda::CUDAGuard guard(x.device());
        ctx->set_materialize_grads(false);
        const Tensor xm = rows_of(x), rm = residual.defined() ? rows_of(residual) : Tensor();
        Tensor y = make(x, x.sizes()), sum, rstd = floats(x, {xm.size(0)});
        if (residual.defined()) sum = make(x, x.sizes());
        norm_into(xm, weight, rm, eps, &y, residual.defined() ? &sum : nullptr, &rstd, nullptr, nullptr);
        ctx->save_for_backward({xm, weight, rm, rstd});
        return residual.defined() ? variable_list{y, sum} : variable_list{y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return first_derivative([&] { return first_backward(ctx, grads); });
    }
    static variable_list first_backward(AutogradContext* ctx, const variable_list& grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &residual = saved[2], &rstd = saved[3];
        const Tensor grad_sum = grads.size() > 1 ? grads[1] : Tensor();
        const c10::cuda::CUDAGuard guard(x.device());
        if (!grads[0].defined()) return {grad_sum, grad_sum.defined() ? torch::zeros_like(weight) : Tensor(), residual.defined() ? grad_sum : Tensor(), Tensor()};
        const Tensor gy = rows_of(grads[0]), gs = grad_sum.defined() ? rows_of(grad_sum) : Tensor(), w = weight.contiguous();
        const int64_t rows = x.size(0), width = x.size(1);
        Tensor grad_x = make(x, grads[0].sizes()), grad_weight = make(x, {width});
        const size_t size = htgs_add_rms_norm_backward_scratch_bytes(rows, int32_t(width));
        Tensor scratch = bytes(x, size);
        check(htgs_add_rms_norm_backward(gy.data_ptr(), gy.stride(0), gs.defined() ? gs.data_ptr() : nullptr, gs.defined() ? gs.stride(0) : 0, x.data_ptr(), x.stride(0),
                                         residual.defined() ? residual.data_ptr() : nullptr, residual.defined() ? residual.stride(0) : 0, w.data_ptr(),
                                         rstd.data_ptr<float>(), type_of(x.scalar_type()), rows, int32_t(width), grad_x.data_ptr(), width, grad_weight.data_ptr(),
                                         scratch.data_ptr(), size, stream_of(x)));
        return {grad_x, grad_weight, residual.defined() ? grad_x : Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps) {
    check_norm(x, weight, residual);
    if (c10::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(residual))) {
        variable_list out = AddRmsNorm::apply(x, weight, residual, eps);
        return {out[0], residual ? out[1] : x};
    }
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor y = make(x, x.sizes()), sum;
    if (residual) sum = make(x, x.sizes());
    norm_into(rows_of(x), weight, residual ? rows_of(*residual) : Tensor(), eps, &y, residual ? &sum : nullptr, nullptr, nullptr, nullptr);
    return {y, residual ? sum : x};
}

// ---- 8-bit matrices -------------------------------------------------------------------------------------------------------------

int64_t up(int64_t n, int64_t unit) { return (n + unit - 1) / unit * unit; }
int64_t blocks(int64_t n, int64_t unit) { return (n + unit - 1) / unit; }

struct Matrix { Tensor codes, scales; int64_t rows_per_scale = 1; };

Matrix empty_matrix(int64_t rows, int64_t width, int64_t rows_per_scale, const Tensor& like) {
    const int64_t across = blocks(width, kBlock);
    return {at::detail::empty_strided_cuda({rows, width}, {up(width, 16), 1}, torch::kFloat8_e4m3fn, like.device()),
            at::detail::empty_strided_cuda({blocks(rows, rows_per_scale), across}, {up(across, 4), 1}, torch::kFloat8_e8m0fnu, like.device()), rows_per_scale};
}
HtgsFp8Matrix view_of(const Matrix& m) {       // the stride of a single row says nothing
    const int64_t rows = m.codes.size(0), width = m.codes.size(1);
    return {static_cast<const uint8_t*>(m.codes.data_ptr()), static_cast<const uint8_t*>(m.scales.data_ptr()), rows, width, rows > 1 ? m.codes.stride(0) : up(width, 16),
            m.scales.size(0) > 1 ? m.scales.stride(0) : up(m.scales.size(1), 4), int32_t(m.rows_per_scale)};
}
void check_rows(const Tensor& t, const char* name, int64_t unit) {
    TORCH_CHECK_VALUE(t.numel() == 0 || (reinterpret_cast<uintptr_t>(t.data_ptr()) % unit == 0 && (t.size(1) <= 1 || t.stride(1) == 1) &&
                                         (t.size(0) <= 1 || (t.stride(0) % unit == 0 && t.stride(0) >= t.size(1)))),
                      name, " must have dense rows that begin on multiples of ", unit, " bytes");
}
void check_matrix(const Tensor& codes, const Tensor& scales, int64_t rows_per_scale) {
    TORCH_CHECK_TYPE(codes.defined() && scales.defined(), "codes and scales must be torch.Tensors");
    TORCH_CHECK_VALUE(codes.is_cuda(), "codes must live on a CUDA device");
    check_like(codes, "codes", torch::kFloat8_e4m3fn, codes.device());
    check_like(scales, "scales", torch::kFloat8_e8m0fnu, codes.device());
    TORCH_CHECK_VALUE(rows_per_scale == 1 || rows_per_scale == kBlock, "rows_per_scale must be 1 or 128");
    TORCH_CHECK_VALUE(codes.dim() == 2 && scales.dim() == 2, "codes and scales must be matrices");
    TORCH_CHECK_VALUE(scales.size(0) == blocks(codes.size(0), rows_per_scale) && scales.size(1) == blocks(codes.size(1), kBlock), "scales must have shape (",
                      blocks(codes.size(0), rows_per_scale), ", ", blocks(codes.size(1), kBlock), "), got ", scales.sizes());
    check_rows(codes, "codes", 16);
    check_rows(scales, "scales", 4);
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_fp8(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps) {
    check_norm(x, weight, residual);
    TORCH_CHECK(!(c10::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(residual))),
                "add_rms_norm_fp8 has no gradient: use add_rms_norm and fp8_linear in training, or torch.no_grad()");
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor xm = rows_of(x);
    Matrix q = empty_matrix(xm.size(0), xm.size(1), 1, x);
    Tensor sum;
    if (residual) sum = make(x, x.sizes());
    norm_into(xm, weight, residual ? rows_of(*residual) : Tensor(), eps, nullptr, residual ? &sum : nullptr, nullptr, &q.codes, &q.scales);
    return {q.codes, q.scales, residual ? sum : x};
}

void quantize_into(const Tensor& x, int64_t rows_per_scale, const Matrix* straight, const Matrix* turned) {
    const auto code = [](const Matrix* m) { return m ? static_cast<uint8_t*>(m->codes.data_ptr()) : nullptr; };
    const auto scale = [](const Matrix* m) { return m ? static_cast<uint8_t*>(m->scales.data_ptr()) : nullptr; };
    if (x.numel() == 0) return;
    check(htgs_quantize_fp8(x.data_ptr(), x.stride(0), type_of(x.scalar_type()), x.size(0), x.size(1), int(rows_per_scale), code(straight), straight ? straight->codes.stride(0) : 0,
                            scale(straight), straight ? straight->scales.stride(0) : 0, code(turned), turned ? turned->codes.stride(0) : 0, scale(turned),
                            turned ? turned->scales.stride(0) : 0, stream_of(x)));
}

std::tuple<Tensor, Tensor> quantize_fp8(const Tensor& x, int64_t rows_per_scale, bool transpose) {
    check_value(x, "x");
    TORCH_CHECK_VALUE(rows_per_scale == 1 || rows_per_scale == kBlock, "rows_per_scale must be 1 or 128");
    TORCH_CHECK_VALUE(x.dim() >= 1 && (!transpose || x.dim() == 2), "x must have a dimension to quantise along (and be a matrix to be transposed)");
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor xm = rows_of(x);
    Matrix q = transpose ? empty_matrix(xm.size(1), xm.size(0), rows_per_scale, x) : empty_matrix(xm.size(0), xm.size(1), rows_per_scale, x);
    quantize_into(xm, rows_per_scale, transpose ? nullptr : &q, transpose ? &q : nullptr);
    return {q.codes, q.scales};
}

Tensor dequantize_fp8(const Tensor& codes, const Tensor& scales, int64_t rows_per_scale, c10::ScalarType dtype) {
    TORCH_CHECK_TYPE(type_of(dtype) >= 0, "dtype must be float32, float16 or bfloat16, got ", dtype);
    const c10::cuda::CUDAGuard guard(codes.device());
    Tensor out = make(codes, codes.sizes(), dtype);
    const HtgsFp8Matrix m = view_of({codes, scales, rows_per_scale});
    check(htgs_dequantize_fp8(&m, out.data_ptr(), out.size(1), type_of(dtype), stream_of(codes)));
    return out;
}

void multiply_into(const Matrix& a, const Matrix& b, Tensor& out) {
    const HtgsFp8Matrix av = view_of(a), bv = view_of(b);
    check(htgs_fp8_matmul(&av, &bv, out.data_ptr(), b.codes.size(0), type_of(out.scalar_type()), stream_of(out)));
}

// x: codes with `x_scales`, or values that are quantised first.
Tensor fp8_matmul(const Tensor& x, const OptTensor& x_scales, int64_t x_rows_per_scale, const Tensor& codes, const Tensor& scales, int64_t rows_per_scale,
                  c10::optional<c10::ScalarType> dtype) {
    TORCH_CHECK_TYPE(!dtype || type_of(*dtype) >= 0, "dtype must be float32, float16 or bfloat16");
    const int64_t width = codes.size(1);
    const Matrix w{codes, scales, rows_per_scale};
    if (x_scales) {
        TORCH_CHECK_VALUE(x.device() == codes.device(), "x is on ", x.device(), ", expected ", codes.device());
        TORCH_CHECK_VALUE(x.size(1) == width, "x has width ", x.size(1), ", weight ", width);
        const c10::cuda::CUDAGuard guard(x.device());
        Tensor out = make(x, {x.size(0), codes.size(0)}, dtype.value_or(torch::kBFloat16));
        multiply_into({x, *x_scales, x_rows_per_scale}, w, out);
        return out;
    }
    check_value(x, "x");
    TORCH_CHECK_VALUE(x.device() == codes.device(), "x is on ", x.device(), ", expected ", codes.device());
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == width, "x must have a last dimension of ", width, " values");
    no_tangent(x);
    TORCH_CHECK(!(c10::GradMode::is_enabled() && x.requires_grad()), "fp8_matmul has no gradient: use fp8_linear in training, or torch.no_grad()");
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor xm = rows_of(x);
    Tensor out = make(x, with_last(x, codes.size(0)), dtype.value_or(x.scalar_type()));
    const int64_t rows = xm.size(0);
    if (rows >= 1 && rows <= 8 && width >= 1 && rows * up(width, kBlock) <= 32768) {       // one kernel codes and multiplies
        const HtgsFp8Matrix b = view_of(w);
        check(htgs_fp8_matmul_values(xm.data_ptr(), xm.stride(0), type_of(x.scalar_type()), rows, &b, out.data_ptr(), codes.size(0), type_of(out.scalar_type()), stream_of(x)));
        return out;
    }
    Matrix q = empty_matrix(rows, width, 1, x);
    quantize_into(xm, 1, &q, nullptr);
    multiply_into(q, w, out);
    return out;
}

struct Fp8Linear : torch::autograd::Function<Fp8Linear> {
    // need_x, need_weight: which gradients will be asked for; their operands are coded along with the product's, from one read
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, bool need_x, bool need_weight) {
        const c10::cuda::CUDAGuard guard(x.device());
        const Tensor xm = rows_of(x), wm = rows_of(weight);
        const int64_t rows = xm.size(0), width = xm.size(1), out = wm.size(0);
        Matrix xq = empty_matrix(rows, width, 1, x), wq = empty_matrix(out, width, kBlock, x), xt, wt;
        if (need_weight) xt = empty_matrix(width, rows, 1, x);
        if (need_x) wt = empty_matrix(width, out, kBlock, x);
        quantize_into(xm, 1, &xq, need_weight ? &xt : nullptr);
        quantize_into(wm, kBlock, &wq, need_x ? &wt : nullptr);
        Tensor y = make(x, with_last(x, out));
        multiply_into(xq, wq, y);
        ctx->save_for_backward({xt.codes, xt.scales, wt.codes, wt.scales});
        ctx->saved_data["type"] = int64_t(x.scalar_type());
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return first_derivative([&] { return first_backward(ctx, grads); });
    }
    static variable_list first_backward(AutogradContext* ctx, const variable_list& grads) {
        const auto saved = ctx->get_saved_variables();
        const Matrix xt{saved[0], saved[1], 1}, wt{saved[2], saved[3], kBlock};
        const Tensor gm = rows_of(grads[0]);
        const c10::cuda::CUDAGuard guard(gm.device());
        const auto type = c10::ScalarType(ctx->saved_data["type"].toInt());
        const bool need_x = wt.codes.defined(), need_weight = xt.codes.defined();
        Matrix gq, gt;
        if (need_x) gq = empty_matrix(gm.size(0), gm.size(1), 1, gm);
        if (need_weight) gt = empty_matrix(gm.size(1), gm.size(0), 1, gm);
        quantize_into(gm, 1, need_x ? &gq : nullptr, need_weight ? &gt : nullptr);
        Tensor grad_x, grad_weight;
        if (need_x) {
            grad_x = make(gm, with_last(grads[0], wt.codes.size(0)), type);
            multiply_into(gq, wt, grad_x);
        }
        if (need_weight) {
            grad_weight = make(gm, {gt.codes.size(0), xt.codes.size(0)}, type);
            multiply_into(gt, xt, grad_weight);
        }
        return {grad_x, grad_weight, Tensor(), Tensor()};
    }
};

Tensor fp8_linear(const Tensor& x, const Tensor& weight) {
    check_value(x, "x");
    check_like(weight, "weight", x.scalar_type(), x.device());
    TORCH_CHECK_VALUE(weight.dim() == 2 && x.dim() >= 1 && x.size(-1) == weight.size(1), "weight must have shape (out, width), and x a last dimension of width values");
    no_tangent(x); no_tangent(weight);
    const bool grad = c10::GradMode::is_enabled(), need_x = grad && x.requires_grad(), need_weight = grad && weight.requires_grad();
    if (need_x || need_weight) return Fp8Linear::apply(x, weight, need_x, need_weight);
    const c10::cuda::CUDAGuard guard(x.device());
    Matrix wq = empty_matrix(weight.size(0), weight.size(1), kBlock, x);
    quantize_into(rows_of(weight), kBlock, &wq, nullptr);
    return fp8_matmul(x, c10::nullopt, 1, wq.codes, wq.scales, kBlock, c10::nullopt);
}

// ---- recurrence -------------------------------------------------------------------------------------------------------------------

Tensor scan_rows(const Tensor& t) {           // row strides are at most 2^22
    const Tensor m = rows_of(t);
    return m.stride(0) > (1 << 22) ? m.clone(at::MemoryFormat::Contiguous) : m;
}

HtgsScan scan_of(const Tensor& x, const Tensor& gate, const Tensor& initial, const Tensor& offsets, int64_t sequences, bool reverse) {
    return {x.data_ptr(), gate.data_ptr(), initial.defined() ? initial.data_ptr<float>() : nullptr, offsets.defined() ? offsets.data_ptr<int32_t>() : nullptr, x.stride(0),
            gate.stride(0), x.size(0), int32_t(x.size(1)), int32_t(sequences), type_of(x.scalar_type()), reverse ? 1 : 0};
}

void scan_into(const Tensor& x, const Tensor& gate, const Tensor& initial, const Tensor& offsets, int64_t sequences, bool reverse, Tensor& h, Tensor& last, Tensor* states) {
    const int64_t rows = x.size(0), width = x.size(1);
    const HtgsScan scan = scan_of(x, gate, initial, offsets, sequences, reverse);
    const size_t size = htgs_gated_scan_workspace_bytes(rows, int32_t(width));
    Tensor workspace = bytes(x, size);
    check(htgs_gated_scan(&scan, h.data_ptr(), width, last.data_ptr<float>(), states ? states->data_ptr<float>() : nullptr, workspace.data_ptr(), size, stream_of(x)));
}

struct GatedScan : torch::autograd::Function<GatedScan> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const OptTensor& given_initial, const OptTensor& given_offsets,
                                 int64_t sequences, bool reverse) {
        const Tensor initial = given_initial ? *given_initial : Tensor(), offsets = given_offsets ? *given_offsets : Tensor();
        const c10::cuda::CUDAGuard guard(x.device());
        ctx->set_materialize_grads(false);
        const Tensor xm = scan_rows(x), gm = scan_rows(gate), start = initial.defined() ? initial.contiguous() : Tensor();
        Tensor h = make(x, x.sizes()), last = floats(x, {sequences, xm.size(1)});
        Tensor states = floats(x, {int64_t(htgs_gated_scan_state_bytes(xm.size(0), int32_t(xm.size(1))) / 4)});
        scan_into(xm, gm, start, offsets, sequences, reverse, h, last, &states);
        ctx->save_for_backward({xm, gm, start, offsets, states});
        ctx->saved_data["sequences"] = sequences;
        ctx->saved_data["reverse"] = reverse;
        ctx->saved_data["initial"] = wants_grad(initial);
        ctx->saved_data["sizes"] = x.sizes().vec();
        return {h, last};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return first_derivative([&] { return first_backward(ctx, grads); });
    }
    static variable_list first_backward(AutogradContext* ctx, const variable_list& grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &gate = saved[1], &initial = saved[2], &offsets = saved[3], &states = saved[4];
        const auto sizes = ctx->saved_data["sizes"].toIntVector();
        const c10::cuda::CUDAGuard guard(x.device());
        const int64_t rows = x.size(0), width = x.size(1);
        const Tensor gh = grads[0].defined() ? scan_rows(grads[0]) : torch::zeros({rows, width}, x.options());
        const Tensor gl = grads[1].defined() ? grads[1].contiguous() : Tensor();
        Tensor grad_x = make(x, sizes), grad_gate = make(x, sizes), grad_initial;
        if (ctx->saved_data["initial"].toBool()) grad_initial = torch::empty_like(initial);
        const HtgsScan scan = scan_of(x, gate, initial, offsets, ctx->saved_data["sequences"].toInt(), ctx->saved_data["reverse"].toBool());
        const size_t size = htgs_gated_scan_workspace_bytes(rows, int32_t(width));
        Tensor workspace = bytes(x, size);
        check(htgs_gated_scan_backward(&scan, states.data_ptr<float>(), gh.data_ptr(), gh.stride(0), gl.defined() ? gl.data_ptr<float>() : nullptr, grad_x.data_ptr(), width,
                                       grad_gate.data_ptr(), width, grad_initial.defined() ? grad_initial.data_ptr<float>() : nullptr, workspace.data_ptr(), size, stream_of(x)));
        return {grad_x, grad_gate, grad_initial, Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor& x, const Tensor& gate, const OptTensor& initial, const OptTensor& offsets, bool reverse) {
    check_value(x, "x");
    check_like(gate, "gate", x.scalar_type(), x.device());
    TORCH_CHECK_VALUE(gate.sizes() == x.sizes() && (x.dim() == 2 || x.dim() == 3), "x and gate must have one shape, [rows, width] or [batch, rows, width]");
    const int64_t width = x.size(-1);
    TORCH_CHECK_VALUE(width >= 1 && width <= 65536, "x must have 1 to 65536 channels");
    Tensor off;
    if (offsets) {
        check_like(*offsets, "offsets", torch::kInt32, x.device());
        TORCH_CHECK_VALUE(x.dim() == 2 && offsets->dim() == 1 && offsets->numel() >= 2, "offsets must hold sequences + 1 row numbers, for x of shape [rows, width]");
        off = offsets->contiguous();
    }
    const int64_t sequences = x.dim() == 3 ? x.size(0) : off.defined() ? off.numel() - 1 : 1;
    if (initial) {
        check_like(*initial, "initial", torch::kFloat32, x.device());
        TORCH_CHECK_VALUE(initial->dim() == 2 && initial->size(0) == sequences && initial->size(1) == width, "initial must have shape (", sequences, ", ", width, "), got ",
                          initial->sizes());
    }
    no_tangent(x); no_tangent(gate); no_tangent(initial);
    if (sequences == 0) return {torch::empty_like(x), floats(x, {0, width})};
    const Tensor start = initial ? *initial : Tensor();
    if (c10::GradMode::is_enabled() && (wants_grad(x) || wants_grad(gate) || wants_grad(start))) {
        variable_list out = GatedScan::apply(x, gate, initial, off.defined() ? OptTensor(off) : OptTensor(), sequences, reverse);
        return {out[0], out[1]};
    }
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor h = make(x, x.sizes()), last = floats(x, {sequences, width});
    scan_into(scan_rows(x), scan_rows(gate), start.defined() ? start.contiguous() : start, off, sequences, reverse, h, last, nullptr);
    return {h, last};
}

Tensor gated_scan_step(const Tensor& x, const Tensor& gate, const Tensor& state) {
    check_value(x, "x");
    check_like(gate, "gate", x.scalar_type(), x.device());
    check_like(state, "state", torch::kFloat32, x.device());
    TORCH_CHECK_VALUE(x.dim() == 2 && gate.sizes() == x.sizes() && state.sizes() == x.sizes() && x.size(1) >= 1, "x, gate and state must have one shape, [rows, width]");
    TORCH_CHECK_VALUE((state.stride(1) == 1 || state.size(1) == 1) && (state.size(0) <= 1 || state.stride(0) >= state.size(1)),
                      "state must have dense rows: it is updated in place");
    no_tangent(x); no_tangent(gate); no_tangent(state);
    TORCH_CHECK(!(c10::GradMode::is_enabled() && (wants_grad(x) || wants_grad(gate) || wants_grad(state))),
                "gated_scan_step has no gradient: use gated_scan in training, or torch.no_grad()");
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor xm = rows_of(x), gm = rows_of(gate);
    Tensor h = make(x, x.sizes());
    check(htgs_gated_scan_step(xm.data_ptr(), xm.stride(0), gm.data_ptr(), gm.stride(0), state.data_ptr<float>(), state.stride(0), h.data_ptr(), x.size(1),
                               type_of(x.scalar_type()), x.size(0), int32_t(x.size(1)), stream_of(x)));
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();       // autograd learns of it; what inference mode made is kept by no gradient
    return h;
}

void define(pybind11::module_& m) {
    m.def("add_rms_norm", &add_rms_norm);
    m.def("add_rms_norm_fp8", &add_rms_norm_fp8);
    m.def("check_fp8_matrix", &check_matrix);
    m.def("quantize_fp8", &quantize_fp8);
    m.def("dequantize_fp8", [](const Tensor& codes, const Tensor& scales, int64_t rows_per_scale, const pybind11::object& dtype) {
        TORCH_CHECK_TYPE(THPDtype_Check(dtype.ptr()), "dtype must be a torch.dtype");
        return dequantize_fp8(codes, scales, rows_per_scale, reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type);
    });
    m.def("fp8_matmul", [](const Tensor& x, const OptTensor& x_scales, int64_t x_rows_per_scale, const Tensor& codes, const Tensor& scales, int64_t rows_per_scale,
                           const pybind11::object& dtype) {
        TORCH_CHECK_TYPE(dtype.is_none() || THPDtype_Check(dtype.ptr()), "dtype must be a torch.dtype");
        return fp8_matmul(x, x_scales, x_rows_per_scale, codes, scales, rows_per_scale,
                          dtype.is_none() ? c10::optional<c10::ScalarType>() : c10::optional<c10::ScalarType>(reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type));
    });
    m.def("fp8_linear", &fp8_linear);
    m.def("gated_scan", &gated_scan);
    m.def("gated_scan_step", &gated_scan_step);
}

}  // namespace sequence
