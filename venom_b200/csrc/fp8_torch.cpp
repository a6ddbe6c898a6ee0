// The block-scaled 8-bit operators in the `spatha` extension: checks, allocations and the C ABI's calls, on torch's current stream, and the
// differentiable operators as autograd nodes (a step of a small layer takes as long as the host takes to queue it: in Python 85 us for a GELU and its
// gradient, see fp8.py for what the calls mean).
#include <torch/extension.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include "../../include/venom_b200.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

Tensor device_empty(at::IntArrayRef shape, c10::ScalarType type, const Tensor &like) { return at::detail::empty_cuda(shape, type, like.device(), c10::nullopt); }

void check(int rc, const char *what) { TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", vnm_last_error_string()); }

int type_code(c10::ScalarType t, const char *what)
{
    if (t == torch::kFloat16) return VNM_F16;
    if (t == torch::kBFloat16) return VNM_BF16;
    TORCH_CHECK(t == torch::kFloat32, what, ": fp16, bf16 or fp32 expected");
    return VNM_F32;
}

int f8_code(c10::ScalarType t, const char *what)
{
    if (t == torch::kFloat8_e5m2) return VNM_E5M2;
    TORCH_CHECK(t == torch::kFloat8_e4m3fn, what, ": float8_e4m3fn or float8_e5m2 expected");
    return VNM_E4M3;
}

int to_int(int64_t v, const char *what)
{
    TORCH_CHECK(v >= 0 && v <= INT32_MAX, what, ": a size of ", v, " is too large");
    return (int)v;
}

// x as rows of unit inner stride; anything else is copied.
Tensor as_rows(const Tensor &x, const char *what)
{
    TORCH_CHECK(x.is_cuda(), what, ": a CUDA tensor expected (there is no CPU path)");
    TORCH_CHECK(x.dim() == 2, what, ": a matrix expected");
    if ((x.stride(1) == 1 || x.size(1) <= 1) && (x.stride(0) >= x.size(1) || x.size(0) <= 1)) return x;
    return x.contiguous();
}
int64_t row_stride(const Tensor &x) { return x.size(0) > 1 ? x.stride(0) : x.size(1) > 1 ? x.size(1) : 1; }

struct Packed {
    Tensor data, scales;
    int64_t ld = 16;
    void *values() { return data.defined() ? data.data_ptr() : nullptr; }
    void *scale() { return data.defined() ? scales.data_ptr() : nullptr; }
};

// A tensor on part of a storage, without the dispatcher (a view of a tensor takes 1.5 us).
Tensor on_storage(const c10::Storage &storage, c10::ScalarType type, int64_t byte_offset, at::IntArrayRef shape, at::IntArrayRef strides)
{
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(byte_offset);      // of types of one byte
    t.unsafeGetTensorImpl()->set_sizes_and_strides(shape, strides);
    return t;
}

// Values and scales in one allocation.
Packed pack(int64_t rows, int64_t cols, c10::ScalarType f8, const Tensor &like)
{
    Packed p;
    p.ld = std::max<int64_t>(16, (cols + 15) / 16 * 16);
    const int64_t groups = (cols + 511) / 512;
    const Tensor bytes = device_empty({rows * p.ld + groups * rows * 4}, torch::kUInt8, like);
    p.data = on_storage(bytes.storage(), f8, 0, {rows, cols}, {p.ld, 1});
    p.scales = on_storage(bytes.storage(), torch::kFloat8_e8m0fnu, rows * p.ld, {groups, rows, 4}, {rows * 4, 4, 1});
    return p;
}

void check_packed(const Tensor &data, const Tensor &scales, const char *what)
{
    TORCH_CHECK(data.is_cuda() && scales.is_cuda() && data.device() == scales.device(), what, ": values and scales on one CUDA device expected");
    TORCH_CHECK(data.dim() == 2 && (data.stride(1) == 1 || data.size(1) <= 1) && (data.size(0) <= 1 || (data.stride(0) >= data.size(1) && data.stride(0) % 16 == 0)), what,
                ": rows of 8-bit values expected, a multiple of 16 bytes apart");
    TORCH_CHECK(scales.scalar_type() == torch::kFloat8_e8m0fnu && scales.is_contiguous() && scales.dim() == 3 && scales.size(0) == (data.size(1) + 511) / 512 &&
                    scales.size(1) == data.size(0) && scales.size(2) == 4,
                what, ": scales must be float8_e8m0fnu [ceil(cols / 512), rows, 4]");
}
// Leading dimension of packed values: one row's own does not matter, but is checked like the others'.
int64_t packed_ld(const Tensor &data) { return data.size(0) > 1 ? data.stride(0) : (data.size(1) + 15) / 16 * 16; }

Tensor undefined_or_sums(c10::optional<c10::ScalarType> type, int64_t cols, const Tensor &like) { return type.has_value() ? device_empty({cols}, *type, like) : Tensor(); }
Tensor sums_workspace(const Tensor &sums, int64_t rows, int64_t cols, const Tensor &like)
{
    return sums.defined() ? device_empty({(rows + 127) / 128 * cols}, torch::kFloat32, like) : Tensor();
}
void *ptr(const Tensor &t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
OptTensor opt(const Tensor &t) { return t.defined() ? OptTensor(t) : c10::nullopt; }

using Quantized = std::tuple<OptTensor, OptTensor, OptTensor, OptTensor, OptTensor>;

// (data, scales, data_t, scales_t, column sums), None for what is not wanted
Quantized quantize(const Tensor &x_in, c10::ScalarType f8, bool square, bool rows_wanted, bool cols_wanted, c10::optional<c10::ScalarType> sums_type)
{
    const Tensor x = as_rows(x_in, "fp8.quantize");
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t rows = x.size(0), cols = x.size(1);
    const int code = f8_code(f8, "fp8.quantize"), type = type_code(x.scalar_type(), "fp8.quantize");
    const int r = to_int(rows, "fp8.quantize"), c = to_int(cols, "fp8.quantize");
    Packed a, t;
    if (rows_wanted) a = pack(rows, cols, f8, x);
    if (cols_wanted) t = pack(cols, rows, f8, x);
    const Tensor sums = undefined_or_sums(sums_type, cols, x), ws = sums_workspace(sums, rows, cols, x);
    check(vnm_fp8_quantize(x.data_ptr(), type, row_stride(x), r, c, code, square, a.values(), a.ld, a.scale(), t.values(), t.ld, t.scale(), ptr(sums),
                           sums_type.has_value() ? type_code(*sums_type, "fp8.quantize") : VNM_F32, ptr(ws), c10::cuda::getCurrentCUDAStream().stream()),
          "vnm_fp8_quantize");
    return Quantized(opt(a.data), opt(a.scales), opt(t.data), opt(t.scales), opt(sums));
}

Tensor dequantize(const Tensor &data, const Tensor &scales, c10::ScalarType type)
{
    check_packed(data, scales, "fp8.dequantize");
    c10::cuda::CUDAGuard guard(data.device());
    Tensor out = device_empty({data.size(0), data.size(1)}, type, data);
    check(vnm_fp8_dequantize(data.data_ptr(), packed_ld(data), scales.data_ptr(), f8_code(data.scalar_type(), "fp8.dequantize"), to_int(data.size(0), "fp8.dequantize"),
                             to_int(data.size(1), "fp8.dequantize"), out.data_ptr(), type_code(type, "fp8.dequantize"), std::max<int64_t>(1, data.size(1)),
                             c10::cuda::getCurrentCUDAStream().stream()),
          "vnm_fp8_dequantize");
    return out;
}

// aligned_rows: the result's rows begin on 16-byte boundaries, for what stays inside an operator (the quantiser reads such rows faster).
Tensor matmul(const Tensor &a, const Tensor &sa, const Tensor &b, const Tensor &sb, const OptTensor &bias, c10::ScalarType type, bool aligned_rows = false)
{
    check_packed(a, sa, "fp8.matmul");
    check_packed(b, sb, "fp8.matmul");
    TORCH_CHECK(a.device() == b.device(), "fp8.matmul: operands on one device expected");
    TORCH_CHECK(a.size(1) == b.size(1), "fp8.matmul: ", a.size(1), " and ", b.size(1), " columns do not match");
    const bool with_bias = bias.has_value() && bias->defined();
    if (with_bias)
        TORCH_CHECK(bias->device() == a.device() && bias->dim() == 1 && bias->numel() == b.size(0) && bias->is_contiguous(), "fp8.matmul: bias must be a contiguous vector of ", b.size(0),
                    " values on the operands' device");
    c10::cuda::CUDAGuard guard(a.device());
    const int M = to_int(a.size(0), "fp8.matmul"), N = to_int(b.size(0), "fp8.matmul"), K = to_int(a.size(1), "fp8.matmul");
    const int64_t ld = aligned_rows ? ((int64_t)N + 7) / 8 * 8 : N;
    Tensor out = device_empty({M, ld}, type, a);
    if (ld != N) out = out.narrow(1, 0, N);
    check(vnm_fp8_matmul(a.data_ptr(), packed_ld(a), sa.data_ptr(), f8_code(a.scalar_type(), "fp8.matmul"), b.data_ptr(), packed_ld(b), sb.data_ptr(),
                         f8_code(b.scalar_type(), "fp8.matmul"), M, N, K, with_bias ? bias->data_ptr() : nullptr, with_bias ? type_code(bias->scalar_type(), "fp8.matmul: bias") : VNM_F32,
                         out.data_ptr(), type_code(type, "fp8.matmul"), std::max<int64_t>(1, ld), c10::cuda::getCurrentCUDAStream().stream()),
          "vnm_fp8_matmul");
    return out;
}

using Gelu = std::tuple<OptTensor, OptTensor, OptTensor, OptTensor, OptTensor, OptTensor, OptTensor>;

// (y, data, scales, data_t, scales_t, checkpoint, its scales), None for what is not wanted
Gelu gelu(const Tensor &x_in, bool tanh_form, bool y_wanted, bool rows_wanted, bool cols_wanted, bool ckpt_wanted)
{
    const Tensor x = as_rows(x_in, "fp8.gelu");
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t rows = x.size(0), cols = x.size(1);
    const int type = type_code(x.scalar_type(), "fp8.gelu"), r = to_int(rows, "fp8.gelu"), c = to_int(cols, "fp8.gelu");
    Packed a, t, k;
    Tensor y;
    if (y_wanted) y = device_empty({rows, cols}, x.scalar_type(), x);
    if (rows_wanted) a = pack(rows, cols, torch::kFloat8_e4m3fn, x);
    if (cols_wanted) t = pack(cols, rows, torch::kFloat8_e4m3fn, x);
    if (ckpt_wanted) k = pack(rows, cols, torch::kFloat8_e4m3fn, x);
    check(vnm_fp8_gelu(x.data_ptr(), type, row_stride(x), r, c, tanh_form, ptr(y), std::max<int64_t>(1, cols), a.values(), a.ld, a.scale(), t.values(), t.ld, t.scale(), k.values(), k.ld,
                       k.scale(), c10::cuda::getCurrentCUDAStream().stream()),
          "vnm_fp8_gelu");
    return Gelu(opt(y), opt(a.data), opt(a.scales), opt(t.data), opt(t.scales), opt(k.data), opt(k.scales));
}

using GeluGrad = std::tuple<OptTensor, OptTensor, OptTensor, OptTensor, OptTensor, OptTensor>;

// (dx, data, scales, data_t, scales_t, column sums), None for what is not wanted
GeluGrad gelu_grad(const Tensor &dy_in, const Tensor &ckpt, const Tensor &ckpt_scales, bool tanh_form, bool dx_wanted, c10::ScalarType f8, bool rows_wanted, bool cols_wanted,
                   c10::optional<c10::ScalarType> sums_type)
{
    const Tensor dy = as_rows(dy_in, "fp8.gelu");
    check_packed(ckpt, ckpt_scales, "fp8.gelu: checkpoint");
    TORCH_CHECK(ckpt.scalar_type() == torch::kFloat8_e4m3fn && ckpt.size(0) == dy.size(0) && ckpt.size(1) == dy.size(1) && ckpt.device() == dy.device(),
                "fp8.gelu: the checkpoint does not belong to this gradient");
    c10::cuda::CUDAGuard guard(dy.device());
    const int64_t rows = dy.size(0), cols = dy.size(1);
    const int type = type_code(dy.scalar_type(), "fp8.gelu"), r = to_int(rows, "fp8.gelu"), c = to_int(cols, "fp8.gelu"), code = f8_code(f8, "fp8.gelu");
    Packed a, t;
    Tensor dx;
    if (dx_wanted) dx = device_empty({rows, cols}, dy.scalar_type(), dy);
    if (rows_wanted) a = pack(rows, cols, f8, dy);
    if (cols_wanted) t = pack(cols, rows, f8, dy);
    const Tensor sums = undefined_or_sums(sums_type, cols, dy), ws = sums_workspace(sums, rows, cols, dy);
    check(vnm_fp8_gelu_grad(dy.data_ptr(), type, row_stride(dy), r, c, tanh_form, ckpt.data_ptr(), packed_ld(ckpt), ckpt_scales.data_ptr(), ptr(dx), std::max<int64_t>(1, cols), code,
                            a.values(), a.ld, a.scale(), t.values(), t.ld, t.scale(), ptr(sums), sums_type.has_value() ? type_code(*sums_type, "fp8.gelu") : VNM_F32, ptr(ws),
                            c10::cuda::getCurrentCUDAStream().stream()),
          "vnm_fp8_gelu_grad");
    return GeluGrad(opt(dx), opt(a.data), opt(a.scales), opt(t.data), opt(t.scales), opt(sums));
}

// ---- differentiable operators ----

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }

// A call that records a graph while its stream is being captured: the node that takes a leaf's gradient lives as long as any graph of the leaf, and belongs to
// the stream of the graph that made it.  A backward pass inside the capture that meets one of another stream waits for that stream, which ends the
// capture (and, thrown from the autograd engine's threads, may end the process), so it is refused here.
void check_capture(std::initializer_list<const Tensor *> inputs)
{
    if (!at::GradMode::is_enabled() || c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
    for (const Tensor *t : inputs) {
        if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (!node) continue;
        const auto stream = node->stream();
        TORCH_CHECK(!stream.has_value() || *stream == c10::cuda::getCurrentCUDAStream(t->device().index()).unwrap(),
                    "a graph of the same leaf recorded on another stream still lives: free it (the tensors that hold it) before this call is captured");
    }
}

// Gradients that can not be differentiated again: doing so raises instead of giving zeros.
variable_list once(variable_list grads, const variable_list &incoming)
{
    if (!at::GradMode::is_enabled()) return grads;
    bool any = false;
    for (const Tensor &g : incoming) any = any || wants_grad(g);
    if (!any) return grads;
    variable_list defined;
    for (Tensor &g : grads)
        if (g.defined()) defined.push_back(g.detach().requires_grad_());
    auto node = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function of venom_b200.fp8", (int64_t)defined.size());
    variable_list out = (*node)(std::move(defined));
    size_t i = 0;
    for (Tensor &g : grads)
        if (g.defined()) g = out[i++];
    return grads;
}

bool is_float(c10::ScalarType t) { return t == torch::kFloat16 || t == torch::kBFloat16 || t == torch::kFloat32; }

void check_input(const Tensor &x, const char *what)
{
    TORCH_CHECK(x.is_cuda(), what, ": a CUDA tensor expected (there is no CPU path)");
    TORCH_CHECK(is_float(x.scalar_type()), what, ": float16, bfloat16 or float32 expected, not ", x.scalar_type());
    TORCH_CHECK(x.dim() >= 1, what, ": at least one dimension expected");
}
void check_weight(const Tensor &x, int64_t features, const Tensor &w, const Tensor &bias, const char *what)
{
    TORCH_CHECK(w.dim() == 2 && is_float(w.scalar_type()) && w.device() == x.device(), what, ": a weight must be a float16, bfloat16 or float32 matrix on the input's device");
    TORCH_CHECK(features == w.size(1) && features >= 1, what, ": ", features, " features do not match a weight of ", w.sizes());
    TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == w.size(0) && is_float(bias.scalar_type()) && bias.device() == x.device()), what,
                ": the bias must be a vector of ", w.size(0), " values on the input's device");
}
void check_grad_dtype(c10::ScalarType t, const char *what)
{
    TORCH_CHECK(t == torch::kFloat8_e4m3fn || t == torch::kFloat8_e5m2, what, ": gradients are kept in float8_e4m3fn or float8_e5m2, not ", t);
}

Tensor flat(const Tensor &x) { return x.dim() == 2 ? x : x.reshape({x.size(-1) ? x.numel() / x.size(-1) : x.numel(), x.size(-1)}); }
Tensor shaped(const Tensor &y, at::IntArrayRef shape)
{
    if (shape.size() == 2) return y;
    std::vector<int64_t> s(shape.begin(), shape.end());
    s.back() = y.size(1);
    return y.view(s);
}

struct Operand {
    Tensor data, scales;
};
struct Both {
    Operand rows, cols;
    Tensor sums;
};
Tensor or_undefined(const OptTensor &t) { return t.has_value() ? *t : Tensor(); }
c10::optional<c10::ScalarType> type_of(bool wanted, c10::ScalarType t) { return wanted ? c10::optional<c10::ScalarType>(t) : c10::nullopt; }

Both quantized(const Tensor &x, c10::ScalarType f8, bool square, bool rows, bool cols, c10::optional<c10::ScalarType> sums)
{
    if (!rows && !cols) return {};
    const Quantized q = quantize(x, f8, square, rows, cols, sums);
    return {{or_undefined(std::get<0>(q)), or_undefined(std::get<1>(q))}, {or_undefined(std::get<2>(q)), or_undefined(std::get<3>(q))}, or_undefined(std::get<4>(q))};
}
Tensor product(const Operand &a, const Operand &b, const Tensor &bias, c10::ScalarType type, bool aligned_rows = false)
{
    return matmul(a.data, a.scales, b.data, b.scales, bias.defined() ? OptTensor(bias.detach().contiguous()) : c10::nullopt, type, aligned_rows);
}
// dy^T x from the transposes; zeros without any token
Tensor weight_grad(const Operand &dy_t, const Operand &x_t, c10::ScalarType type)
{
    if (dy_t.data.size(1) == 0) return torch::zeros({dy_t.data.size(0), x_t.data.size(0)}, dy_t.data.options().dtype(type));
    return product(dy_t, x_t, Tensor(), type);
}

struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const OptTensor &opt_bias, c10::ScalarType grad_type, bool record)
    {
        const Tensor bias = or_undefined(opt_bias);
        const bool need_x = record && wants_grad(x), need_w = record && wants_grad(w);
        Both xs = quantized(flat(x), torch::kFloat8_e4m3fn, false, true, need_w, c10::nullopt);
        Both ws = quantized(w, torch::kFloat8_e4m3fn, true, true, need_x, c10::nullopt);
        const Tensor y = product(xs.rows, ws.rows, bias, x.scalar_type());
        ctx->save_for_backward({xs.cols.data, xs.cols.scales, ws.cols.data, ws.cols.scales});
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["x"] = (int64_t)x.scalar_type();
        ctx->saved_data["w"] = (int64_t)w.scalar_type();
        ctx->saved_data["b"] = (int64_t)(bias.defined() ? bias.scalar_type() : x.scalar_type());
        ctx->saved_data["grad"] = (int64_t)grad_type;
        ctx->saved_data["bias"] = bias.defined();
        return shaped(y, x.sizes());
    }
    static variable_list backward(AutogradContext *ctx, variable_list dys)
    {
        const variable_list saved = ctx->get_saved_variables();
        // counted over the tensors that there are
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
        auto type = [&](const char *k) { return (c10::ScalarType)ctx->saved_data[k].toInt(); };
        const Both g = quantized(flat(dys[0]), type("grad"), false, need_x, need_w || need_b, type_of(need_b, type("b")));
        Tensor dx, dw;
        if (need_x) dx = product(g.rows, {saved[2], saved[3]}, Tensor(), type("x")).view(ctx->saved_data["shape"].toIntVector());
        if (need_w) dw = weight_grad(g.cols, {saved[0], saved[1]}, type("w"));
        return once({dx, dw, g.sums, Tensor(), Tensor()}, dys);
    }
};

Tensor linear(const Tensor &x, const Tensor &w, const OptTensor &bias, c10::ScalarType grad_type)
{
    const Tensor b = or_undefined(bias);
    check_input(x, "fp8.linear");
    check_weight(x, x.size(-1), w, b, "fp8.linear");
    check_grad_dtype(grad_type, "fp8.linear");
    check_capture({&x, &w, &b});
    return Linear::apply(x, w, bias, grad_type, at::GradMode::is_enabled());
}

struct Gelu8 : torch::autograd::Function<Gelu8> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, bool tanh_form, bool record)
    {
        const Gelu g = gelu(flat(x), tanh_form, true, false, false, record && wants_grad(x));
        ctx->save_for_backward({or_undefined(std::get<5>(g)), or_undefined(std::get<6>(g))});
        ctx->saved_data["tanh"] = tanh_form;
        ctx->saved_data["shape"] = x.sizes().vec();
        return std::get<0>(g)->view(x.sizes());
    }
    static variable_list backward(AutogradContext *ctx, variable_list dys)
    {
        const variable_list saved = ctx->get_saved_variables();
        const GeluGrad g = gelu_grad(flat(dys[0]), saved[0], saved[1], ctx->saved_data["tanh"].toBool(), true, torch::kFloat8_e4m3fn, false, false, c10::nullopt);
        return once({std::get<0>(g)->view(ctx->saved_data["shape"].toIntVector()), Tensor(), Tensor()}, dys);
    }
};

Tensor gelu8(const Tensor &x, bool tanh_form)
{
    check_input(x, "fp8.gelu");
    check_capture({&x});
    return Gelu8::apply(x, tanh_form, at::GradMode::is_enabled());
}

struct Mlp : torch::autograd::Function<Mlp> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w1, const OptTensor &opt_b1, const Tensor &w2, const OptTensor &opt_b2, bool tanh_form,
                          c10::ScalarType grad_type, bool record)
    {
        const Tensor b1 = or_undefined(opt_b1), b2 = or_undefined(opt_b2);
        const bool need_x = record && wants_grad(x), need_w1 = record && wants_grad(w1), need_b1 = record && wants_grad(b1), need_w2 = record && wants_grad(w2);
        const bool inner = need_x || need_w1 || need_b1;      // whether the gradient goes back through the GELU
        Both xs = quantized(flat(x), torch::kFloat8_e4m3fn, false, true, need_w1, c10::nullopt);
        Both w1s = quantized(w1, torch::kFloat8_e4m3fn, true, true, need_x, c10::nullopt);
        Gelu a = gelu(product(xs.rows, w1s.rows, b1, x.scalar_type(), true), tanh_form, false, true, need_w2, inner);
        Both w2s = quantized(w2, torch::kFloat8_e4m3fn, true, true, inner, c10::nullopt);
        const Tensor y = product({*std::get<1>(a), *std::get<2>(a)}, w2s.rows, b2, x.scalar_type());
        ctx->save_for_backward({xs.cols.data, xs.cols.scales, w1s.cols.data, w1s.cols.scales, or_undefined(std::get<3>(a)), or_undefined(std::get<4>(a)),
                                or_undefined(std::get<5>(a)), or_undefined(std::get<6>(a)), w2s.cols.data, w2s.cols.scales});
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["x"] = (int64_t)x.scalar_type();
        ctx->saved_data["w1"] = (int64_t)w1.scalar_type();
        ctx->saved_data["w2"] = (int64_t)w2.scalar_type();
        ctx->saved_data["b1"] = (int64_t)(b1.defined() ? b1.scalar_type() : x.scalar_type());
        ctx->saved_data["b2"] = (int64_t)(b2.defined() ? b2.scalar_type() : x.scalar_type());
        ctx->saved_data["grad"] = (int64_t)grad_type;
        ctx->saved_data["tanh"] = tanh_form;
        ctx->saved_data["bias1"] = b1.defined();
        ctx->saved_data["bias2"] = b2.defined();
        return shaped(y, x.sizes());
    }
    static variable_list backward(AutogradContext *ctx, variable_list dys)
    {
        const variable_list s = ctx->get_saved_variables();
        const bool has_b1 = ctx->saved_data["bias1"].toBool(), has_b2 = ctx->saved_data["bias2"].toBool();
        const size_t at_w2 = has_b1 ? 3 : 2;      // counted over the tensors that there are
        const bool need_x = ctx->needs_input_grad(0), need_w1 = ctx->needs_input_grad(1), need_b1 = has_b1 && ctx->needs_input_grad(2), need_w2 = ctx->needs_input_grad(at_w2),
                   need_b2 = has_b2 && ctx->needs_input_grad(at_w2 + 1), inner = need_x || need_w1 || need_b1;
        auto type = [&](const char *k) { return (c10::ScalarType)ctx->saved_data[k].toInt(); };
        const Both g = quantized(flat(dys[0]), type("grad"), false, inner, need_w2 || need_b2, type_of(need_b2, type("b2")));
        Tensor dx, dw1, db1, dw2;
        if (need_w2) dw2 = weight_grad(g.cols, {s[4], s[5]}, type("w2"));
        if (inner) {
            const Tensor da = product(g.rows, {s[8], s[9]}, Tensor(), type("x"), true);
            const GeluGrad h = gelu_grad(da, s[6], s[7], ctx->saved_data["tanh"].toBool(), false, type("grad"), need_x, need_w1 || need_b1, type_of(need_b1, type("b1")));
            db1 = or_undefined(std::get<5>(h));
            if (need_x) dx = product({*std::get<1>(h), *std::get<2>(h)}, {s[2], s[3]}, Tensor(), type("x")).view(ctx->saved_data["shape"].toIntVector());
            if (need_w1) dw1 = weight_grad({*std::get<3>(h), *std::get<4>(h)}, {s[0], s[1]}, type("w1"));
        }
        return once({dx, dw1, db1, dw2, g.sums, Tensor(), Tensor(), Tensor()}, dys);
    }
};

Tensor mlp(const Tensor &x, const Tensor &w1, const OptTensor &bias1, const Tensor &w2, const OptTensor &bias2, bool tanh_form, c10::ScalarType grad_type)
{
    const Tensor b1 = or_undefined(bias1), b2 = or_undefined(bias2);
    check_input(x, "fp8.mlp");
    check_weight(x, x.size(-1), w1, b1, "fp8.mlp");
    check_weight(x, w1.size(0), w2, b2, "fp8.mlp");
    check_grad_dtype(grad_type, "fp8.mlp");
    check_capture({&x, &w1, &b1, &w2, &b2});
    return Mlp::apply(x, w1, bias1, w2, bias2, tanh_form, grad_type, at::GradMode::is_enabled());
}

int64_t device_status()
{
    int status = 0;
    check(vnm_fp8_device_status(&status, c10::cuda::getCurrentCUDAStream().stream()), "vnm_fp8_device_status");
    return status;
}

// fp8.quantize() and fp8.matmul() as plain C functions of the module: at decoding sizes they take as long as the host takes to queue them, and pybind11's conversions of
// arguments and results were 1 us of 5.4.
const Tensor &tensor_of(PyObject *o)
{
    TORCH_CHECK_TYPE(THPVariable_Check(o), "expected a tensor");
    return THPVariable_Unpack(o);
}
c10::ScalarType dtype_of(PyObject *o)
{
    TORCH_CHECK_TYPE(THPDtype_Check(o), "expected a dtype");
    return reinterpret_cast<THPDtype *>(o)->scalar_type;
}

// (x, dtype, square, both) -> (data, scales) or (data, scales, data_t, scales_t)
PyObject *py_quantize(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 4, "quantize(x, dtype, square, both)");
    const Tensor &x = tensor_of(args[0]);
    const c10::ScalarType f8 = dtype_of(args[1]);
    const bool square = args[2] == Py_True, both = args[3] == Py_True;
    Quantized q;
    {
        pybind11::gil_scoped_release no_gil;
        q = quantize(x, f8, square, true, both, c10::nullopt);
    }
    PyObject *out = PyTuple_New(both ? 4 : 2);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(*std::get<0>(q))));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(*std::get<1>(q))));
    if (both) {
        PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(*std::get<2>(q))));
        PyTuple_SET_ITEM(out, 3, THPVariable_Wrap(std::move(*std::get<3>(q))));
    }
    return out;
    END_HANDLE_TH_ERRORS
}

// (a, a's scales, b, b's scales, bias or None, dtype) -> a b^T (+ bias)
PyObject *py_matmul(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 6, "matmul(a, a_scales, b, b_scales, bias, dtype)");
    const Tensor &a = tensor_of(args[0]), &sa = tensor_of(args[1]), &b = tensor_of(args[2]), &sb = tensor_of(args[3]);
    const OptTensor bias = args[4] == Py_None ? c10::nullopt : OptTensor(tensor_of(args[4]));
    const c10::ScalarType type = dtype_of(args[5]);
    Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        out = matmul(a, sa, b, sb, bias, type);
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

PyMethodDef fast_calls[] = {
    {"fp8_quantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&py_quantize)), METH_FASTCALL, "vnm_fp8_quantize with its allocations"},
    {"fp8_matmul", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&py_matmul)), METH_FASTCALL, "vnm_fp8_matmul with its allocation"},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

void define_fp8(pybind11::module &mod)
{
    using release = pybind11::call_guard<pybind11::gil_scoped_release>;
    if (PyModule_AddFunctions(mod.ptr(), fast_calls) != 0) throw pybind11::error_already_set();
    mod.def("fp8_dequantize", &dequantize, "vnm_fp8_dequantize with its allocation", release());
    mod.def("fp8_gelu", &gelu, "vnm_fp8_gelu with its allocations", release());
    mod.def("fp8_linear", &linear, "A differentiable linear layer in 8 bits", release());
    mod.def("fp8_gelu8", &gelu8, "GELU with an 8-bit checkpoint for its gradient", release());
    mod.def("fp8_mlp", &mlp, "A differentiable feed-forward block in 8 bits", release());
    mod.def("fp8_device_status", &device_status, "vnm_fp8_device_status", release());
}
