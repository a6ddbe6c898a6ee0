// The block-scaled 8-bit operators in the `spatha` extension: checks, allocations and the C ABI's calls, on torch's current stream, and the
// differentiable operators as autograd nodes (see fp8.py for what the calls mean).  A step of a small layer takes as long as the host takes to queue it: a GELU and
// its gradient 85 us as a Python node, 53 here, of which torch's engine is 45.
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

#include <array>

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

// A tensor on part of a storage, without the dispatcher (a view of a tensor takes 1.5 us).
Tensor on_storage(const c10::Storage &storage, c10::ScalarType type, int64_t byte_offset, at::IntArrayRef shape, at::IntArrayRef strides)
{
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(byte_offset);      // of types of one byte
    t.unsafeGetTensorImpl()->set_sizes_and_strides(shape, strides);
    return t;
}

// A matrix in 8 bits: values and scales in one allocation.
struct Packed {
    Tensor bytes;                // undefined: not wanted
    c10::ScalarType f8 = torch::kFloat8_e4m3fn;
    int64_t rows = 0, cols = 0, ld = 16;
    bool wanted() const { return bytes.defined(); }
    void *values() const { return wanted() ? bytes.data_ptr() : nullptr; }
    void *scale() const { return wanted() ? static_cast<char *>(bytes.data_ptr()) + rows * ld : nullptr; }
    Tensor data() const { return on_storage(bytes.storage(), f8, 0, {rows, cols}, {ld, 1}); }
    Tensor scales() const { return on_storage(bytes.storage(), torch::kFloat8_e8m0fnu, rows * ld, {(cols + 511) / 512, rows, 4}, {rows * 4, 4, 1}); }
};
Packed packed(const Tensor &bytes, int64_t rows, int64_t cols, c10::ScalarType f8) { return {bytes, f8, rows, cols, std::max<int64_t>(16, (cols + 15) / 16 * 16)}; }
int64_t packed_bytes(const Packed &p) { return p.rows * p.ld + (p.cols + 511) / 512 * p.rows * 4; }
Packed pack(bool wanted, int64_t rows, int64_t cols, c10::ScalarType f8, const Tensor &like)
{
    Packed p = packed(Tensor(), rows, cols, f8);
    if (wanted) p.bytes = device_empty({packed_bytes(p)}, torch::kUInt8, like);
    return p;
}
// What a backward pass gets back of one: the bytes may have been elsewhere meanwhile (hooks on saved tensors).
Packed unpacked(const Tensor &bytes, int64_t rows, int64_t cols)
{
    const Packed p = packed(bytes, rows, cols, torch::kFloat8_e4m3fn);
    TORCH_CHECK(bytes.defined() && bytes.is_cuda() && bytes.scalar_type() == torch::kUInt8 && bytes.is_contiguous() && bytes.numel() == packed_bytes(p),
                "a saved tensor came back from its hooks in another form");
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

struct Both {
    Packed rows, cols;           // of a matrix and of its transpose
    Tensor sums;                 // of its columns
};

Both quantize(const Tensor &x_in, c10::ScalarType f8, bool square, bool rows_wanted, bool cols_wanted, c10::optional<c10::ScalarType> sums_type)
{
    const Tensor x = as_rows(x_in, "fp8.quantize");
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t rows = x.size(0), cols = x.size(1);
    const int code = f8_code(f8, "fp8.quantize"), type = type_code(x.scalar_type(), "fp8.quantize");
    const int r = to_int(rows, "fp8.quantize"), c = to_int(cols, "fp8.quantize");
    Both q = {pack(rows_wanted, rows, cols, f8, x), pack(cols_wanted, cols, rows, f8, x), undefined_or_sums(sums_type, cols, x)};
    const Tensor ws = sums_workspace(q.sums, rows, cols, x);
    check(vnm_fp8_quantize(x.data_ptr(), type, row_stride(x), r, c, code, square, q.rows.values(), q.rows.ld, q.rows.scale(), q.cols.values(), q.cols.ld, q.cols.scale(), ptr(q.sums),
                           sums_type.has_value() ? type_code(*sums_type, "fp8.quantize") : VNM_F32, ptr(ws), c10::cuda::getCurrentCUDAStream().stream()),
          "vnm_fp8_quantize");
    return q;
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

struct Operand {
    const void *data;
    int64_t ld;
    const void *scales;
    c10::ScalarType f8;
    int64_t rows, cols;
    Operand(const void *data_, int64_t ld_, const void *scales_, c10::ScalarType f8_, int64_t rows_, int64_t cols_) : data(data_), ld(ld_), scales(scales_), f8(f8_), rows(rows_), cols(cols_) {}
    Operand(const Packed &p) : data(p.values()), ld(p.ld), scales(p.scale()), f8(p.f8), rows(p.rows), cols(p.cols) {}
    Operand(const Tensor &d, const Tensor &s) : data(d.data_ptr()), ld(packed_ld(d)), scales(s.data_ptr()), f8(d.scalar_type()), rows(d.size(0)), cols(d.size(1)) {}
};

// On the current device.  aligned_rows: the result's rows begin on 16-byte boundaries, for what stays inside an operator (the quantiser reads such rows faster).
Tensor multiply(const Operand &a, const Operand &b, const Tensor &bias, c10::ScalarType type, const Tensor &like, bool aligned_rows = false)
{
    const int M = to_int(a.rows, "fp8.matmul"), N = to_int(b.rows, "fp8.matmul"), K = to_int(a.cols, "fp8.matmul");
    const int64_t ld = aligned_rows ? ((int64_t)N + 7) / 8 * 8 : N;
    Tensor out = device_empty({M, ld}, type, like);
    if (ld != N) out = out.narrow(1, 0, N);
    check(vnm_fp8_matmul(a.data, a.ld, a.scales, f8_code(a.f8, "fp8.matmul"), b.data, b.ld, b.scales, f8_code(b.f8, "fp8.matmul"), M, N, K, ptr(bias),
                         bias.defined() ? type_code(bias.scalar_type(), "fp8.matmul: bias") : VNM_F32, out.data_ptr(), type_code(type, "fp8.matmul"), std::max<int64_t>(1, ld),
                         c10::cuda::getCurrentCUDAStream().stream()),
          "vnm_fp8_matmul");
    return out;
}

void check_bias(const Tensor &bias, int64_t rows, const at::Device &device, const char *what)
{
    if (bias.defined())
        TORCH_CHECK(bias.device() == device && bias.dim() == 1 && bias.numel() == rows && bias.is_contiguous(), what, ": bias must be a contiguous vector of ", rows,
                    " values on the operands' device");
}

Tensor matmul(const Tensor &a, const Tensor &sa, const Tensor &b, const Tensor &sb, const Tensor &bias, c10::ScalarType type)
{
    check_packed(a, sa, "fp8.matmul");
    check_packed(b, sb, "fp8.matmul");
    TORCH_CHECK(a.device() == b.device(), "fp8.matmul: operands on one device expected");
    TORCH_CHECK(a.size(1) == b.size(1), "fp8.matmul: ", a.size(1), " and ", b.size(1), " columns do not match");
    check_bias(bias, b.size(0), a.device(), "fp8.matmul");
    c10::cuda::CUDAGuard guard(a.device());
    return multiply({a, sa}, {b, sb}, bias, type, a);
}

struct Gelu {
    Tensor y;
    Packed rows, cols, ckpt;
};

Gelu gelu(const Tensor &x_in, bool tanh_form, bool y_wanted, bool rows_wanted, bool cols_wanted, bool ckpt_wanted)
{
    const Tensor x = as_rows(x_in, "fp8.gelu");
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t rows = x.size(0), cols = x.size(1);
    const int type = type_code(x.scalar_type(), "fp8.gelu"), r = to_int(rows, "fp8.gelu"), c = to_int(cols, "fp8.gelu");
    Gelu g = {Tensor(), pack(rows_wanted, rows, cols, torch::kFloat8_e4m3fn, x), pack(cols_wanted, cols, rows, torch::kFloat8_e4m3fn, x),
              pack(ckpt_wanted, rows, cols, torch::kFloat8_e4m3fn, x)};
    if (y_wanted) g.y = device_empty({rows, cols}, x.scalar_type(), x);
    check(vnm_fp8_gelu(x.data_ptr(), type, row_stride(x), r, c, tanh_form, ptr(g.y), std::max<int64_t>(1, cols), g.rows.values(), g.rows.ld, g.rows.scale(), g.cols.values(), g.cols.ld,
                       g.cols.scale(), g.ckpt.values(), g.ckpt.ld, g.ckpt.scale(), c10::cuda::getCurrentCUDAStream().stream()),
          "vnm_fp8_gelu");
    return g;
}

struct GeluGrad {
    Tensor dx;
    Both both;                   // of dx in 8 bits
};

GeluGrad gelu_grad(const Tensor &dy_in, const Packed &ckpt, bool tanh_form, bool dx_wanted, c10::ScalarType f8, bool rows_wanted, bool cols_wanted, c10::optional<c10::ScalarType> sums_type)
{
    const Tensor dy = as_rows(dy_in, "fp8.gelu");
    TORCH_CHECK(ckpt.rows == dy.size(0) && ckpt.cols == dy.size(1) && ckpt.bytes.device() == dy.device(), "fp8.gelu: the checkpoint does not belong to this gradient");
    c10::cuda::CUDAGuard guard(dy.device());
    const int64_t rows = dy.size(0), cols = dy.size(1);
    const int type = type_code(dy.scalar_type(), "fp8.gelu"), r = to_int(rows, "fp8.gelu"), c = to_int(cols, "fp8.gelu"), code = f8_code(f8, "fp8.gelu");
    GeluGrad g = {Tensor(), {pack(rows_wanted, rows, cols, f8, dy), pack(cols_wanted, cols, rows, f8, dy), undefined_or_sums(sums_type, cols, dy)}};
    if (dx_wanted) g.dx = device_empty({rows, cols}, dy.scalar_type(), dy);
    const Tensor ws = sums_workspace(g.both.sums, rows, cols, dy);
    check(vnm_fp8_gelu_grad(dy.data_ptr(), type, row_stride(dy), r, c, tanh_form, ckpt.values(), ckpt.ld, ckpt.scale(), ptr(g.dx), std::max<int64_t>(1, cols), code, g.both.rows.values(),
                            g.both.rows.ld, g.both.rows.scale(), g.both.cols.values(), g.both.cols.ld, g.both.cols.scale(), ptr(g.both.sums),
                            sums_type.has_value() ? type_code(*sums_type, "fp8.gelu") : VNM_F32, ptr(ws), c10::cuda::getCurrentCUDAStream().stream()),
          "vnm_fp8_gelu_grad");
    return g;
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

Tensor or_undefined(const OptTensor &t) { return t.has_value() ? *t : Tensor(); }
c10::optional<c10::ScalarType> type_of(bool wanted, c10::ScalarType t) { return wanted ? c10::optional<c10::ScalarType>(t) : c10::nullopt; }

Both quantized(const Tensor &x, c10::ScalarType f8, bool square, bool rows, bool cols, c10::optional<c10::ScalarType> sums)
{
    if (!rows && !cols) return {};
    return quantize(x, f8, square, rows, cols, sums);
}
// a b^T (+ bias); zeros where there is nothing to sum (a gradient without any token or output)
Tensor product(const Packed &a, const Packed &b, const Tensor &bias, c10::ScalarType type, bool aligned_rows = false)
{
    TORCH_CHECK(a.bytes.device() == b.bytes.device(), "a saved tensor came back from its hooks on another device");
    c10::cuda::CUDAGuard guard(a.bytes.device());
    if (a.cols == 0) return torch::zeros({a.rows, b.rows}, a.bytes.options().dtype(type));
    return multiply(a, b, bias.defined() ? bias.detach().contiguous() : bias, type, a.bytes, aligned_rows);
}

// What a node keeps besides tensors, as one list: a shape behind N numbers.
template <size_t N>
void keep(AutogradContext *ctx, const std::array<int64_t, N> &numbers, at::IntArrayRef shape)
{
    std::vector<int64_t> v(numbers.begin(), numbers.end());
    v.insert(v.end(), shape.begin(), shape.end());
    ctx->saved_data["kept"] = std::move(v);
}
struct Kept {
    std::vector<int64_t> v;
    size_t n;
    Kept(AutogradContext *ctx, size_t numbers) : v(ctx->saved_data["kept"].toIntVector()), n(numbers) {}
    int64_t operator[](size_t i) const { return v[i]; }
    c10::ScalarType type(size_t i) const { return (c10::ScalarType)v[i]; }
    at::IntArrayRef shape() const { return at::IntArrayRef(v).slice(n); }
};
Tensor viewed(const Tensor &t, at::IntArrayRef shape) { return t.sizes() == shape ? t : t.view(shape); }

// What a backward pass needs of a weight is its transpose in 8 bits, in . out bytes.  It is written beside the forward operand from one read and kept while that is no
// more than a 16-bit layer keeps: its input takes in . tokens bytes here and 2 in . tokens there, so for out <= tokens; where input and weight differ in type such a layer keeps a
// cast weight as well.  Elsewhere a leaf, which lives anyway, is kept itself and quantised again (12288 x 12288 with 2048 tokens: 176 -> 25 MB kept, for a second pass over
// the weight).  What is not a leaf is kept in 8 bits, half of its own size; so are tensors made in inference mode, which no graph may hold.
bool again_later(const Tensor &w, const Tensor &x, int64_t tokens) { return w.size(0) > tokens && w.is_leaf() && !w.is_inference() && w.scalar_type() == x.scalar_type(); }
Packed transposed_weight(const Tensor &saved, bool again, int64_t rows, int64_t cols)
{
    if (!again) return unpacked(saved, cols, rows);
    TORCH_CHECK(saved.defined() && saved.is_cuda() && saved.dim() == 2 && saved.size(0) == rows && saved.size(1) == cols && is_float(saved.scalar_type()),
                "a saved tensor came back from its hooks in another form");
    return quantize(saved, torch::kFloat8_e4m3fn, true, false, true, c10::nullopt).cols;
}

struct Linear : torch::autograd::Function<Linear> {
    enum { X_TYPE, W_TYPE, BIAS_TYPE, GRAD_TYPE, HAS_BIAS, AGAIN, TOKENS, IN, OUT, NUMBERS };
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const OptTensor &opt_bias, c10::ScalarType grad_type, bool record)
    {
        const Tensor bias = or_undefined(opt_bias);
        const bool need_x = record && wants_grad(x), need_w = record && wants_grad(w);
        const Both xs = quantized(flat(x), torch::kFloat8_e4m3fn, false, true, need_w, c10::nullopt);
        const bool again = need_x && again_later(w, x, xs.rows.rows);
        const Both ws = quantized(w, torch::kFloat8_e4m3fn, true, true, need_x && !again, c10::nullopt);
        const Tensor y = product(xs.rows, ws.rows, bias, x.scalar_type());
        ctx->save_for_backward({xs.cols.bytes, again ? w : ws.cols.bytes});
        keep<NUMBERS>(ctx, {(int64_t)x.scalar_type(), (int64_t)w.scalar_type(), (int64_t)(bias.defined() ? bias.scalar_type() : x.scalar_type()), (int64_t)grad_type, bias.defined(),
                            again, xs.rows.rows, w.size(1), w.size(0)}, x.sizes());
        return shaped(y, x.sizes());
    }
    static variable_list backward(AutogradContext *ctx, variable_list dys)
    {
        const variable_list saved = ctx->get_saved_variables();
        const Kept kept(ctx, NUMBERS);
        // counted over the tensors that there are
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = kept[HAS_BIAS] && ctx->needs_input_grad(2);
        const Both g = quantized(flat(dys[0]), kept.type(GRAD_TYPE), false, need_x, need_w || need_b, type_of(need_b, kept.type(BIAS_TYPE)));
        Tensor dx, dw;
        if (need_x) dx = viewed(product(g.rows, transposed_weight(saved[1], kept[AGAIN] != 0, kept[OUT], kept[IN]), Tensor(), kept.type(X_TYPE)), kept.shape());
        if (need_w) dw = product(g.cols, unpacked(saved[0], kept[IN], kept[TOKENS]), Tensor(), kept.type(W_TYPE));
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
    enum { TANH, ROWS, COLS, NUMBERS };
    static Tensor forward(AutogradContext *ctx, const Tensor &x, bool tanh_form, bool record)
    {
        const Gelu g = gelu(flat(x), tanh_form, true, false, false, record && wants_grad(x));
        ctx->save_for_backward({g.ckpt.bytes});
        keep<NUMBERS>(ctx, {tanh_form, g.ckpt.rows, g.ckpt.cols}, x.sizes());
        return viewed(g.y, x.sizes());
    }
    static variable_list backward(AutogradContext *ctx, variable_list dys)
    {
        const variable_list saved = ctx->get_saved_variables();
        const Kept kept(ctx, NUMBERS);
        const GeluGrad g = gelu_grad(flat(dys[0]), unpacked(saved[0], kept[ROWS], kept[COLS]), kept[TANH] != 0, true, torch::kFloat8_e4m3fn, false, false, c10::nullopt);
        return once({viewed(g.dx, kept.shape()), Tensor(), Tensor()}, dys);
    }
};

Tensor gelu8(const Tensor &x, bool tanh_form)
{
    check_input(x, "fp8.gelu");
    check_capture({&x});
    return Gelu8::apply(x, tanh_form, at::GradMode::is_enabled());
}

struct Mlp : torch::autograd::Function<Mlp> {
    enum { X_TYPE, W1_TYPE, B1_TYPE, W2_TYPE, B2_TYPE, GRAD_TYPE, TANH, HAS_B1, HAS_B2, AGAIN1, AGAIN2, TOKENS, IN, HIDDEN, OUT, NUMBERS };
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w1, const OptTensor &opt_b1, const Tensor &w2, const OptTensor &opt_b2, bool tanh_form,
                          c10::ScalarType grad_type, bool record)
    {
        const Tensor b1 = or_undefined(opt_b1), b2 = or_undefined(opt_b2);
        const bool need_x = record && wants_grad(x), need_w1 = record && wants_grad(w1), need_b1 = record && wants_grad(b1), need_w2 = record && wants_grad(w2);
        const bool inner = need_x || need_w1 || need_b1;      // whether the gradient goes back through the GELU
        const Both xs = quantized(flat(x), torch::kFloat8_e4m3fn, false, true, need_w1, c10::nullopt);
        const bool again1 = need_x && again_later(w1, x, xs.rows.rows), again2 = inner && again_later(w2, x, xs.rows.rows);
        const Both w1s = quantized(w1, torch::kFloat8_e4m3fn, true, true, need_x && !again1, c10::nullopt);
        const Gelu a = gelu(product(xs.rows, w1s.rows, b1, x.scalar_type(), true), tanh_form, false, true, need_w2, inner);
        const Both w2s = quantized(w2, torch::kFloat8_e4m3fn, true, true, inner && !again2, c10::nullopt);
        const Tensor y = product(a.rows, w2s.rows, b2, x.scalar_type());
        ctx->save_for_backward({xs.cols.bytes, again1 ? w1 : w1s.cols.bytes, a.cols.bytes, a.ckpt.bytes, again2 ? w2 : w2s.cols.bytes});
        keep<NUMBERS>(ctx, {(int64_t)x.scalar_type(), (int64_t)w1.scalar_type(), (int64_t)(b1.defined() ? b1.scalar_type() : x.scalar_type()), (int64_t)w2.scalar_type(),
                            (int64_t)(b2.defined() ? b2.scalar_type() : x.scalar_type()), (int64_t)grad_type, tanh_form, b1.defined(), b2.defined(), again1, again2, xs.rows.rows, w1.size(1),
                            w1.size(0), w2.size(0)}, x.sizes());
        return shaped(y, x.sizes());
    }
    static variable_list backward(AutogradContext *ctx, variable_list dys)
    {
        const variable_list s = ctx->get_saved_variables();
        const Kept kept(ctx, NUMBERS);
        const int64_t tokens = kept[TOKENS], hidden = kept[HIDDEN];
        const bool has_b1 = kept[HAS_B1] != 0, has_b2 = kept[HAS_B2] != 0;
        const size_t at_w2 = has_b1 ? 3 : 2;      // counted over the tensors that there are
        const bool need_x = ctx->needs_input_grad(0), need_w1 = ctx->needs_input_grad(1), need_b1 = has_b1 && ctx->needs_input_grad(2), need_w2 = ctx->needs_input_grad(at_w2),
                   need_b2 = has_b2 && ctx->needs_input_grad(at_w2 + 1), inner = need_x || need_w1 || need_b1;
        const Both g = quantized(flat(dys[0]), kept.type(GRAD_TYPE), false, inner, need_w2 || need_b2, type_of(need_b2, kept.type(B2_TYPE)));
        Tensor dx, dw1, db1, dw2;
        if (need_w2) dw2 = product(g.cols, unpacked(s[2], hidden, tokens), Tensor(), kept.type(W2_TYPE));
        if (inner) {
            const Tensor da = product(g.rows, transposed_weight(s[4], kept[AGAIN2] != 0, kept[OUT], hidden), Tensor(), kept.type(X_TYPE), true);
            const GeluGrad h = gelu_grad(da, unpacked(s[3], tokens, hidden), kept[TANH] != 0, false, kept.type(GRAD_TYPE), need_x, need_w1 || need_b1, type_of(need_b1, kept.type(B1_TYPE)));
            db1 = h.both.sums;
            if (need_x) dx = viewed(product(h.both.rows, transposed_weight(s[1], kept[AGAIN1] != 0, hidden, kept[IN]), Tensor(), kept.type(X_TYPE)), kept.shape());
            if (need_w1) dw1 = product(h.both.cols, unpacked(s[0], kept[IN], tokens), Tensor(), kept.type(W1_TYPE));
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

// ---- frozen weights, as modules hold them: e4m3 values as bytes [rows, padded columns], scales as bytes [ceil(columns / 512), rows, 4] ----

Operand held(const Tensor &w, const Tensor &scales, int64_t cols, const Tensor &bias, const at::Device &device, const char *what)
{
    TORCH_CHECK(w.device() == device && scales.device() == device, what, ": the weight's values and scales must be on the input's CUDA device");
    TORCH_CHECK(w.scalar_type() == torch::kUInt8 && w.dim() == 2 && w.is_contiguous() && w.size(1) == packed(w, 0, cols, torch::kFloat8_e4m3fn).ld, what,
                ": a weight's values must be bytes in rows of ", cols, " padded to 16");
    TORCH_CHECK(scales.scalar_type() == torch::kUInt8 && scales.dim() == 3 && scales.is_contiguous() && scales.size(0) == (cols + 511) / 512 && scales.size(1) == w.size(0) &&
                    scales.size(2) == 4,
                what, ": a weight's scales must be bytes [ceil(columns / 512), rows, 4]");
    check_bias(bias, w.size(0), device, what);
    return {w.data_ptr(), w.size(1), scales.data_ptr(), torch::kFloat8_e4m3fn, w.size(0), cols};
}
Packed held_input(const Tensor &x, int64_t features, const char *what)
{
    check_input(x, what);
    TORCH_CHECK(x.size(-1) == features, what, ": ", x.size(-1), " features do not match a weight of ", features);
    return quantize(flat(x), torch::kFloat8_e4m3fn, false, true, false, c10::nullopt).rows;
}

Tensor held_linear(const Tensor &x, const Tensor &w, const Tensor &sw, int64_t cols, const OptTensor &bias)
{
    const Tensor b = or_undefined(bias);
    const Packed q = held_input(x, cols, "Fp8Linear");
    const Operand weight = held(w, sw, cols, b, x.device(), "Fp8Linear");
    c10::cuda::CUDAGuard guard(x.device());
    return shaped(multiply(q, weight, b, x.scalar_type(), x), x.sizes());
}

Tensor held_mlp(const Tensor &x, const Tensor &w1, const Tensor &sw1, int64_t cols1, const OptTensor &bias1, const Tensor &w2, const Tensor &sw2, int64_t cols2, const OptTensor &bias2,
                bool tanh_form)
{
    const Tensor b1 = or_undefined(bias1), b2 = or_undefined(bias2);
    const Packed q = held_input(x, cols1, "Fp8Mlp");
    const Operand fc = held(w1, sw1, cols1, b1, x.device(), "Fp8Mlp"), proj = held(w2, sw2, cols2, b2, x.device(), "Fp8Mlp");
    TORCH_CHECK(fc.rows == cols2, "Fp8Mlp: ", fc.rows, " features do not match a weight of ", cols2);
    c10::cuda::CUDAGuard guard(x.device());
    const Gelu g = gelu(multiply(q, fc, b1, x.scalar_type(), x, true), tanh_form, false, true, false, false);
    return shaped(multiply(g.rows, proj, b2, x.scalar_type(), x), x.sizes());
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
    Tensor parts[4];
    {
        pybind11::gil_scoped_release no_gil;
        const Both q = quantize(x, f8, square, true, both, c10::nullopt);
        parts[0] = q.rows.data();
        parts[1] = q.rows.scales();
        if (both) {
            parts[2] = q.cols.data();
            parts[3] = q.cols.scales();
        }
    }
    const int count = both ? 4 : 2;
    PyObject *out = PyTuple_New(count);
    if (!out) return nullptr;
    for (int i = 0; i < count; i++) PyTuple_SET_ITEM(out, i, THPVariable_Wrap(std::move(parts[i])));
    return out;
    END_HANDLE_TH_ERRORS
}

// (a, a's scales, b, b's scales, bias or None, dtype) -> a b^T (+ bias)
PyObject *py_matmul(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 6, "matmul(a, a_scales, b, b_scales, bias, dtype)");
    const Tensor &a = tensor_of(args[0]), &sa = tensor_of(args[1]), &b = tensor_of(args[2]), &sb = tensor_of(args[3]);
    const Tensor bias = args[4] == Py_None ? Tensor() : tensor_of(args[4]);
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
    mod.def("fp8_held_linear", &held_linear, "A linear layer whose weight is held in 8 bits", release());
    mod.def("fp8_held_mlp", &held_mlp, "A feed-forward block whose weights are held in 8 bits", release());
    mod.def("fp8_linear", &linear, "A differentiable linear layer in 8 bits", release());
    mod.def("fp8_gelu8", &gelu8, "GELU with an 8-bit checkpoint for its gradient", release());
    mod.def("fp8_mlp", &mlp, "A differentiable feed-forward block in 8 bits", release());
    mod.def("fp8_device_status", &device_status, "vnm_fp8_device_status", release());
}
