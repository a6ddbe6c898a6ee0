// The block-scaled 8-bit operators in the `spatha` extension: checks, allocations and the C ABI's calls, on torch's current stream.
// The autograd functions and modules on top are in fp8.py.
#include <torch/extension.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
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

Packed pack(int64_t rows, int64_t cols, c10::ScalarType f8, const Tensor &like)
{
    Packed p;
    p.ld = std::max<int64_t>(16, (cols + 15) / 16 * 16);
    p.data = device_empty({rows, p.ld}, f8, like);
    if (p.ld != cols) p.data = p.data.narrow(1, 0, cols);
    p.scales = device_empty({(cols + 511) / 512, rows, 4}, torch::kFloat8_e8m0fnu, like);
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

Tensor matmul(const Tensor &a, const Tensor &sa, const Tensor &b, const Tensor &sb, const OptTensor &bias, c10::ScalarType type)
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
    Tensor out = device_empty({M, N}, type, a);
    check(vnm_fp8_matmul(a.data_ptr(), packed_ld(a), sa.data_ptr(), f8_code(a.scalar_type(), "fp8.matmul"), b.data_ptr(), packed_ld(b), sb.data_ptr(),
                         f8_code(b.scalar_type(), "fp8.matmul"), M, N, K, with_bias ? bias->data_ptr() : nullptr, with_bias ? type_code(bias->scalar_type(), "fp8.matmul: bias") : VNM_F32,
                         out.data_ptr(), type_code(type, "fp8.matmul"), std::max(1, N), c10::cuda::getCurrentCUDAStream().stream()),
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

// A call that records a graph while its stream is being captured: the node that takes a leaf's gradient lives as long as any graph of the leaf, and belongs to
// the stream of the graph that made it.  A backward pass inside the capture that meets one of another stream waits for that stream, which ends the
// capture (and, thrown from the autograd engine's threads, may end the process), so it is refused here.
void check_capture(const std::vector<OptTensor> &inputs)
{
    for (const OptTensor &t : inputs) {
        if (!t.has_value() || !t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (!node) continue;
        const auto stream = node->stream();
        TORCH_CHECK(!stream.has_value() || *stream == c10::cuda::getCurrentCUDAStream(t->device().index()).unwrap(),
                    "a graph of the same leaf recorded on another stream still lives: free it (the tensors that hold it) before this call is captured");
    }
}

int64_t device_status()
{
    int status = 0;
    check(vnm_fp8_device_status(&status, c10::cuda::getCurrentCUDAStream().stream()), "vnm_fp8_device_status");
    return status;
}

}  // namespace

void define_fp8(pybind11::module &mod)
{
    using release = pybind11::call_guard<pybind11::gil_scoped_release>;
    mod.def("fp8_quantize", &quantize, "vnm_fp8_quantize with its allocations", release());
    mod.def("fp8_dequantize", &dequantize, "vnm_fp8_dequantize with its allocation", release());
    mod.def("fp8_matmul", &matmul, "vnm_fp8_matmul with its allocation", release());
    mod.def("fp8_gelu", &gelu, "vnm_fp8_gelu with its allocations", release());
    mod.def("fp8_gelu_grad", &gelu_grad, "vnm_fp8_gelu_grad with its allocations", release());
    mod.def("fp8_check_capture", &check_capture, "Refuses to record a graph under capture beside a graph of the same leaves on another stream");
    mod.def("fp8_device_status", &device_status, "vnm_fp8_device_status", release());
}
