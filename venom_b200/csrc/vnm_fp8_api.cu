// C ABI of the block-scaled 8-bit operators (see include/venom_b200.h): argument checks, tensor maps and the choice of kernel.
#include "../../include/venom_b200.h"
#include "vnm_fp8.h"

#include <cstdarg>
#include <cstdio>
#include <mutex>

using namespace vnm;

namespace {

int fail(int code, const char *fmt, ...)
{
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return set_last_error(code, buf);
}

int done(cudaError_t e, const char *what) { return e == cudaSuccess ? VNM_OK : fail(VNM_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e)); }

int64_t elem_size(int type) { return type == VNM_F32 ? 4 : 2; }
bool known_type(int type) { return type == VNM_F32 || type == VNM_F16 || type == VNM_BF16; }
bool aligned(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// The tiles kernel has a block for each 128 x 128, the rows kernel counts pieces of 512 columns (and runs a grid past the last one): both in 32 bits.
int check_shape(const char *name, const void *x, int type, int64_t ldx, int rows, int cols)
{
    if (rows < 0 || cols < 0) return fail(VNM_ERR_BAD_ARG, "%s: negative size (%d, %d)", name, rows, cols);
    if (!known_type(type)) return fail(VNM_ERR_BAD_ARG, "%s: unknown type %d", name, type);
    if (rows == 0 || cols == 0) return VNM_OK;
    if (!x) return fail(VNM_ERR_BAD_ARG, "%s: null input", name);
    if (ldx < cols) return fail(VNM_ERR_BAD_ARG, "%s: leading dimension %lld is less than %d columns", name, (long long)ldx, cols);
    if (!aligned(x, (uintptr_t)elem_size(type))) return fail(VNM_ERR_BAD_ARG, "%s: input is not aligned to its type", name);
    if (((int64_t)rows + 127) / 128 * (((int64_t)cols + 127) / 128) > INT32_MAX || (int64_t)rows * (((int64_t)cols + 511) / 512) > INT32_MAX - (1 << 20) || cols > INT32_MAX - 512)
        return fail(VNM_ERR_UNSUPPORTED, "%s: %d x %d is too large", name, rows, cols);
    return VNM_OK;
}

int check_f8(const char *name, const char *what, const void *data, int64_t ld, const void *scales, int rows, int cols)
{
    if (!data && !scales) return VNM_OK;
    if (rows == 0 || cols == 0) return VNM_OK;
    if (!data || !scales) return fail(VNM_ERR_BAD_ARG, "%s: %s needs both values and scales", name, what);
    if (ld < cols || ld % 16 || !aligned(data, 16)) return fail(VNM_ERR_BAD_ARG, "%s: %s must lie in rows of a multiple of 16 bytes, at least %d, on a 16-byte boundary", name, what, cols);
    if (!aligned(scales, 4)) return fail(VNM_ERR_BAD_ARG, "%s: scales of %s must be 4-byte aligned", name, what);
    return VNM_OK;
}

int check_value(const char *name, const char *what, const void *y, int64_t ld, int type, int rows, int cols)
{
    if (!y || rows == 0 || cols == 0) return VNM_OK;
    if (ld < cols || !aligned(y, (uintptr_t)elem_size(type))) return fail(VNM_ERR_BAD_ARG, "%s: %s needs a leading dimension of at least %d and its type's alignment", name, what, cols);
    return VNM_OK;
}

int check_sums(const char *name, const void *colsum, int type, const void *workspace, const void *data_t, int rows, int cols)
{
    if (!colsum) return VNM_OK;
    if (!known_type(type)) return fail(VNM_ERR_BAD_ARG, "%s: unknown type %d of the column sums", name, type);
    if (!aligned(colsum, (uintptr_t)elem_size(type)) || !aligned(workspace, 4)) return fail(VNM_ERR_BAD_ARG, "%s: column sums or workspace are not aligned", name);
    if (rows && cols && (!workspace || !data_t)) return fail(VNM_ERR_BAD_ARG, "%s: column sums need a workspace and the transpose", name);
    return VNM_OK;
}

int check_product_size(const char *name, int M, int N, int K)
{
    if (K > INT32_MAX - 256 || M > INT32_MAX - 256 || N > INT32_MAX - 256 || ((int64_t)M + 15) / 16 * (((int64_t)N + 127) / 128) > INT32_MAX / 8)
        return fail(VNM_ERR_UNSUPPORTED, "%s: %d x %d x %d is too large", name, M, N, K);
    return VNM_OK;
}

bool pieces(const void *x, int type, int64_t ld) { return aligned(x, 16) && ld * elem_size(type) % 16 == 0; }

int row_alignment(const void *x, int type, int64_t ld)
{
    const uintptr_t both = reinterpret_cast<uintptr_t>(x) | (uintptr_t)(ld * elem_size(type));
    return (both & 15) == 0 ? 16 : (both & 3) == 0 ? 4 : 2;
}

void set_input(Fp8QuantParams *p, const void *x, int type, int64_t ldx, int rows, int cols)
{
    p->x = x; p->ldx = ldx; p->rows = rows; p->cols = cols;
    p->align_x = row_alignment(x, type, ldx);
}

#define VNM_TRY(call)               \
    do {                            \
        const int rc__ = (call);    \
        if (rc__ != VNM_OK) return rc__; \
    } while (0)

int empty_sums(void *colsum, int type, int cols, cudaStream_t stream)
{
    if (!colsum || cols == 0) return VNM_OK;
    return done(cudaMemsetAsync(colsum, 0, (size_t)cols * elem_size(type), stream), "column sums of no rows");
}

// What a device needs once: shared-memory limits, the status word's address, what plans depend on.  Not written again once it is ready.
constexpr int kMaxDevices = 64;
struct Device {
    bool ready;
    int *status;
    Fp8Device plans;
};
Device g_devices[kMaxDevices];
std::mutex g_mutex;
__device__ int g_status;

int device_ready(const Device **ready)
{
    int dev = -1;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return done(e, "cudaGetDevice");
    if (dev < 0 || dev >= kMaxDevices) return fail(VNM_ERR_UNSUPPORTED, "device index %d not supported", dev);
    std::lock_guard<std::mutex> lock(g_mutex);
    Device &d = g_devices[dev];
    if (!d.ready) {
        // settings of the kernels are not work that a capture on this thread must not miss
        struct Relaxed {
            cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
            Relaxed() { (void)cudaThreadExchangeStreamCaptureMode(&mode); }
            ~Relaxed() { (void)cudaThreadExchangeStreamCaptureMode(&mode); }
        } relaxed;
        if ((e = cudaDeviceGetAttribute(&d.plans.sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return done(e, "cudaDeviceGetAttribute");
        if ((e = fp8_small_init()) != cudaSuccess || (e = fp8_pair_init(d.plans.sms, &d.plans.clusters)) != cudaSuccess) return done(e, "cudaFuncSetAttribute(max dynamic shared memory)");
        void *at = nullptr;
        if ((e = cudaGetSymbolAddress(&at, g_status)) != cudaSuccess) return done(e, "cudaGetSymbolAddress");
        d.status = static_cast<int *>(at);
        d.ready = true;
    }
    *ready = &d;
    return VNM_OK;
}

// [rows, K] bytes as boxes of 128 bytes x `box` rows, 128-byte swizzle; rows and k past the end read as zeros.
CUresult encode_operand(EncodeTiledFn enc, CUtensorMap *map, const void *data, int64_t ld, int rows, int K, int box)
{
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    const cuuint32_t boxes[2] = {128, (cuuint32_t)box}, steps[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(data), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// The kernel and tile with the smaller estimate.
int choose_plan(int M, int N, int K, bool wide_out, bool whole, bool bias, const Fp8Device &device, Fp8Plan *plan, bool *on_pairs)
{
    Fp8Plan small = {}, pair = {};
    const float small_us = fp8_small_config(M, N, (int)(((int64_t)K + 127) / 128), wide_out, device, &small),
                pair_us = fp8_pair_config(M, N, K, wide_out, whole, bias, device, &pair);
    if (small_us < 0.0f && pair_us < 0.0f) return fail(VNM_ERR_UNSUPPORTED, "vnm_fp8_matmul: no kernel for %d x %d x %d", M, N, K);
    *on_pairs = small_us < 0.0f || (pair_us >= 0.0f && pair_us < small_us);
    *plan = *on_pairs ? pair : small;
    return VNM_OK;
}

// Band of the tile order of the pair kernel.  A band's operand stays in L2 while the other one streams past: row bands read A once and B once per
// band, column bands the other way round.
int tile_band(int M, int N, int K, int mt, int nt, int bn)
{
    const int64_t room = 32 << 20;
    int64_t g = room / (256 * (int64_t)K), q = room / (bn * (int64_t)K);
    g = g < 1 ? 1 : g > mt ? mt : g;
    q = q < 1 ? 1 : q > nt ? nt : q;
    const int64_t a = (int64_t)M * K, b = (int64_t)N * K;
    return a + b * ((mt + g - 1) / g) <= b + a * ((nt + q - 1) / q) ? (int)g : -(int)q;
}

}  // namespace

extern "C" int64_t vnm_fp8_scale_bytes(int rows, int cols)
{
    if (rows <= 0 || cols <= 0) return 0;
    return (((int64_t)cols + 511) / 512) * rows * 4;
}

extern "C" int vnm_fp8_quantize(const void *x, int x_type, int64_t ldx, int rows, int cols, int f8_type, int square, void *data, int64_t ldd, void *scales,
                                void *data_t, int64_t ldt, void *scales_t, void *colsum, int colsum_type, void *workspace, void *stream)
{
    const char *name = "vnm_fp8_quantize";
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    VNM_TRY(check_shape(name, x, x_type, ldx, rows, cols));
    if (f8_type != VNM_E4M3 && f8_type != VNM_E5M2) return fail(VNM_ERR_BAD_ARG, "%s: unknown 8-bit type %d", name, f8_type);
    VNM_TRY(check_f8(name, "the result", data, ldd, scales, rows, cols));
    VNM_TRY(check_f8(name, "the transpose", data_t, ldt, scales_t, cols, rows));
    VNM_TRY(check_sums(name, colsum, colsum_type, workspace, data_t, rows, cols));
    if (rows == 0 || cols == 0) return empty_sums(colsum, colsum_type, cols, s);
    if (!data && !data_t) return fail(VNM_ERR_BAD_ARG, "%s: nothing is wanted", name);
    Fp8QuantParams p = {};
    set_input(&p, x, x_type, ldx, rows, cols);
    p.f8 = f8_type;
    p.data = static_cast<uint8_t *>(data); p.ldd = ldd; p.scales = static_cast<uint8_t *>(scales);
    p.data_t = static_cast<uint8_t *>(data_t); p.ldt = ldt; p.scales_t = static_cast<uint8_t *>(scales_t);
    p.partial = colsum ? static_cast<float *>(workspace) : nullptr;
    if (!data_t && !square) return done(launch_fp8_rows(p, x_type, FP8_PLAIN, s), name);
    VNM_TRY(done(launch_fp8_tiles(p, x_type, FP8_PLAIN, square != 0, s), name));
    return colsum ? done(launch_fp8_colsum(p.partial, (int)(((int64_t)rows + 127) / 128), cols, colsum, colsum_type, s), name) : VNM_OK;
}

extern "C" int vnm_fp8_dequantize(const void *data, int64_t ldd, const void *scales, int f8_type, int rows, int cols, void *out, int out_type, int64_t ldo, void *stream)
{
    const char *name = "vnm_fp8_dequantize";
    VNM_TRY(check_shape(name, data, VNM_BF16, ldd, rows, cols));
    if (!known_type(out_type)) return fail(VNM_ERR_BAD_ARG, "%s: unknown type %d", name, out_type);
    if (f8_type != VNM_E4M3 && f8_type != VNM_E5M2) return fail(VNM_ERR_BAD_ARG, "%s: unknown 8-bit type %d", name, f8_type);
    if (rows == 0 || cols == 0) return VNM_OK;
    if (!out) return fail(VNM_ERR_BAD_ARG, "%s: null result", name);
    VNM_TRY(check_f8(name, "the input", data, ldd, scales, rows, cols));
    VNM_TRY(check_value(name, "the result", out, ldo, out_type, rows, cols));
    return done(launch_fp8_dequantize(static_cast<const uint8_t *>(data), ldd, static_cast<const uint8_t *>(scales), f8_type, rows, cols, out, out_type, ldo,
                                      row_alignment(out, out_type, ldo), static_cast<cudaStream_t>(stream)), name);
}

extern "C" int vnm_fp8_gelu(const void *x, int x_type, int64_t ldx, int rows, int cols, int tanh_form, void *y, int64_t ldy, void *data, int64_t ldd, void *scales,
                            void *data_t, int64_t ldt, void *scales_t, void *ckpt, int64_t ldc, void *ckpt_scales, void *stream)
{
    const char *name = "vnm_fp8_gelu";
    VNM_TRY(check_shape(name, x, x_type, ldx, rows, cols));
    VNM_TRY(check_value(name, "the result", y, ldy, x_type, rows, cols));
    VNM_TRY(check_f8(name, "the 8-bit result", data, ldd, scales, rows, cols));
    VNM_TRY(check_f8(name, "the transpose", data_t, ldt, scales_t, cols, rows));
    VNM_TRY(check_f8(name, "the checkpoint", ckpt, ldc, ckpt_scales, rows, cols));
    if (rows == 0 || cols == 0) return VNM_OK;
    if (y && data_t) return fail(VNM_ERR_UNSUPPORTED, "%s: the result in its own type together with a transpose", name);
    if (!y && !data && !data_t) return fail(VNM_ERR_BAD_ARG, "%s: nothing is wanted", name);
    Fp8QuantParams p = {};
    set_input(&p, x, x_type, ldx, rows, cols);
    p.f8 = VNM_E4M3; p.tanh_form = tanh_form != 0;
    p.y = y; p.ldy = ldy; p.align_y = row_alignment(y, x_type, ldy);
    p.data = static_cast<uint8_t *>(data); p.ldd = ldd; p.scales = static_cast<uint8_t *>(scales);
    p.data_t = static_cast<uint8_t *>(data_t); p.ldt = ldt; p.scales_t = static_cast<uint8_t *>(scales_t);
    p.ckpt = static_cast<uint8_t *>(ckpt); p.ldc = ldc; p.ckpt_scales = static_cast<uint8_t *>(ckpt_scales);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return done(data_t ? launch_fp8_tiles(p, x_type, FP8_GELU, false, s) : launch_fp8_rows(p, x_type, FP8_GELU, s), name);
}

extern "C" int vnm_fp8_gelu_grad(const void *dy, int dy_type, int64_t ldy, int rows, int cols, int tanh_form, const void *ckpt, int64_t ldc, const void *ckpt_scales, void *dx,
                                 int64_t lddx, int f8_type, void *data, int64_t ldd, void *scales, void *data_t, int64_t ldt, void *scales_t, void *colsum,
                                 int colsum_type, void *workspace, void *stream)
{
    const char *name = "vnm_fp8_gelu_grad";
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    VNM_TRY(check_shape(name, dy, dy_type, ldy, rows, cols));
    if (f8_type != VNM_E4M3 && f8_type != VNM_E5M2) return fail(VNM_ERR_BAD_ARG, "%s: unknown 8-bit type %d", name, f8_type);
    VNM_TRY(check_value(name, "the result", dx, lddx, dy_type, rows, cols));
    VNM_TRY(check_f8(name, "the 8-bit result", data, ldd, scales, rows, cols));
    VNM_TRY(check_f8(name, "the transpose", data_t, ldt, scales_t, cols, rows));
    VNM_TRY(check_f8(name, "the checkpoint", ckpt, ldc, ckpt_scales, rows, cols));
    VNM_TRY(check_sums(name, colsum, colsum_type, workspace, data_t, rows, cols));
    if (rows == 0 || cols == 0) return empty_sums(colsum, colsum_type, cols, s);
    if (!ckpt) return fail(VNM_ERR_BAD_ARG, "%s: no checkpoint", name);
    if (dx && data_t) return fail(VNM_ERR_UNSUPPORTED, "%s: the result in its own type together with a transpose", name);
    if (!dx && !data && !data_t) return fail(VNM_ERR_BAD_ARG, "%s: nothing is wanted", name);
    Fp8QuantParams p = {};
    set_input(&p, dy, dy_type, ldy, rows, cols);
    p.f8 = f8_type; p.tanh_form = tanh_form != 0;
    p.y = dx; p.ldy = lddx; p.align_y = row_alignment(dx, dy_type, lddx);
    p.data = static_cast<uint8_t *>(data); p.ldd = ldd; p.scales = static_cast<uint8_t *>(scales);
    p.data_t = static_cast<uint8_t *>(data_t); p.ldt = ldt; p.scales_t = static_cast<uint8_t *>(scales_t);
    p.ckpt = static_cast<uint8_t *>(const_cast<void *>(ckpt)); p.ldc = ldc; p.ckpt_scales = static_cast<uint8_t *>(const_cast<void *>(ckpt_scales));
    p.partial = colsum ? static_cast<float *>(workspace) : nullptr;
    if (!data_t) return done(launch_fp8_rows(p, dy_type, FP8_GELU_GRAD, s), name);
    VNM_TRY(done(launch_fp8_tiles(p, dy_type, FP8_GELU_GRAD, false, s), name));
    return colsum ? done(launch_fp8_colsum(p.partial, (int)(((int64_t)rows + 127) / 128), cols, colsum, colsum_type, s), name) : VNM_OK;
}

extern "C" int vnm_fp8_matmul(const void *a, int64_t lda, const void *a_scales, int a_type, const void *b, int64_t ldb, const void *b_scales, int b_type, int M, int N, int K,
                              const void *bias, int bias_type, void *out, int out_type, int64_t ldo, void *stream)
{
    const char *name = "vnm_fp8_matmul";
    if (M < 0 || N < 0 || K < 1) return fail(VNM_ERR_BAD_ARG, "%s: sizes must not be negative and K at least 1 (got %d, %d, %d)", name, M, N, K);
    if ((a_type != VNM_E4M3 && a_type != VNM_E5M2) || (b_type != VNM_E4M3 && b_type != VNM_E5M2)) return fail(VNM_ERR_BAD_ARG, "%s: unknown 8-bit type", name);
    if (!known_type(out_type) || (bias && !known_type(bias_type))) return fail(VNM_ERR_BAD_ARG, "%s: unknown type of the result or bias", name);
    if (M == 0 || N == 0) return VNM_OK;
    if (!a || !b || !out) return fail(VNM_ERR_BAD_ARG, "%s: null operand", name);
    VNM_TRY(check_f8(name, "A", a, lda, a_scales, M, K));
    VNM_TRY(check_f8(name, "B", b, ldb, b_scales, N, K));
    VNM_TRY(check_value(name, "the result", out, ldo, out_type, M, N));
    if (bias && !aligned(bias, (uintptr_t)elem_size(bias_type))) return fail(VNM_ERR_BAD_ARG, "%s: bias is not aligned to its type", name);
    VNM_TRY(check_product_size(name, M, N, K));
    const Device *device = nullptr;
    VNM_TRY(device_ready(&device));
    const EncodeTiledFn enc = get_encode_fn();
    if (!enc) return fail(VNM_ERR_CUDA, "cuTensorMapEncodeTiled not available");
    Fp8MatmulParams p = {};
    p.sa = static_cast<const uint32_t *>(a_scales); p.sb = static_cast<const uint32_t *>(b_scales);
    p.bias = bias; p.bias_type = bias_type;
    p.out = out; p.out_type = out_type; p.ldo = ldo;
    p.whole_pieces = pieces(out, out_type, ldo);
    p.M = M; p.N = N; p.K = K; p.ktiles = (K + 127) / 128;
    p.a_f8 = a_type; p.b_f8 = b_type;
    p.status = device->status;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    Fp8Plan plan = {};
    bool on_pairs = false;
    VNM_TRY(choose_plan(M, N, K, out_type == VNM_F32, p.whole_pieces != 0, bias != nullptr, device->plans, &plan, &on_pairs));
    CUtensorMap map_a, map_b;
    if (encode_operand(enc, &map_a, a, lda, M, K, on_pairs ? 128 : plan.bn) != CUDA_SUCCESS || encode_operand(enc, &map_b, b, ldb, N, K, on_pairs ? plan.bn / 2 : 128) != CUDA_SUCCESS)
        return fail(VNM_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed", name);
    p.split = plan.split;
    if (on_pairs) {
        p.mt = (M + 255) / 256;
        p.nt = (N + plan.bn - 1) / plan.bn;
        p.order = TileOrder(p.mt, p.nt, tile_band(M, N, K, p.mt, p.nt, plan.bn));
        return done(launch_fp8_pair(plan, map_a, map_b, p, s), name);
    }
    p.mt = (M + plan.bn - 1) / plan.bn;
    p.nt = (N + 127) / 128;
    return done(launch_fp8_small(plan, map_a, map_b, p, s), name);
}

extern "C" int vnm_fp8_matmul_config(int M, int N, int K, int out_type, int whole, int bias, int *tile_m, int *tile_n, int *split, int *grid)
{
    const char *name = "vnm_fp8_matmul_config";
    if (M < 1 || N < 1 || K < 1) return fail(VNM_ERR_BAD_ARG, "%s: sizes must be positive (got %d, %d, %d)", name, M, N, K);
    if (!known_type(out_type)) return fail(VNM_ERR_BAD_ARG, "%s: unknown type %d", name, out_type);
    VNM_TRY(check_product_size(name, M, N, K));
    const Device *device = nullptr;
    VNM_TRY(device_ready(&device));
    Fp8Plan plan = {};
    bool on_pairs = false;
    VNM_TRY(choose_plan(M, N, K, out_type == VNM_F32, whole != 0, bias != 0, device->plans, &plan, &on_pairs));
    if (tile_m) *tile_m = on_pairs ? 256 : plan.bn;
    if (tile_n) *tile_n = on_pairs ? plan.bn : 128;
    if (split) *split = plan.split;
    if (grid) *grid = plan.grid;
    return VNM_OK;
}

extern "C" int vnm_fp8_device_status(int *status, void *stream)
{
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const Device *device = nullptr;
    VNM_TRY(device_ready(&device));
    int *const dev = device->status;
    int got = 0;
    cudaError_t e = cudaMemcpyAsync(&got, dev, sizeof(got), cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return done(e, "vnm_fp8_device_status");
    if (status) *status = got;
    if (!got) return VNM_OK;
    if ((e = cudaMemsetAsync(dev, 0, sizeof(got), s)) != cudaSuccess || (e = cudaStreamSynchronize(s)) != cudaSuccess) return done(e, "vnm_fp8_device_status");
    return fail(VNM_ERR_DEVICE_TIMEOUT, "a bounded device-side wait of an 8-bit product gave up (status %d)", got);
}
