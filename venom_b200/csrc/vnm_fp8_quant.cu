// Quantiser of the block-scaled 8-bit operators, with the GELU and its gradient in the same pass.
//
// A block is 128 values of a row (or of a column for the transpose, or 128 x 128).  Its scale is the smallest power of two s = 2^e with amax / s <= T,
// T = 448 = 1.75 2^8 (e4m3) or 57344 = 1.75 2^15 (e5m2).  With amax = f 2^k, 1 <= f < 2, that is e = k - 8 (or 15), one more where f > 1.75: an addition to
// the bits of amax that carries into the exponent.  x / s is exact in fp32 (a power of two, and what underflows is far below the 8-bit type's smallest
// value), so each value is rounded once.  amax is taken over finite values; NaN and, in e4m3, infinities become NaN, in e5m2 infinities stay.
// e >= -127, the smallest scale there is.
//
// Built without --use_fast_math: denormal inputs count.
#include "vnm_fp8.h"

#include <cuda_bf16.h>
#include <cuda_fp8.h>

namespace vnm {

namespace {

template <int TYPE> struct Elem;
template <> struct Elem<T_F32> { using type = float; };
template <> struct Elem<T_F16> { using type = __half; };
template <> struct Elem<T_BF16> { using type = __nv_bfloat16; };

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <int TYPE>
__device__ __forceinline__ typename Elem<TYPE>::type from_float(float x)
{
    if constexpr (TYPE == T_F32) return x;
    else if constexpr (TYPE == T_F16) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}

// Eight neighbouring values of a row from column c on; what lies past `cols` is zero.
template <int TYPE>
__device__ __forceinline__ void load8(const void *x, int64_t at, int c, int cols, bool vec, float (&v)[8])
{
    using E = typename Elem<TYPE>::type;
    const E *src = reinterpret_cast<const E *>(x) + at + c;
    if (vec && c + 8 <= cols) {
        if constexpr (TYPE == T_F32) {
            const float4 a = __ldg(reinterpret_cast<const float4 *>(src)), b = __ldg(reinterpret_cast<const float4 *>(src) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 q = __ldg(reinterpret_cast<const uint4 *>(src));
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (TYPE == T_F16) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                    v[2 * i] = f.x;
                    v[2 * i + 1] = f.y;
                } else {
                    v[2 * i] = __uint_as_float(w[i] << 16);
                    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = c + i < cols ? to_float(src[i]) : 0.0f;
    }
}

template <int TYPE>
__device__ __forceinline__ void store8(void *y, int64_t at, int c, int cols, bool vec, const float (&v)[8])
{
    using E = typename Elem<TYPE>::type;
    E *dst = reinterpret_cast<E *>(y) + at + c;
    if (vec && c + 8 <= cols) {
        if constexpr (TYPE == T_F32) {
            reinterpret_cast<float4 *>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4 *>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (TYPE == T_F16) {
                    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                    w[i] = *reinterpret_cast<const uint32_t *>(&h);
                } else {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                    w[i] = *reinterpret_cast<const uint32_t *>(&h);
                }
            }
            *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (c + i < cols) dst[i] = from_float<TYPE>(v[i]);
    }
}

// ---- scales ----
constexpr uint32_t INF_BITS = 0x7F800000u;

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t finite_bits(float x) { const uint32_t b = abs_bits(x); return b < INF_BITS ? b : 0u; }

// The scale's byte (its exponent + 127) for a block whose largest finite magnitude has these bits.
__device__ __forceinline__ uint32_t scale_code(uint32_t amax_bits, int f8)
{
    const int e = (int)((amax_bits + 0x1FFFFFu) >> 23) - (f8 == F8_E4M3 ? 8 : 15);
    return e > 0 ? (uint32_t)e : 0u;
}
__device__ __forceinline__ float inverse_scale(uint32_t code) { return __uint_as_float((254u - code) << 23); }
__device__ __forceinline__ float scale_value(uint32_t code) { return code ? __uint_as_float(code << 23) : __uint_as_float(0x00400000u); }

// (a, b) / s in 8 bits, a in the low byte.  `odd`: the block holds values that are not finite.
__device__ __forceinline__ uint32_t round2(float a, float b, float inv, int f8, bool odd)
{
    const float2 v = make_float2(a * inv, b * inv);
    const __nv_fp8_interpretation_t kind = f8 == F8_E4M3 ? __NV_E4M3 : __NV_E5M2;
    if (odd) return __nv_cvt_float2_to_fp8x2(v, __NV_NOSAT, kind);   // an infinity stays one or becomes NaN
    if (f8 == F8_E4M3) return __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
    return __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E5M2);
}
__device__ __forceinline__ uint2 round8(const float (&v)[8], float inv, int f8, bool odd)
{
    uint2 r;
    r.x = round2(v[0], v[1], inv, f8, odd) | (round2(v[2], v[3], inv, f8, odd) << 16);
    r.y = round2(v[4], v[5], inv, f8, odd) | (round2(v[6], v[7], inv, f8, odd) << 16);
    return r;
}

// Largest of the sixteen lanes that share a row's block.
__device__ __forceinline__ uint32_t max16(uint32_t b)
{
#pragma unroll
    for (int o = 8; o; o >>= 1) {
        const uint32_t n = __shfl_xor_sync(0xffffffffu, b, o);
        b = n > b ? n : b;
    }
    return b;
}
// The block of eight values a lane: bits of the largest finite magnitude, and whether others are in it.
__device__ __forceinline__ uint32_t row_amax(const float (&v)[8], bool *odd)
{
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) { const uint32_t a = abs_bits(v[i]); b = a > b ? a : b; }
    b = max16(b);
    *odd = b >= INF_BITS;
    if (__any_sync(0xffffffffu, *odd)) {
        uint32_t f = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) { const uint32_t a = finite_bits(v[i]); f = a > f ? a : f; }
        f = max16(f);
        if (*odd) b = f;
    }
    return b;
}

// Byte of block `kb` in the scales of a matrix of `n` rows; the last block's writer also sets what pads its word.
__device__ __forceinline__ void store_scale(uint8_t *scales, int64_t n, int64_t row, int kb, int blocks, uint32_t code)
{
    uint8_t *w = scales + ((int64_t)(kb >> 2) * n + row) * 4;
    w[kb & 3] = (uint8_t)code;
    if (kb == blocks - 1)
        for (int j = (kb & 3) + 1; j < 4; j++) w[j] = 0;
}

// ---- GELU ----
// The exact form by a published approximation of erfc (Abramowitz and Stegun, 7.1.26, |error| <= 1.5e-7): with t = 1 / (1 + p |z|), z = x / sqrt 2,
// erfc |z| = (a1 t + .. + a5 t^5) exp(-z^2).  The exponential is the density's as well, which the derivative needs, so one exponential and one reciprocal
// give both.  The tail of negative x has no cancellation.
__device__ __forceinline__ void gelu_erf(float x, float *cdf, float *density)
{
    const float z = fabsf(x) * 0.70710678118654752f;
    const float t = __fdividef(1.0f, fmaf(0.3275911f, z, 1.0f));
    const float e = exp2f(x * x * -0.72134752044448170f);
    float poly = fmaf(1.061405429f, t, -1.453152027f);
    poly = fmaf(poly, t, 1.421413741f);
    poly = fmaf(poly, t, -0.284496736f);
    poly = fmaf(poly, t, 0.254829592f);
    const float half_erfc = 0.5f * poly * t * e;
    *cdf = x < 0.0f ? half_erfc : 1.0f - half_erfc;
    *density = e * 0.39894228040143268f;
}
// The tanh form: (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3)
__device__ __forceinline__ float gelu_sigmoid(float x, float *du2)
{
    x = x > 64.0f ? 64.0f : x < -64.0f ? -64.0f : x;   // the square of a large x would overflow beside a zero; NaN stays
    const float x2 = x * x;
    const float u2 = x * fmaf(0.0713548162726f, x2, 1.59576912160573f);
    *du2 = fmaf(0.214064448817801f, x2, 1.59576912160573f);
    return __fdividef(1.0f, 1.0f + exp2f(-1.4426950408889634f * u2));
}
__device__ __forceinline__ float gelu(float x, int tanh_form)
{
    if (tanh_form) {
        float d;
        return x * gelu_sigmoid(x, &d);
    }
    float cdf, density;
    gelu_erf(x, &cdf, &density);
    return x * cdf;
}
__device__ __forceinline__ float gelu_grad(float x, int tanh_form)
{
    if (tanh_form) {
        float d;
        const float s = gelu_sigmoid(x, &d);
        x = x > 64.0f ? 64.0f : x < -64.0f ? -64.0f : x;
        return fmaf(x * s * (1.0f - s), d, s);
    }
    float cdf, density;
    gelu_erf(x, &cdf, &density);
    return fmaf(x, density, cdf);
}

// Eight values of an e4m3 checkpoint.
__device__ __forceinline__ void load_ckpt8(const Fp8QuantParams &p, int64_t row, int c, float (&h)[8])
{
    const uint2 q = __ldg(reinterpret_cast<const uint2 *>(p.ckpt + row * p.ldc + c));
    const int kb = c >> 7;
    const float s = scale_value(__ldg(p.ckpt_scales + ((int64_t)(kb >> 2) * p.rows + row) * 4 + (kb & 3)));
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = (i < 2 ? q.x : q.y) >> (16 * (i & 1));
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFFu), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r));
        h[2 * i] = f.x * s;
        h[2 * i + 1] = f.y * s;
    }
}

// ---- rows only: sixteen lanes a block, several blocks a lane ----
// Reads and writes every value once; bound by HBM, and by launch and latency for few rows.
constexpr int ROWS_THREADS = 256;
constexpr int ROWS_UNROLL = 4;

template <int TYPE, int OP>
__global__ void __launch_bounds__(ROWS_THREADS) fp8_rows_kernel(const Fp8QuantParams p)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const int blocks = (int)(((int64_t)p.cols + 127) >> 7);
    const int64_t total = (int64_t)p.rows * blocks;
    const int64_t first = ((int64_t)blockIdx.x * ROWS_THREADS + threadIdx.x) >> 4;
    const int64_t step = (int64_t)gridDim.x * (ROWS_THREADS / 16);
    const int sub = (int)(threadIdx.x & 15) * 8;
    const bool vec_y = OP != FP8_PLAIN && p.y && ((p.ldy * (int64_t)sizeof(typename Elem<TYPE>::type)) & 15) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
    for (int64_t u0 = first; u0 - (threadIdx.x >> 4) % 2 < total; u0 += step * ROWS_UNROLL) {   // both halves of a warp stay until its first one is through
        float v[ROWS_UNROLL][8];
#pragma unroll
        for (int j = 0; j < ROWS_UNROLL; j++) {
            const int64_t u = u0 + j * step;
            const int64_t row = u / blocks;
            const int c = (int)(u - row * blocks) * 128 + sub;
            load8<TYPE>(p.x, row * p.ldx, c, u < total ? p.cols : 0, p.vec_in != 0, v[j]);
        }
#pragma unroll
        for (int j = 0; j < ROWS_UNROLL; j++) {
            const int64_t u = u0 + j * step;
            const bool on = u < total;
            const int64_t row = on ? u / blocks : 0;
            const int kb = on ? (int)(u - row * blocks) : 0, c = kb * 128 + sub;
            const bool in = on && c < p.cols;
            bool odd;
            if constexpr (OP == FP8_GELU) {
                if (p.ckpt) {
                    const uint32_t code = scale_code(row_amax(v[j], &odd), F8_E4M3);
                    if (in) *reinterpret_cast<uint2 *>(p.ckpt + row * p.ldc + c) = round8(v[j], inverse_scale(code), F8_E4M3, odd);
                    if (on && sub == 0) store_scale(p.ckpt_scales, p.rows, row, kb, blocks, code);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) v[j][i] = gelu(v[j][i], p.tanh_form);
            } else if constexpr (OP == FP8_GELU_GRAD) {
                if (in) {
                    float h[8];
                    load_ckpt8(p, row, c, h);
#pragma unroll
                    for (int i = 0; i < 8; i++) v[j][i] *= gelu_grad(h[i], p.tanh_form);
                }
            }
            if (OP != FP8_PLAIN && p.y && in) store8<TYPE>(p.y, row * p.ldy, c, p.cols, vec_y, v[j]);
            if (p.data) {
                const uint32_t code = scale_code(row_amax(v[j], &odd), p.f8);
                if (in) *reinterpret_cast<uint2 *>(p.data + row * p.ldd + c) = round8(v[j], inverse_scale(code), p.f8, odd);
                if (on && sub == 0) store_scale(p.scales, p.rows, row, kb, blocks, code);
            }
        }
    }
}

// ---- tiles of 128 x 128: the matrix and its transpose from one read ----
// A thread holds four rows x eight columns.  The transposed bytes pass through shared memory: column c's 32 words of four rows each, word w at
// w ^ 2 (c / 8), so that the lanes of a warp (sixteen groups of eight columns, two of four rows) write to 32 banks, and read back whole columns.
constexpr int TILE_THREADS = 512;

template <int TYPE, int OP, bool SQUARE>
__global__ void __launch_bounds__(TILE_THREADS, 2) fp8_tiles_kernel(const Fp8QuantParams p)
{
    __shared__ uint32_t image[128 * 32];
    __shared__ uint32_t amax_of[16][128];
    __shared__ float inv_of[128];
    __shared__ uint32_t all[16], all_finite[16];
    grid_dependency_wait();
    grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = lane & 15, half = lane >> 4;
    const int cblocks = (int)(((int64_t)p.cols + 127) >> 7), rblocks = (int)(((int64_t)p.rows + 127) >> 7);
    const int tr = (int)(blockIdx.x / (unsigned)cblocks), tc = (int)blockIdx.x - tr * cblocks;
    const int c = tc * 128 + group * 8;
    const int64_t r0 = (int64_t)tr * 128 + warp * 8 + half * 4;
    const bool in = c < p.cols;

    float v[4][8];
#pragma unroll
    for (int j = 0; j < 4; j++) load8<TYPE>(p.x, (r0 + j) * p.ldx, c, r0 + j < p.rows ? p.cols : 0, p.vec_in != 0, v[j]);
    if constexpr (OP == FP8_GELU) {
        if (p.ckpt) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                bool odd;
                const uint32_t code = scale_code(row_amax(v[j], &odd), F8_E4M3);
                if (in && r0 + j < p.rows) *reinterpret_cast<uint2 *>(p.ckpt + (r0 + j) * p.ldc + c) = round8(v[j], inverse_scale(code), F8_E4M3, odd);
                if (group == 0 && r0 + j < p.rows) store_scale(p.ckpt_scales, p.rows, r0 + j, tc, cblocks, code);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) v[j][i] = gelu(v[j][i], p.tanh_form);   // of the zeros that pad: zero
    } else if constexpr (OP == FP8_GELU_GRAD) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (in && r0 + j < p.rows) {
                float h[8];
                load_ckpt8(p, r0 + j, c, h);
#pragma unroll
                for (int i = 0; i < 8; i++) v[j][i] *= gelu_grad(h[i], p.tanh_form);
            }
        }
    }

    uint32_t tile_code = 0;
    bool tile_odd = false;
    if constexpr (SQUARE) {
        uint32_t b = 0, f = 0;
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t a = abs_bits(v[j][i]), g = finite_bits(v[j][i]);
                b = a > b ? a : b;
                f = g > f ? g : f;
            }
        b = __reduce_max_sync(0xffffffffu, b);
        f = __reduce_max_sync(0xffffffffu, f);
        if (lane == 0) { all[warp] = b; all_finite[warp] = f; }
        __syncthreads();
        b = f = 0;
#pragma unroll
        for (int w = 0; w < 16; w++) { b = all[w] > b ? all[w] : b; f = all_finite[w] > f ? all_finite[w] : f; }
        tile_odd = b >= INF_BITS;
        tile_code = scale_code(f, p.f8);
    }

    if (p.data) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            bool odd = tile_odd;
            uint32_t code = tile_code;
            if constexpr (!SQUARE) code = scale_code(row_amax(v[j], &odd), p.f8);
            if (in && r0 + j < p.rows) *reinterpret_cast<uint2 *>(p.data + (r0 + j) * p.ldd + c) = round8(v[j], inverse_scale(code), p.f8, odd);
            if (group == 0 && r0 + j < p.rows) store_scale(p.scales, p.rows, r0 + j, tc, cblocks, code);
        }
    }

    if (p.data_t) {
        float inv[8];
        if constexpr (!SQUARE) {
#pragma unroll
            for (int pass = 0; pass < 2; pass++) {   // the second one only for columns with values that are not finite: see below
                if (pass == 1 && !__syncthreads_or(threadIdx.x < 128 && inv_of[threadIdx.x & 127] < 0.0f)) break;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    uint32_t b = 0;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t a = pass ? finite_bits(v[j][i]) : abs_bits(v[j][i]);
                        b = a > b ? a : b;
                    }
                    const uint32_t n = __shfl_xor_sync(0xffffffffu, b, 16);
                    if (half == 0) amax_of[warp][group * 8 + i] = n > b ? n : b;
                }
                __syncthreads();
                if (threadIdx.x < 128) {
                    uint32_t b = 0;
#pragma unroll
                    for (int w = 0; w < 16; w++) b = amax_of[w][threadIdx.x] > b ? amax_of[w][threadIdx.x] : b;
                    const bool odd = pass == 0 ? b >= INF_BITS : inv_of[threadIdx.x] < 0.0f;
                    const uint32_t code = scale_code(b < INF_BITS ? b : 0u, p.f8);
                    inv_of[threadIdx.x] = odd ? -inverse_scale(code) : inverse_scale(code);   // the sign says that some are not finite
                    const int col = tc * 128 + (int)threadIdx.x;
                    if (col < p.cols) store_scale(p.scales_t, p.cols, col, tr, rblocks, code);
                }
                __syncthreads();
            }
#pragma unroll
            for (int i = 0; i < 8; i++) inv[i] = inv_of[group * 8 + i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) inv[i] = tile_odd ? -inverse_scale(tile_code) : inverse_scale(tile_code);
            if (threadIdx.x < 128 && tc * 128 + (int)threadIdx.x < p.cols) store_scale(p.scales_t, p.cols, tc * 128 + threadIdx.x, tr, rblocks, tile_code);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const bool odd = inv[i] < 0.0f;
            const float s = fabsf(inv[i]);
            image[(group * 8 + i) * 32 + ((warp * 2 + half) ^ (2 * group))] = round2(v[0][i], v[1][i], s, p.f8, odd) | (round2(v[2][i], v[3][i], s, p.f8, odd) << 16);
        }
        __syncthreads();
        const int64_t padded = ((int64_t)p.rows + 15) & ~(int64_t)15;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int e = k * TILE_THREADS + threadIdx.x;
            const int col = e >> 4, piece = e & 15;
            const uint2 q = *reinterpret_cast<const uint2 *>(&image[col * 32 + 2 * (piece ^ (col >> 3))]);
            const int64_t row = (int64_t)tr * 128 + piece * 8;
            if (tc * 128 + col < p.cols && row < padded) *reinterpret_cast<uint2 *>(p.data_t + (int64_t)(tc * 128 + col) * p.ldt + row) = q;
        }
    }

    if (p.partial) {
        __syncthreads();   // amax_of is read no more
        float (*sum_of)[128] = reinterpret_cast<float (*)[128]>(amax_of);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float s = (v[0][i] + v[1][i]) + (v[2][i] + v[3][i]);
            s += __shfl_xor_sync(0xffffffffu, s, 16);
            if (half == 0) sum_of[warp][group * 8 + i] = s;
        }
        __syncthreads();
        const int col = tc * 128 + (int)threadIdx.x;
        if (threadIdx.x < 128 && col < p.cols) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < 16; w++) s += sum_of[w][threadIdx.x];
            p.partial[(int64_t)tr * p.cols + col] = s;
        }
    }
}

// Sums of the blocks' partial sums, always in the same order: eight threads a column, each every eighth block.
template <int TYPE>
__global__ void __launch_bounds__(256) fp8_colsum_kernel(const float *__restrict__ partial, int blocks, int cols, void *out)
{
    __shared__ float sums[8][33];
    grid_dependency_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (col < cols)
        for (int b = part; b < blocks; b += 8) s += partial[(int64_t)b * cols + col];
    sums[part][lane] = s;
    __syncthreads();
    if (part == 0 && col < cols) {
#pragma unroll
        for (int k = 1; k < 8; k++) s += sums[k][lane];
        reinterpret_cast<typename Elem<TYPE>::type *>(out)[col] = from_float<TYPE>(s);
    }
}

template <int TYPE>
__global__ void __launch_bounds__(256) fp8_dequantize_kernel(const uint8_t *__restrict__ data, int64_t ldd, const uint8_t *__restrict__ scales, int f8, int rows, int cols,
                                                             void *out, int64_t ldo)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const int per_row = (cols + 3) >> 2;
    const int64_t total = (int64_t)rows * per_row;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += (int64_t)gridDim.x * 256) {
        const int64_t row = u / per_row;
        const int c = (int)(u - row * per_row) * 4, kb = c >> 7;
        const uint32_t w = __ldg(reinterpret_cast<const uint32_t *>(data + row * ldd + c));
        const float s = scale_value(__ldg(scales + ((int64_t)(kb >> 2) * rows + row) * 4 + (kb & 3)));
        typename Elem<TYPE>::type *dst = reinterpret_cast<typename Elem<TYPE>::type *>(out) + row * ldo + c;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half_raw r = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)((w >> (8 * i)) & 0xFFu), f8 == F8_E4M3 ? __NV_E4M3 : __NV_E5M2);
            if (c + i < cols) dst[i] = from_float<TYPE>(__half2float(*reinterpret_cast<const __half *>(&r)) * s);
        }
    }
}

template <typename... Args>
cudaError_t launch(void (*kernel)(Args...), dim3 grid, int threads, cudaStream_t stream, std::common_type_t<Args>... args)
{
    cudaLaunchConfig_t lc = {};
    lc.gridDim = grid;
    lc.blockDim = dim3((unsigned)threads, 1, 1);
    lc.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0] = early_launch();
    lc.attrs = attr;
    lc.numAttrs = 1;
    return cudaLaunchKernelEx(&lc, kernel, args...);
}

int device_sms()
{
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    return sms;
}

template <int TYPE>
cudaError_t rows_of(const Fp8QuantParams &p, int op, cudaStream_t stream)
{
    const int64_t units = (int64_t)p.rows * (((int64_t)p.cols + 127) / 128), per_cta = ROWS_THREADS / 16;
    // one pass of the loop where that fills the GPU, so that every load is on its way at once
    int64_t ctas = (units + per_cta * ROWS_UNROLL - 1) / (per_cta * ROWS_UNROLL);
    const int64_t wave = (int64_t)device_sms() * 8;
    if (ctas < wave / 8) ctas = (units + per_cta - 1) / per_cta < wave / 8 ? (units + per_cta - 1) / per_cta : wave / 8;
    if (ctas > wave) ctas = wave;
    const dim3 grid((unsigned)ctas);
    if (op == FP8_PLAIN) return launch(fp8_rows_kernel<TYPE, FP8_PLAIN>, grid, ROWS_THREADS, stream, p);
    if (op == FP8_GELU) return launch(fp8_rows_kernel<TYPE, FP8_GELU>, grid, ROWS_THREADS, stream, p);
    return launch(fp8_rows_kernel<TYPE, FP8_GELU_GRAD>, grid, ROWS_THREADS, stream, p);
}

template <int TYPE>
cudaError_t tiles_of(const Fp8QuantParams &p, int op, bool square, cudaStream_t stream)
{
    const dim3 grid((unsigned)((((int64_t)p.cols + 127) / 128) * (((int64_t)p.rows + 127) / 128)));
    if (op == FP8_GELU) return launch(fp8_tiles_kernel<TYPE, FP8_GELU, false>, grid, TILE_THREADS, stream, p);
    if (op == FP8_GELU_GRAD) return launch(fp8_tiles_kernel<TYPE, FP8_GELU_GRAD, false>, grid, TILE_THREADS, stream, p);
    if (square) return launch(fp8_tiles_kernel<TYPE, FP8_PLAIN, true>, grid, TILE_THREADS, stream, p);
    return launch(fp8_tiles_kernel<TYPE, FP8_PLAIN, false>, grid, TILE_THREADS, stream, p);
}

}  // namespace

cudaError_t launch_fp8_rows(const Fp8QuantParams &p, int type, int op, cudaStream_t stream)
{
    return type == T_F32 ? rows_of<T_F32>(p, op, stream) : type == T_F16 ? rows_of<T_F16>(p, op, stream) : rows_of<T_BF16>(p, op, stream);
}

cudaError_t launch_fp8_tiles(const Fp8QuantParams &p, int type, int op, bool square, cudaStream_t stream)
{
    return type == T_F32 ? tiles_of<T_F32>(p, op, square, stream) : type == T_F16 ? tiles_of<T_F16>(p, op, square, stream) : tiles_of<T_BF16>(p, op, square, stream);
}

cudaError_t launch_fp8_colsum(const float *partial, int blocks, int cols, void *out, int type, cudaStream_t stream)
{
    const dim3 grid((unsigned)((cols + 31) / 32));
    if (type == T_F32) return launch(fp8_colsum_kernel<T_F32>, grid, 256, stream, partial, blocks, cols, out);
    if (type == T_F16) return launch(fp8_colsum_kernel<T_F16>, grid, 256, stream, partial, blocks, cols, out);
    return launch(fp8_colsum_kernel<T_BF16>, grid, 256, stream, partial, blocks, cols, out);
}

cudaError_t launch_fp8_dequantize(const uint8_t *data, int64_t ldd, const uint8_t *scales, int f8, int rows, int cols, void *out, int type, int64_t ldo, cudaStream_t stream)
{
    const int64_t units = (int64_t)rows * ((cols + 3) / 4);
    const int64_t most = (int64_t)device_sms() * 8;
    const int64_t ctas = (units + 255) / 256 < most ? (units + 255) / 256 : most;
    const dim3 grid((unsigned)ctas);
    if (type == T_F32) return launch(fp8_dequantize_kernel<T_F32>, grid, 256, stream, data, ldd, scales, f8, rows, cols, out, ldo);
    if (type == T_F16) return launch(fp8_dequantize_kernel<T_F16>, grid, 256, stream, data, ldd, scales, f8, rows, cols, out, ldo);
    return launch(fp8_dequantize_kernel<T_BF16>, grid, 256, stream, data, ldd, scales, f8, rows, cols, out, ldo);
}

}  // namespace vnm
