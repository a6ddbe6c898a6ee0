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

#include <climits>
#include <type_traits>

namespace vnm {

namespace {

template <int TYPE> struct Elem;
template <> struct Elem<T_F32> { using type = float; };
template <> struct Elem<T_F16> { using type = __half; };
template <> struct Elem<T_BF16> { using type = __nv_bfloat16; };

template <int TYPE>
__device__ __forceinline__ typename Elem<TYPE>::type from_float(float x)
{
    if constexpr (TYPE == T_F32) return x;
    else if constexpr (TYPE == T_F16) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}

// Eight neighbouring values of a row as they lie: four words of 16-bit values or eight of 32.
template <int TYPE>
struct Raw {
    static constexpr int WORDS = TYPE == T_F32 ? 8 : 4;
    uint32_t w[WORDS];
};
// `align`: what the rows' addresses are a multiple of, 16, 4 or 2 bytes.  What lies past `cols` is zero.  inner: rows lie ahead of this one and behind it, so that a row
// which begins inside a word may be read in whole words, with two bytes too many at either end: five of them, the last in `extra`, out of which settle() takes the
// values when they are wanted (taken here, they would be waited for).  8191 x 4095 fp16: value by value 35 us.
// Loading whole pieces of 16 bytes and exchanging words between lanes instead is slower for such rows, and its registers slow the others down.
template <int TYPE>
__device__ __forceinline__ Raw<TYPE> load_raw(const void *x, int64_t at, int c, int cols, int align, bool inner, uint32_t &extra)
{
    using E = typename Elem<TYPE>::type;
    Raw<TYPE> r;
    const E *src = reinterpret_cast<const E *>(x) + at + c;
    if (c + 8 <= cols && align >= 4) {
        if (align == 16) {
#pragma unroll
            for (int i = 0; i < Raw<TYPE>::WORDS / 4; i++) {
                const uint4 q = __ldg(reinterpret_cast<const uint4 *>(src) + i);
                r.w[4 * i] = q.x; r.w[4 * i + 1] = q.y; r.w[4 * i + 2] = q.z; r.w[4 * i + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < Raw<TYPE>::WORDS; i++) r.w[i] = __ldg(reinterpret_cast<const uint32_t *>(src) + i);
        }
    } else if constexpr (TYPE == T_F32) {
#pragma unroll
        for (int i = 0; i < 8; i++) r.w[i] = c + i < cols ? __ldg(reinterpret_cast<const uint32_t *>(src) + i) : 0u;
    } else if (c + 8 <= cols && inner) {
        const uint32_t odd = (uint32_t)(reinterpret_cast<uintptr_t>(src) & 2);
        const uint32_t *word = reinterpret_cast<const uint32_t *>(reinterpret_cast<const uint8_t *>(src) - odd);
#pragma unroll
        for (int i = 0; i < 4; i++) r.w[i] = __ldg(word + i);
        extra = __ldg(word + (odd ? 4 : 3));
    } else {
        const unsigned short *h = reinterpret_cast<const unsigned short *>(src);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = c + 2 * i < cols ? __ldg(h + 2 * i) : 0u, hi = c + 2 * i + 1 < cols ? __ldg(h + 2 * i + 1) : 0u;
            r.w[i] = lo | (hi << 16);
        }
    }
    return r;
}
template <int TYPE>
__device__ __forceinline__ void settle(Raw<TYPE> &r, uint32_t extra, const void *x, int64_t at, int c, int cols, int align, bool inner)
{
    if constexpr (TYPE != T_F32) {
        if (align < 4 && inner && c + 8 <= cols && ((reinterpret_cast<uintptr_t>(x) + 2 * (uintptr_t)(at + c)) & 2)) {
#pragma unroll
            for (int i = 0; i < 4; i++) r.w[i] = __byte_perm(r.w[i], i < 3 ? r.w[i < 3 ? i + 1 : 3] : extra, 0x5432);
        }
    }
}
template <int TYPE>
__device__ __forceinline__ void to_floats(const Raw<TYPE> &r, float (&v)[8])
{
#pragma unroll
    for (int i = 0; i < Raw<TYPE>::WORDS; i++) {
        if constexpr (TYPE == T_F32) {
            v[i] = __uint_as_float(r.w[i]);
        } else if constexpr (TYPE == T_F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r.w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        } else {
            v[2 * i] = __uint_as_float(r.w[i] << 16);
            v[2 * i + 1] = __uint_as_float(r.w[i] & 0xFFFF0000u);
        }
    }
}

// The pair of words' values.
template <int TYPE>
__device__ __forceinline__ float2 pair_of(const Raw<TYPE> &r, int k)
{
    if constexpr (TYPE == T_F32) {
        return make_float2(__uint_as_float(r.w[2 * k]), __uint_as_float(r.w[2 * k + 1]));
    } else if constexpr (TYPE == T_F16) {
        // volatile: converted anew for each use.  Kept between the uses, 32 values of a thread cost the tiles kernel its third CTA of an SM.
        float2 f;
        asm volatile("{\n\t.reg .b16 l, h;\n\t"
                     "mov.b32 {l, h}, %2;\n\t"
                     "cvt.f32.f16 %0, l;\n\t"
                     "cvt.f32.f16 %1, h;\n\t}"
                     : "=f"(f.x), "=f"(f.y)
                     : "r"(r.w[k]));
        return f;
    } else return make_float2(__uint_as_float(r.w[k] << 16), __uint_as_float(r.w[k] & 0xFFFF0000u));
}
// Larger magnitudes of two words, passing over NaN.
template <int TYPE>
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b)
{
    if constexpr (TYPE == T_F16) {
        const __half2 m = __hmax2(__habs2(*reinterpret_cast<const __half2 *>(&a)), __habs2(*reinterpret_cast<const __half2 *>(&b)));
        return *reinterpret_cast<const uint32_t *>(&m);
    } else {
        const __nv_bfloat162 m = __hmax2(__habs2(*reinterpret_cast<const __nv_bfloat162 *>(&a)), __habs2(*reinterpret_cast<const __nv_bfloat162 *>(&b)));
        return *reinterpret_cast<const uint32_t *>(&m);
    }
}
template <int TYPE>
__device__ __forceinline__ float2 word_values(uint32_t w)
{
    if constexpr (TYPE == T_F16) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
// Four rows x eight columns of a thread: as they were loaded (16-bit types whose values are only rounded: half of the registers, and maxima of two values an
// instruction), or in 32 bits.
template <int TYPE, bool AS_LOADED>
struct Block4;
template <int TYPE>
struct Block4<TYPE, true> {
    static constexpr bool SHORT = true;        // of registers
    Raw<TYPE> raw[4];
    __device__ __forceinline__ float2 at(int j, int k) const { return pair_of<TYPE>(raw[j], k); }
    __device__ __forceinline__ float row_amax(int j) const
    {
        const uint32_t *w = raw[j].w;
        const float2 m = word_values<TYPE>(max_word<TYPE>(max_word<TYPE>(w[0], w[1]), max_word<TYPE>(w[2], w[3])));
        return fmaxf(m.x, m.y);
    }
    __device__ __forceinline__ float2 col_amax(int k) const
    {
        return word_values<TYPE>(max_word<TYPE>(max_word<TYPE>(raw[0].w[k], raw[1].w[k]), max_word<TYPE>(raw[2].w[k], raw[3].w[k])));
    }
};
template <int TYPE>
struct Block4<TYPE, false> {
    static constexpr bool SHORT = false;
    float v[4][8];
    __device__ __forceinline__ float2 at(int j, int k) const { return make_float2(v[j][2 * k], v[j][2 * k + 1]); }
    __device__ __forceinline__ float row_amax(int j) const
    {
        const float a = fmaxf(fmaxf(fabsf(v[j][0]), fabsf(v[j][1])), fmaxf(fabsf(v[j][2]), fabsf(v[j][3])));
        return fmaxf(a, fmaxf(fmaxf(fabsf(v[j][4]), fabsf(v[j][5])), fmaxf(fabsf(v[j][6]), fabsf(v[j][7]))));
    }
    __device__ __forceinline__ float2 col_amax(int k) const
    {
        return make_float2(fmaxf(fmaxf(fabsf(v[0][2 * k]), fabsf(v[1][2 * k])), fmaxf(fabsf(v[2][2 * k]), fabsf(v[3][2 * k]))),
                           fmaxf(fmaxf(fabsf(v[0][2 * k + 1]), fabsf(v[1][2 * k + 1])), fmaxf(fabsf(v[2][2 * k + 1]), fabsf(v[3][2 * k + 1]))));
    }
};

template <int TYPE>
__device__ __forceinline__ void store8(void *y, int64_t at, int c, int cols, int align, const float (&v)[8])
{
    using E = typename Elem<TYPE>::type;
    E *dst = reinterpret_cast<E *>(y) + at + c;
    if (c + 8 <= cols && align >= 4) {
        uint32_t w[Raw<TYPE>::WORDS];
#pragma unroll
        for (int i = 0; i < Raw<TYPE>::WORDS; i++) {
            if constexpr (TYPE == T_F32) {
                w[i] = __float_as_uint(v[i]);
            } else if constexpr (TYPE == T_F16) {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        if (align == 16) {
#pragma unroll
            for (int i = 0; i < Raw<TYPE>::WORDS / 4; i++) reinterpret_cast<uint4 *>(dst)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < Raw<TYPE>::WORDS; i++) reinterpret_cast<uint32_t *>(dst)[i] = w[i];
        }
    } else if (TYPE != T_F32 && c + 8 <= cols && (reinterpret_cast<uintptr_t>(dst) & 2)) {
        // inside a word: the first and the last value alone, three words between them
        dst[0] = from_float<TYPE>(v[0]);
#pragma unroll
        for (int i = 0; i < 3; i++) {
            uint32_t w;
            if constexpr (TYPE == T_F16) {
                const __half2 h = __floats2half2_rn(v[2 * i + 1], v[2 * i + 2]);
                w = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i + 1], v[2 * i + 2]);
                w = *reinterpret_cast<const uint32_t *>(&h);
            }
            *reinterpret_cast<uint32_t *>(dst + 2 * i + 1) = w;
        }
        dst[7] = from_float<TYPE>(v[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (c + i < cols) dst[i] = from_float<TYPE>(v[i]);
    }
}

// ---- two 32-bit operations an instruction, each rounded to nearest ----
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 p, q;\n\t"
        "mov.b64 p, {%2, %3};\n\t"
        "mov.b64 q, {%4, %5};\n\t"
        "mul.rn.f32x2 p, p, q;\n\t"
        "mov.b64 {%0, %1}, p;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 r;
    asm("{\n\t.reg .b64 p, q, s;\n\t"
        "mov.b64 p, {%2, %3};\n\t"
        "mov.b64 q, {%4, %5};\n\t"
        "mov.b64 s, {%6, %7};\n\t"
        "fma.rn.f32x2 p, p, q, s;\n\t"
        "mov.b64 {%0, %1}, p;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// ---- scales ----
// The scale's byte (its exponent + 127) for a block whose largest finite magnitude is amax.
template <int F8>
__device__ __forceinline__ uint32_t scale_code(float amax)
{
    const int e = (int)((__float_as_uint(amax) + 0x1FFFFFu) >> 23) - (F8 == F8_E4M3 ? 8 : 15);
    return e > 0 ? (uint32_t)e : 0u;
}
__device__ __forceinline__ float inverse_scale(uint32_t code) { return __uint_as_float((254u - code) << 23); }
// 0 stands for 2^-127, which is denormal in fp32.
__device__ __forceinline__ float scale_value(uint32_t code) { return code ? __uint_as_float(code << 23) : __uint_as_float(0x00400000u); }
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < __uint_as_float(0x7F800000u); }

// The maximum passes over NaN; an infinity shows in it, and takes its block (`odd`) through the slow forms below.
__device__ __forceinline__ float finite_max(float m, float x) { return finite(x) ? fmaxf(m, fabsf(x)) : m; }
template <typename B>
__device__ __forceinline__ float finite_row_amax(const B &v, int j)
{
    float m = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; k++) m = finite_max(finite_max(m, v.at(j, k).x), v.at(j, k).y);
    return m;
}

template <int F8>
__device__ __forceinline__ uint32_t round2(float a, float b)
{
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, F8 == F8_E4M3 ? __NV_E4M3 : __NV_E5M2);
}
template <int F8, typename B>
__device__ __forceinline__ uint2 round8(const B &v, int j, float inv)
{
    uint32_t h[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float2 s = mul2(v.at(j, k), both(inv));
        h[k] = round2<F8>(s.x, s.y);
    }
    return make_uint2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410));
}
// Four rounded values of a block with infinities, which the conversion has made the largest value: they stay infinities in e5m2 and become NaN in e4m3.
template <int F8>
__device__ __forceinline__ uint32_t mend4_here(uint32_t w, float a, float b, float c, float d)
{
    const float v[4] = {a, b, c, d};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t bits = __float_as_uint(v[i]);
        if ((bits & 0x7FFFFFFFu) == 0x7F800000u) w = (w & ~(0xFFu << (8 * i))) | ((((bits >> 24) & 0x80u) | (F8 == F8_E4M3 ? 0x7Fu : 0x7Cu)) << (8 * i));
    }
    return w;
}
// The same as a call: where registers are short (three CTAs an SM) this rare way shall take none from the usual one.
template <int F8>
__device__ __noinline__ uint32_t mend4_call(uint32_t w, float a, float b, float c, float d) { return mend4_here<F8>(w, a, b, c, d); }
template <int F8, bool CALL>
__device__ __forceinline__ uint32_t mend4(uint32_t w, float a, float b, float c, float d)
{
    if constexpr (CALL) return mend4_call<F8>(w, a, b, c, d);
    else return mend4_here<F8>(w, a, b, c, d);
}
template <int F8, typename B>
__device__ __forceinline__ uint2 mend8(uint2 r, const B &v, int j)
{
    const float2 a = v.at(j, 0), b = v.at(j, 1), c = v.at(j, 2), d = v.at(j, 3);
    return make_uint2(mend4<F8, B::SHORT>(r.x, a.x, a.y, b.x, b.y), mend4<F8, B::SHORT>(r.y, c.x, c.y, d.x, d.y));
}

// Largest of sixteen lanes for four values at once: lanes exchange the values that they do not keep, so that five shuffles do, and each lane ends with
// value (lane >> 2) & 3 ...
__device__ __forceinline__ float max16_of4(float a0, float a1, float a2, float a3)
{
    const bool h8 = (threadIdx.x & 8) != 0, h4 = (threadIdx.x & 4) != 0;
    const float r0 = __shfl_xor_sync(0xffffffffu, h8 ? a0 : a2, 8), r1 = __shfl_xor_sync(0xffffffffu, h8 ? a1 : a3, 8);
    const float b0 = fmaxf(h8 ? a2 : a0, r0), b1 = fmaxf(h8 ? a3 : a1, r1);
    float c = fmaxf(h4 ? b1 : b0, __shfl_xor_sync(0xffffffffu, h4 ? b0 : b1, 4));
    c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, 2));
    return fmaxf(c, __shfl_xor_sync(0xffffffffu, c, 1));
}
// ... whose byte goes back to all sixteen: byte i of the result belongs to value i.
__device__ __forceinline__ uint32_t bytes_of4(uint32_t code)
{
    uint32_t w = code << (8 * ((threadIdx.x >> 2) & 3));
    w |= __shfl_xor_sync(0xffffffffu, w, 4);
    w |= __shfl_xor_sync(0xffffffffu, w, 8);
    return w;
}
// Codes of four blocks of eight values a lane; byte i of *odd: block i has an infinity.  Returns whether any block of the warp has one: that way lies off the
// usual one (selected by value instead, it took a third of all instructions).
template <int F8, typename B>
__device__ __forceinline__ bool codes_of4(const B &v, uint32_t *codes, uint32_t *odd)
{
    float m = max16_of4(v.row_amax(0), v.row_amax(1), v.row_amax(2), v.row_amax(3));
    const bool any = __any_sync(0xffffffffu, !finite(m));
    if (any) {
        *odd = bytes_of4(finite(m) ? 0u : 1u);
        m = max16_of4(finite_row_amax(v, 0), finite_row_amax(v, 1), finite_row_amax(v, 2), finite_row_amax(v, 3));
    }
    *codes = bytes_of4(scale_code<F8>(m));
    return any;
}
__device__ __forceinline__ uint32_t byte_of(uint32_t w, int i) { return (w >> (8 * i)) & 0xFFu; }

// Byte of block `kb` in the scales of a matrix of `n` rows; the last block's writer also sets what pads its word.
__device__ __forceinline__ void store_scale(uint8_t *scales, int64_t n, int64_t row, int kb, int blocks, uint32_t code)
{
    uint8_t *w = scales + ((int64_t)(kb >> 2) * n + row) * 4;
    w[kb & 3] = (uint8_t)code;
    if (kb == blocks - 1)
        for (int j = (kb & 3) + 1; j < 4; j++) w[j] = 0;
}

// ---- GELU ----
__device__ __forceinline__ float fast_exp2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float fast_rcp(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b)   // a NaN stays
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b)
{
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Beyond 64 either form is x or 0 and the derivative 1 or 0: values are cut off there, ahead of squares that would overflow beside a zero.  So -inf gives 0.
__device__ __forceinline__ float near(float x) { return max_nan(min_nan(x, 64.0f), -64.0f); }

// The exact form: Phi(-a) = R(t) exp(-a^2 / 2), a = |x|, t = 1 / (1 + p a), the form of Abramowitz and Stegun, 7.1.26, with polynomials R that bound the relative error
// instead of the absolute one: minimax over 0 <= a <= 13.3, where fp32 ends, by exchange of the extrema in 40 digits (against 2^q with the rounded constant of q).  7.1.26 itself
// is off by 5e-5 of the value at a = 3 and 1.6e-3 at 5, and one in 1e4 of a GELU's 8-bit results was another than the formula's.  FINE, for values of 32 bits and for the
// derivative: degree 7, 2.7e-7, and one half at t = 1 to the last bit, because a gradient of 16 bits times the derivative at 0 often lies between two 8-bit values.  Else degree 6,
// 1.5e-6, a hundredth of fp16's half step (a GELU step of 16384 x 4096 fp16: 133 us if both take it, 137 if neither does).  The exponential is the density's as well, which the
// derivative needs, so one exponential and one reciprocal give both.  gelu(x) = max(x, 0) - a Phi(-a): no cancellation for negative x, where it is off by 2.5e-6 (FINE:
// 1.6e-6) + a^2 2^-24 of itself at most.  The result is S Phi(-a), S = 1 or -1; a is cut off.
template <int S, bool FINE>
__device__ __forceinline__ float2 normal_tail(float2 a, float2 *e)
{
    const float2 d = fma2(both(FINE ? 0.255f : 0.2975f), a, both(1.0f));
    const float2 t = make_float2(fast_rcp(d.x), fast_rcp(d.y));
    const float2 q = mul2(mul2(a, a), both(-0.72134752044448170f));
    *e = make_float2(fast_exp2(q.x), fast_exp2(q.y));
    float2 poly;
    if (FINE) {
        poly = fma2(both(S * -0.0861255229f), t, both(S * 0.300162017f));
        poly = fma2(poly, t, both(S * -0.213580772f));
        poly = fma2(poly, t, both(S * 0.251812041f));
        poly = fma2(poly, t, both(S * 0.0317303129f));
        poly = fma2(poly, t, both(S * 0.115937077f));
        poly = fma2(poly, t, both(S * 0.0999727994f));
        poly = fma2(poly, t, both(S * 9.20295715e-05f));
    } else {
        poly = fma2(both(S * -0.0874843597f), t, both(S * 0.257873505f));
        poly = fma2(poly, t, both(S * -0.0690223277f));
        poly = fma2(poly, t, both(S * 0.175907403f));
        poly = fma2(poly, t, both(S * 0.101962328f));
        poly = fma2(poly, t, both(S * 0.12088152f));
        poly = fma2(poly, t, both(S * -0.000118785138f));
    }
    return mul2(poly, *e);
}
// The tanh form: (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3); x cut off.  -2 u log2 e = x (c1 x^2 + c0).
__device__ __forceinline__ float2 gelu_sigmoid(float2 x, float2 x2)
{
    const float2 q = mul2(x, fma2(both(-0.10294324f), x2, both(-2.3022082f)));
    return make_float2(fast_rcp(1.0f + fast_exp2(q.x)), fast_rcp(1.0f + fast_exp2(q.y)));
}
template <bool TANH, bool FINE>
__device__ __forceinline__ void gelu2(float &x, float &y)
{
    float2 r;
    if (TANH) {
        const float2 lo = make_float2(max_nan(x, -64.0f), max_nan(y, -64.0f)), n = make_float2(min_nan(lo.x, 64.0f), min_nan(lo.y, 64.0f));
        r = mul2(lo, gelu_sigmoid(n, mul2(n, n)));
    } else {
        const float2 a = make_float2(min_nan(fabsf(x), 64.0f), min_nan(fabsf(y), 64.0f));
        float2 e;
        const float2 h = normal_tail<-1, FINE>(a, &e);
        r = fma2(a, h, make_float2(max_nan(x, 0.0f), max_nan(y, 0.0f)));
    }
    x = r.x;
    y = r.y;
}
// (x, y) times the derivative at (a, b)
template <bool TANH>
__device__ __forceinline__ void times_gelu_grad2(float &x, float &y, float a, float b)
{
    const float2 n = make_float2(near(a), near(b));
    float2 g;
    if (TANH) {
        // from 1 - s of |n|, which keeps its bits where s is next to 1
        const float2 n2 = mul2(n, n), s = gelu_sigmoid(make_float2(-fabsf(n.x), -fabsf(n.y)), n2), c = fma2(both(-1.0f), s, both(1.0f));
        const float2 du = fma2(both(0.21406445f), n2, both(1.59576912f));
        g = fma2(mul2(mul2(n, s), c), du, make_float2(n.x < 0.0f ? s.x : c.x, n.y < 0.0f ? s.y : c.y));
    } else {
        float2 e;
        const float2 h = normal_tail<1, true>(make_float2(fabsf(n.x), fabsf(n.y)), &e);
        const float2 far = make_float2(n.x < 0.0f ? h.x : 1.0f - h.x, n.y < 0.0f ? h.y : 1.0f - h.y);
        g = fma2(n, mul2(e, both(0.39894228040143268f)), far);
    }
    const float2 r = mul2(make_float2(x, y), g);
    x = r.x;
    y = r.y;
}

// Two 8-bit values in the low half of a word, times their scale.
template <int F8>
__device__ __forceinline__ float2 block_pair(uint32_t w, float s)
{
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFFu), F8 == F8_E4M3 ? __NV_E4M3 : __NV_E5M2);
    return mul2(__half22float2(*reinterpret_cast<const __half2 *>(&r)), both(s));
}
// Eight values of an e4m3 checkpoint whose block has this code.
__device__ __forceinline__ void ckpt_values(uint2 q, uint32_t code, float (&h)[8])
{
    const float s = scale_value(code);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = block_pair<F8_E4M3>((i < 2 ? q.x : q.y) >> (16 * (i & 1)), s);
        h[2 * i] = f.x;
        h[2 * i + 1] = f.y;
    }
}

// ---- rows only ----
// Sixteen lanes take four blocks of a row, whose bytes are one scale word; a lane holds eight values of each.  The next four blocks are on their way while these
// are worked on.  Every value is read and written once; bound by HBM, and by launch and latency for few rows.
constexpr int ROWS_THREADS = 256;

template <int TYPE, int OP, int F8, bool TANH>
__global__ void __launch_bounds__(ROWS_THREADS, TYPE == T_F32 || OP != FP8_PLAIN ? 2 : 3) fp8_rows_kernel(const Fp8QuantParams p)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t groups = (uint32_t)(((int64_t)p.cols + 511) >> 9), total = groups * (uint32_t)p.rows;
    const uint32_t first = (blockIdx.x * ROWS_THREADS + threadIdx.x) >> 4, step = gridDim.x * (ROWS_THREADS / 16);
    const uint32_t step_rows = step / groups, step_groups = step - step_rows * groups;
    const int sub = (int)(threadIdx.x & 15) * 8;
    uint32_t u = first, row = first / groups, g = first - row * groups;

    Raw<TYPE> next[4];
    uint32_t extra[4];
    uint2 next_h[4];
    uint32_t next_codes = 0;
    auto fetch = [&](uint32_t unit, uint32_t r, uint32_t gr) {
        const int c = (int)gr * 512 + sub;
#pragma unroll
        for (int i = 0; i < 4; i++) next[i] = load_raw<TYPE>(p.x, (int64_t)r * p.ldx, c + 128 * i, unit < total ? p.cols : 0, p.align_x, r > 0 && r + 1 < (uint32_t)p.rows, extra[i]);
        if constexpr (OP == FP8_GELU_GRAD) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                next_h[i] = unit < total && c + 128 * i < p.cols ? __ldg(reinterpret_cast<const uint2 *>(p.ckpt + (int64_t)r * p.ldc + c + 128 * i)) : make_uint2(0u, 0u);
            next_codes = unit < total ? __ldg(reinterpret_cast<const uint32_t *>(p.ckpt_scales) + (int64_t)gr * p.rows + r) : 0u;
        }
    };
    fetch(u, row, g);
    for (; u - ((threadIdx.x >> 4) & 1) < total;) {          // the halves of a warp stay together
        const bool on = u < total;
        const int64_t r = row;
        const int c = (int)g * 512 + sub;
        const int64_t word = (int64_t)g * p.rows + r;
        constexpr bool AS_LOADED = OP == FP8_PLAIN && TYPE != T_F32;
        Block4<TYPE, AS_LOADED> v;
        if (TYPE != T_F32 && p.align_x < 4 && on) {
#pragma unroll
            for (int i = 0; i < 4; i++) settle<TYPE>(next[i], extra[i], p.x, r * p.ldx, c + 128 * i, p.cols, p.align_x, r > 0 && r + 1 < p.rows);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (AS_LOADED) v.raw[i] = next[i];
            else to_floats<TYPE>(next[i], v.v[i]);
        }
        uint2 h[4];
        uint32_t h_codes = 0;
        if constexpr (OP == FP8_GELU_GRAD) {
#pragma unroll
            for (int i = 0; i < 4; i++) h[i] = next_h[i];
            h_codes = next_codes;
        }
        u += step;
        row += step_rows;
        g += step_groups;
        if (g >= groups) { g -= groups; row++; }
        fetch(u, row, g);

        auto store = [&](uint8_t *data, int64_t ld, uint8_t *scales, auto type) {
            constexpr int T8 = decltype(type)::value;
            uint32_t codes, odd = 0;
            const bool any = codes_of4<T8>(v, &codes, &odd);
            uint2 q[4];
#pragma unroll
            for (int i = 0; i < 4; i++) q[i] = round8<T8>(v, i, inverse_scale(byte_of(codes, i)));
            if (any) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (byte_of(odd, i)) q[i] = mend8<T8>(q[i], v, i);
            }
            if (on) {
                uint8_t *dst = data + r * ld + c;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (c + 128 * i < p.cols) *reinterpret_cast<uint2 *>(dst + 128 * i) = q[i];
                // blocks past the last one are zeros, whose code is 0
                if (sub == 0) reinterpret_cast<uint32_t *>(scales)[word] = codes;
            }
        };
        if constexpr (OP == FP8_GELU) {
            if (p.ckpt) store(p.ckpt, p.ldc, p.ckpt_scales, std::integral_constant<int, F8_E4M3>());
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 8; j += 2) gelu2<TANH, TYPE == T_F32>(v.v[i][j], v.v[i][j + 1]);
        } else if constexpr (OP == FP8_GELU_GRAD) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float x[8];
                ckpt_values(h[i], byte_of(h_codes, i), x);
#pragma unroll
                for (int j = 0; j < 8; j += 2) times_gelu_grad2<TANH>(v.v[i][j], v.v[i][j + 1], x[j], x[j + 1]);
            }
        }
        if constexpr (OP != FP8_PLAIN) {
            if (p.y && on) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (c + 128 * i < p.cols) store8<TYPE>(p.y, r * p.ldy, c + 128 * i, p.cols, p.align_y, v.v[i]);
            }
        }
        if (p.data) store(p.data, p.ldd, p.scales, std::integral_constant<int, F8>());
    }
}

// ---- tiles of 128 x 128: the matrix and its transpose from one read ----
// A thread holds four rows x eight columns.  The transposed bytes pass through shared memory: column c's 32 words of four rows each, word w at
// w ^ 2 (c / 8), so that the lanes of a warp (sixteen groups of eight columns, two of four rows) write to 32 banks, and read back whole columns.
constexpr int TILE_THREADS = 512;
constexpr int AMAX_PITCH = 136;    // four rows side by side lie in different banks

struct TileShared {
    uint32_t image[128 * 32];
    float amax_of[32][AMAX_PITCH];   // of each four rows; later their sums
    float inv_of[128];
    float all[16];
};

// WHOLE: a tile of 128 x 128 values whose rows are 16-byte aligned; nothing is checked.
template <int TYPE, int OP, int F8, bool SQUARE, bool TANH, bool WHOLE>
__device__ __forceinline__ void fp8_tile(const Fp8QuantParams &p, TileShared &sh, int tr, int tc)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = lane & 15, half = lane >> 4;
    const int cblocks = (int)(((int64_t)p.cols + 127) >> 7), rblocks = (int)(((int64_t)p.rows + 127) >> 7);
    const int c = tc * 128 + group * 8;
    const int64_t r0 = (int64_t)tr * 128 + warp * 8 + half * 4;
    const bool in = WHOLE || c < p.cols;
    const int left = WHOLE ? 4 : (int)(p.rows - r0 < 4 ? p.rows - r0 : 4);   // rows that there are, or fewer than one
    const int own_row = (lane >> 2) & 3;                       // the row whose code this lane stores (lanes 0, 4, 8, 12 of a half)

    constexpr bool AS_LOADED = OP == FP8_PLAIN && TYPE != T_F32;
    Block4<TYPE, AS_LOADED> v;
    {
        Raw<TYPE> raw[4];
        if (WHOLE || p.align_x >= 4) {
            uint32_t extra;
#pragma unroll
            for (int j = 0; j < 4; j++) raw[j] = load_raw<TYPE>(p.x, (r0 + j) * p.ldx, c, WHOLE ? c + 8 : j < left ? p.cols : 0, WHOLE ? 16 : p.align_x, false, extra);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t extra;
                const bool inner = r0 + j > 0 && r0 + j + 1 < p.rows;
                const int cols = j < left ? p.cols : 0;
                raw[j] = load_raw<TYPE>(p.x, (r0 + j) * p.ldx, c, cols, 2, inner, extra);
                settle<TYPE>(raw[j], extra, p.x, (r0 + j) * p.ldx, c, cols, 2, inner);
            }
        }
        uint2 q[4];
        uint32_t codes[4];
        if constexpr (OP == FP8_GELU_GRAD) {
            const uint8_t *src = p.ckpt + r0 * p.ldc + c, *code = p.ckpt_scales + ((int64_t)(tc >> 2) * p.rows + r0) * 4 + (tc & 3);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bool there = WHOLE || (in && j < left);
                q[j] = there ? __ldg(reinterpret_cast<const uint2 *>(src + j * p.ldc)) : make_uint2(0u, 0u);
                codes[j] = there ? __ldg(code + 4 * j) : 0u;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (AS_LOADED) v.raw[j] = raw[j];
            else to_floats<TYPE>(raw[j], v.v[j]);
            if constexpr (OP == FP8_GELU_GRAD) {
                float h[8];
                ckpt_values(q[j], codes[j], h);
#pragma unroll
                for (int i = 0; i < 8; i += 2) times_gelu_grad2<TANH>(v.v[j][i], v.v[j][i + 1], h[i], h[i + 1]);
            }
        }
    }
    auto store_rows = [&](uint8_t *data, int64_t ld, uint8_t *scales, auto type, uint32_t codes, uint32_t odd, bool any) {
        constexpr int T8 = decltype(type)::value;
        uint8_t *dst = data + r0 * ld + c;
        uint2 q[4];
#pragma unroll
        for (int j = 0; j < 4; j++) q[j] = round8<T8>(v, j, inverse_scale(byte_of(codes, j)));
        if (any) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (byte_of(odd, j)) q[j] = mend8<T8>(q[j], v, j);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (in && (WHOLE || j < left)) *reinterpret_cast<uint2 *>(dst + j * ld) = q[j];
        if ((lane & 3) == 0 && own_row < left) store_scale(scales, p.rows, r0 + own_row, tc, cblocks, byte_of(codes, own_row));
    };
    if constexpr (OP == FP8_GELU) {
        if (p.ckpt) {
            uint32_t codes, odd = 0;
            const bool any = codes_of4<F8_E4M3>(v, &codes, &odd);
            store_rows(p.ckpt, p.ldc, p.ckpt_scales, std::integral_constant<int, F8_E4M3>(), codes, odd, any);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < 8; i += 2) gelu2<TANH, TYPE == T_F32>(v.v[j][i], v.v[j][i + 1]);   // of the zeros that pad: zero
    }

    uint32_t tile_code = 0;
    bool tile_odd = false;
    if constexpr (SQUARE) {
        // values that are not negative are ordered like their bits; a thread without a number has NaN, whose bits are above all of them
        auto over_tile = [&](float m) {
            m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(m, 0.0f))));
            if (lane == 0) sh.all[warp] = m;
            __syncthreads();
            m = 0.0f;
#pragma unroll
            for (int w = 0; w < 16; w++) m = fmaxf(m, sh.all[w]);
            return m;
        };
        float m = over_tile(fmaxf(fmaxf(v.row_amax(0), v.row_amax(1)), fmaxf(v.row_amax(2), v.row_amax(3))));
        tile_odd = !finite(m);
        if (tile_odd) {
            __syncthreads();
            m = over_tile(fmaxf(fmaxf(finite_row_amax(v, 0), finite_row_amax(v, 1)), fmaxf(finite_row_amax(v, 2), finite_row_amax(v, 3))));
        }
        tile_code = scale_code<F8>(m);
    }

    if (p.data) {
        uint32_t odd = 0x01010101u, codes = tile_code * 0x01010101u;
        bool any = tile_odd;
        if constexpr (!SQUARE) any = codes_of4<F8>(v, &codes, &odd);
        store_rows(p.data, p.ldd, p.scales, std::integral_constant<int, F8>(), codes, odd, any);
    }

    // four threads a column: rows of sh.amax_of taken in turn
    const int own_col = threadIdx.x >> 2, part = threadIdx.x & 3;
    auto put8 = [&](const float (&m)[8]) {
        float4 *at = reinterpret_cast<float4 *>(&sh.amax_of[warp * 2 + half][group * 8]);
        at[0] = make_float4(m[0], m[1], m[2], m[3]);
        at[1] = make_float4(m[4], m[5], m[6], m[7]);
    };
    if (p.data_t) {
        float inv[8];
        bool any = tile_odd;
        if constexpr (!SQUARE) {
            // scales of the tile's columns from what put8() has laid out
            auto column_scales = [&](bool finite_only) {
                __syncthreads();
                float a = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; k++) a = fmaxf(a, sh.amax_of[4 * k + part][own_col]);
                a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
                a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
                const bool odd = finite_only ? sh.inv_of[own_col] < 0.0f : !finite(a);
                __syncwarp();
                if (part == 0) {
                    const uint32_t code = scale_code<F8>(finite(a) ? a : 0.0f);
                    sh.inv_of[own_col] = odd ? -inverse_scale(code) : inverse_scale(code);   // the sign says that it has an infinity
                    const int col = tc * 128 + own_col;
                    if (WHOLE || col < p.cols) store_scale(p.scales_t, p.cols, col, tr, rblocks, code);
                }
                return __syncthreads_or(odd) != 0;
            };
            float m[8];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float2 a = v.col_amax(k);
                m[2 * k] = a.x;
                m[2 * k + 1] = a.y;
            }
            put8(m);
            any = column_scales(false);
            if (any) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    m[2 * k] = m[2 * k + 1] = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        m[2 * k] = finite_max(m[2 * k], v.at(j, k).x);
                        m[2 * k + 1] = finite_max(m[2 * k + 1], v.at(j, k).y);
                    }
                }
                put8(m);
                (void)column_scales(true);
            }
            const float4 lo = *reinterpret_cast<const float4 *>(&sh.inv_of[group * 8]), hi = *reinterpret_cast<const float4 *>(&sh.inv_of[group * 8 + 4]);
            inv[0] = lo.x; inv[1] = lo.y; inv[2] = lo.z; inv[3] = lo.w;
            inv[4] = hi.x; inv[5] = hi.y; inv[6] = hi.z; inv[7] = hi.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) inv[i] = tile_odd ? -inverse_scale(tile_code) : inverse_scale(tile_code);
            if (threadIdx.x < 128 && tc * 128 + (int)threadIdx.x < p.cols) store_scale(p.scales_t, p.cols, tc * 128 + threadIdx.x, tr, rblocks, tile_code);
        }
        uint32_t *const image = &sh.image[group * 256 + ((warp * 2 + half) ^ (2 * group))];
        if (!any) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                float2 s[4];
#pragma unroll
                for (int j = 0; j < 4; j++) s[j] = mul2(v.at(j, i / 2), make_float2(inv[i], inv[i + 1]));
                image[i * 32] = __byte_perm(round2<F8>(s[0].x, s[1].x), round2<F8>(s[2].x, s[3].x), 0x5410);
                image[i * 32 + 32] = __byte_perm(round2<F8>(s[0].y, s[1].y), round2<F8>(s[2].y, s[3].y), 0x5410);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float a = fabsf(inv[i]);
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = i & 1 ? v.at(j, i / 2).y : v.at(j, i / 2).x;
                uint32_t w = __byte_perm(round2<F8>(x[0] * a, x[1] * a), round2<F8>(x[2] * a, x[3] * a), 0x5410);
                if (inv[i] < 0.0f) w = mend4<F8, AS_LOADED>(w, x[0], x[1], x[2], x[3]);
                image[i * 32] = w;
            }
        }
        __syncthreads();
        // sixteen lanes a column: eight rows each
        const int64_t padded = ((int64_t)p.rows + 15) & ~(int64_t)15;
        const int piece = lane & 15, col0 = threadIdx.x >> 4;
        const int64_t row = (int64_t)tr * 128 + piece * 8;
        uint8_t *dst = p.data_t + ((int64_t)tc * 128 + col0) * p.ldt + row;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int col = col0 + 32 * k;
            const uint2 q = *reinterpret_cast<const uint2 *>(&sh.image[col * 32 + 2 * (piece ^ (col >> 3))]);
            if (WHOLE || (tc * 128 + col < p.cols && row < padded)) *reinterpret_cast<uint2 *>(dst + (int64_t)(32 * k) * p.ldt) = q;
        }
    }

    if (p.partial) {                       // amax_of has been read by all: the image is complete
        float s[8];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float2 a = v.at(0, k), b = v.at(1, k), c = v.at(2, k), d = v.at(3, k);
            s[2 * k] = (a.x + b.x) + (c.x + d.x);
            s[2 * k + 1] = (a.y + b.y) + (c.y + d.y);
        }
        put8(s);
        __syncthreads();
        float a = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) a += sh.amax_of[4 * k + part][own_col];
        a += __shfl_xor_sync(0xffffffffu, a, 1);
        a += __shfl_xor_sync(0xffffffffu, a, 2);
        const int col = tc * 128 + own_col;
        if (part == 0 && (WHOLE || col < p.cols)) p.partial[(int64_t)tr * p.cols + col] = a;
    }
}

template <int TYPE, int OP, int F8, bool SQUARE, bool TANH>
__global__ void __launch_bounds__(TILE_THREADS, OP == FP8_PLAIN && TYPE != T_F32 ? 3 : 2) fp8_tiles_kernel(const Fp8QuantParams p)
{
    __shared__ TileShared sh;
    grid_dependency_wait();
    grid_launch_dependents();
    const int cblocks = (int)(((int64_t)p.cols + 127) >> 7);
    const int tr = (int)(blockIdx.x / (unsigned)cblocks), tc = (int)blockIdx.x - tr * cblocks;
    if (p.align_x == 16 && (int64_t)tr * 128 + 128 <= p.rows && (int64_t)tc * 128 + 128 <= p.cols) fp8_tile<TYPE, OP, F8, SQUARE, TANH, true>(p, sh, tr, tc);
    else fp8_tile<TYPE, OP, F8, SQUARE, TANH, false>(p, sh, tr, tc);
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

// A warp takes four blocks of a row, whose scales are one word; lanes lie along the row with V values each, as many as the result's alignment lets one store write (16
// bytes, 4 or a value), so that a warp's store covers neighbouring sectors whatever V.  Bound by HBM.  16384 x 4096 to fp16 37 us, to fp32 64 (floors 31 and 51),
// 8191 x 4095 to fp16 28 (15); eight values a lane for every type and alignment: 41, 96 and 107.
template <int TYPE, int F8, int V>
__global__ void __launch_bounds__(ROWS_THREADS) fp8_dequantize_kernel(const uint8_t *__restrict__ data, int64_t ldd, const uint32_t *__restrict__ scales, int rows, int cols,
                                                                      void *out, int64_t ldo)
{
    using E = typename Elem<TYPE>::type;
    using Bytes = std::conditional_t<V == 8, uint2, std::conditional_t<V == 4, uint32_t, std::conditional_t<V == 2, uint16_t, uint8_t>>>;
    constexpr int STEPS = 16 / V;
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t groups = (uint32_t)(((int64_t)cols + 511) >> 9), total = groups * (uint32_t)rows;
    const uint32_t step = gridDim.x * (ROWS_THREADS / 32);
    for (uint32_t u = (blockIdx.x * ROWS_THREADS + threadIdx.x) >> 5; u < total; u += step) {
        const uint32_t r = u / groups, g = u - r * groups;
        const int c0 = (int)g * 512 + (int)(threadIdx.x & 31) * V;
        const uint8_t *src = data + (int64_t)r * ldd + c0;
        E *dst = reinterpret_cast<E *>(out) + (int64_t)r * ldo + c0;
        const uint32_t codes = __ldg(scales + (int64_t)g * rows + r);
        // a block's scale as half a word: bf16 has them all, and NaN for 255
        uint32_t pair[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const __nv_bfloat162_raw b = __nv_cvt_e8m0x2_to_bf162raw((__nv_fp8x2_storage_t)(codes >> (16 * i)));
            pair[i] = (uint32_t)b.x | ((uint32_t)b.y << 16);
        }
        Bytes q[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; i++) q[i] = c0 + 32 * V * i < cols ? __ldg(reinterpret_cast<const Bytes *>(src + 32 * V * i)) : Bytes{};
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            const int c = c0 + 32 * V * i;
            const int kb = ((int)(threadIdx.x & 31) * V + 32 * V * i) >> 7;
            const float s = __uint_as_float(kb & 1 ? pair[kb >> 1] & 0xFFFF0000u : pair[kb >> 1] << 16);
            float v[V];
            if constexpr (V == 1) {
                const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)q[i], F8 == F8_E4M3 ? __NV_E4M3 : __NV_E5M2);
                v[0] = __half2float(*reinterpret_cast<const __half *>(&h)) * s;
            } else {
#pragma unroll
                for (int k = 0; k < V; k += 2) {
                    uint32_t w;
                    if constexpr (V == 8) w = (k < 4 ? q[i].x : q[i].y) >> (8 * (k & 3));
                    else w = (uint32_t)q[i] >> (8 * k);
                    const float2 f = block_pair<F8>(w, s);
                    v[k] = f.x;
                    v[k + 1] = f.y;
                }
            }
            if (c + V <= cols) {
                if constexpr (TYPE == T_F32 && V == 4) {
                    *reinterpret_cast<float4 *>(dst + 32 * V * i) = make_float4(v[0], v[1], v[2], v[3]);
                } else if constexpr (V == 8) {
                    store8<TYPE>(dst, 0, 32 * V * i, INT_MAX, 16, v);
                } else if constexpr (V == 2) {
                    E pair[2] = {from_float<TYPE>(v[0]), from_float<TYPE>(v[1])};
                    *reinterpret_cast<uint32_t *>(dst + 32 * V * i) = *reinterpret_cast<const uint32_t *>(pair);
                } else {
                    dst[32 * V * i] = from_float<TYPE>(v[0]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < V; k++)
                    if (c + k < cols) dst[32 * V * i + k] = from_float<TYPE>(v[k]);
            }
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
    const int64_t units = (int64_t)p.rows * (((int64_t)p.cols + 511) / 512), per_cta = ROWS_THREADS / 16;
    const int64_t wave = (int64_t)device_sms() * (TYPE == T_F32 || op != FP8_PLAIN ? 2 : 3);
    const int64_t ctas = (units + per_cta - 1) / per_cta < wave ? (units + per_cta - 1) / per_cta : wave;
    const dim3 grid((unsigned)ctas);
    const bool e4 = p.f8 == F8_E4M3;
#define VNM_ROWS(OP, F8, TANH) launch(fp8_rows_kernel<TYPE, OP, F8, TANH>, grid, ROWS_THREADS, stream, p)
    if (op == FP8_PLAIN) return e4 ? VNM_ROWS(FP8_PLAIN, F8_E4M3, false) : VNM_ROWS(FP8_PLAIN, F8_E5M2, false);
    if (op == FP8_GELU) return p.tanh_form ? VNM_ROWS(FP8_GELU, F8_E4M3, true) : VNM_ROWS(FP8_GELU, F8_E4M3, false);
    if (e4) return p.tanh_form ? VNM_ROWS(FP8_GELU_GRAD, F8_E4M3, true) : VNM_ROWS(FP8_GELU_GRAD, F8_E4M3, false);
    return p.tanh_form ? VNM_ROWS(FP8_GELU_GRAD, F8_E5M2, true) : VNM_ROWS(FP8_GELU_GRAD, F8_E5M2, false);
#undef VNM_ROWS
}

template <int TYPE>
cudaError_t tiles_of(const Fp8QuantParams &p, int op, bool square, cudaStream_t stream)
{
    const dim3 grid((unsigned)((((int64_t)p.cols + 127) / 128) * (((int64_t)p.rows + 127) / 128)));
    const bool e4 = p.f8 == F8_E4M3;
#define VNM_TILES(OP, F8, SQUARE, TANH) launch(fp8_tiles_kernel<TYPE, OP, F8, SQUARE, TANH>, grid, TILE_THREADS, stream, p)
    if (op == FP8_GELU) return p.tanh_form ? VNM_TILES(FP8_GELU, F8_E4M3, false, true) : VNM_TILES(FP8_GELU, F8_E4M3, false, false);
    if (op == FP8_GELU_GRAD) {
        if (e4) return p.tanh_form ? VNM_TILES(FP8_GELU_GRAD, F8_E4M3, false, true) : VNM_TILES(FP8_GELU_GRAD, F8_E4M3, false, false);
        return p.tanh_form ? VNM_TILES(FP8_GELU_GRAD, F8_E5M2, false, true) : VNM_TILES(FP8_GELU_GRAD, F8_E5M2, false, false);
    }
    if (square) return e4 ? VNM_TILES(FP8_PLAIN, F8_E4M3, true, false) : VNM_TILES(FP8_PLAIN, F8_E5M2, true, false);
    return e4 ? VNM_TILES(FP8_PLAIN, F8_E4M3, false, false) : VNM_TILES(FP8_PLAIN, F8_E5M2, false, false);
#undef VNM_TILES
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

cudaError_t launch_fp8_dequantize(const uint8_t *data, int64_t ldd, const uint8_t *scales, int f8, int rows, int cols, void *out, int type, int64_t ldo, int align,
                                  cudaStream_t stream)
{
    const int64_t units = (int64_t)rows * (((int64_t)cols + 511) / 512), per_cta = ROWS_THREADS / 32, wave = (int64_t)device_sms() * 8;
    const dim3 grid((unsigned)((units + per_cta - 1) / per_cta < wave ? (units + per_cta - 1) / per_cta : wave));
    const uint32_t *words = reinterpret_cast<const uint32_t *>(scales);
#define VNM_DEQUANTIZE(TYPE, V)                                                                                                                                    \
    return f8 == F8_E4M3 ? launch(fp8_dequantize_kernel<TYPE, F8_E4M3, V>, grid, ROWS_THREADS, stream, data, ldd, words, rows, cols, out, ldo)                      \
                         : launch(fp8_dequantize_kernel<TYPE, F8_E5M2, V>, grid, ROWS_THREADS, stream, data, ldd, words, rows, cols, out, ldo);
    if (type == T_F32) {
        if (align == 16) { VNM_DEQUANTIZE(T_F32, 4) }
        VNM_DEQUANTIZE(T_F32, 1)
    }
    if (type == T_F16) {
        if (align == 16) { VNM_DEQUANTIZE(T_F16, 8) }
        if (align == 4) { VNM_DEQUANTIZE(T_F16, 2) }
        VNM_DEQUANTIZE(T_F16, 1)
    }
    if (align == 16) { VNM_DEQUANTIZE(T_BF16, 8) }
    if (align == 4) { VNM_DEQUANTIZE(T_BF16, 2) }
    VNM_DEQUANTIZE(T_BF16, 1)
#undef VNM_DEQUANTIZE
}

}  // namespace vnm
