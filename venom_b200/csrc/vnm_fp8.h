// Internal interface of the block-scaled 8-bit operators: parameters of their kernels, and the tensor-core wrappers they share.
#pragma once

#include "vnm_internal.h"

namespace vnm {

enum : int { T_F32 = 0, T_F16 = 1, T_BF16 = 2 };   // as VNM_F32, VNM_F16, VNM_BF16
enum : int { F8_E4M3 = 0, F8_E5M2 = 1 };           // as VNM_E4M3, VNM_E5M2

// What is done to the values between their load and their rounding to 8 bits.
enum : int {
    FP8_PLAIN = 0,      // x
    FP8_GELU = 1,       // gelu(x)
    FP8_GELU_GRAD = 2   // x gelu'(h) with h from an 8-bit checkpoint
};

struct Fp8QuantParams {
    const void *x;           // [rows, cols], rows ldx elements apart
    int64_t ldx;
    int rows, cols;
    int f8;                  // type of data and data_t
    int tanh_form;           // GELU by tanh
    int align_x, align_y;    // what the addresses of the rows of x and y are a multiple of: 16, 4 or 2 bytes
    uint8_t *data;           // [rows, ldd] or null
    int64_t ldd;
    uint8_t *scales;         // [groups][rows][4]
    uint8_t *data_t;         // [cols, ldt] or null
    int64_t ldt;
    uint8_t *scales_t;       // [groups of row blocks][cols][4]
    uint8_t *ckpt;           // e4m3 checkpoint of x (FP8_GELU: written where not null, FP8_GELU_GRAD: read), [rows, ldc]
    int64_t ldc;
    uint8_t *ckpt_scales;
    void *y;                 // the values themselves, in the type of x (null: not wanted)
    int64_t ldy;
    float *partial;          // tile kernel: [row blocks][cols] sums over the rows of a block (null: not wanted)
};

cudaError_t launch_fp8_rows(const Fp8QuantParams &p, int type, int op, cudaStream_t stream);
cudaError_t launch_fp8_tiles(const Fp8QuantParams &p, int type, int op, bool square, cudaStream_t stream);
cudaError_t launch_fp8_colsum(const float *partial, int blocks, int cols, void *out, int type, cudaStream_t stream);
cudaError_t launch_fp8_dequantize(const uint8_t *data, int64_t ldd, const uint8_t *scales, int f8, int rows, int cols, void *out, int type, int64_t ldo, int align,
                                  cudaStream_t stream);

// n / d of 0 <= n < 2^31 by a multiplication: with 2^(s - 1) < d <= 2^s and m = floor(2^(31 + s) / d) + 1, m d - 2^(31 + s) is at most 2^s, so that
// floor(n m / 2^(31 + s)) is the quotient (Granlund and Montgomery, 1994).
struct FastDiv {
    uint32_t d, m;
    int s;
    FastDiv() = default;
    explicit FastDiv(uint32_t divisor) : d(divisor), s(0)
    {
        while ((1ull << s) < d) s++;
        m = (uint32_t)((1ull << (31 + s)) / d + 1);
    }
    __host__ __device__ uint32_t quotient(uint32_t n) const { return (uint32_t)(((uint64_t)n * m) >> (31 + s)); }
};
// The order of tile_coords() with its divisions prepared: a tile's place is on the way of every role of a kernel with short tiles (two divisions
// took 600 of 5000 clocks a tile).
struct TileOrder {
    FastDiv band, full, last;   // tiles of a band, lines of a band and of the last one
    int lines, other, rows;     // lines banded (row or column tiles), the other count, whether lines are row tiles
    TileOrder() = default;
    TileOrder(int mt, int nt, int group) : rows(group >= 0)
    {
        const int g = group >= 0 ? group : -group;
        lines = rows ? mt : nt;
        other = rows ? nt : mt;
        band = FastDiv((uint32_t)g * (uint32_t)other);
        full = FastDiv((uint32_t)g);
        last = FastDiv((uint32_t)(lines % g ? lines % g : g));
    }
    __host__ __device__ void at(int tile, int *tm, int *tn) const
    {
        const uint32_t b = band.quotient((uint32_t)tile), within = (uint32_t)tile - b * band.d, first = b * full.d;
        const FastDiv size = first + full.d <= (uint32_t)lines ? full : last;
        const uint32_t across = size.quotient(within), line = first + within - across * size.d;
        *tm = (int)(rows ? line : across);
        *tn = (int)(rows ? across : line);
    }
};

// out[m, n] = sum over k of A[m, k] B[n, k] (+ bias[n]), A [M, K] and B [N, K] in 8 bits with a scale for each 128 k of a row.
struct Fp8MatmulParams {
    const uint32_t *sa, *sb;  // scale words [groups][M] and [groups][N]: byte j of word (g, r) is block 4 g + j of row r
    const void *bias;
    void *out;
    int64_t ldo;
    int M, N, K, ktiles;
    int out_type, bias_type;
    int whole_pieces;         // pair kernel: rows of the result lie on 16-byte boundaries
    int a_f8, b_f8;
    int mt, nt;               // tiles along M and N
    int split;                // CTAs of a cluster that share one tile's k
    TileOrder order;          // pair kernel
    int *status;
};

// What a plan depends on of the device that it is for.
struct Fp8Device {
    int sms;
    int clusters;  // of two CTAs of the pair kernel that run side by side; 0: it does not run here
};

struct Fp8Plan {
    int bn;        // columns of the accumulator
    int split;
    int grid;
};

// On pairs of SMs: tiles of 256 x (192 .. 256).
cudaError_t fp8_pair_init(int sms, int *clusters);      // for the current device
// wide_out: results of 32 bits; whole: their rows are stored in whole pieces (see whole_pieces).  Both return an estimate in microseconds, < 0: not for this problem.
float fp8_pair_config(int M, int N, int K, bool wide_out, bool whole, bool bias, const Fp8Device &device, Fp8Plan *plan);
cudaError_t launch_fp8_pair(const Fp8Plan &plan, const CUtensorMap &map_a, const CUtensorMap &map_b, const Fp8MatmulParams &p, cudaStream_t stream);
// One SM a tile: 128 rows of B x (16 .. 128) rows of A, k split over a cluster where tiles are few.
cudaError_t fp8_small_init();
float fp8_small_config(int M, int N, int ktiles, bool wide_out, const Fp8Device &device, Fp8Plan *plan);
cudaError_t launch_fp8_small(const Fp8Plan &plan, const CUtensorMap &map_a, const CUtensorMap &map_b, const Fp8MatmulParams &p, cudaStream_t stream);

#if defined(__CUDACC__)
// Instruction descriptor of tcgen05.mma kind::mxf8f6f4 with a power of two (ue8m0) as scale, fp32 accumulators, both operands K-major:
// bits 4-5 byte of B's scale word, 7-9 type of A (0 = e4m3, 1 = e5m2), 10-12 type of B, 17-22 N >> 3, 23 scale type (1 = ue8m0), 27-28 M >> 7,
// 29-30 byte of A's scale word.
__device__ __forceinline__ uint32_t make_idesc_mxf8(int M, int N, int a_f8, int b_f8)
{
    return ((uint32_t)a_f8 << 7) | ((uint32_t)b_f8 << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27);
}
__device__ __forceinline__ uint32_t idesc_scale_byte(int j) { return ((uint32_t)j << 4) | ((uint32_t)j << 29); }

// D[tmem] (+)= (scale_a A[smem]) (scale_b B[smem])^T over 32 k: one scale byte a row of either operand, from tensor memory.
__device__ __forceinline__ void tc_mma_mxf8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sa_tmem, uint32_t sb_tmem, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sa_tmem), "r"(sb_tmem), "r"(accumulate)
        : "memory");
}
// One register of every lane of the warp -> one column of the warp's 32 lanes of tensor memory.
template <int N>
__device__ __forceinline__ void tc_st_32x32b(uint32_t taddr, const uint32_t *r)
{
    if constexpr (N == 1) {
        asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(r[0]) : "memory");
    } else if constexpr (N == 2) {
        asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1, %2};" ::"r"(taddr), "r"(r[0]), "r"(r[1]) : "memory");
    } else if constexpr (N == 4) {
        asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
    } else {
        static_assert(N == 8, "widths of a store");
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                     "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                     : "memory");
    }
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
#endif

}  // namespace vnm
