// Matrix product of block-scaled 8-bit operands on PAIRS of SMs (clusters of two CTAs, tcgen05 cta_group::2): see vnm_fp8_small.cu for the arithmetic.
//
// A pair tile is 256 rows of A x BN rows of B; each CTA loads its 128 rows of A and half of the rows of B for a k-tile of 128, 31 KiB for 480 clocks of
// MMAs (BN = 240).  Two accumulators of up to 240 columns alternate between tiles, so that one drains while the other fills; 256 columns leave tensor memory for
// one.  Scale words of four k-tiles lie in one of two sets of twelve columns beside them: four for the CTA's rows of A, eight for all rows of B, which both CTAs hold.
//
// Protocol (rank 0 = leader):
//   * the peer's loads report to the leader's barriers themselves (cta_group::2 form of the copy, without multicast), whose expected bytes count both CTAs';
//   * only the leader issues MMAs; its commits arrive on the ring-free, scale-free and accumulator-full barriers of both CTAs;
//   * scale and epilogue warps of the peer arrive remotely on the leader's scale-full and accumulator-empty barriers.
// Every wait is bounded, and the CTAs meet at a cluster barrier before either leaves.
//
// Bound by power: 2048 x 12288 x 12288 239 to 261 us in long runs = 2.4-2.6 PFLOP/s at 1.0-1.4 GHz, 203 in short ones; 16384 x 4096 x 1024 with a bias 62 to 65 by
// itself (2.2 PFLOP/s), 73 to 81 among other calls: eight k-tiles for the epilogue of 256 x 240 values.
#include "vnm_fp8.h"

#include <cuda_bf16.h>

#include <cmath>
#include <type_traits>

namespace vnm {

namespace {

constexpr int A_BYTES = 128 * 128;
constexpr int NUM_THREADS = 512;
constexpr int SCALE_WARP0 = 4, EPI_WARP0 = 8;
constexpr int TMEM_COLS = 512;
constexpr int SF_SETS = 2;

// Epilogue, rows that begin anywhere: words between the rows of the windows (forty are used), an odd number of 16-byte pieces, so that eight rows lie in different banks;
// every eight rows are a piece further, so that rows of different phases do, too.
constexpr int WINDOW = 44;
__host__ __device__ constexpr int window_at(int row) { return row * WINDOW + 4 * (row >> 3); }

template <int BN, bool WHOLE>
struct Fp8Pair {
    static_assert(BN % 16 == 0 && BN <= 256 && BN > 128, "accumulator columns");
    static constexpr bool ONE = BN > 240;                // one accumulator
    static constexpr int HALF_N = BN / 2;
    static constexpr int B_BYTES = HALF_N * 128;
    static constexpr int B_SLOT = (B_BYTES + 1023) / 1024 * 1024;
    static constexpr int STAGE_BYTES = A_BYTES + B_SLOT;
    static constexpr int WARP_BYTES = (WHOLE ? 4096 : 4 * window_at(31) + 4 * WINDOW) + 640;   // an epilogue warp's 32 rows, and the bias of its columns and 32 before
    static constexpr int OUT_BYTES = 8 * WARP_BYTES;
    static constexpr int STAGES = (227 * 1024 - OUT_BYTES - 512 - 1024) / STAGE_BYTES;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + OUT_BYTES + 512 + 1024;
    static_assert(SMEM_BYTES <= 227 * 1024, "shared memory per CTA");
    static_assert((2 * STAGES + 2 * SF_SETS + 4) * 8 + 8 <= 512, "barriers");
};
__device__ __forceinline__ uint32_t acc_col(int a) { return (uint32_t)a * 256u; }
template <int BN>
__device__ __forceinline__ uint32_t sf_col(int set) { return Fp8Pair<BN, true>::ONE ? 256u + 16u * (uint32_t)set : 240u + 256u * (uint32_t)set; }

__device__ __forceinline__ uint32_t cluster_ctarank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t mapa_shared(uint32_t saddr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory"); }
__device__ __forceinline__ void cluster_sync_all() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_alloc2(uint32_t *smem_result, uint32_t ncols)
{
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_result)), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish2() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_dealloc2(uint32_t taddr, uint32_t ncols)
{
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// Arrives on the barrier at this offset in both CTAs once every tcgen05 operation issued so far by this thread has completed.
__device__ __forceinline__ void tc_commit2(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3)
                 : "memory");
}
// Box at (col, row) into this CTA's shared memory; the bytes are reported to the barrier at `bar` (an address of the cluster, here the leader's).
__device__ __forceinline__ void tma_load_2d_pair(void *smem_dst, const void *tmap, int col, int row, uint32_t bar, uint64_t policy)
{
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(
                     smem_u32(smem_dst)),
                 "l"(tmap), "r"(col), "r"(row), "r"(bar), "l"(policy)
                 : "memory");
}
// 256 rows: 0-127, their scales and accumulator in the leader, 128-255 in the peer; rows of B: the first half in the leader's shared memory, the rest in the peer's
__device__ __forceinline__ void tc_mma2_mxf8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sa_tmem, uint32_t sb_tmem, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sa_tmem), "r"(sb_tmem), "r"(accumulate)
        : "memory");
}

// ---- epilogue of one warp: 32 accumulator lanes (rows of the result), `cols` columns from n0 on ----
// 128 bytes of each row at a time pass through shared memory and leave in pieces of 16 bytes, eight lanes a row.  Exchanging words between lanes instead, so
// that nothing passes through shared memory, needs 2.4 times the instructions, and the epilogue's eight warps are what short tiles wait for: 16384 x 4096 x
// 1024 with a bias 83 us (62 this way).
// Rows that begin anywhere (odd numbers of columns) leave in the same pieces, aligned where they go and not where they come from: the lane that owns a row writes it
// into its window word by word, as far behind a sector's begin as it will lie in memory (16 bits: words shifted by a half where it begins inside one).  What
// a step leaves behind its last whole 128 bytes is where the next one begins, so that a sector between two steps is written once and whole; what costs
// is sectors written in parts (11844 x 15043, K = 116, bf16: 348 us with words of 4 bytes a lane and single values at the edges of each 128 bytes), and only a tile's edges
// are.  Windows as the columns lie, and pieces cut out of five words when they are read: 8191 x 4095 x 1023, fp16 41.9 us against
// 37.4, 2978 x 2039 x 1371, fp32 19.0 against 14.3.
template <int TYPE>
__device__ __forceinline__ uint32_t pack16(float a, float b)
{
    if constexpr (TYPE == T_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
__device__ __forceinline__ uint32_t bias_bits(const void *bias, int type, int n)
{
    return type == T_F32 ? __ldg(reinterpret_cast<const uint32_t *>(bias) + n) : (uint32_t)__ldg(reinterpret_cast<const unsigned short *>(bias) + n);
}
__device__ __forceinline__ float bias_float(uint32_t bits, int type)
{
    return type == T_F32 ? __uint_as_float(bits) : type == T_F16 ? __half2float(__ushort_as_half((unsigned short)bits)) : __uint_as_float(bits << 16);
}

// (a, b) += (x, y), both rounded to nearest
__device__ __forceinline__ void add2(uint32_t &a, uint32_t &b, float x, float y)
{
    asm("{\n\t.reg .b64 p, q;\n\t"
        "mov.b64 p, {%0, %1};\n\t"
        "mov.b64 q, {%2, %3};\n\t"
        "add.rn.f32x2 p, p, q;\n\t"
        "mov.b64 {%0, %1}, p;\n\t}"
        : "+r"(a), "+r"(b)
        : "f"(x), "f"(y));
}
// 32 columns of `v`, behind the wait for them, rounded and packed.  The bias is read ahead of the wait.
template <int TYPE, bool BIAS>
__device__ __forceinline__ void round32(uint32_t (&v)[32], const float4 *bias, uint32_t (&word)[TYPE == T_F32 ? 32 : 16])
{
    float4 b[BIAS ? 8 : 1];
    if constexpr (BIAS) {
#pragma unroll
        for (int i = 0; i < 8; i++) b[i] = bias[i];
    }
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i++) asm volatile("" : "+r"(v[i]));
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (BIAS) {
            add2(v[4 * i], v[4 * i + 1], b[i].x, b[i].y);
            add2(v[4 * i + 2], v[4 * i + 3], b[i].z, b[i].w);
        }
        if constexpr (TYPE == T_F32) {
#pragma unroll
            for (int k = 0; k < 4; k++) word[4 * i + k] = v[4 * i + k];
        } else {
            word[2 * i] = pack16<TYPE>(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]));
            word[2 * i + 1] = pack16<TYPE>(__uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
        }
    }
}

// Bytes [from, to) of a 16-byte piece at `dst`, both even: at most six stores, for the edges of a tile.
__device__ __forceinline__ void store_part(uint8_t *dst, const uint32_t (&y)[4], int from, int to)
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const bool lo = from <= 4 * i && to >= 4 * i + 2, hi = from <= 4 * i + 2 && to >= 4 * i + 4;
        if (lo && hi) *reinterpret_cast<uint32_t *>(dst + 4 * i) = y[i];
        else if (lo) *reinterpret_cast<uint16_t *>(dst + 4 * i) = (uint16_t)y[i];
        else if (hi) *reinterpret_cast<uint16_t *>(dst + 4 * i + 2) = (uint16_t)(y[i] >> 16);
    }
}

// `part`: 0 the first 128 columns of a tile, 1 the rest; WHOLE: rows lie on 16-byte boundaries.  HOLD (128 columns of 16 bits): all of them are
// rounded into registers before the first is stored, where the next tile's MMAs wait for this accumulator.
template <int TYPE, bool BIAS, bool WHOLE, bool HOLD, typename Release>
__device__ __forceinline__ void store_columns(uint32_t tacc, int64_t row0, int n0, int cols, int part, uint4 *stage, const float4 *bias, const Fp8MatmulParams &p, Release release)
{
    constexpr int SIZE = TYPE == T_F32 ? 4 : 2, WIDTH = 128 / SIZE, PIECES = TYPE == T_F32 ? 8 : 4;   // pieces of 32 columns
    const int lane = threadIdx.x & 31;
    const int64_t pitch = p.ldo * SIZE;
    uint8_t *out = reinterpret_cast<uint8_t *>(p.out) + row0 * pitch + (int64_t)n0 * SIZE;
    const int rows = p.M - row0 < 32 ? (int)(p.M - row0) : 32;     // that there are; may be none
    const int bytes = (p.N - n0 < cols ? p.N - n0 : cols) * SIZE;   // of a row to store; may be none
    uint4 *const mine = stage + lane * 8;                          // WHOLE
    uint32_t *const words = reinterpret_cast<uint32_t *>(stage), *const own = words + window_at(lane);   // !WHOLE
    const int phase = (int)(reinterpret_cast<uintptr_t>(out + lane * pitch) & 31), at = phase >> 2;     // of this lane's row in its sector; the same in each step
    const uint32_t shifted = phase & 2 ? 0x5432u : 0x7654u;        // the word before and this one, or this one
    uint32_t last = 0;                                             // word before the next one
    if constexpr (!WHOLE) {
        if (part == 1) {                                           // the first part leaves the sector between the two to this one
            uint32_t u[32];
            tc_ld_32x32b_x32(tacc - 32u, u);
            uint32_t w[TYPE == T_F32 ? 32 : 16];
            round32<TYPE, BIAS>(u, bias - 8, w);
            __syncwarp();                                          // the tile before has been read
#pragma unroll
            for (int i = 1; i < 8; i++) {
                constexpr int FROM = TYPE == T_F32 ? 24 : 8;
                if (at - 8 + i >= 0) own[at - 8 + i] = TYPE == T_F32 ? w[FROM + i] : __byte_perm(w[FROM + i - 1], w[FROM + i], shifted);
            }
            last = w[TYPE == T_F32 ? 31 : 15];
        }
    }
    uint32_t v[32];
    tc_ld_32x32b_x32(tacc, v);
    uint32_t held[HOLD ? 64 : 1];
    if constexpr (HOLD) {
#pragma unroll
        for (int h = 0; h < 4; h++) {
            uint32_t word[16];
            round32<TYPE, BIAS>(v, bias + 8 * h, word);
            if (h < 3) tc_ld_32x32b_x32(tacc + (uint32_t)(32 * (h + 1)), v);
            else release();
#pragma unroll
            for (int i = 0; i < 16; i++) held[16 * h + i] = word[i];
        }
    }
#pragma unroll(HOLD ? 2 : 1)
    for (int c0 = 0; c0 < (HOLD ? 128 : cols); c0 += WIDTH, out += 128) {
        // 32 columns at a time, the next ones on their way while these are rounded
#pragma unroll
        for (int h = 0; h < WIDTH / 32; h++) {
            uint32_t word[TYPE == T_F32 ? 32 : 16];
            if constexpr (HOLD) {
#pragma unroll
                for (int i = 0; i < 16; i++) word[i] = held[c0 / 2 + 16 * h + i];
            } else {
                round32<TYPE, BIAS>(v, bias + c0 / 4 + 8 * h, word);
                const int c1 = c0 + 32 * (h + 1);
                if (c1 < cols) tc_ld_32x32b_x32(tacc + (uint32_t)c1, v);
                else if (c1 - 32 < cols) release();                // once: behind the last columns that belong to the tile
            }
            if (h == 0) {
                __syncwarp();                                      // the columns before have been read
                if constexpr (!WHOLE) {
                    if (c0 > 0) {
                        uint4 *const piece = reinterpret_cast<uint4 *>(own);
                        const uint4 q0 = piece[8], q1 = piece[9];
                        piece[0] = q0;
                        piece[1] = q1;
                    }
                }
            }
            if constexpr (WHOLE) {
#pragma unroll
                for (int i = 0; i < PIECES; i++) mine[(PIECES * h + i) ^ (lane & 7)] = make_uint4(word[4 * i], word[4 * i + 1], word[4 * i + 2], word[4 * i + 3]);
            } else if constexpr (TYPE == T_F32) {
#pragma unroll
                for (int i = 0; i < 32; i++) own[at + i] = word[i];
            } else {
#pragma unroll
                for (int i = 0; i < 16; i++) own[at + 16 * h + i] = __byte_perm(i ? word[i ? i - 1 : 0] : last, word[i], shifted);
                last = word[15];
                if (h == WIDTH / 32 - 1) own[at + 32] = last >> 16;      // the half that a shift leaves over
            }
        }
        __syncwarp();
        const int left = bytes - c0 * SIZE;                         // bytes of a row from here on
        const int piece = lane & 7, first = lane >> 3;
        if constexpr (WHOLE) {
            uint8_t *dst = out + first * pitch + piece * 16;
            const int end = left - piece * 16;                      // bytes of a row from this piece on
            if (left >= 128 || (left & 15) == 0) {
                const bool on = end > 0;
#pragma unroll
                for (int i = 0; i < 8; i++, dst += 4 * pitch) {
                    const int r = 4 * i + first;
                    const uint4 q = stage[r * 8 + (piece ^ (r & 7))];
                    if (on && r < rows) *reinterpret_cast<uint4 *>(dst) = q;
                }
            } else if (end > 0) {                                   // the matrix ends inside a piece
#pragma unroll 1
                for (int i = 0; i < 8; i++, dst += 4 * pitch) {
                    const int r = 4 * i + first;
                    const uint4 q = stage[r * 8 + (piece ^ (r & 7))];
                    if (r >= rows) break;
                    if (end >= 16) {
                        *reinterpret_cast<uint4 *>(dst) = q;
                    } else {
                        const uint32_t y[4] = {q.x, q.y, q.z, q.w};
                        store_part(dst, y, 0, end);
                    }
                }
            }
        } else if (left > 0) {
            const bool head = c0 == 0 && part == 0;                                // the sector that the row begins in is another tile's as well
            {
                uint8_t *row = out + first * pitch;
#pragma unroll 4
                for (int i = 0; i < 8; i++, row += 4 * pitch) {
                    const int r = 4 * i + first, s = (int)(reinterpret_cast<uintptr_t>(row) & 31);
                    const uint4 q = *reinterpret_cast<const uint4 *>(words + window_at(r) + 4 * piece);
                    if (r < rows && 16 * piece >= (head ? s : 0) && 16 * piece + 16 <= s + left) *reinterpret_cast<uint4 *>(row - s + 16 * piece) = q;
                }
            }
            // The last sector, where it is not left to the next columns or the other part; and pieces that begin or end inside: a lane a row.
            const bool tail = left <= 128 && !(part == 0 && p.N - n0 > 128);
            if ((head || tail) && lane < rows) {
                uint8_t *row = out + lane * pitch - phase;
                const int end = phase + left;
                auto part_of = [&](int q, int from, int to) {
                    const uint4 v4 = reinterpret_cast<const uint4 *>(own)[q];
                    const uint32_t y[4] = {v4.x, v4.y, v4.z, v4.w};
                    store_part(row + 16 * q, y, from, to);
                };
                if (head && (phase & 15)) part_of(phase >> 4, phase & 15, end - (phase & 16) < 16 ? end - (phase & 16) : 16);
                if (tail && end >= 144) *reinterpret_cast<uint4 *>(row + 128) = reinterpret_cast<const uint4 *>(own)[8];
                if (tail && (end & 15) && !(head && end < ((phase + 15) & ~15))) part_of(end >> 4, 0, end & 15);      // not where head and tail are one piece
            }
        }
    }
}

// Warps: 0 loads A, 1 loads B, 2 issues the MMAs (leader), 3 owns tensor memory, 4..7 scale words, 8..15 epilogue: columns 0..127 and the rest.
template <int BN, bool WHOLE>
__global__ void __launch_bounds__(NUM_THREADS, 1) fp8_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Fp8MatmulParams p)
{
    using T = Fp8Pair<BN, WHOLE>;
    constexpr int S = T::STAGES;
    extern __shared__ uint8_t smem_raw[];
    // Through a pointer that the compiler knows to be shared memory: 16384 x 4096 x 256 34.9 -> 31.8 us, with a bias 41.3 -> 37.0.  The other epilogues are scheduled worse then
    // (11844 x 15043 x 116 130 -> 140, in tiles of 256 columns 16384 x 4096 x 256 36 -> 41): theirs goes through an integer.
    uint8_t *smem = WHOLE && !T::ONE ? smem_raw + (-smem_u32(smem_raw) & 1023u) : reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *a_ring = smem, *b_ring = smem + S * A_BYTES;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + S * T::STAGE_BYTES + T::OUT_BYTES);
    uint64_t *freed = full + S;
    uint64_t *sf_full = freed + S, *sf_free = sf_full + SF_SETS;
    uint64_t *acc_full = sf_free + SF_SETS, *acc_empty = acc_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t crank = cluster_ctarank();
    const bool leader = crank == 0;
    const int pair = (int)blockIdx.x >> 1, npairs = (int)gridDim.x >> 1;
    const int total = p.mt * p.nt;
    const int my_tiles = pair < total ? (total - pair + npairs - 1) / npairs : 0;
    const int total_it = my_tiles * p.ktiles;
    const int groups = (p.ktiles + 3) >> 2;             // of scale words, a tile

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(&full[s], 2);
            mbar_init(&freed[s], 1);
        }
        for (int s = 0; s < SF_SETS; s++) {
            mbar_init(&sf_full[s], 8);
            mbar_init(&sf_free[s], 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(&acc_full[a], 1);
            mbar_init(&acc_empty[a], 16);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    cluster_sync_all();                                 // both CTAs' barriers exist before anyone arrives on them remotely
    grid_dependency_wait();
    // The loads begin at once; whoever uses tensor memory meets behind its allocation.  (The first MMA waits for the scale words of both CTAs, so for both allocations.)
    if (warp >= 2) {
        if (warp == 3) {
            tmem_alloc2(tmem_slot, TMEM_COLS);
            tmem_relinquish2();
        }
        tc_fence_before();
        named_barrier_sync(1, NUM_THREADS - 64);
        tc_fence_after();
        grid_launch_dependents();
    }

    if (warp < 2) {
        // ---------------- loads ----------------
        if (elect_one()) {
            const bool is_a = warp == 0;
            const CUtensorMap *map = is_a ? &map_a : &map_b;
            uint8_t *ring = is_a ? a_ring : b_ring;
            const int slot = is_a ? A_BYTES : T::B_SLOT;
            const uint32_t bytes = is_a ? A_BYTES : T::B_BYTES;
            const uint64_t policy = (p.order.rows != 0) == is_a ? L2_EVICT_LAST : L2_EVICT_NORMAL;   // the banded operand is read again soon
            const uint32_t report = mapa_shared(smem_u32(full), 0);
            tma_prefetch_desc(map);
            int s = 0, it = 0;
            uint32_t ph = 1;
            bool alive = true;
            for (int tile = pair; alive && tile < total; tile += npairs) {
                int tm, tn;
                p.order.at(tile, &tm, &tn);
                const int row = is_a ? tm * 256 + (int)crank * 128 : tn * BN + (int)crank * T::HALF_N;
                for (int kt = 0; kt < p.ktiles; ++kt, ++it) {
                    if (!wait_quiet(&freed[s], ph, abort_flag, p.status, DEV_TIMEOUT_PRODUCER)) { alive = false; break; }
                    if (leader) mbar_arrive_expect_tx(&full[s], 2 * bytes);
                    tma_load_2d_pair(ring + s * slot, map, kt * 128, row, report + (uint32_t)s * 8u, policy);
                    if (++s == S) { s = 0; ph ^= 1; }
                }
            }
            if (*abort_flag && leader) {
                // both CTAs' copies report here: those of every slot that has been filled land before this CTA meets the other one and leaves
                for (int k = it > S ? it - S : 0; k < it; ++k) drain_slot(&full[k % S], (uint32_t)(k / S) & 1u, p.status);
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        // ---------------- MMA issuer ----------------
        if (leader && elect_one()) {
            const uint32_t tmem_base = *tmem_slot;
            const uint32_t idesc0 = make_idesc_mxf8(256, BN, p.a_f8, p.b_f8);
            const uint64_t adesc0 = make_smem_desc(smem_u32(a_ring), 16, 1024, 2), bdesc0 = make_smem_desc(smem_u32(b_ring), 16, 1024, 2);
            int s = 0, left = total_it, gleft = my_tiles * groups, set = 0;
            uint32_t ph = 0, sf_ph = 0;
            bool alive = true;
            for (int ti = 0; alive && ti < my_tiles; ++ti) {
                const int acc = T::ONE ? 0 : ti & 1;
                const uint32_t acc_ph = T::ONE ? (uint32_t)ti & 1u : (uint32_t)(ti >> 1) & 1u;
                if (!wait_one(&acc_empty[acc], acc_ph ^ 1u, abort_flag, p.status, DEV_TIMEOUT_MMA)) break;
                for (int kt = 0; kt < p.ktiles; ++kt) {
                    if ((kt & 3) == 0 && !wait_one(&sf_full[set], sf_ph, abort_flag, p.status, DEV_TIMEOUT_MMA)) { alive = false; break; }
                    if (!wait_one(&full[s], ph, abort_flag, p.status, DEV_TIMEOUT_MMA)) { alive = false; break; }
                    tc_fence_after();
                    const uint32_t sf = tmem_base + sf_col<BN>(set);
                    const uint32_t idesc = idesc0 | idesc_scale_byte(kt & 3);
                    const uint64_t adesc = adesc0 + (uint32_t)((s * A_BYTES) >> 4), bdesc = bdesc0 + (uint32_t)((s * T::B_SLOT) >> 4);
#pragma unroll
                    for (int kb = 0; kb < 4; kb++)
                        tc_mma2_mxf8(tmem_base + acc_col(acc), adesc + (uint32_t)(kb * 2), bdesc + (uint32_t)(kb * 2), idesc, sf, sf + 4u, (kt | kb) != 0 ? 1u : 0u);
                    // slots and sets are reported free only where they will be filled again: nothing arrives at the peer after its last wait
                    if (left > S) tc_commit2(&freed[s]);
                    --left;
                    if (++s == S) { s = 0; ph ^= 1; }
                    if ((kt & 3) == 3 || kt == p.ktiles - 1) {
                        if (gleft > SF_SETS) tc_commit2(&sf_free[set]);
                        --gleft;
                        if (++set == SF_SETS) { set = 0; sf_ph ^= 1; }
                    }
                }
                if (alive) tc_commit2(&acc_full[acc]);
            }
        }
        __syncwarp();
    } else if (warp >= SCALE_WARP0 && warp < EPI_WARP0) {
        // ---------------- scale words ----------------
        const uint32_t quarter = *tmem_slot + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t ready = mapa_shared(smem_u32(sf_full), 0);
        uint32_t next[12];
        auto fetch = [&](int tile, int g) {
            int tm, tn;
            p.order.at(tile, &tm, &tn);
            const int m0 = tm * 256 + (int)crank * 128 + lane, n0 = tn * BN + lane;
            const uint32_t *sa = p.sa + (int64_t)g * p.M, *sb = p.sb + (int64_t)g * p.N;
#pragma unroll
            for (int i = 0; i < 4; i++) next[i] = m0 + 32 * i < p.M ? __ldg(sa + m0 + 32 * i) : 0u;
#pragma unroll
            for (int i = 0; i < 8; i++) next[4 + i] = 32 * i + lane < BN && n0 + 32 * i < p.N ? __ldg(sb + n0 + 32 * i) : 0u;
        };
        int set = 0;
        uint32_t ph = 1;
        bool alive = true;
        if (my_tiles > 0) fetch(pair, 0);
        for (int tile = pair; alive && tile < total; tile += npairs) {
            for (int g = 0; g < groups; ++g) {
                if (!wait_warp(&sf_free[set], ph, abort_flag, p.status, DEV_TIMEOUT_EPILOGUE)) { alive = false; break; }
                tc_fence_after();
                tc_st_32x32b<4>(quarter + sf_col<BN>(set), next);
                tc_st_32x32b<8>(quarter + sf_col<BN>(set) + 4u, next + 4);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(ready + (uint32_t)set * 8u);
                if (++set == SF_SETS) { set = 0; ph ^= 1; }
                if (g + 1 < groups) fetch(tile, g + 1);
                else if (tile + npairs < total) fetch(tile + npairs, 0);
            }
        }
    } else if (warp >= EPI_WARP0) {
        // ---------------- epilogue ----------------
        const int q = warp & 3, part = (warp - EPI_WARP0) >> 2;
        constexpr int REST = BN - 128;
        const int cols = part == 0 ? 128 : REST;
        const uint32_t tmem_base = *tmem_slot;
        uint8_t *own = smem + S * T::STAGE_BYTES + (warp - EPI_WARP0) * T::WARP_BYTES;
        uint4 *stage = reinterpret_cast<uint4 *>(own);
        // 32 columns before: part 1, !WHOLE.  Known to be shared memory in every epilogue: 11844 x 15043 x 116 159 -> 150 us.
        float4 *bias = reinterpret_cast<float4 *>(smem_raw + (-smem_u32(smem_raw) & 1023u) + S * T::STAGE_BYTES + (warp - EPI_WARP0) * T::WARP_BYTES + T::WARP_BYTES - 512);
        // bias of four columns a lane (and of one of the 32 before), on its way while the tile before is stored: as it lies, for a conversion would wait for it
        uint32_t next[5];
        auto fetch = [&](int tile) {
            int tm, tn;
            p.order.at(tile, &tm, &tn);
            const int n = tn * BN + part * 128 + 4 * lane;
#pragma unroll
            for (int i = 0; i < 4; i++) next[i] = bias_bits(p.bias, p.bias_type, n + i < p.N ? n + i : p.N - 1);      // past the end: not stored
            if (!WHOLE && part == 1) next[4] = bias_bits(p.bias, p.bias_type, n - 3 * lane - 32 < p.N ? n - 3 * lane - 32 : p.N - 1);
        };
        if (p.bias && my_tiles > 0) fetch(pair);
        int ti = 0;
        for (int tile = pair; tile < total; tile += npairs, ++ti) {
            const int acc = T::ONE ? 0 : ti & 1;
            int tm, tn;
            p.order.at(tile, &tm, &tn);
            if (p.bias) {
                __syncwarp();
                bias[lane] = make_float4(bias_float(next[0], p.bias_type), bias_float(next[1], p.bias_type), bias_float(next[2], p.bias_type), bias_float(next[3], p.bias_type));
                if (!WHOLE && part == 1) reinterpret_cast<float *>(bias)[lane - 32] = bias_float(next[4], p.bias_type);
                __syncwarp();
                if (tile + npairs < total) fetch(tile + npairs);
            }
            if (!wait_warp(&acc_full[acc], T::ONE ? (uint32_t)ti & 1u : (uint32_t)(ti >> 1) & 1u, abort_flag, p.status, DEV_TIMEOUT_EPILOGUE)) break;
            tc_fence_after();
            const uint32_t empty = mapa_shared(smem_u32(&acc_empty[acc]), 0);
            auto release = [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(empty);
            };
            const uint32_t tacc = tmem_base + ((uint32_t)(q * 32) << 16) + acc_col(acc) + (uint32_t)(part * 128);
            const int64_t row0 = (int64_t)tm * 256 + (int)crank * 128 + q * 32;
            const int n0 = tn * BN + part * 128;
            auto store = [&](auto type) {
                constexpr int TYPE = decltype(type)::value;
                constexpr bool HOLD = T::ONE && TYPE != T_F32;
                if (p.bias) store_columns<TYPE, true, WHOLE, HOLD>(tacc, row0, n0, cols, part, stage, bias, p, release);
                else store_columns<TYPE, false, WHOLE, HOLD>(tacc, row0, n0, cols, part, stage, bias, p, release);
            };
            if (p.out_type == T_F16) store(std::integral_constant<int, T_F16>());
            else if (p.out_type == T_BF16) store(std::integral_constant<int, T_BF16>());
            else store(std::integral_constant<int, T_F32>());
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync_all();      // the peer's shared and tensor memory stay until the leader's last MMA is done: the epilogues have seen its accumulator full
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc2(*tmem_slot, TMEM_COLS);
    }
}

}  // namespace

#define VNM_FP8_PAIR(X) X(192, true) X(224, true) X(240, true) X(256, true) X(192, false) X(224, false) X(240, false) X(256, false)

cudaError_t fp8_pair_init(int sms, int *clusters)
{
    cudaError_t e;
#define VNM_ATTR(BN, WHOLE) \
    if ((e = cudaFuncSetAttribute(fp8_pair_kernel<BN, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Fp8Pair<BN, WHOLE>::SMEM_BYTES)) != cudaSuccess) return e;
    VNM_FP8_PAIR(VNM_ATTR)
#undef VNM_ATTR
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(sms & ~1));
    lc.blockDim = dim3(NUM_THREADS);
    lc.dynamicSmemBytes = Fp8Pair<256, true>::SMEM_BYTES;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(clusters, fp8_pair_kernel<256, true>, &lc);
    if (e != cudaSuccess) { (void)cudaGetLastError(); *clusters = 0; }
    return cudaSuccess;
}

// The cost of a call, us: a start, waves of tiles (between the whole number that the last one makes and the fraction that the power limit sees), and the last
// tile's epilogue.  A tile takes its k-tiles' time or its epilogue's, whichever is longer (a smooth maximum), or with one accumulator both.  Both
// kernels' costs were fitted to steady calls on inputs that change, 802 shapes of 1 to 16384 x 8 to 36864 x 64 to 12288, odd ones and round ones, with and without a bias,
// fp16 and fp32 results, for the choice that they make: over 366 others the plan that is taken was measured at 1.014 of the fastest one's time on average, 1.29 at most (few rows,
// few columns or few k: 4527 x 56 x 560 7.5 us against 5.8, 10 x 21128 x 5102 29.7 against 23.1, where one CTA a tile would do).
float fp8_pair_config(int M, int N, int K, bool wide_out, bool whole, bool bias, const Fp8Device &device, Fp8Plan *plan)
{
    const int clusters = device.clusters;
    if (clusters <= 0) return -1.0f;
    static const int widths[4] = {192, 224, 240, 256};
    static const float ktile[4] = {0.352f, 0.380f, 0.388f, 0.410f};
    const int64_t mt = ((int64_t)M + 255) / 256;
    const float kt = (float)(((int64_t)K + 127) / 128);
    const float edge = 1.69f + (wide_out ? 1.20f : 0.0f) + (whole ? 0.0f : 0.98f) + (bias ? 0.58f : 0.0f);
    float best = -1.0f;
    for (int i = 0; i < 4; i++) {
        const int w = widths[i];
        const int64_t nt = ((int64_t)N + w - 1) / w, tiles = mt * nt;
        if (tiles > INT32_MAX / 2) continue;
        const float waves = 0.715f * (float)((tiles + clusters - 1) / clusters) + 0.285f * (float)tiles / (float)clusters;
        const float mma = kt * ktile[i], out = edge * (float)w / 240.0f;
        const float one = w == 256 ? mma + 1.12f * out : powf(powf(mma, 1.1f) + powf(out, 1.1f), 1.0f / 1.1f);
        const float us = 3.19f + waves * one + 0.26f * out;
        if (best < 0.0f || us < best) {
            best = us;
            plan->bn = w;
            plan->grid = 2 * (int)(tiles < clusters ? tiles : clusters);
        }
    }
    plan->split = 1;
    return best;
}

cudaError_t launch_fp8_pair(const Fp8Plan &plan, const CUtensorMap &map_a, const CUtensorMap &map_b, const Fp8MatmulParams &p, cudaStream_t stream)
{
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)plan.grid);
    lc.blockDim = dim3(NUM_THREADS);
    lc.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1] = early_launch();
    lc.attrs = attr;
    lc.numAttrs = 2;
#define VNM_LAUNCH(BN, WHOLE)                                      \
    if (plan.bn == BN && (p.whole_pieces != 0) == WHOLE) {         \
        lc.dynamicSmemBytes = Fp8Pair<BN, WHOLE>::SMEM_BYTES;      \
        return cudaLaunchKernelEx(&lc, fp8_pair_kernel<BN, WHOLE>, map_a, map_b, p); \
    }
    VNM_FP8_PAIR(VNM_LAUNCH)
#undef VNM_LAUNCH
    return cudaErrorInvalidValue;
}

}  // namespace vnm
