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
#include "vnm_fp8.h"

#include <cuda_bf16.h>

#include <type_traits>

namespace vnm {

namespace {

constexpr int A_BYTES = 128 * 128;
constexpr int NUM_THREADS = 512;
constexpr int SCALE_WARP0 = 4, EPI_WARP0 = 8;
constexpr int TMEM_COLS = 512;
constexpr int SF_SETS = 2;

template <int BN>
struct Fp8Pair {
    static_assert(BN % 16 == 0 && BN <= 256 && BN > 128, "accumulator columns");
    static constexpr bool ONE = BN > 240;                // one accumulator
    static constexpr int HALF_N = BN / 2;
    static constexpr int B_BYTES = HALF_N * 128;
    static constexpr int B_SLOT = (B_BYTES + 1023) / 1024 * 1024;
    static constexpr int STAGE_BYTES = A_BYTES + B_SLOT;
    static constexpr int STAGES = 7;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 512 + 1024;
    static_assert(SMEM_BYTES <= 227 * 1024, "shared memory per CTA");
    static_assert((2 * STAGES + 2 * SF_SETS + 4) * 8 + 8 <= 512, "barriers");
};
__device__ __forceinline__ uint32_t acc_col(int a) { return (uint32_t)a * 256u; }
template <int BN>
__device__ __forceinline__ uint32_t sf_col(int set) { return Fp8Pair<BN>::ONE ? 256u + 16u * (uint32_t)set : 240u + 256u * (uint32_t)set; }

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

// ---- epilogue of one warp: 32 accumulator lanes (rows of the result) x up to 128 columns, straight from tensor memory ----
// Read in fragment order: thread t holds columns 2 (t % 4), + 1 of every eight for lanes t / 4 and t / 4 + 8 of a 16-lane group.  Two 4 x 4 exchanges inside a
// quad give each thread 16 neighbouring columns of a row in 16 bits, so that a store instruction writes 128 contiguous bytes of eight rows; 32-bit
// results leave as pairs, a sector a quad.
__device__ __forceinline__ void quad_swap(uint32_t &a, uint32_t &b, bool up, int mask)
{
    const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? a : b, mask);
    if (up) a = got; else b = got;
}
__device__ __forceinline__ float2 bias_pair(const void *bias, int type, int n, int N)
{
    float2 r;
    if (type == T_F32) {
        const float *b = reinterpret_cast<const float *>(bias);
        r.x = n < N ? __ldg(b + n) : 0.0f;
        r.y = n + 1 < N ? __ldg(b + n + 1) : 0.0f;
    } else {
        const unsigned short *b = reinterpret_cast<const unsigned short *>(bias);
        const unsigned short x = n < N ? __ldg(b + n) : (unsigned short)0, y = n + 1 < N ? __ldg(b + n + 1) : (unsigned short)0;
        if (type == T_F16) r = make_float2(__half2float(__ushort_as_half(x)), __half2float(__ushort_as_half(y)));
        else r = make_float2(__uint_as_float((uint32_t)x << 16), __uint_as_float((uint32_t)y << 16));
    }
    return r;
}
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

template <int TYPE, int COLS, typename Release>
__device__ __forceinline__ void store_columns(uint32_t tacc, int64_t row0, int n0, const Fp8MatmulParams &p, Release release)
{
    const int lane = threadIdx.x & 31, quad = lane & 3, w = lane >> 2;
    const bool odd = (lane & 1) != 0, upper = (lane & 2) != 0;
    const int64_t size = TYPE == T_F32 ? 4 : 2;
    const uintptr_t base = reinterpret_cast<uintptr_t>(p.out);
    const bool wide = ((base | (uintptr_t)(p.ldo * size)) & 31) == 0, half_wide = ((base | (uintptr_t)(p.ldo * size)) & 15) == 0, pairs = ((base | (uintptr_t)(p.ldo * size)) & (2 * size - 1)) == 0;
    constexpr int CHUNKS = (COLS + 63) / 64;
#pragma unroll 1
    for (int k = 0; k < CHUNKS; k++) {
        const int cols = COLS - 64 * k;                     // a last chunk of fewer reads on into columns that it does not store
        const int c0 = n0 + 64 * k;
#pragma unroll
        for (int g = 0; g < 2; g++) {
            uint32_t v[32];
            tc_ld_16x256b(tacc + ((uint32_t)(16 * g) << 16) + (uint32_t)(64 * k), v);
            tc_wait_ld();
            if (k == CHUNKS - 1 && g == 1) release();
            if (p.bias) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float2 b = bias_pair(p.bias, p.bias_type, c0 + 8 * j + 2 * quad, p.N);
                    v[4 * j] = __float_as_uint(__uint_as_float(v[4 * j]) + b.x);
                    v[4 * j + 1] = __float_as_uint(__uint_as_float(v[4 * j + 1]) + b.y);
                    v[4 * j + 2] = __float_as_uint(__uint_as_float(v[4 * j + 2]) + b.x);
                    v[4 * j + 3] = __float_as_uint(__uint_as_float(v[4 * j + 3]) + b.y);
                }
            }
            if constexpr (TYPE == T_F32) {
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const int64_t row = row0 + 16 * g + 8 * r + w;
                    float *dst = reinterpret_cast<float *>(p.out) + row * p.ldo;
                    if (row < p.M) {
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const int n = c0 + 8 * j + 2 * quad;
                            const float x = __uint_as_float(v[4 * j + 2 * r]), y = __uint_as_float(v[4 * j + 2 * r + 1]);
                            if (8 * j >= cols) break;
                            if (pairs && n + 1 < p.N) {
                                *reinterpret_cast<float2 *>(dst + n) = make_float2(x, y);
                            } else {
                                if (n < p.N) dst[n] = x;
                                if (n + 1 < p.N) dst[n + 1] = y;
                            }
                        }
                    }
                }
            } else {
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    uint32_t x[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) x[j] = pack16<TYPE>(__uint_as_float(v[4 * j + 2 * r]), __uint_as_float(v[4 * j + 2 * r + 1]));
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        quad_swap(x[0 + h], x[2 + h], odd, 1);
                        quad_swap(x[4 + h], x[6 + h], odd, 1);
                        quad_swap(x[0 + h], x[4 + h], upper, 2);
                        quad_swap(x[2 + h], x[6 + h], upper, 2);
                    }
                    const uint32_t o[8] = {x[0], x[2], x[4], x[6], x[1], x[3], x[5], x[7]};
                    const int64_t row = row0 + 16 * g + 8 * r + w;
                    const int n = c0 + 16 * quad, rest = p.N - n;
                    if (row >= p.M || rest <= 0 || 16 * quad >= cols) continue;
                    uint16_t *dst = reinterpret_cast<uint16_t *>(p.out) + row * p.ldo + n;
                    if (wide && rest >= 16) {
                        st_global_v8(dst, o);
                    } else if (half_wide && rest >= 16) {
                        *reinterpret_cast<uint4 *>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
                        *reinterpret_cast<uint4 *>(dst + 8) = make_uint4(o[4], o[5], o[6], o[7]);
                    } else if (pairs) {
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            if (2 * i + 1 < rest) *reinterpret_cast<uint32_t *>(dst + 2 * i) = o[i];
                            else if (2 * i < rest) dst[2 * i] = (uint16_t)o[i];
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            if (2 * i < rest) dst[2 * i] = (uint16_t)o[i];
                            if (2 * i + 1 < rest) dst[2 * i + 1] = (uint16_t)(o[i] >> 16);
                        }
                    }
                }
            }
        }
    }
}

// Warps: 0 loads A, 1 loads B, 2 issues the MMAs (leader), 3 owns tensor memory, 4..7 scale words, 8..15 epilogue: columns 0..127 and the rest.
template <int BN>
__global__ void __launch_bounds__(NUM_THREADS, 1) fp8_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Fp8MatmulParams p)
{
    using T = Fp8Pair<BN>;
    constexpr int S = T::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *a_ring = smem, *b_ring = smem + S * A_BYTES;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + S * T::STAGE_BYTES);
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
    grid_dependency_wait();
    if (warp == 3) {
        tmem_alloc2(tmem_slot, TMEM_COLS);
        tmem_relinquish2();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                 // both CTAs' barriers exist before anyone arrives on them remotely
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    grid_launch_dependents();

    if (warp < 2) {
        // ---------------- loads ----------------
        if (elect_one()) {
            const bool is_a = warp == 0;
            const CUtensorMap *map = is_a ? &map_a : &map_b;
            uint8_t *ring = is_a ? a_ring : b_ring;
            const int slot = is_a ? A_BYTES : T::B_SLOT;
            const uint32_t bytes = is_a ? A_BYTES : T::B_BYTES;
            const uint64_t policy = (p.band >= 0) == is_a ? L2_EVICT_LAST : L2_EVICT_NORMAL;   // the banded operand is read again soon
            const uint32_t report = mapa_shared(smem_u32(full), 0);
            tma_prefetch_desc(map);
            int s = 0, it = 0;
            uint32_t ph = 1;
            bool alive = true;
            for (int tile = pair; alive && tile < total; tile += npairs) {
                int tm, tn;
                tile_coords(tile, p.mt, p.nt, p.band, &tm, &tn);
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
        const uint32_t quarter = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t ready = mapa_shared(smem_u32(sf_full), 0);
        uint32_t next[12];
        auto fetch = [&](int tile, int g) {
            int tm, tn;
            tile_coords(tile, p.mt, p.nt, p.band, &tm, &tn);
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
        int ti = 0;
        for (int tile = pair; tile < total; tile += npairs, ++ti) {
            const int acc = T::ONE ? 0 : ti & 1;
            int tm, tn;
            tile_coords(tile, p.mt, p.nt, p.band, &tm, &tn);
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
                if (part == 0) store_columns<TYPE, 128>(tacc, row0, n0, p, release);
                else store_columns<TYPE, BN - 128>(tacc, row0, n0, p, release);
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
        tmem_dealloc2(tmem_base, TMEM_COLS);
    }
}

int g_clusters = 0;          // co-resident clusters of two CTAs on this device (0 = not queried yet)

}  // namespace

#define VNM_FP8_PAIR(X) X(192) X(224) X(240) X(256)

cudaError_t fp8_pair_init()
{
    cudaError_t e;
#define VNM_ATTR(BN) \
    if ((e = cudaFuncSetAttribute(fp8_pair_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Fp8Pair<BN>::SMEM_BYTES)) != cudaSuccess) return e;
    VNM_FP8_PAIR(VNM_ATTR)
#undef VNM_ATTR
    int dev = 0, sms = 0;
    if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(sms & ~1));
    lc.blockDim = dim3(NUM_THREADS);
    lc.dynamicSmemBytes = Fp8Pair<256>::SMEM_BYTES;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
    int clusters = 0;
    e = cudaOccupancyMaxActiveClusters(&clusters, fp8_pair_kernel<256>, &lc);
    if (e != cudaSuccess) { (void)cudaGetLastError(); clusters = 0; }
    g_clusters = clusters;
    return cudaSuccess;
}

float fp8_pair_config(int M, int N, int K, Fp8Plan *plan)
{
    if (g_clusters <= 0) return -1.0f;
    static const int widths[4] = {256, 240, 224, 192};
    const int64_t mt = ((int64_t)M + 255) / 256;
    float best = -1.0f;
    for (int w : widths) {
        const int64_t nt = ((int64_t)N + w - 1) / w, tiles = mt * nt;
        if (tiles > INT32_MAX / 2) continue;
        const int64_t waves = (tiles + g_clusters - 1) / g_clusters;
        const float us = (float)waves * ((float)((K + 127) / 128) * w / 900.0f + (w == 256 ? 0.4f : 0.2f));
        if (best < 0.0f || us < best) {
            best = us;
            plan->bn = w;
            plan->grid = 2 * (int)(tiles < g_clusters ? tiles : g_clusters);
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
#define VNM_LAUNCH(BN)                                   \
    if (plan.bn == BN) {                                 \
        lc.dynamicSmemBytes = Fp8Pair<BN>::SMEM_BYTES;   \
        return cudaLaunchKernelEx(&lc, fp8_pair_kernel<BN>, map_a, map_b, p); \
    }
    VNM_FP8_PAIR(VNM_LAUNCH)
#undef VNM_LAUNCH
    return cudaErrorInvalidValue;
}

}  // namespace vnm
