// Matrix product of block-scaled 8-bit operands, one SM a tile: out[m, n] = sum over k of A[m, k] B[n, k] (+ bias[n]), with sums in fp32.
//
// tcgen05.mma kind::mxf8f6f4 multiplies every row of A and of B by a power of two for each 32 k, in the tensor core; here four such blocks in a row
// have the same scale, the byte of their block of 128 k.  So a k-tile of 128 (128 bytes, the swizzle's span) is four MMAs that read the same byte, and a word
// of four bytes a row lasts for four k-tiles.  Nothing is rescaled outside of the tensor core, and one accumulator holds the whole sum.
//
// The rows of B (a weight's output features) are the 128 lanes of a tile, the rows of A (tokens) its BN columns: a decoding step reads the weight once,
// whatever its few tokens, in tiles of 128 x 16.  Where tiles are few a cluster of CTAs splits the k-tiles of one, and the partial sums travel through distributed
// shared memory and are added in rank order, so that results are the same on every call.
//
// Warps: 0 loads B, 1 loads A (TMA boxes of 128 bytes, 128-byte swizzle), 2 issues the MMAs, 3 owns tensor memory, 4..7 bring the scale words into tensor
// memory (coalesced loads, one register store for each 32 rows, every warp its quarter of the lanes: the tensor core wants four copies) and are the epilogue.
// Every wait is bounded.
#include "vnm_fp8.h"

#include <cuda_bf16.h>

namespace vnm {

namespace {

constexpr int W_TILE_BYTES = 128 * 128;   // rows of B
constexpr int SMALL_THREADS = 256;
constexpr int EPI_WARP0 = 4;

template <int BN>
struct Fp8Small {
    static constexpr int X_BYTES = BN * 128;
    static constexpr int STAGE_BYTES = W_TILE_BYTES + X_BYTES;
    static constexpr int STAGES = 104 * 1024 / STAGE_BYTES;
    static constexpr int RED_BYTES = (BN + 8) * 128 * 4;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 256 + 1024;
    static constexpr int SFB_COLS = (BN + 31) / 32;
    static constexpr int SF_SETS = 2;
    static constexpr int SF_COL = BN < 32 ? 32 : BN;              // the epilogue reads 32 columns at a time
    static constexpr int SF_WIDTH = 8;                            // four columns for the 128 rows of B, up to four for the rows of A
    static constexpr int TMEM_COLS = SF_COL + SF_SETS * SF_WIDTH <= 64 ? 64 : SF_COL + SF_SETS * SF_WIDTH <= 128 ? 128 : 256;
    static_assert(2 * (SMEM_BYTES + 1024) <= 227 * 1024, "two CTAs an SM");
    static_assert(RED_BYTES <= STAGES * STAGE_BYTES, "partial sums lie in the rings");
};

__device__ __forceinline__ uint32_t cluster_ctarank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t mapa_shared(uint32_t saddr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

__device__ __forceinline__ float bias_at(const void *bias, int type, int64_t n)
{
    if (!bias) return 0.0f;
    if (type == T_F16) return __half2float(reinterpret_cast<const __half *>(bias)[n]);
    if (type == T_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(bias)[n]);
    return reinterpret_cast<const float *>(bias)[n];
}
__device__ __forceinline__ uint32_t pack2(float a, float b, int type)
{
    if (type == T_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void store_one(const Fp8MatmulParams &p, int64_t m, int64_t n, float v)
{
    const int64_t at = m * p.ldo + n;
    if (p.out_type == T_F32) reinterpret_cast<float *>(p.out)[at] = v;
    else if (p.out_type == T_F16) reinterpret_cast<__half *>(p.out)[at] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(v);
}

template <int BN>
__global__ void __launch_bounds__(SMALL_THREADS, 2) fp8_small_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Fp8MatmulParams p)
{
    using T = Fp8Small<BN>;
    constexpr int S = T::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
    uint8_t *w_ring = smem, *x_ring = smem + S * W_TILE_BYTES;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + S * T::STAGE_BYTES);
    uint64_t *freed = full + S;
    uint64_t *sf_full = freed + S, *sf_free = sf_full + T::SF_SETS;
    uint64_t *acc_full = sf_free + T::SF_SETS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_full + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *fills = reinterpret_cast<int *>(tmem_slot + 2);
    float *red = reinterpret_cast<float *>(smem);
    static_assert((2 * S + 2 * T::SF_SETS + 1) * 8 + 12 <= 256 && T::X_BYTES % 1024 == 0, "shared-memory plan");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = p.split;
    const uint32_t rank = split > 1 ? cluster_ctarank() : 0u;
    const int tile = (int)blockIdx.x / split;
    const int tn = tile / p.mt, tm = tile - tn * p.mt;    // the tiles of one weight tile run side by side
    const int n0 = tn * 128, m0 = tm * BN;
    const int k0 = (int)((int64_t)p.ktiles * rank / split), k1 = (int)((int64_t)p.ktiles * (rank + 1) / split);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(&full[s], 2);
            mbar_init(&freed[s], 1);
        }
        for (int s = 0; s < T::SF_SETS; s++) {
            mbar_init(&sf_full[s], 4);
            mbar_init(&sf_free[s], 1);
        }
        mbar_init(acc_full, 1);
        *abort_flag = 0;
        *fills = 0;
        fence_barrier_init();
    }
    __syncthreads();
    grid_dependency_wait();
    // The loads begin at once; whoever uses tensor memory meets behind its allocation.
    uint32_t tmem_base = 0;
    if (warp >= 2) {
        if (warp == 3) {
            tmem_alloc(tmem_slot, T::TMEM_COLS);
            tmem_relinquish();
        }
        tc_fence_before();
        named_barrier_sync(1, SMALL_THREADS - 64);
        tc_fence_after();
        tmem_base = *tmem_slot;
        grid_launch_dependents();
    }

    if (warp < 2) {
        // ---------------- loads: warp 0 rows of B, warp 1 rows of A ----------------
        if (elect_one()) {
            const CUtensorMap *map = warp == 0 ? &map_b : &map_a;
            uint8_t *ring = warp == 0 ? w_ring : x_ring;
            const int bytes = warp == 0 ? W_TILE_BYTES : T::X_BYTES, row = warp == 0 ? n0 : m0;
            tma_prefetch_desc(map);
            int s = 0;
            uint32_t ph = 1;
            int kt = k0;
            for (; kt < k1; ++kt) {
                if (!wait_quiet(&freed[s], ph, abort_flag, p.status, DEV_TIMEOUT_PRODUCER)) break;
                mbar_arrive_expect_tx(&full[s], (uint32_t)bytes);
                tma_load_2d(ring + s * bytes, map, kt * 128, row, &full[s]);
                if (++s == S) { s = 0; ph ^= 1; }
            }
            atomicMax(fills, kt - k0);
        }
        __syncwarp();
    } else if (warp == 2) {
        // ---------------- MMA issuer ----------------
        if (elect_one()) {
            const uint32_t idesc0 = make_idesc_mxf8(128, BN, p.b_f8, p.a_f8);
            const uint64_t wdesc0 = make_smem_desc(smem_u32(w_ring), 16, 1024, 2), xdesc0 = make_smem_desc(smem_u32(x_ring), 16, 1024, 2);
            int s = 0;
            uint32_t ph = 0;
            for (int kt = k0; kt < k1; ++kt) {
                const int g = (kt >> 2) - (k0 >> 2), set = g % T::SF_SETS;
                if ((kt == k0 || (kt & 3) == 0) && !wait_one(&sf_full[set], (uint32_t)(g / T::SF_SETS) & 1u, abort_flag, p.status, DEV_TIMEOUT_MMA)) break;
                if (!wait_one(&full[s], ph, abort_flag, p.status, DEV_TIMEOUT_MMA)) break;
                tc_fence_after();
                const uint32_t sf = tmem_base + (uint32_t)(T::SF_COL + set * T::SF_WIDTH);
                const uint32_t idesc = idesc0 | idesc_scale_byte(kt & 3);
                const uint64_t wdesc = wdesc0 + (uint32_t)((s * W_TILE_BYTES) >> 4), xdesc = xdesc0 + (uint32_t)((s * T::X_BYTES) >> 4);
#pragma unroll
                for (int kb = 0; kb < 4; kb++)
                    tc_mma_mxf8(tmem_base, wdesc + (uint32_t)(kb * 2), xdesc + (uint32_t)(kb * 2), idesc, sf, sf + 4u, (kt != k0 || kb != 0) ? 1u : 0u);
                tc_commit(&freed[s]);
                if ((kt & 3) == 3) tc_commit(&sf_free[set]);
                if (++s == S) { s = 0; ph ^= 1; }
            }
            tc_commit(acc_full);   // on an abort, too: nothing of this thread is in flight when the CTA leaves
        }
        __syncwarp();
    } else if (warp >= EPI_WARP0) {
        // ---------------- scale words ----------------
        const int q = warp & 3;
        const uint32_t quarter = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)T::SF_COL;
        auto word = [&](const uint32_t *scales, int rows, int row, int g) -> uint32_t { return row < rows ? __ldg(scales + (int64_t)g * rows + row) : 0u; };
        uint32_t next[8] = {};
        auto fetch = [&](int g) {
#pragma unroll
            for (int i = 0; i < 4; i++) next[i] = word(p.sb, p.N, n0 + 32 * i + lane, g);
#pragma unroll
            for (int i = 0; i < T::SFB_COLS; i++) next[4 + i] = 32 * i + lane < BN ? word(p.sa, p.M, m0 + 32 * i + lane, g) : 0u;
        };
        const int g0 = k0 >> 2, g1 = k1 > k0 ? ((k1 - 1) >> 2) + 1 : g0;
        if (g0 < g1) fetch(g0);
        for (int g = g0; g < g1; ++g) {
            const int set = (g - g0) % T::SF_SETS;
            if (!wait_warp(&sf_free[set], ((uint32_t)((g - g0) / T::SF_SETS) & 1u) ^ 1u, abort_flag, p.status, DEV_TIMEOUT_EPILOGUE)) break;
            tc_fence_after();
            tc_st_32x32b<4>(quarter + (uint32_t)(set * T::SF_WIDTH), next);
            tc_st_32x32b<T::SFB_COLS>(quarter + (uint32_t)(set * T::SF_WIDTH + 4), next + 4);
            if (g + 1 < g1) fetch(g + 1);
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sf_full[set]);
        }
    }

    if (split == 1) {
        if (warp >= EPI_WARP0) {
            const int q = warp & 3;
            if (wait_warp(acc_full, 0u, abort_flag, p.status, DEV_TIMEOUT_EPILOGUE) && *abort_flag == 0) {
                tc_fence_after();
                const int n = n0 + q * 32 + lane;
                const float bias = n < p.N ? bias_at(p.bias, p.bias_type, n) : 0.0f;
                // 16 bits: neighbouring lanes exchange, so that each stores pairs of features of every other token
                const bool pairs = p.out_type != T_F32 && (p.ldo & 1) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 3) == 0;
#pragma unroll 1
                for (int c0 = 0; c0 < BN && m0 + c0 < p.M; c0 += 32) {
                    uint32_t v[32];
                    tc_ld_32x32b_x32(tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)c0, v);
                    tc_wait_ld();
                    const int count = BN - c0 < 32 ? BN - c0 : 32;
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        if (i >= count) break;
                        const float a = __uint_as_float(v[i]) + bias, b = __uint_as_float(v[i + 1]) + bias;
                        if (pairs) {
                            const bool up = (lane & 1) != 0;
                            const float got = __shfl_xor_sync(0xffffffffu, up ? a : b, 1);
                            const int m = m0 + c0 + i + (up ? 1 : 0);
                            const int nn = n & ~1;
                            if (m < p.M) {
                                const uint32_t w = up ? pack2(got, b, p.out_type) : pack2(a, got, p.out_type);
                                uint16_t *dst = reinterpret_cast<uint16_t *>(p.out) + (int64_t)m * p.ldo + nn;
                                if (nn + 1 < p.N) *reinterpret_cast<uint32_t *>(dst) = w;
                                else if (nn < p.N) *dst = (uint16_t)w;
                            }
                        } else if (n < p.N) {
                            if (m0 + c0 + i < p.M) store_one(p, m0 + c0 + i, n, a);
                            if (m0 + c0 + i + 1 < p.M) store_one(p, m0 + c0 + i + 1, n, b);
                        }
                    }
                }
            }
        }
    } else {
        // ---------------- split over K: rank d adds up columns [d * share, (d + 1) * share) of all ranks ----------------
        // A CTA whose waits ran out still takes part in the barriers; its sums are meaningless and the status word says so.
        const int share = (BN + split - 1) / split;
        if (warp >= EPI_WARP0) {
            (void)wait_warp(acc_full, 0u, abort_flag, p.status, DEV_TIMEOUT_EPILOGUE);
            tc_fence_after();
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();                  // every MMA of every rank is done: the rings are free
        if (warp >= EPI_WARP0) {
            const int q = warp & 3;
            const uint32_t red0 = smem_u32(red) + (uint32_t)(q * 32 + lane) * 4u;
            for (int c0 = 0; c0 < BN; c0 += 8) {
                uint32_t v[8];
                tc_ld_32x32b_x8(tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)c0, v);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int m = c0 + i, d = m / share;
                    st_cluster(mapa_shared(red0, (uint32_t)d) + (uint32_t)(((int)rank * share + m - d * share) * 128 * 4), v[i]);
                }
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();                  // all partial sums have arrived, and nobody writes here any more
        const int first = (int)rank * share, count = first + share <= BN ? share : (BN > first ? BN - first : 0);
        for (int e = threadIdx.x; e < count * 128; e += SMALL_THREADS) {
            const int m = e >> 7, r = e & 127;
            float sum = 0.0f;
            for (int d = 0; d < split; d++) sum += red[(d * share + m) * 128 + r];
            const int row = m0 + first + m, col = n0 + r;
            if (row < p.M && col < p.N) store_one(p, row, col, sum + bias_at(p.bias, p.bias_type, col));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0 && *abort_flag) drain_ring(full, S, *fills, p.status);
    __syncthreads();
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem_base, T::TMEM_COLS);
    }
}

}  // namespace

#define VNM_FP8_SMALL(X) X(16) X(32) X(64) X(128)

cudaError_t fp8_small_init()
{
    cudaError_t e;
#define VNM_ATTR(BN) \
    if ((e = cudaFuncSetAttribute(fp8_small_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Fp8Small<BN>::SMEM_BYTES)) != cudaSuccess) return e;
    VNM_FP8_SMALL(VNM_ATTR)
#undef VNM_ATTR
    return cudaSuccess;
}

// The cost of a call, us: a start, then a CTA's k-tiles (one CTA an SM, or two that share it) or the operands' bytes, whichever takes longer, its epilogue, and the exchange
// of partial sums.  See fp8_pair_config for what they were fitted to.  (512 x 4096 x 4096: 128 x 64 16.2 us, pairs 12.6;  16 x 36864 x 12288: 128 x 16 68.2, all of it
// the weight's bytes;  128 x 4096 x 1024: 128 x 32 6.2, pairs 6.4;  8 x 1024 x 1024: 128 x 16 alone 4.6, split by eight 3.8.)
float fp8_small_config(int M, int N, int ktiles, bool wide_out, const Fp8Device &device, Fp8Plan *plan)
{
    struct Cost { float start, kt1, kt2, out, split, bytes; };
    static const Cost cost[4] = {{1.75f, 0.189f, 0.554f, 1.93f, 0.51f, 0.094f}, {1.83f, 0.204f, 0.492f, 2.53f, 0.54f, 0.084f}, {2.46f, 0.257f, 0.496f, 3.95f, 0.21f, 0.077f},
                                 {5.28f, 0.399f, 0.760f, 2.85f, 1.34f, 0.118f}};
    const int64_t nt = ((int64_t)N + 127) / 128;
    const int sms = device.sms;
    float best = -1.0f;
    for (int i = 0; i < 4; i++) {
        const int bn = 16 << i;
        if (i > 0 && bn >= 2 * (int64_t)M) break;
        const int64_t tiles = ((int64_t)M + bn - 1) / bn * nt;
        if (tiles > INT32_MAX / 8) continue;
        const float mem = (float)tiles * (float)ktiles * (float)(128 + bn) * 128e-6f * cost[i].bytes;
        for (int split = 1; split <= 8 && split <= ktiles; split *= 2) {
            const int64_t ctas = tiles * split;
            if (split > 1 && ctas > 8 * sms) break;
            const int64_t waves = (ctas + 2 * sms - 1) / (2 * sms);
            const float per = (float)((ktiles + split - 1) / split);
            const float work = ctas <= sms ? per * cost[i].kt1 : (float)waves * per * cost[i].kt2;
            const float us = cost[i].start + (work > mem ? work : mem) + (float)waves * cost[i].out * (wide_out ? 1.6f : 1.0f) + (split > 1 ? cost[i].split : 0.0f);
            if (best < 0.0f || us < best) {
                best = us;
                plan->bn = bn;
                plan->split = split;
                plan->grid = (int)ctas;
            }
        }
    }
    return best;
}

cudaError_t launch_fp8_small(const Fp8Plan &plan, const CUtensorMap &map_a, const CUtensorMap &map_b, const Fp8MatmulParams &p, cudaStream_t stream)
{
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)plan.grid);
    lc.blockDim = dim3(SMALL_THREADS);
    lc.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0] = early_launch();
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)plan.split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    lc.attrs = attr;
    lc.numAttrs = plan.split > 1 ? 2 : 1;
#define VNM_LAUNCH(BN)                                    \
    if (plan.bn == BN) {                                  \
        lc.dynamicSmemBytes = Fp8Small<BN>::SMEM_BYTES;   \
        return cudaLaunchKernelEx(&lc, fp8_small_kernel<BN>, map_a, map_b, p); \
    }
    VNM_FP8_SMALL(VNM_LAUNCH)
#undef VNM_LAUNCH
    return cudaErrorInvalidValue;
}

}  // namespace vnm
