// mx4_gemm.cu — products of microscaled 4-bit matrices on tcgen05 (mx4.cuh): weights are the
// 128 rows of the tensor cores' tile (the lanes of TMEM), tokens its columns, so that a few
// tokens are a narrow tile, each thread has one output feature, and gate and up of a feature,
// two sums in TMEM, meet in one thread.
//
// out[t, n] = sum over k of x[t, k] w[n, k], both c * 2^s in groups of 32 along k: kind::mxf4
// multiplies codes and scales and adds in f32.  One producer thread brings stages of 256
// columns by bulk copies (the tiles lie in memory as shared memory wants them), one thread
// copies their scales to TMEM and issues the products, four warps write the results.  Where the
// tiles are fewer than the SMs, the CTAs of a cluster share a tile's columns and add their sums
// over distributed shared memory, in rank order.
#include <cooperative_groups.h>

#include "mx4_tc.cuh"

namespace cg = cooperative_groups;

namespace sg {
using namespace mx4;
using namespace tiled;

namespace {

constexpr uint32_t THREADS = 192;
constexpr uint32_t HDR = 1024;  // barriers, TMEM base, place in the experts

// A launch's shape: up to NT tokens a tile, DUAL: gate and up.
template <int NT, bool DUAL>
struct Cfg {
    static constexpr uint32_t XT = NT > 128 ? 2 : 1;                       // tiles of x a stage
    static constexpr uint32_t XROWS = NT / XT;
    static constexpr uint32_t X_BYTES = mx4_tile_bytes(XROWS);
    static constexpr uint32_t W_BYTES = MX4_TILE * (DUAL ? 2 : 1);
    static constexpr uint32_t STAGE = W_BYTES + XT * X_BYTES;
    static constexpr uint32_t FIT = (NT == 32 ? 112u * 1024 : 226u * 1024) - HDR;
    static constexpr uint32_t STAGES = FIT / STAGE < 8 ? FIT / STAGE : 8;
    static constexpr uint32_t SMEM = HDR + STAGES * STAGE;
    // TMEM columns: sums, then each stage's scales: eight a tile of 256 columns and 128 rows
    static constexpr uint32_t SUMS = NT * (DUAL ? 2 : 1), SC = 8 * ((DUAL ? 2 : 1) + XT);
    static constexpr uint32_t WANT = SUMS + STAGES * SC;
    static constexpr uint32_t COLS = WANT <= 128 ? 128 : WANT <= 256 ? 256 : 512;
    static_assert(WANT <= 512 && STAGES >= 2, "TMEM");
    static_assert((STAGES * STAGE) >= (DUAL ? 2 : 1) * 128 * (NT < 128 ? NT : 1) * 4, "partial sums");
};

// A result of feature f of row t
__device__ __forceinline__ void put(const Mx4GemmArgs &a, uint64_t t, uint32_t f, float v) {
    const uint64_t at = t * a.ldo + f;
    if (a.type == SG_F32) static_cast<float *>(a.out)[at] = v;
    else if (a.type == SG_F16) static_cast<__half *>(a.out)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(v);
}

template <int NT, bool DUAL>
__global__ void __launch_bounds__(THREADS) mx4_gemm_kernel(const __grid_constant__ Mx4GemmArgs a) {
    using C = Cfg<NT, DUAL>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t *full = reinterpret_cast<uint64_t *>(smem), *empty = full + 8, *done = empty + 8;
    uint32_t *slot = reinterpret_cast<uint32_t *>(smem + 256);
    uint32_t *where = slot + 1;  // expert, its first tile of x, valid rows, and the first row of the output
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t parts = cluster.num_blocks(), part = cluster.block_rank();
    if (blockDim.x != THREADS || dynamic_smem_size() < C::SMEM || (smem_u32(smem) & 1023u) || a.nk == 0 || parts > a.nk) {
        if (tid == 0) atomicExch(&g_dev_status, (unsigned)DEV_BAD_LAUNCH);
        return;  // (the whole grid alike)
    }
    const uint32_t tile = blockIdx.x / parts, ft = tile % a.feat_tiles, tt = tile / a.feat_tiles;

    // what this tile is: of experts, the one whose tiles of NT tokens reach past tt
    uint32_t e = 0, x_tile = tt * C::XT, rows = 0, row0 = tt * NT;
    if (a.first) {
        if (warp == 0) {
            if (lane == 0) where[2] = 0;
            __syncwarp();
            uint32_t before = 0;
            for (uint32_t base = 0; base < a.n_expert && before <= tt; base += 32) {
                const uint32_t i = base + lane;
                const uint32_t f0 = i < a.n_expert ? __ldg(a.first + i) : 0, f1 = i < a.n_expert ? __ldg(a.first + i + 1) : 0;
                const uint32_t n = (f1 - f0 + NT - 1) / NT;
                uint32_t upto = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= (uint32_t)o) upto += v;
                }
                const uint32_t from = before + upto - n;
                if (tt >= from && tt < from + n) {
                    const uint32_t r = (tt - from) * NT;
                    where[0] = i;
                    where[1] = __ldg(a.tiles + i) + (tt - from) * C::XT;
                    where[2] = min(f1 - f0 - r, (uint32_t)NT);
                    where[3] = f0 + r;
                }
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        __syncthreads();
        e = where[0], x_tile = where[1], rows = where[2], row0 = where[3];
        if (rows == 0) return;  // past the last tile: all CTAs of the cluster alike
    } else {
        rows = (uint32_t)(a.n_tok - (uint64_t)tt * NT < NT ? a.n_tok - (uint64_t)tt * NT : NT);
    }
    const uint32_t n = (rows + 15) & ~15u;  // the tile's columns: of rows past the last nothing is kept
    const uint32_t k0 = a.nk * part / parts, k1 = a.nk * (part + 1) / parts;

    if (tid == 0) {
        for (uint32_t i = 0; i < C::STAGES; i++) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        mbar_init(done, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc<1>(slot, C::COLS);
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *slot;

    bool ok = true;
    if (tid == 0) {
        const uint64_t w_at = (uint64_t)e * a.expert_bytes + (uint64_t)ft * a.nk * MX4_TILE;
        const uint64_t x_at = (uint64_t)x_tile * a.nk * C::X_BYTES;
        const uint32_t xts = C::XT == 2 && rows > 128 ? 2 : 1;
        const uint32_t bytes = C::W_BYTES + xts * C::X_BYTES;
        bool waited = false;
        uint32_t i = 0;
        for (uint32_t k = k0; k < k1 && ok; k++, i++) {
            const uint32_t s = i % C::STAGES;
            if (i >= C::STAGES) ok = mbar_wait_bounded(&empty[s], (i / C::STAGES - 1) & 1, WAIT_LIMIT_NS);
            if (!ok) break;
            uint8_t *st = smem + HDR + s * C::STAGE;
            mbar_arrive_expect_tx(&full[s], bytes);
            bulk_g2s(st, a.w + w_at + (uint64_t)k * MX4_TILE, MX4_TILE, &full[s]);
            if (DUAL) bulk_g2s(st + MX4_TILE, a.up + w_at + (uint64_t)k * MX4_TILE, MX4_TILE, &full[s]);
            if (!waited) {  // x comes from the launch before
                grid_dependency_wait();
                waited = true;
            }
            const uint8_t *x = a.x + x_at + (uint64_t)k * C::X_BYTES;
            if (C::XT == 1) bulk_g2s(st + C::W_BYTES, x, C::X_BYTES, &full[s]);
            else  // all codes, then all scales
                for (uint32_t t = 0; t < xts; t++, x += (uint64_t)a.nk * C::X_BYTES) {
                    bulk_g2s(st + C::W_BYTES + t * C::XROWS * 128, x, C::XROWS * 128, &full[s]);
                    bulk_g2s(st + C::W_BYTES + NT * 128 + t * MX4_SCALES, x + C::XROWS * 128, MX4_SCALES, &full[s]);
                }
        }
        if (!ok) {  // the copies in flight end before the memory is given up
            for (uint32_t j = i > C::STAGES ? i - C::STAGES : 0; j < i; j++)
                mbar_wait_bounded(&full[j % C::STAGES], (j / C::STAGES) & 1, WAIT_LIMIT_NS);
        }
    } else if (tid == 32) {
        uint32_t i = 0;
        for (uint32_t k = k0; k < k1 && ok; k++, i++) {
            const uint32_t s = i % C::STAGES;
            ok = mbar_wait_bounded(&full[s], (i / C::STAGES) & 1, WAIT_LIMIT_NS);
            if (!ok) break;
            fence_after();
            const uint32_t st = smem_u32(smem + HDR + s * C::STAGE), sc = tmem + C::SUMS + s * C::SC, sx = sc + 8 * (DUAL ? 2 : 1);
#pragma unroll
            for (uint32_t h = 0; h < 2; h++) {
                copy_scales<1>(sc + 4 * h, desc_scales(st + MX4_ROWS * 128 + 512 * h));
                if (DUAL) copy_scales<1>(sc + 8 + 4 * h, desc_scales(st + MX4_TILE + MX4_ROWS * 128 + 512 * h));
#pragma unroll
                for (uint32_t t = 0; t < C::XT; t++)
                    copy_scales<1>(sx + 4 * C::XT * h + 4 * t, desc_scales(st + C::W_BYTES + NT * 128 + t * MX4_SCALES + 512 * h));
            }
            // a product has 64 columns: 32 bytes of a row, half of a word of four scales
#pragma unroll
            for (uint32_t q = 0; q < 4; q++) {
                const uint32_t h = q >> 1, id = idesc(128, n, q & 1), add = i > 0 || q > 0;
                const uint64_t x = desc_operand(st + C::W_BYTES + 32 * q);
                mma<1>(tmem, desc_operand(st + 32 * q), x, id, sc + 4 * h, sx + 4 * C::XT * h, add);
                if (DUAL) mma<1>(tmem + NT, desc_operand(st + MX4_TILE + 32 * q), x, id, sc + 8 + 4 * h, sx + 4 * C::XT * h, add);
            }
            commit<1>(&empty[s]);
        }
        if (ok) commit<1>(done);
    }
    if (warp >= 2) {
        ok = mbar_wait_bounded(done, 0, 2 * WAIT_LIMIT_NS);
        fence_after();
        ok = __all_sync(0xffffffffu, ok);
    }
    if (!ok) atomicExch(&g_dev_status, (unsigned)DEV_TIMEOUT_TMA);
    __syncwarp();
    const uint32_t lane_at = (warp & 3) * 32, f = ft * MX4_ROWS + lane_at + lane;
    if (parts == 1) {
        if (warp >= 2 && ok) {
            for (uint32_t c = 0; c < n; c += 16) {
                float v[16], u[16];
                tmem_ld16(tmem + (lane_at << 16) + c, v);
                if (DUAL) {
                    tmem_ld16(tmem + (lane_at << 16) + NT + c, u);
#pragma unroll
                    for (int j = 0; j < 16; j++) v[j] = silu_times(v[j], u[j]);
                }
                if (f < a.feats)
#pragma unroll
                    for (uint32_t j = 0; j < 16; j++)
                        if (c + j < rows) put(a, row0 + c + j, f, v[j]);
            }
        }
    } else {
        // the stages have been read: this part's sums take their place, [tokens][128 features], gate then up
        float *mine = reinterpret_cast<float *>(smem + HDR);
        if (warp >= 2 && ok)
            for (uint32_t c = 0; c < n; c += 16)
#pragma unroll
                for (uint32_t d = 0; d < (DUAL ? 2 : 1); d++) {
                    float v[16];
                    tmem_ld16(tmem + (lane_at << 16) + d * NT + c, v);
#pragma unroll
                    for (uint32_t j = 0; j < 16; j++) mine[(d * NT + c + j) * MX4_ROWS + lane_at + lane] = v[j];
                }
        cluster.sync();
        if (warp >= 2 && ok && f < a.feats)
            for (uint32_t t = part; t < rows; t += parts) {
                float v[2] = {};
                for (uint32_t p = 0; p < parts; p++) {
                    const float *theirs = cluster.map_shared_rank(mine, p);
#pragma unroll
                    for (uint32_t d = 0; d < (DUAL ? 2 : 1); d++) v[d] += theirs[(d * NT + t) * MX4_ROWS + lane_at + lane];
                }
                put(a, row0 + t, f, DUAL ? silu_times(v[0], v[1]) : v[0]);
            }
        cluster.sync();
    }
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        tmem_free<1>(tmem, C::COLS);
    }
}

template <int NT, bool DUAL>
cudaError_t launch_as(const Mx4GemmArgs &a, uint64_t tiles, uint32_t parts, cudaStream_t s) {
    using C = Cfg<NT, DUAL>;
    auto fn = mx4_gemm_kernel<NT, DUAL>;
    static bool ready[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!ready[dev & 63]) {
        if ((e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) != cudaSuccess) return e;
        ready[dev & 63] = true;
    }
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((uint32_t)(tiles * parts));
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = C::SMEM;
    c.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {parts, 1, 1};
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = at;
    c.numAttrs = 2;
    return cudaLaunchKernelEx(&c, fn, a);
}

}  // namespace

cudaError_t mx4_gemm_launch(const Mx4GemmArgs &a, uint32_t tile_shift, uint64_t token_tiles, int sms, cudaStream_t s) {
    const uint64_t tiles = token_tiles * a.feat_tiles;
    // few tiles of few tokens: the columns of a tile in 2, 4 or 8 parts
    uint32_t parts = 1;
    if (tile_shift == 5)
        while (parts < 8 && tiles * parts <= (uint64_t)sms && a.nk >= 2 * parts * 2) parts *= 2;
    if (tile_shift == 5) return a.up ? launch_as<32, true>(a, tiles, parts, s) : launch_as<32, false>(a, tiles, parts, s);
    if (tile_shift == 7) return a.up ? launch_as<128, true>(a, tiles, parts, s) : launch_as<128, false>(a, tiles, parts, s);
    return cudaErrorInvalidValue;
}

}  // namespace sg
