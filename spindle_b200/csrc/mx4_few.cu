// mx4_few.cu — products of microscaled 4-bit matrices for a few tokens (mx4.cuh): what bounds them
// is bringing the weights, so the weights are the 128 rows of tcgen05's tile (the lanes of TMEM), the
// tokens its columns, as narrow as they are, and the copies never pause.
//
// One CTA an SM.  One thread brings the weights of a tile of 128 features, stage after stage of 256
// columns, on into the next tile, up to 200 KB ahead; another the tokens' codes (the weights do not
// wait for them, or for the launch before that quantizes them); one thread copies scales to TMEM and
// issues the products; four warps write the results.  Where the tiles are fewer than the SMs, the
// CTAs of a cluster take a part of the columns each and add their sums over distributed shared
// memory, in rank order.
// One row of 4096 to 14336 (31 MB of weights, 4.8 us): 10.3 us, 8.1 with its quantizing launch in a graph;
// 33 rows of 14336 to 4096 (32 MB): 12.6, 10.4 in a graph: launches, the first copies' way and the last
// sums; the copies between go at 5 to 6 TB/s.  Gate and up of 16 tokens' 8 of 128 experts (131 MB, 20 us): 27 us.
#include <cooperative_groups.h>

#include "mx4_tc.cuh"

namespace cg = cooperative_groups;

namespace sg {
using namespace mx4;
using namespace tiled;

namespace {

constexpr uint32_t FIRST_EPI = 4, THREADS = 32 * (FIRST_EPI + 4);
constexpr uint32_t HDR = 1024 + EXPERTS_BYTES;  // barriers and TMEM base; what is looked up of the experts

// Up to NT tokens a tile, which is also the rows of a tile of x; DUAL: gate and up.
template <uint32_t NT, bool DUAL>
struct Cfg {
    static constexpr uint32_t W_BYTES = MX4_TILE * (DUAL ? 2 : 1), X_BYTES = mx4_tile_bytes(NT), STAGE = W_BYTES + X_BYTES;
    static constexpr uint32_t FIT = (227 * 1024 - HDR - OUT_BYTES) / STAGE, STAGES = FIT < 9 ? FIT : 9;
    static constexpr uint32_t OUT_AT = HDR + STAGES * STAGE, SMEM = OUT_AT + OUT_BYTES;
    // TMEM columns: sums, in two buffers in turn unless they are gate and up of many, then each stage's scales
    static constexpr uint32_t BUFS = DUAL && NT > 64 ? 1 : 2, SUMS = NT * (DUAL ? 2 : 1) * BUFS, SC = 8 * (DUAL ? 3 : 2);
    static constexpr uint32_t WANT = SUMS + STAGES * SC, COLS = WANT <= 256 ? 256 : 512;
    static_assert(WANT <= 512 && STAGE % 1024 == 0 && STAGES * STAGE >= NT * (DUAL ? 2 : 1) * MX4_ROWS * 4, "shapes, partial sums");
};

struct Shared {
    uint64_t full[9], empty[9], sums_full[2], sums_empty[2];
    uint32_t tmem;
};
static_assert(sizeof(Shared) <= 1024 && sizeof(Experts) <= EXPERTS_BYTES, "places");

__device__ __forceinline__ void arrive(uint64_t *bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }

template <uint32_t NT, bool DUAL>
__global__ void __launch_bounds__(THREADS, 1) mx4_few_kernel(const __grid_constant__ Mx4GemmArgs a) {
    using C = Cfg<NT, DUAL>;
    extern __shared__ __align__(1024) uint8_t smem[];
    Shared &sh = *reinterpret_cast<Shared *>(smem);
    Experts &ex = *reinterpret_cast<Experts *>(smem + 1024);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t parts = cluster.num_blocks(), part = cluster.block_rank(), step = gridDim.x / parts;
    if (blockDim.x != THREADS || dynamic_smem_size() < C::SMEM || (smem_u32(smem) & 1023u) || parts > a.nk || a.n_expert > MAX_E) {
        if (tid == 0) atomicExch(&g_dev_status, (unsigned)DEV_BAD_LAUNCH);
        return;  // (the whole grid alike)
    }
    if (tid == 0) {
        for (uint32_t i = 0; i < C::STAGES; i++) mbar_init(&sh.full[i], 2), mbar_init(&sh.empty[i], 1);
        for (uint32_t i = 0; i < 2; i++) mbar_init(&sh.sums_full[i], 1), mbar_init(&sh.sums_empty[i], 4);
        fence_mbar_init();
    }
    if (warp == 2) tmem_alloc<1>(&sh.tmem, C::COLS);
    if (a.first && warp == 1) find_experts(a, ex, NT, lane);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;
    // (a part of a cluster has its one tile: the launch makes no more)
    const uint32_t tiles = (a.first ? ex.upto[a.n_expert - 1] : (uint32_t)((a.n_tok + NT - 1) / NT)) * a.feat_tiles, me = blockIdx.x / parts;
    const uint32_t k0 = a.nk * part / parts, k1 = a.nk * (part + 1) / parts;
    auto tile_at = [&](uint32_t i) { return tile_of<NT>(a, ex, i / a.feat_tiles); };

    bool ok = true;
    if (warp < 2) {
        uint32_t s = 0, turn = 0, issued = 0;
        if (warp) grid_dependency_wait();  // x comes from the launch before
        for (uint32_t i = me; i < tiles && ok; i += step) {
            const Tile t = tile_at(i);
            const uint64_t w_at = (uint64_t)t.e * a.expert_bytes + ((uint64_t)(i % a.feat_tiles) * a.nk + k0) * MX4_TILE;
            const uint8_t *w = a.w + w_at, *up = DUAL ? a.up + w_at : nullptr, *x = a.x + ((uint64_t)t.x_tile * a.nk + k0) * C::X_BYTES;
            const uint32_t n = (t.rows + 15) & ~15u;
            for (uint32_t k = k0; k < k1; k++) {
                if (turn) ok = wait(&sh.empty[s], (turn - 1) & 1);
                if (!ok) break;
                uint8_t *st = smem + HDR + s * C::STAGE;
                uint64_t *full = &sh.full[s];
                if (warp == 0) {
                    if (elect_one()) {
                        mbar_arrive_expect_tx(full, C::W_BYTES);
                        bulk_g2s(st, w, MX4_TILE, full);
                        if (DUAL) bulk_g2s(st + MX4_TILE, up, MX4_TILE, full);
                    }
                    w += MX4_TILE, up += MX4_TILE;
                } else {
                    if (elect_one()) {
                        mbar_arrive_expect_tx(full, n * 128 + MX4_SCALES);
                        if (n == NT) bulk_g2s(st + C::W_BYTES, x, C::X_BYTES, full);
                        else {
                            bulk_g2s(st + C::W_BYTES, x, n * 128, full);
                            bulk_g2s(st + C::W_BYTES + NT * 128, x + NT * 128, MX4_SCALES, full);
                        }
                    }
                    x += C::X_BYTES;
                }
                __syncwarp();
                issued = min(issued + 1, C::STAGES);
                if (++s == C::STAGES) s = 0, turn++;
            }
        }
        if (!ok && warp == 0)  // the copies in flight end before the memory is given up
            for (; issued; issued--) {
                const bool back = s == 0;
                s = back ? C::STAGES - 1 : s - 1;
                turn -= back;
                mbar_wait_bounded(&sh.full[s], turn & 1, WAIT_LIMIT_NS);
            }
    } else if (warp == 2) {
        uint32_t s = 0, turn = 0, count = 0;
        // what changes in a descriptor from stage to stage is its address
        const uint32_t base = smem_u32(smem + HDR);
        const uint64_t w_desc = desc_operand(base), x_desc = desc_operand(base + C::W_BYTES);
        const uint64_t ws_desc = desc_scales(base + MX4_ROWS * 128), xs_desc = desc_scales(base + C::W_BYTES + NT * 128);
        for (uint32_t i = me; i < tiles && ok; i += step, count++) {
            const uint32_t n = (tile_at(i).rows + 15) & ~15u, id = idesc(128, n, 0), b = count % C::BUFS, sums = tmem + b * NT * (DUAL ? 2 : 1);
            if (count >= C::BUFS) ok = wait(&sh.sums_empty[b], (count / C::BUFS - 1) & 1);
            if (!ok) break;
            fence_after();
            for (uint32_t k = k0; k < k1; k++) {
                ok = wait(&sh.full[s], turn & 1);
                if (!ok) break;
                fence_after();
                const uint32_t at = (s * C::STAGE) >> 4, sc = tmem + C::SUMS + s * C::SC, sx = sc + 8 * (DUAL ? 2 : 1);
                if (elect_one()) {
#pragma unroll
                    for (uint32_t h = 0; h < 2; h++) {
                        copy_scales<1>(sc + 4 * h, ws_desc + at + 32 * h);
                        if (DUAL) copy_scales<1>(sc + 8 + 4 * h, ws_desc + at + (MX4_TILE >> 4) + 32 * h);
                        copy_scales<1>(sx + 4 * h, xs_desc + at + 32 * h);
                    }
                    // a product has 64 columns: 32 bytes of a row, half of a word of four scales
#pragma unroll
                    for (uint32_t q = 0; q < 4; q++) {
                        const uint32_t h = q >> 1, iq = id | (q & 1 ? idesc(0, 0, 1) ^ idesc(0, 0, 0) : 0u), add = k > k0 || q > 0;
                        mma<1>(sums, w_desc + at + 2 * q, x_desc + at + 2 * q, iq, sc + 4 * h, sx + 4 * h, add);
                        if (DUAL) mma<1>(sums + NT, w_desc + at + (MX4_TILE >> 4) + 2 * q, x_desc + at + 2 * q, iq, sc + 8 + 4 * h, sx + 4 * h, add);
                    }
                    commit<1>(&sh.empty[s]);
                }
                __syncwarp();
                if (++s == C::STAGES) s = 0, turn++;
            }
            if (ok && elect_one()) commit<1>(&sh.sums_full[b]);
            __syncwarp();
        }
    } else if (warp >= FIRST_EPI && parts == 1) {
        const uint32_t q = warp & 3;
        uint8_t *buf = smem + C::OUT_AT;
        uint32_t count = 0, turn = 0;
        for (uint32_t i = me; i < tiles; i += step, count++) {
            const Tile t = tile_at(i);
            const uint32_t b = count % C::BUFS;
            // one warp waits, the others for it; they go on together, or not at all
            uint32_t bad = q == 0 && !wait(&sh.sums_full[b], (count / C::BUFS) & 1);
            asm volatile("{\n .reg .pred p, r;\n setp.ne.u32 p, %0, 0;\n barrier.cta.red.or.pred r, %1, 128, p;\n selp.u32 %0, 1, 0, r;\n}"
                         : "+r"(bad)
                         : "r"(1)
                         : "memory");
            if (bad) {
                ok = false;
                break;
            }
            fence_after();
            const uint32_t at = tmem + b * NT * (DUAL ? 2 : 1) + ((32 * q) << 16), f0 = i % a.feat_tiles * MX4_ROWS;
            auto put = [&](auto type) {
                const Out<decltype(type), 2> o(a, t.row0, f0, q, lane);
                for (uint32_t c = 0; c < t.rows; c += 16) {
                    float v[16], u[16];
                    tmem_ld32x16(at + c, v);
                    if (DUAL) tmem_ld32x16(at + NT + c, u);
                    tmem_wait(v);
                    if (DUAL) {
                        tmem_wait(u);
#pragma unroll
                        for (int j = 0; j < 16; j++) v[j] = silu_times(v[j], u[j]);
                    }
                    put_piece(a, o, sizeof(type) == 2 ? buf + (turn & 1) * (OUT_BYTES / 2) : buf, v, c, t.rows - c, q, lane, 0);
                    turn++;
                }
            };
            if (a.type == SG_F32) put(float());
            else if (a.type == SG_F16) put(__half());
            else put(__nv_bfloat16());
            fence_before();
            __syncwarp();
            if (elect_one()) arrive(&sh.sums_empty[b]);
            __syncwarp();
        }
    } else if (warp >= FIRST_EPI && me < tiles) {
        // the stages have been read: this part's sums take their place, [tokens][128 features], gate then up
        ok = wait(&sh.sums_full[0], 0);
        fence_after();
        const uint32_t q = warp & 3, n = tile_at(me).rows;
        float *mine = reinterpret_cast<float *>(smem + HDR) + 32 * q + (lane >> 2);
        if (ok)
            for (uint32_t c = 0; c < n; c += 16)
#pragma unroll
                for (uint32_t d = 0; d < (DUAL ? 2 : 1); d++) {
                    float v[16];
                    tmem_ld32x16(tmem + ((32 * q) << 16) + d * NT + c, v);
                    tmem_wait(v);
#pragma unroll
                    for (uint32_t j = 0; j < 16; j++)  // feature 8 (j / 2 % 2) + 16 (j / 8), token 8 (j / 4 % 2) + 2 (lane % 4) + j % 2
                        mine[(d * NT + c + 8 * (j >> 2 & 1) + 2 * (lane & 3) + (j & 1)) * MX4_ROWS + 8 * (j >> 1 & 1) + 16 * (j >> 3)] = v[j];
                }
    }
    if (!ok) atomicExch(&g_dev_status, (unsigned)DEV_TIMEOUT_TMA);
    __syncwarp();
    if (parts > 1) {
        cluster.sync();
        if (me < tiles) {
            // four features a thread, token after token
            const Tile t = tile_at(me);
            const uint32_t f0 = me % a.feat_tiles * MX4_ROWS + 4 * lane;
            float *sums = reinterpret_cast<float *>(smem + HDR) + 4 * lane;
            for (uint32_t j = part * (THREADS / 32) + warp; j < t.rows; j += parts * (THREADS / 32)) {
                float4 v[2] = {};
                for (uint32_t p = 0; p < parts; p++) {
                    const float *theirs = cluster.map_shared_rank(sums, p);
#pragma unroll
                    for (uint32_t d = 0; d < (DUAL ? 2 : 1); d++) {
                        const float4 w = *reinterpret_cast<const float4 *>(theirs + (d * NT + j) * MX4_ROWS);
                        v[d].x += w.x, v[d].y += w.y, v[d].z += w.z, v[d].w += w.w;
                    }
                }
                float r[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
                if (DUAL) {
                    const float u[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
                    for (int i = 0; i < 4; i++) r[i] = silu_times(r[i], u[i]);
                }
                const uint64_t at = (t.row0 + j) * a.ldo + f0;
#pragma unroll
                for (uint32_t i = 0; i < 4; i++)
                    if (f0 + i < a.feats) {
                        if (a.type == SG_F32) static_cast<float *>(a.out)[at + i] = r[i];
                        else if (a.type == SG_F16) static_cast<__half *>(a.out)[at + i] = __float2half_rn(r[i]);
                        else static_cast<__nv_bfloat16 *>(a.out)[at + i] = __float2bfloat16_rn(r[i]);
                    }
            }
        }
        cluster.sync();  // nobody reads here any more
    }
    fence_before();
    __syncthreads();
    if (warp == 2) {
        fence_after();
        tmem_free<1>(tmem, C::COLS);
    }
}

template <uint32_t NT, bool DUAL>
cudaError_t launch_as(const Mx4GemmArgs &a, uint32_t grid, uint32_t parts, cudaStream_t s) {
    using C = Cfg<NT, DUAL>;
    auto fn = mx4_few_kernel<NT, DUAL>;
    static bool ready[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!ready[dev & 63]) {
        if ((e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) != cudaSuccess) return e;
        ready[dev & 63] = true;
    }
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(grid);
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

cudaError_t mx4_few_launch(const Mx4GemmArgs &a, uint32_t x_rows, uint64_t token_tiles, int sms, cudaStream_t s) {
    const uint64_t tiles = token_tiles * a.feat_tiles;
    // few tiles: their columns in 2, 4 or 8 parts, while a part has four stages or more
    uint32_t parts = 1;
    while (parts < 8 && tiles * parts * 2 <= (uint64_t)sms && a.nk >= parts * 8) parts *= 2;
    const uint32_t grid = parts > 1 ? (uint32_t)tiles * parts : (uint32_t)(tiles < (uint64_t)sms ? tiles : sms);
    if (x_rows == 32) return a.up ? launch_as<32, true>(a, grid, parts, s) : launch_as<32, false>(a, grid, parts, s);
    return a.up ? launch_as<128, true>(a, grid, parts, s) : launch_as<128, false>(a, grid, parts, s);
}

}  // namespace sg
