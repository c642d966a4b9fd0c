// mx4_many.cu — products of microscaled 4-bit matrices for many tokens (mx4.cuh): tcgen05 on pairs
// of SMs, persistent.
//
// A pair of CTAs has a tile of 256 features (128 of TMEM's lanes in each) by up to NT tokens: each
// brings its own rows of the weights and half of the tokens, the tensor cores of both read both
// halves.  That halves what a token's codes cost to bring: reading the operands out of L2 is what
// bounds such products (all SMs together get 17.9 TB/s by bulk copies, 64 bytes a cycle each, while
// the tensor cores eat a stage of 256 columns and 256 tokens, 35 KB, in 512 cycles).
//   - three threads issue the bulk copies (a copy takes its thread about 70 ns, a wait 80): weights,
//     tokens, the tokens' scales (both halves': the scales of all columns stand in each CTA);
//   - one thread of the pair's first CTA issues scales' copies to TMEM and products for both; the
//     other CTA's tells it when its operands are there;
//   - eight warps take the sums out of TMEM into registers, at once, so that the next tile's products
//     can begin, then round them and write them by way of shared memory, 16 bytes a lane.
#include <cooperative_groups.h>

#include "mx4_tc.cuh"

namespace cg = cooperative_groups;

namespace sg {
using namespace mx4;
using namespace tiled;

namespace {

constexpr uint32_t EPI_WARPS = 8, FIRST_EPI = 4, THREADS = 32 * (FIRST_EPI + EPI_WARPS);
constexpr uint32_t MAX_E = MOE_SORT_MAX_EXPERTS;
constexpr uint32_t HDR = 1024 + (MAX_E + 4) * 4 / 1024 * 1024 + 1024;  // barriers and TMEM base; the experts' first tiles
constexpr uint32_t OUT_ROW = 144;                                      // a token's 32 features of a warp, and padding
constexpr uint32_t OUT_BYTES = 32 * OUT_ROW;

template <bool DUAL>
struct Cfg {
    static constexpr uint32_t NT = DUAL ? 128 : 256, XT = NT / 128;
    static constexpr uint32_t W_BYTES = MX4_TILE * (DUAL ? 2 : 1), X_BYTES = NT / 2 * 128, XS_BYTES = XT * MX4_SCALES;
    static constexpr uint32_t STAGE = W_BYTES + X_BYTES + XS_BYTES;
    static constexpr uint32_t STAGES = DUAL ? 4 : 5;
    static constexpr uint32_t OUT_AT = HDR + STAGES * STAGE, SMEM = OUT_AT + EPI_WARPS * OUT_BYTES;
    static constexpr uint32_t SUMS = 256, SC = 8 * ((DUAL ? 2 : 1) + XT), COLS = 512;
    static_assert(SUMS + STAGES * SC <= COLS && SMEM <= 227 * 1024 && STAGE % 1024 == 0, "shapes");
};

struct Shared {
    uint64_t full[8], empty[8], sums_full, sums_empty;
    uint32_t tmem;
};

__device__ __forceinline__ bool try_wait_cluster(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded: a wait that does not end is recorded, and everybody goes home.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity) {
    for (int i = 0; i < 16; i++)
        if (try_wait_cluster(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (;;) {
        for (int i = 0; i < 64; i++)
            if (try_wait_cluster(bar, parity)) return true;
        if (globaltimer_ns() - t0 > WAIT_LIMIT_NS) return false;
    }
}
// Arrives at the barrier of the pair's CTA `rank` that lies where bar does here.  Relaxed: what it tells of are bulk copies
// and TMEM loads, whose end this thread has seen; nothing that it wrote itself is handed over.  (With release each arrival
// takes 500 ns, which made a stage of the pipeline 640 to 800 ns long instead of 330.)
__device__ __forceinline__ void arrive_at(uint64_t *bar, uint32_t rank) {
    asm volatile(
        "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, %1;\n mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [a];\n}" ::"r"(smem_u32(bar)),
        "r"(rank)
        : "memory");
}

// A tile: up to NT rows of x, those of one expert, from row row0 of the output on.
struct Tile {
    uint32_t e, x_tile, rows, fp;
    uint64_t row0;
};

template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 32 tokens of 32 features, a feature a lane, to rows of the output; n of the tokens are there.
template <typename T>
__device__ __forceinline__ void put32(const Mx4GemmArgs &a, uint8_t *buf, const float *v, uint64_t row, uint32_t n, uint32_t f0, uint32_t lane) {
    T *out = static_cast<T *>(a.out);
    if (a.vec && f0 + 32 <= a.feats) {
#pragma unroll
        for (uint32_t j = 0; j < 32; j++) *reinterpret_cast<T *>(buf + j * OUT_ROW + lane * sizeof(T)) = narrow<T>(v[j]);
        __syncwarp();
        constexpr uint32_t PER = 2 * sizeof(T), AT_ONCE = 32 / PER;  // lanes a token
#pragma unroll
        for (uint32_t j = 0; j < 32; j += AT_ONCE) {
            const uint32_t t = j + lane / PER, c = lane % PER;
            const uint4 w = *reinterpret_cast<const uint4 *>(buf + t * OUT_ROW + 16 * c);
            if (t < n) *reinterpret_cast<uint4 *>(reinterpret_cast<uint8_t *>(out + (row + t) * a.ldo + f0) + 16 * c) = w;
        }
        __syncwarp();
    } else if (f0 + lane < a.feats) {
#pragma unroll
        for (uint32_t j = 0; j < 32; j++)
            if (j < n) out[(row + j) * a.ldo + f0 + lane] = narrow<T>(v[j]);
    }
}

template <bool DUAL>
__global__ void __launch_bounds__(THREADS, 1) mx4_many_kernel(const __grid_constant__ Mx4GemmArgs a) {
    using C = Cfg<DUAL>;
    extern __shared__ __align__(1024) uint8_t smem[];
    Shared &sh = *reinterpret_cast<Shared *>(smem);
    uint32_t *upto = reinterpret_cast<uint32_t *>(smem + 1024);  // experts: tiles of the ones up to each
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank();
    if (cluster.num_blocks() != 2 || blockDim.x != THREADS || dynamic_smem_size() < C::SMEM || (smem_u32(smem) & 1023u) || a.nk == 0 ||
        a.n_expert > MAX_E) {
        if (tid == 0) atomicExch(&g_dev_status, (unsigned)DEV_BAD_LAUNCH);
        return;  // (the whole grid alike)
    }
    if (tid == 0) {
        for (uint32_t i = 0; i < C::STAGES; i++) mbar_init(&sh.full[i], rank ? 3 : 4), mbar_init(&sh.empty[i], 1);
        mbar_init(&sh.sums_full, 1);
        mbar_init(&sh.sums_empty, 2 * EPI_WARPS);
        fence_mbar_init();
    }
    if (warp == 3) tmem_alloc<2>(&sh.tmem, C::COLS);
    uint32_t token_tiles;
    if (a.first) {
        if (warp == 0) {
            uint32_t before = 0;
            for (uint32_t base = 0; base < a.n_expert; base += 32) {
                const uint32_t i = base + lane;
                uint32_t n = i < a.n_expert ? ((uint32_t)__ldg(a.first + i + 1) - (uint32_t)__ldg(a.first + i) + C::NT - 1) / C::NT : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, n, o);
                    if (lane >= (uint32_t)o) n += v;
                }
                if (i < a.n_expert) upto[i] = before + n;
                before += __shfl_sync(0xffffffffu, n, 31);
            }
        }
    }
    fence_before();
    __syncthreads();
    cluster.sync();
    fence_after();
    token_tiles = a.first ? upto[a.n_expert - 1] : (uint32_t)((a.n_tok + C::NT - 1) / C::NT);
    const uint32_t tmem = sh.tmem, pairs = gridDim.x / 2, me = blockIdx.x / 2;
    const uint32_t fps = (a.feat_tiles + 1) / 2;
    const uint64_t tiles = (uint64_t)token_tiles * fps;

    auto tile_at = [&](uint64_t i) {
        Tile t;
        const uint32_t tt = (uint32_t)(i / fps);
        t.fp = (uint32_t)(i - (uint64_t)tt * fps);
        if (a.first) {
            uint32_t lo = 0, hi = a.n_expert - 1;  // the first expert whose tiles reach past tt
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                if (upto[mid] > tt) hi = mid;
                else lo = mid + 1;
            }
            const uint32_t k = tt - (lo ? upto[lo - 1] : 0), f0 = (uint32_t)__ldg(a.first + lo), n = (uint32_t)__ldg(a.first + lo + 1) - f0;
            t.e = lo;
            t.x_tile = (uint32_t)__ldg(a.tiles + lo) + k * C::XT;
            t.rows = min(n - k * C::NT, C::NT);
            t.row0 = f0 + k * C::NT;
        } else {
            t.e = 0;
            t.x_tile = tt * C::XT;
            t.row0 = (uint64_t)tt * C::NT;
            t.rows = (uint32_t)(a.n_tok - t.row0 < C::NT ? a.n_tok - t.row0 : C::NT);
        }
        return t;
    };

    bool ok = true;
    if (warp < 3) {
        uint32_t s = 0, turn = 0, issued = 0;
        if (warp) grid_dependency_wait();  // x comes from the launch before
        for (uint64_t i = me; i < tiles && ok; i += pairs) {
            const Tile t = tile_at(i);
            const uint32_t n = (t.rows + 31) & ~31u, half = n / 2, r0 = rank * half;  // this CTA's tokens: r0 .. r0 + half
            const uint32_t ft = min(2 * t.fp + rank, a.feat_tiles - 1);
            const uint64_t w_at = (uint64_t)t.e * a.expert_bytes + (uint64_t)ft * a.nk * MX4_TILE, next = (uint64_t)a.nk * MX4_TILE;
            const uint8_t *w = a.w + w_at, *up = DUAL ? a.up + w_at : nullptr, *x = a.x + (uint64_t)t.x_tile * next;
            // rows from the first of them on in its tile of 128, and what is left of it
            const uint32_t in = r0 & 127u, part = min(half, 128 - in), xts = C::XT == 2 && n > 128 ? 2 : 1;
            const uint8_t *xr = x + (r0 >> 7) * next + in * 128, *xr2 = x + next;
            if (warp == 2) x += MX4_ROWS * 128;
            for (uint32_t k = 0; k < a.nk; k++) {
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
                } else if (warp == 1) {
                    if (elect_one()) {
                        mbar_arrive_expect_tx(full, half * 128);
                        bulk_g2s(st + C::W_BYTES, xr, part * 128, full);
                        if (part < half) bulk_g2s(st + C::W_BYTES + part * 128, xr2, (half - part) * 128, full);
                    }
                    xr += MX4_TILE, xr2 += MX4_TILE;
                } else {
                    if (elect_one()) {
                        mbar_arrive_expect_tx(full, xts * MX4_SCALES);
                        bulk_g2s(st + C::W_BYTES + C::X_BYTES, x, MX4_SCALES, full);
                        if (xts == 2) bulk_g2s(st + C::W_BYTES + C::X_BYTES + MX4_SCALES, x + next, MX4_SCALES, full);
                    }
                    x += MX4_TILE;
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
    } else if (warp == 3) {
        uint32_t s = 0, turn = 0, count = 0;
        if (rank) {  // the other CTA's operands are there: the first one is told
            for (uint64_t i = me; i < tiles && ok; i += pairs)
                for (uint32_t k = 0; k < a.nk; k++) {
                    ok = wait(&sh.full[s], turn & 1);
                    if (!ok) break;
                    if (elect_one()) arrive_at(&sh.full[s], 0);
                    __syncwarp();
                    if (++s == C::STAGES) s = 0, turn++;
                }
        } else {
            // what changes in a descriptor from stage to stage is its address
            const uint32_t base = smem_u32(smem + HDR);
            const uint64_t w_desc = desc_operand(base), x_desc = desc_operand(base + C::W_BYTES);
            const uint64_t ws_desc = desc_scales(base + MX4_ROWS * 128), xs_desc = desc_scales(base + C::W_BYTES + C::X_BYTES);
            for (uint64_t i = me; i < tiles && ok; i += pairs, count++) {
                const uint32_t n = (tile_at(i).rows + 31) & ~31u, id = idesc(256, n, 0);
                if (count) ok = wait(&sh.sums_empty, (count - 1) & 1);
                if (!ok) break;
                fence_after();
                for (uint32_t k = 0; k < a.nk; k++) {
                    ok = wait(&sh.full[s], turn & 1);
                    if (!ok) break;
                    fence_after();
                    const uint32_t at = (s * C::STAGE) >> 4, sc = tmem + C::SUMS + s * C::SC, sx = sc + 8 * (DUAL ? 2 : 1);
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t h = 0; h < 2; h++) {
                            copy_scales<2>(sc + 4 * h, ws_desc + at + 32 * h);
                            if (DUAL) copy_scales<2>(sc + 8 + 4 * h, ws_desc + at + (MX4_TILE >> 4) + 32 * h);
#pragma unroll
                            for (uint32_t j = 0; j < C::XT; j++) copy_scales<2>(sx + 4 * C::XT * h + 4 * j, xs_desc + at + j * (MX4_SCALES >> 4) + 32 * h);
                        }
                        // a product has 64 columns: 32 bytes of a row, half of a word of four scales
#pragma unroll
                        for (uint32_t q = 0; q < 4; q++) {
                            const uint32_t h = q >> 1, iq = id | (q & 1 ? idesc(0, 0, 1) ^ idesc(0, 0, 0) : 0u), add = k > 0 || q > 0;
                            mma<2>(tmem, w_desc + at + 2 * q, x_desc + at + 2 * q, iq, sc + 4 * h, sx + 4 * C::XT * h, add);
                            if (DUAL)
                                mma<2>(tmem + 128, w_desc + at + (MX4_TILE >> 4) + 2 * q, x_desc + at + 2 * q, iq, sc + 8 + 4 * h, sx + 4 * h, add);
                        }
                        commit<2>(&sh.empty[s]);
                    }
                    __syncwarp();
                    if (++s == C::STAGES) s = 0, turn++;
                }
                if (ok && elect_one()) commit<2>(&sh.sums_full);
                __syncwarp();
            }
        }
    } else {
        const uint32_t q = warp & 3, g = (warp - FIRST_EPI) >> 2;  // lanes 32 q on; which half of the tokens
        uint8_t *buf = smem + C::OUT_AT + (warp - FIRST_EPI) * OUT_BYTES;
        constexpr uint32_t HALF = C::NT / 2;
        uint32_t count = 0;
        for (uint64_t i = me; i < tiles; i += pairs, count++) {
            const Tile t = tile_at(i);
            ok = __all_sync(0xffffffffu, wait(&sh.sums_full, count & 1));
            if (!ok) break;
            fence_after();
            float v[128];
            const uint32_t from = g * HALF, at = tmem + ((32 * q) << 16) + from;
            if (t.rows > from) {
                tmem_ld64(at, v);
                if (DUAL) tmem_ld64(at + 128, v + 64);
                else if (t.rows > from + 64) tmem_ld64(at + 64, v + 64);
            }
            fence_before();
            __syncwarp();
            if (elect_one()) arrive_at(&sh.sums_empty, 0);
            __syncwarp();
            if (t.rows <= from) continue;
            const uint32_t f0 = (2 * t.fp + rank) * MX4_ROWS + 32 * q;
            if (f0 >= a.feats) continue;
            if (DUAL) {
#pragma unroll
                for (int j = 0; j < 64; j++) v[j] = silu_times(v[j], v[64 + j]);
            }
#pragma unroll
            for (uint32_t c = 0; c < HALF; c += 32)
                if (t.rows > from + c) {
                    const uint32_t n = t.rows - from - c;
                    if (a.type == SG_F32) put32<float>(a, buf, v + c, t.row0 + from + c, n, f0, lane);
                    else if (a.type == SG_F16) put32<__half>(a, buf, v + c, t.row0 + from + c, n, f0, lane);
                    else put32<__nv_bfloat16>(a, buf, v + c, t.row0 + from + c, n, f0, lane);
                }
        }
    }
    if (!ok) atomicExch(&g_dev_status, (unsigned)DEV_TIMEOUT_TMA);
    __syncwarp();
    fence_before();
    cluster.sync();  // (the pair's products have read this CTA's memory, its arrivals have been made)
    if (warp == 3) {
        fence_after();
        tmem_free<2>(tmem, C::COLS);
    }
}

template <bool DUAL>
cudaError_t launch_as(const Mx4GemmArgs &a, uint64_t tiles, int sms, cudaStream_t s) {
    using C = Cfg<DUAL>;
    auto fn = mx4_many_kernel<DUAL>;
    static bool ready[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!ready[dev & 63]) {
        if ((e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) != cudaSuccess) return e;
        ready[dev & 63] = true;
    }
    cudaLaunchConfig_t c = {};
    const uint64_t pairs = tiles < (uint64_t)sms / 2 ? tiles : sms / 2;
    c.gridDim = dim3((uint32_t)pairs * 2);
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = C::SMEM;
    c.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {2, 1, 1};
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = at;
    c.numAttrs = 2;
    return cudaLaunchKernelEx(&c, fn, a);
}

}  // namespace

cudaError_t mx4_many_launch(const Mx4GemmArgs &a, uint64_t token_tiles, int sms, cudaStream_t s) {
    const uint64_t tiles = token_tiles * ((a.feat_tiles + 1) / 2);
    return a.up ? launch_as<true>(a, tiles, sms, s) : launch_as<false>(a, tiles, sms, s);
}

}  // namespace sg
