// mx4_many.cu — products of microscaled 4-bit matrices for many tokens (mx4.cuh): tcgen05 on pairs
// of SMs, persistent.
//
// A pair of CTAs has a tile of 256 features (128 of TMEM's lanes in each) by up to NT tokens: each
// brings its own rows of the weights and half of the tokens, the tensor cores of both read both
// halves.  That halves what a token's codes cost to bring: reading the operands out of L2 is what
// bounds such products (all SMs together get 17.9 TB/s by bulk copies, 64 bytes a cycle each, while
// the tensor cores eat a stage of 256 columns and 256 tokens, 35 KB, in 512 cycles).
//   - three warps issue the bulk copies, a stage each 17 KB of weights (twice with gate and up), half of
//     the tokens, all tokens' scales (the scales of all columns stand in each CTA): a copy takes its
//     warp 20 ns, the wait before it 95;
//   - one thread of the pair's first CTA issues scales' copies to TMEM and products for both; the
//     other CTA's tells it when its operands are there;
//   - sixteen warps take the sums out of TMEM into registers, at once, so that the next tile's products
//     can begin, then round them and write them by way of shared memory, 16 bytes a lane.
// 4096 x 4096 x 14336 in bf16: 91 us, 5.3 PFLOP/s (3.2 times the measured bf16 rate), 1.04 GB out of L2, tensor
// pipe busy 64 % of the time: a stage's way round (load 0.5 to 1.2 us, the other CTA's word 0.2, products 0.3,
// the word back 0.2) times the 180 KB of stages is what holds it, and 0.6 us a tile between two tiles' products.
// In a loop of such calls the card's power limit does (1.55 GHz).  Gate and up of 4096 tokens' 8 of 128 experts
// (2048 to 768): 63 us, 290 MB of HBM (44 us) and 650 MB out of L2; back (768 to 2048): 52 us, 241 MB (37 us).
#include <cooperative_groups.h>

#include "mx4_tc.cuh"

namespace cg = cooperative_groups;

namespace sg {
using namespace mx4;
using namespace tiled;

namespace {

constexpr uint32_t EPI_WARPS = 16, FIRST_EPI = 4, THREADS = 32 * (FIRST_EPI + EPI_WARPS);
constexpr uint32_t HDR = 1024 + EXPERTS_BYTES;  // barriers and TMEM base; what is looked up of the experts
constexpr uint32_t GROUPS = EPI_WARPS / 4;      // four warps take a piece of 16 tokens, 32 features each

// Up to NT tokens a tile; DUAL: gate and up.
template <uint32_t N, bool D>
struct Cfg {
    static constexpr uint32_t NT = N, XT = (NT + 127) / 128, X_TILE = mx4_tile_bytes(NT);
    static constexpr bool DUAL = D;
    static constexpr uint32_t W_BYTES = MX4_TILE * (DUAL ? 2 : 1), X_BYTES = NT / 2 * 128, XS_BYTES = mx4_scale_bytes(NT);
    static constexpr uint32_t STAGE = W_BYTES + X_BYTES + XS_BYTES;
    static constexpr uint32_t STAGES = DUAL ? 4 : 5;
    static constexpr uint32_t PIECES = NT / 16 / GROUPS;
    static constexpr uint32_t OUT_AT = HDR + STAGES * STAGE, SMEM = OUT_AT + GROUPS * OUT_BYTES;
    // TMEM: sums, in two buffers in turn where there is room beside the scales
    static constexpr uint32_t SC = 8 * ((DUAL ? 2 : 1) + XT), COLS = 512, ONE = NT * (DUAL ? 2 : 1), BUFS = 2 * ONE + STAGES * SC <= COLS ? 2 : 1;
    static constexpr uint32_t SUMS = ONE * BUFS;
    static_assert(DUAL ? PIECES == 2 : PIECES == 3 || PIECES == 4, "what tmem_ld32x32 and so on are for");
    static_assert(SUMS + STAGES * SC <= COLS && SMEM <= 227 * 1024 && STAGE % 1024 == 0 && NT % (16 * GROUPS) == 0, "shapes");
};

struct Shared {
    uint64_t full[8], empty[8], sums_full[2], sums_empty[2];
    uint32_t tmem;
};
static_assert(sizeof(Shared) <= 1024 && sizeof(Experts) <= EXPERTS_BYTES, "places");

// Arrives at the barrier of the pair's CTA `rank` that lies where bar does here.  Release at the scope of the CTA, the
// instruction's default.  What it tells of are bulk copies into this SM's shared memory, whose end this thread has seen and
// which this SM's own tensor cores read there, and TMEM loads that have ended (ordered by the fence before); nothing that a
// thread wrote is handed over.  The memory model orders the other CTA behind a thread's own view by a release at cluster
// scope only: that bytes which have arrived here are there for products that the other CTA issues is an assumption about the
// tensor cores.  At cluster scope an arrival takes 500 ns, the relay of every stage: 4096 x 4096 x 14336 216 to 223 us instead of
// 99 in bursts, gate and up of 4096 tokens 128 to 144 instead of 93 in a loop; relaxed it is no faster than this.
__device__ __forceinline__ void arrive_at(uint64_t *bar, uint32_t rank) {
    asm volatile(
        "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, %1;\n mbarrier.arrive.release.cta.shared::cluster.b64 _, [a];\n}" ::"r"(smem_u32(bar)),
        "r"(rank)
        : "memory");
}

template <typename C, typename T, bool VEC>
__global__ void __launch_bounds__(THREADS, 1) mx4_many_kernel(const __grid_constant__ Mx4GemmArgs a) {
    constexpr bool DUAL = C::DUAL;
    extern __shared__ __align__(1024) uint8_t smem[];
    Shared &sh = *reinterpret_cast<Shared *>(smem);
    Experts &ex = *reinterpret_cast<Experts *>(smem + 1024);
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
        for (uint32_t i = 0; i < 2; i++) mbar_init(&sh.sums_full[i], 1), mbar_init(&sh.sums_empty[i], 2 * EPI_WARPS);
        fence_mbar_init();
    }
    if (warp == 3) tmem_alloc<2>(&sh.tmem, C::COLS);
    if (a.first && warp == 0) find_experts(a, ex, C::NT, lane);
    fence_before();
    __syncthreads();
    cluster.sync();
    fence_after();
    const uint32_t token_tiles = a.first ? ex.upto[a.n_expert - 1] : (uint32_t)((a.n_tok + C::NT - 1) / C::NT);
    const uint32_t tmem = sh.tmem, pairs = gridDim.x / 2, me = blockIdx.x / 2;
    const uint32_t fps = (a.feat_tiles + 1) / 2;
    const uint32_t tiles = token_tiles * fps;

    // (the feature pairs of a token tile follow each other: an expert's weights are read once, by neighbours)
    auto tile_at = [&](uint32_t i) { return tile_of<C::NT>(a, ex, i / fps); };
    auto pair_of = [&](uint32_t i) { return i % fps; };

    bool ok = true;
    if (warp < 3) {
        uint32_t s = 0, turn = 0, issued = 0;
        if (warp) grid_dependency_wait();  // x comes from the launch before
        for (uint32_t i = me; i < tiles && ok; i += pairs) {
            const Tile t = tile_at(i);
            const uint32_t half = ((t.rows + 31) & ~31u) / 2;  // this CTA's tokens: from rank * half on
            const uint32_t ft = min(2 * pair_of(i) + rank, a.feat_tiles - 1);
            const uint64_t w_at = (uint64_t)t.e * a.expert_bytes + (uint64_t)ft * a.nk * MX4_TILE;
            const uint8_t *w = a.w + w_at, *up = DUAL ? a.up + w_at : nullptr, *x = a.x + (uint64_t)t.x_tile * a.nk * C::X_TILE;
            x += warp == 1 ? rank * half * 128 : C::NT * 128;
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
                } else {
                    if (elect_one()) {
                        const uint32_t bytes = warp == 1 ? half * 128 : C::XS_BYTES;
                        mbar_arrive_expect_tx(full, bytes);
                        bulk_g2s(st + C::W_BYTES + (warp == 1 ? 0 : C::X_BYTES), x, bytes, full);
                    }
                    x += C::X_TILE;
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
            for (uint32_t i = me; i < tiles && ok; i += pairs)
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
            for (uint32_t i = me; i < tiles && ok; i += pairs, count++) {
                const Tile t = tile_at(i);
                const uint32_t n = (t.rows + 31) & ~31u, id = idesc(256, n, 0), b = count % C::BUFS, sums = tmem + b * C::ONE;
                if (count >= C::BUFS) ok = wait(&sh.sums_empty[b], (count / C::BUFS - 1) & 1);
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
                            for (uint32_t j = 0; j < C::XT; j++) copy_scales<2>(sx + 4 * C::XT * h + 4 * j, xs_desc + at + 32 * (C::XT * h + j));
                        }
                        // a product has 64 columns: 32 bytes of a row, half of a word of four scales
#pragma unroll
                        for (uint32_t q = 0; q < 4; q++) {
                            const uint32_t h = q >> 1, iq = id | (q & 1 ? idesc(0, 0, 1) ^ idesc(0, 0, 0) : 0u), add = k > 0 || q > 0;
                            mma<2>(sums, w_desc + at + 2 * q, x_desc + at + 2 * q, iq, sc + 4 * h, sx + 4 * C::XT * h, add);
                            if (DUAL)
                                mma<2>(sums + C::NT, w_desc + at + (MX4_TILE >> 4) + 2 * q, x_desc + at + 2 * q, iq, sc + 8 + 4 * h, sx + 4 * h, add);
                        }
                        commit<2>(&sh.empty[s]);
                    }
                    __syncwarp();
                    if (++s == C::STAGES) s = 0, turn++;
                }
                if (ok && elect_one()) commit<2>(&sh.sums_full[b]);
                __syncwarp();
            }
        }
    } else {
        // lanes 32 q on; a quarter of the tile's pieces of 16 tokens
        const uint32_t q = warp & 3, g = (warp - FIRST_EPI) >> 2;
        uint8_t *buf = smem + C::OUT_AT + g * OUT_BYTES;
        uint32_t count = 0, turn = 0;
        for (uint32_t i = me; i < tiles; i += pairs, count++) {
            const Tile t = tile_at(i);
            const uint32_t b = count % C::BUFS;
            // one warp of a group waits, the others for it; they go on together, or not at all
            uint32_t bad = q == 0 && !wait(&sh.sums_full[b], (count / C::BUFS) & 1);
            asm volatile("{\n .reg .pred p, r;\n setp.ne.u32 p, %0, 0;\n barrier.cta.red.or.pred r, %1, 128, p;\n selp.u32 %0, 1, 0, r;\n}"
                         : "+r"(bad)
                         : "r"(1 + g)
                         : "memory");
            if (bad) {
                ok = false;
                break;
            }
            fence_after();
            float v[16 * C::PIECES * (DUAL ? 2 : 1)];  // the sums of the pieces, then those of `up`
            // of a full tile a group takes neighbouring pieces, of another every GROUPS-th
            const bool full = t.rows == C::NT;
            const uint32_t apart = full ? 16 : 16 * GROUPS, first = full ? 16 * C::PIECES * g : 16 * g;
            const uint32_t at = tmem + b * C::ONE + ((32 * q) << 16) + first;
            if (full) {
                if constexpr (C::PIECES == 4) tmem_ld32x64(at, v);
                else {
                    tmem_ld32x32(at, v);
                    if constexpr (C::PIECES == 3) tmem_ld32x16(at + 32, v + 32);
                }
                if (DUAL) tmem_ld32x32(at + C::NT, v + 32);
            } else {
#pragma unroll
                for (uint32_t c = 0; c < C::PIECES; c++)
                    if (t.rows > apart * c + first) {
                        tmem_ld32x16(at + apart * c, v + 16 * c);
                        if (DUAL) tmem_ld32x16(at + C::NT + apart * c, v + 16 * (C::PIECES + c));
                    }
            }
#pragma unroll
            for (uint32_t c = 0; c < C::PIECES * (DUAL ? 2 : 1); c++) tmem_wait(v + 16 * c);
            fence_before();
            __syncwarp();
            if (elect_one()) arrive_at(&sh.sums_empty[b], 0);
            __syncwarp();
            const uint32_t f0 = (2 * pair_of(i) + rank) * MX4_ROWS;
            if (f0 >= a.feats) continue;
            const Out<T, VEC> o(a, t.row0, f0, q, lane);
#pragma unroll
            for (uint32_t c = 0; c < C::PIECES; c++)
                if (t.rows > apart * c + first) {
                    const uint32_t from = apart * c + first;
                    float *p = v + 16 * c;
                    if (DUAL) {
#pragma unroll
                        for (int j = 0; j < 16; j++) p[j] = silu_times(p[j], p[16 * C::PIECES + j]);
                    }
                    put_piece(a, o, sizeof(T) == 2 ? buf + (turn & 1) * (OUT_BYTES / 2) : buf, p, from, t.rows - from, q, lane, g);
                    turn++;
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

template <typename C, typename T, bool VEC>
cudaError_t launch_as(const Mx4GemmArgs &a, uint64_t tiles, int sms, cudaStream_t s) {
    auto fn = mx4_many_kernel<C, T, VEC>;
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

template <typename C, typename T>
cudaError_t launch_vec(const Mx4GemmArgs &a, uint64_t tiles, int sms, cudaStream_t s) {
    return a.vec ? launch_as<C, T, true>(a, tiles, sms, s) : launch_as<C, T, false>(a, tiles, sms, s);
}
template <typename C>
cudaError_t launch_type(const Mx4GemmArgs &a, uint64_t tiles, int sms, cudaStream_t s) {
    return a.type == SG_F32 ? launch_vec<C, float>(a, tiles, sms, s) : a.type == SG_F16 ? launch_vec<C, __half>(a, tiles, sms, s) : launch_vec<C, __nv_bfloat16>(a, tiles, sms, s);
}

}  // namespace

cudaError_t mx4_many_launch(const Mx4GemmArgs &a, uint32_t x_rows, uint64_t token_tiles, int sms, cudaStream_t s) {
    const uint64_t tiles = token_tiles * ((a.feat_tiles + 1) / 2);
    if (a.up) return launch_type<Cfg<128, true>>(a, tiles, sms, s);
    return x_rows == 256 ? launch_type<Cfg<256, false>>(a, tiles, sms, s) : launch_type<Cfg<192, false>>(a, tiles, sms, s);
}

}  // namespace sg
