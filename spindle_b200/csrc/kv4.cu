// kv4.cu — bookkeeping and rows of the paged 4-bit KV cache: block tables and
// slot maps from request lengths, rows quantized into the cache, rows read back.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv4.cuh"

namespace sg {

namespace {

template <typename T>
struct Conv;
template <>
struct Conv<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Conv<__half> {
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <>
struct Conv<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

__device__ __forceinline__ uint32_t warp_scan(uint32_t v, uint32_t lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= (uint32_t)o) v += u;
    }
    return v;
}

}  // namespace

// ---- plan -------------------------------------------------------------------
//
// Every CTA scans all requests (1024 at a time: new positions, blocks wanted,
// blocks given back), so one launch does without a grid-wide step, and fills its
// own stretch of the new positions: the request of a position by a binary search
// of the scan in shared memory.  A new block of a request starts exactly at the
// one new position that is a multiple of the page, so the thread of that
// position writes the table entry, and everyone else computes the block from the
// ring without reading it back.  A decode step of 64 requests is a launch (5 us); 1.5 million positions of 509
// requests 13 to 14 us, 1 TB/s of positions and slots, bound by the searches and the scan that every CTA repeats.
// Where the new lengths take the place of the old ones, which every CTA reads, a second launch of one CTA writes them.
__global__ void __launch_bounds__(KV4_PLAN_THREADS) kv4_plan_kernel(const __grid_constant__ Kv4PlanArgs a) {
    __shared__ uint32_t cu_s[KV4_PLAN_THREADS + 1], want_s[KV4_PLAN_THREADS];
    __shared__ int32_t ctx_s[KV4_PLAN_THREADS];
    __shared__ uint32_t warp_s[3][32], total_s[3];
    const uint32_t tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const uint32_t page = 1u << a.page_shift;
    const uint32_t head = (uint32_t)a.cursor[0], tail = (uint32_t)a.cursor[1], free_blocks = tail - head;
    const uint32_t per = ((a.max_tok + gridDim.x - 1) / gridDim.x + 3) & ~3u;
    const uint32_t t0 = min(a.max_tok, blockIdx.x * per), t1 = min(a.max_tok, t0 + per);
    uint32_t base_come = 0, base_want = 0, base_back = 0;

    for (uint32_t r0 = 0; r0 < a.n_req; r0 += KV4_PLAN_THREADS) {
        const uint32_t r = r0 + tid, n = min((uint32_t)KV4_PLAN_THREADS, a.n_req - r0);
        uint32_t ctx = 0, come = 0, want = 0, kept = 0, back = 0;
        bool ends = false;
        if (r < a.n_req) {
            const int32_t add = a.add[r];
            ctx = (uint32_t)max(a.ctx[r], 0);
            ends = add < 0;
            come = (uint32_t)max(add, 0);
            const uint32_t have = min((ctx + page - 1) >> a.page_shift, a.width);
            const uint32_t need = min((ctx + come + page - 1) >> a.page_shift, a.width);
            want = ends ? 0 : need - have;
            kept = ends ? have : 0;
        }
        // what a request that ends gives back: its entries that are blocks, counted a warp per request
        for (uint32_t todo = __ballot_sync(0xffffffffu, kept > 0); todo; todo &= todo - 1) {
            const int src = __ffs(todo) - 1;
            const uint32_t cnt = __shfl_sync(0xffffffffu, kept, src);
            const int32_t *row = a.tables + (uint64_t)(r0 + wid * 32 + src) * a.ld_tables;
            uint32_t valid = 0;
            for (uint32_t j = lane; j < cnt; j += 32) valid += (uint32_t)row[j] < a.n_blocks;
            valid = __reduce_add_sync(0xffffffffu, valid);
            if (lane == (uint32_t)src) back = valid;
        }
        const uint32_t s0 = warp_scan(come, lane), s1 = warp_scan(want, lane), s2 = warp_scan(back, lane);
        if (lane == 31) warp_s[0][wid] = s0, warp_s[1][wid] = s1, warp_s[2][wid] = s2;
        __syncthreads();
        if (wid < 3) {
            const uint32_t v = warp_s[wid][lane], inc = warp_scan(v, lane);
            warp_s[wid][lane] = inc - v;
            if (lane == 31) total_s[wid] = inc;
        }
        __syncthreads();
        const uint32_t c0 = base_come + warp_s[0][wid] + s0 - come;
        cu_s[tid] = c0;
        want_s[tid] = base_want + warp_s[1][wid] + s1 - want;
        ctx_s[tid] = (int32_t)ctx;
        const uint32_t back_at = base_back + warp_s[2][wid] + s2 - back;
        if (tid == 0) cu_s[KV4_PLAN_THREADS] = base_come + total_s[0];
        if (blockIdx.x == 0 && r < a.n_req && a.lengths) {
            a.cu[r] = (int32_t)c0;
            a.seq[r] = ends ? 0 : (int32_t)(ctx + come);
        }
        __syncthreads();
        // the blocks of the requests that end go back to the ring's tail, in table order, a warp per request
        for (uint32_t todo = __ballot_sync(0xffffffffu, back > 0 && (r % gridDim.x) == blockIdx.x); todo; todo &= todo - 1) {
            const int src = __ffs(todo) - 1;
            const uint32_t cnt = __shfl_sync(0xffffffffu, kept, src);
            uint32_t at = tail + __shfl_sync(0xffffffffu, back_at, src);
            const int32_t *row = a.tables + (uint64_t)(r0 + wid * 32 + src) * a.ld_tables;
            for (uint32_t j0 = 0; j0 < cnt; j0 += 32) {
                const int32_t block = j0 + lane < cnt ? row[j0 + lane] : -1;
                const uint32_t is = __ballot_sync(0xffffffffu, (uint32_t)block < a.n_blocks);
                if ((uint32_t)block < a.n_blocks) a.ring[(at + __popc(is & ((1u << lane) - 1))) % a.n_blocks] = block;
                at += __popc(is);
            }
        }
        // this CTA's new positions among these requests, four neighbours a thread: one search, and a table entry
        // looked up again where the request or the page changes
        const uint32_t lo = max(t0, base_come), hi = min(t1, base_come + total_s[0]);
        for (uint32_t q = (lo & ~3u) + tid * 4; q < hi; q += KV4_PLAN_THREADS * 4) {
            uint32_t x = 0, y = n;  // the last request with cu <= the first position
            const uint32_t first = max(q, lo), last = min(q + 4, hi);
            while (y - x > 1) {
                const uint32_t m = (x + y) >> 1;
                if (cu_s[m] <= first) x = m;
                else y = m;
            }
            int32_t block = -1, pos4[4], slot4[4];
            uint32_t known = ~0u;  // the page that block is of
            for (uint32_t t = first; t < last; t++) {
                while (x + 1 < n && cu_s[x + 1] <= t) x++, known = ~0u;
                const uint32_t c = (uint32_t)ctx_s[x], pos = c + (t - cu_s[x]), j = pos >> a.page_shift;
                if (j != known) {
                    const uint32_t have = min((c + page - 1) >> a.page_shift, a.width);
                    int32_t *row = a.tables + (uint64_t)(r0 + x) * a.ld_tables;
                    block = -1;
                    if (j < have) {
                        block = row[j];
                    } else if (j < a.width) {
                        const uint32_t k = want_s[x] + j - have;
                        if (k < free_blocks) block = a.ring[(head + k) % a.n_blocks];
                        if ((pos & (page - 1)) == 0) row[j] = block;
                    }
                    known = j;
                }
                pos4[t & 3] = (int32_t)pos;
                slot4[t & 3] = (uint32_t)block < a.n_blocks ? block * (int32_t)page + (int32_t)(pos & (page - 1)) : -1;
            }
            if (a.vec && last - first == 4) {
                *reinterpret_cast<int4 *>(a.pos + q) = make_int4(pos4[0], pos4[1], pos4[2], pos4[3]);
                *reinterpret_cast<int4 *>(a.slots + q) = make_int4(slot4[0], slot4[1], slot4[2], slot4[3]);
            } else {
                for (uint32_t t = first; t < last; t++) a.pos[t] = pos4[t & 3], a.slots[t] = slot4[t & 3];
            }
        }
        base_come += total_s[0];
        base_want += total_s[1];
        base_back += total_s[2];
        __syncthreads();
    }
    for (uint32_t t = max(t0, min(base_come, t1)) + tid; t < t1; t += KV4_PLAN_THREADS) a.pos[t] = a.slots[t] = -1;
    if (blockIdx.x == 0 && tid == 0 && a.lengths) {
        const uint32_t taken = min(base_want, free_blocks);
        a.cu[a.n_req] = (int32_t)base_come;
        const uint32_t turn = (head + taken) / a.n_blocks * a.n_blocks;  // the head stays inside the ring
        a.info[0] = (int32_t)(head + taken - turn);
        a.info[1] = (int32_t)(tail + base_back - turn);
        a.info[2] = (int32_t)base_come;
        a.info[3] = (int32_t)(base_want - taken);
    }
}

// ---- append -------------------------------------------------------------------
//
// Two lanes per group of 32 values, sixteen values each: lane i's are the K words
// j = 2 i and 2 i + 1 of the group, and its V half words 4 i .. 4 i + 3.
//   m = f16(min), s = f16((max - m) * f32(1/15)), c = rint(clamp((x - m) * (1 / s), 0, 15))
// with x clamped to f16's finite range, NaN counted as 0, and s the next smaller
// f16 where m + 15 s >= 65520, which is infinity in f16, so that the cache holds
// finite numbers only; groups that had an infinity or a NaN are counted.  Every
// step is one rounded f32 operation, so the codes can be reproduced bit for bit.
// What bounds it is the arithmetic (20 instructions a value by the counters), hence sixteen
// values a lane: the place of a row in the cache is worked out half as often.
// 24001 rows of 8 heads of 128 in bf16: 44 us, 2.9 TB/s (45 % of the measured copy rate); 32 rows are a launch.

// The larger and the smaller one, NaN if either is.
__device__ __forceinline__ float max_nan(float x, float y) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(x), "f"(y));
    return d;
}
__device__ __forceinline__ float min_nan(float x, float y) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(x), "f"(y));
    return d;
}

// Which sixteen values a lane has: token t, head h, K or V, group g, half i of it.
struct Place {
    uint32_t t, h, g, i;
    bool is_v;
};
template <int D>
__device__ __forceinline__ Place place_of(uint32_t f, uint32_t heads) {
    constexpr uint32_t G = D / 32;
    const uint32_t per_tok = heads * G * 4;  // lanes of a token: K's, then V's, head by head, two a group
    const uint32_t t = f / per_tok, u = f - t * per_tok, hv = u / (2 * G);
    return {t, hv >= heads ? hv - heads : hv, u / 2 % G, u % 2, hv >= heads};
}
// The tile of a slot, and the position inside it.
template <int D>
__device__ __forceinline__ uint8_t *tile_of(const Kv4Cache &c, int32_t slot, uint32_t h, uint32_t &p) {
    const uint32_t at = (uint32_t)slot & ((1u << c.page_shift) - 1);
    p = at & 15;
    return c.data + ((((uint64_t)((uint32_t)slot >> c.page_shift) * c.heads + h) << (c.page_shift - 4)) + (at >> 4)) * (uint64_t)Kv4Tile<D>::BYTES;
}

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(KV4_ROW_THREADS) kv4_append_kernel(const __grid_constant__ Kv4RowArgs a) {
    using L = Kv4Tile<D>;
    constexpr uint32_t G = L::G;
    for (uint32_t f = blockIdx.x * KV4_ROW_THREADS + threadIdx.x; f - threadIdx.x % 32 < a.lanes; f += gridDim.x * KV4_ROW_THREADS) {
        const bool live = f < a.lanes;
        const Place q = place_of<D>(live ? f : a.lanes - 1, a.c.heads);
        const int32_t slot = a.slots[q.t];
        const T *src = (const T *)(q.is_v ? a.v : a.k) + q.t * (q.is_v ? a.v_tok : a.k_tok) + q.h * (q.is_v ? a.v_head : a.k_head) +
                       q.g * 32 + q.i * 16;
        alignas(16) T raw[16];
        if (VEC) {
#pragma unroll
            for (int w = 0; w < (int)sizeof(T); w++) reinterpret_cast<uint4 *>(raw)[w] = __ldg(reinterpret_cast<const uint4 *>(src) + w);
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) raw[e] = src[e];
        }
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = Conv<T>::get(raw[e]);
        float lo = x[0], hi = x[0];
#pragma unroll
        for (int e = 1; e < 16; e++) lo = min_nan(lo, x[e]), hi = max_nan(hi, x[e]);
        const bool bad = !(lo >= -3.4028235e38f && hi <= 3.4028235e38f);  // a NaN or an infinity
        if (bad) {
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = x[e] == x[e] ? x[e] : 0.0f;
            lo = hi = x[0];
#pragma unroll
            for (int e = 1; e < 16; e++) lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]);
        }
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, 1));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
        lo = fminf(fmaxf(lo, -65504.0f), 65504.0f);
        hi = fminf(fmaxf(hi, -65504.0f), 65504.0f);
        const __half mh = __float2half_rn(lo + 0.0f);  // + 0: no negative zero
        const float m = __half2float(mh);
        __half sh = __float2half_rn(__fmul_rn(fmaxf(hi - m, 0.0f), 1.0f / 15.0f));
        // a step that was rounded up so far that the largest value would be infinite in f16: the next smaller one
        if (fmaf(15.0f, __half2float(sh), m) >= 65520.0f) sh = __ushort_as_half(__half_as_ushort(sh) - 1);
        const float s = __half2float(sh), r = s > 0.0f ? __frcp_rn(s) : 0.0f;
        uint32_t word[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 16; e++) {
            // to an unsigned number, below 0 and NaN to 0; a value beyond the clamped ends falls on their codes
            const uint32_t c = min(__float2uint_rn(__fmul_rn(__fsub_rn(x[e], m), r)), 15u);
            word[e / 8] += c << (4 * (e % 8));
        }
        const unsigned any = __ballot_sync(0xffffffffu, bad && live) >> (threadIdx.x & 30) & 3;
        if (!live || slot < 0 || (uint32_t)(slot >> a.c.page_shift) >= a.c.n_blocks) continue;
        if (any && q.i == 0 && a.nonfinite) atomicAdd(a.nonfinite, 1);
        uint32_t p;
        uint8_t *tile = tile_of<D>(a.c, slot, q.h, p);
        const uint32_t pair = ((p >> 1) * G + q.g) * 2 + (p & 1);
        if (q.is_v) {
            uint8_t *v = tile + L::VC + (p >> 1) * L::VROW + (p & 1) * 2;
#pragma unroll
            for (int k = 0; k < 4; k++) *reinterpret_cast<uint16_t *>(v + kv4_word(4 * q.i + k, q.g, 8, G) * 4) = (uint16_t)(word[k / 2] >> (k % 2 * 16));
            reinterpret_cast<__half *>(tile + (q.i ? L::VM : L::VS))[pair] = q.i ? mh : sh;
        } else {
#pragma unroll
            for (int k = 0; k < 2; k++) *reinterpret_cast<uint32_t *>(tile + p * L::KROW + kv4_word(2 * q.i + k, q.g, 4, G) * 4) = word[k];
            if (q.i) reinterpret_cast<__half *>(tile + L::KM)[p * G + q.g] = mh;
            else reinterpret_cast<__half *>(tile + L::KS)[pair] = sh;
        }
    }
}

// ---- read ---------------------------------------------------------------------
// The values of given slots, m + s * c rounded once; a slot that is no slot reads as zeros.  The rows above to f16:
// 32 us, 4.0 TB/s, bound by unpacking (13 instructions a value).
template <typename T, int D>
__global__ void __launch_bounds__(KV4_ROW_THREADS) kv4_read_kernel(const __grid_constant__ Kv4RowArgs a) {
    using L = Kv4Tile<D>;
    constexpr uint32_t G = L::G;
    for (uint32_t f = blockIdx.x * KV4_ROW_THREADS + threadIdx.x; f < a.lanes; f += gridDim.x * KV4_ROW_THREADS) {
        const Place q = place_of<D>(f, a.c.heads);
        const int32_t slot = a.slots[q.t];
        uint32_t word[2] = {0, 0};
        float s = 0.0f, m = 0.0f;
        if (slot >= 0 && (uint32_t)(slot >> a.c.page_shift) < a.c.n_blocks) {
            uint32_t p;
            const uint8_t *tile = tile_of<D>(a.c, slot, q.h, p);
            const uint32_t pair = ((p >> 1) * G + q.g) * 2 + (p & 1);
            if (q.is_v) {
                const uint8_t *v = tile + L::VC + (p >> 1) * L::VROW + (p & 1) * 2;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    word[k / 2] |= (uint32_t) * reinterpret_cast<const uint16_t *>(v + kv4_word(4 * q.i + k, q.g, 8, G) * 4) << (k % 2 * 16);
                s = __half2float(reinterpret_cast<const __half *>(tile + L::VS)[pair]);
                m = __half2float(reinterpret_cast<const __half *>(tile + L::VM)[pair]);
            } else {
#pragma unroll
                for (int k = 0; k < 2; k++) word[k] = *reinterpret_cast<const uint32_t *>(tile + p * L::KROW + kv4_word(2 * q.i + k, q.g, 4, G) * 4);
                s = __half2float(reinterpret_cast<const __half *>(tile + L::KS)[pair]);
                m = __half2float(reinterpret_cast<const __half *>(tile + L::KM)[p * G + q.g]);
            }
        }
        alignas(16) T y[16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float c = __uint_as_float((word[e / 8] >> (4 * (e % 8)) & 15u) | 0x4B000000u) - 8388608.0f;  // 2^23 + c
            y[e] = Conv<T>::put(fmaf(s, c, m));
        }
        uint4 *dst = reinterpret_cast<uint4 *>((T *)(q.is_v ? a.v_out : a.k_out) + ((uint64_t)q.t * a.c.heads + q.h) * D + q.g * 32 + q.i * 16);
#pragma unroll
        for (int w = 0; w < (int)sizeof(T); w++) dst[w] = reinterpret_cast<const uint4 *>(y)[w];
    }
}

namespace {
template <typename T, bool VEC>
kv4_row_fn pick_append(uint32_t d) {
    return d == 64 ? kv4_append_kernel<T, 64, VEC> : d == 128 ? kv4_append_kernel<T, 128, VEC> : kv4_append_kernel<T, 256, VEC>;
}
template <typename T>
kv4_row_fn pick_read(uint32_t d) {
    return d == 64 ? kv4_read_kernel<T, 64> : d == 128 ? kv4_read_kernel<T, 128> : kv4_read_kernel<T, 256>;
}
}  // namespace

kv4_row_fn kv4_append_kernel_for(int32_t type, uint32_t d, bool vec) {
    if (type == SG_F32) return vec ? pick_append<float, true>(d) : pick_append<float, false>(d);
    if (type == SG_F16) return vec ? pick_append<__half, true>(d) : pick_append<__half, false>(d);
    return vec ? pick_append<__nv_bfloat16, true>(d) : pick_append<__nv_bfloat16, false>(d);
}

kv4_row_fn kv4_read_kernel_for(int32_t type, uint32_t d) {
    return type == SG_F32 ? pick_read<float>(d) : type == SG_F16 ? pick_read<__half>(d) : pick_read<__nv_bfloat16>(d);
}

}  // namespace sg
