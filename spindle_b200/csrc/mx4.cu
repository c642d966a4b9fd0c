// mx4.cu — rows into microscaled 4-bit tiles (mx4.cuh) and back.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "mx4.cuh"
#include "tiled_block.cuh"

namespace sg {
using namespace tiled;

namespace {

template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Sixteen values of a row, as they are loaded.
template <typename T>
struct Raw {
    static constexpr int N = 16 * sizeof(T) / 16;
    uint4 w[N];
};
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T *p, bool there, Raw<T> &r) {
#pragma unroll
    for (int i = 0; i < Raw<T>::N; i++) r.w[i] = make_uint4(0, 0, 0, 0);
    if (!there) return;
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < Raw<T>::N; i++) r.w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    } else {
        T *t = reinterpret_cast<T *>(r.w);
#pragma unroll
        for (int i = 0; i < 16; i++) t[i] = p[i];
    }
}

// Eight codes, the first in the lowest bits.
__device__ __forceinline__ uint32_t codes8(const float *y) {
    uint32_t w;
    asm("{\n .reg .b8 a, b, c, d;\n"
        " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        " mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(w)
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    return w;
}

// The bits of the largest of sixteen magnitudes as f32 (an infinity or a NaN: at least 0x7F800000).  16-bit magnitudes are
// compared as they are, two at a time.
__device__ __forceinline__ uint32_t top16(const Raw<float> &r) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(r.w);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) top = max(top, w[i] & 0x7FFFFFFFu);
    return top;
}
template <typename T>
__device__ __forceinline__ uint32_t top16(const Raw<T> &r) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(r.w), m = 0x7FFF7FFFu;
    uint32_t t = w[0] & m;
#pragma unroll
    for (int i = 1; i < 7; i += 2) t = __vimax3_u16x2(t, w[i] & m, w[i + 1] & m);
    t = __vimax3_u16x2(t, w[7] & m, 0u);
    const uint32_t most = max(t >> 16, t & 0xFFFFu);
    return std::is_same<T, __nv_bfloat16>::value ? most << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)most)));
}
// The sixteen values times a power of two f.
__device__ __forceinline__ void scaled16(const Raw<float> &r, float f, float (&y)[16]) {
    const float *v = reinterpret_cast<const float *>(r.w);
#pragma unroll
    for (int i = 0; i < 16; i++) y[i] = v[i] * f;
}
__device__ __forceinline__ void scaled16(const Raw<__half> &r, float f, float (&y)[16]) {
    const __half2 *v = reinterpret_cast<const __half2 *>(r.w);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float2 t = __half22float2(v[i]);
        y[2 * i] = t.x * f, y[2 * i + 1] = t.y * f;
    }
}
__device__ __forceinline__ void scaled16(const Raw<__nv_bfloat16> &r, float f, float (&y)[16]) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(r.w);
#pragma unroll
    for (int i = 0; i < 8; i++) y[2 * i] = __uint_as_float(w[i] << 16) * f, y[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u) * f;
}

// Two lanes have the 32 values of a block: each gets its sixteen codes, both its scale byte.
template <typename T>
__device__ __forceinline__ uint2 quantize16(const Raw<T> &raw, uint32_t &scale) {
    uint32_t top = top16(raw);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    // the exponent of the largest, one more from 1.75 times a power of two on, less 2
    const int e = max((int)((top + 0x200000u) >> 23) - 2, 0);
    scale = top >= 0x7F800000u ? 255u : (uint32_t)e;               // (all 32 are NaN then, whatever their codes)
    float y[16];
    scaled16(raw, __uint_as_float((uint32_t)(254 - e) << 23), y);  // times 2^(127 - e), e at most 254
    return make_uint2(codes8(y), codes8(y + 8));
}

// A warp takes 1024 columns of a row, 512 at a time, all loads at once: a lane has sixteen values, two lanes a block of 32.
// A token that goes to several experts is read and quantized once.  What bounds it: instructions (160 for a lane's sixteen
// values, the issue slots 63 % busy) next to reading x (8191 x 4096 bf16: 18.2 us, 85 MB read and written at 4.7 TB/s; with eight
// values a lane 21.5).  Rows that do not begin on 16 bytes are loaded value by value: 41 us, f32 73 instead of 29.
constexpr uint32_t QUANT_TILES = 4, STEPS = QUANT_TILES / 2;

template <typename T, bool VEC>
__global__ void __launch_bounds__(MX4_QUANT_THREADS) mx4_quantize_kernel(const __grid_constant__ Mx4QuantArgs a) {
    // a lane's tile of the two, its chunk there, its half of the chunk's bytes
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, side = lane >> 4, chunk = lane >> 1 & 7u, part = lane & 1u;
    const uint32_t tile_bytes = mx4_tile_bytes(a.x_rows), half = mx4_scale_bytes(a.x_rows) / 2, rows_at_once = gridDim.x * (MX4_QUANT_THREADS / 32);
    if (a.early) grid_launch_dependents();
    // a row's place among the tiles, from its place among the sorted ones (-1: none; a plan that was filled anew for other tokens
    // than the host counts, by a replayed graph, leads nowhere outside)
    auto row_of = [&](int32_t pair, uint32_t place) -> int64_t {
        const uint32_t e = (uint32_t)pair < a.n_pairs ? (uint32_t)__ldg(a.ids + pair) : a.n_expert;
        if (e >= a.n_expert) return -1;
        const uint64_t row = (uint64_t)(uint32_t)__ldg(a.tiles + e) * a.x_rows + (place - (uint32_t)__ldg(a.first + e));
        return row < a.out_rows ? (int64_t)row : -1;
    };
    for (uint32_t kt0 = blockIdx.y * QUANT_TILES; kt0 < a.nk; kt0 += gridDim.y * QUANT_TILES) {
        const uint32_t kt = kt0 + side, col = kt * MX4_COLS + (lane & 15u) * 16;
        uint32_t turn = 0;
        int64_t ahead = -1;
        for (uint64_t i = blockIdx.x * (MX4_QUANT_THREADS / 32) + warp; i < a.n_rows; i += rows_at_once, turn = (turn + 1) & 31) {
            const T *src = static_cast<const T *>(a.x) + col;
            bool row_there = true;
            if (a.n_used) src += i * a.ld;
            else {
                const uint32_t e = (uint32_t)i / a.tile_rows, r = (uint32_t)i - e * a.tile_rows;
                src += e * a.ld_expert + r * a.ld;
                row_there = r < a.rows;
            }
            Raw<T> raw[STEPS];
#pragma unroll
            for (uint32_t u = 0; u < STEPS; u++) load16<T, VEC>(src + u * 2 * MX4_COLS, row_there && col + u * 2 * MX4_COLS < a.cols, raw[u]);
            // where it goes: of sorted rows the lanes look up the places of this one and the warp's next 31, of a token's
            // those of its pairs
            if (a.order) {
                if (turn == 0) {
                    const uint64_t j = i + (uint64_t)lane * rows_at_once;
                    const int32_t pair = j < a.n_rows ? __ldg(a.order + j) : -1;
                    ahead = pair < 0 ? -1 : row_of(pair, (uint32_t)j);
                }
            } else if (a.n_used) {
                const int32_t p = lane < a.n_used ? __ldg(a.place + i * a.n_used + lane) : -1;
                ahead = p < 0 ? -1 : row_of((int32_t)(i * a.n_used + lane), (uint32_t)p);
            }
            uint2 w[STEPS];
            uint32_t scale[STEPS];
#pragma unroll
            for (uint32_t u = 0; u < STEPS; u++)
                if (kt0 + 2 * u < a.nk) {
                    w[u] = quantize16(raw[u], scale[u]);
                    if (!row_there || col + u * 2 * MX4_COLS >= a.cols) scale[u] = 0;
                }
            auto put = [&](uint64_t row) {
                const uint32_t tile = (uint32_t)row / a.x_rows, r = (uint32_t)row - tile * a.x_rows;  // (rows are below 2^32)
                uint8_t *t = a.out + ((uint64_t)tile * a.nk + kt) * tile_bytes;
                uint8_t *code = t + mx4_code_at(r, chunk) + 8 * part, *sc = t + a.x_rows * 128 + mx4_scale_at(r, chunk, half);
#pragma unroll
                for (uint32_t u = 0; u < STEPS; u++)
                    if (kt + 2 * u < a.nk) {
                        *reinterpret_cast<uint2 *>(code + u * 2 * tile_bytes) = w[u];
                        if (part == 0) sc[u * 2 * tile_bytes] = (uint8_t)scale[u];
                    }
            };
            if (!a.n_used) put(i);
            else if (a.order) {
                const int64_t to = __shfl_sync(0xffffffffu, ahead, turn);
                if (to >= 0) put(to);
            } else
                for (uint32_t j = 0; j < a.n_used; j++) {
                    const int64_t to = __shfl_sync(0xffffffffu, ahead, j);
                    if (to >= 0) put(to);
                }
        }
    }
}

// The values of two codes.
__device__ __forceinline__ float2 values2(uint32_t byte) {
    uint32_t h;
    asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %1;\n cvt.rn.f16x2.e2m1x2 %0, a;\n}" : "=r"(h) : "r"(byte));
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// Eight values a lane of each of four tiles: a lane's 16-bit results are one 16-byte store beside its neighbours' (sixteen, as
// above, would be two with gaps: 22 us for 8191 x 4096 to bf16 against 15; value by value, to rows that do not begin on 16 bytes,
// 108).
template <typename T, bool VEC>
__global__ void __launch_bounds__(MX4_QUANT_THREADS) mx4_dequantize_kernel(const __grid_constant__ Mx4ReadArgs a) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, chunk = lane >> 2, rows_at_once = gridDim.x * (MX4_QUANT_THREADS / 32);
    for (uint32_t kt0 = blockIdx.y * QUANT_TILES; kt0 < a.nk; kt0 += gridDim.y * QUANT_TILES)
        for (uint64_t i = blockIdx.x * (MX4_QUANT_THREADS / 32) + warp; i < a.n_rows; i += rows_at_once) {
            const uint32_t e = (uint32_t)i / a.rows, r = (uint32_t)i - e * a.rows, row = e * a.tile_rows + r, in = row % MX4_ROWS;
            const uint8_t *t = a.data + ((uint64_t)(row / MX4_ROWS) * a.nk + kt0) * MX4_TILE;
            T *o = static_cast<T *>(a.out) + e * a.ld_expert + r * a.ld + kt0 * MX4_COLS + lane * 8;
            uint32_t w[QUANT_TILES], sc[QUANT_TILES];
#pragma unroll
            for (uint32_t u = 0; u < QUANT_TILES; u++)
                if (kt0 + u < a.nk) {
                    w[u] = __ldg(reinterpret_cast<const uint32_t *>(t + u * MX4_TILE + mx4_code_at(in, chunk) + 4 * (lane & 3)));
                    sc[u] = __ldg(t + u * MX4_TILE + MX4_ROWS * 128 + mx4_scale_at(in, chunk));
                }
#pragma unroll
            for (uint32_t u = 0; u < QUANT_TILES; u++) {
                if ((kt0 + u) * MX4_COLS + lane * 8 >= a.cols) break;
                const float s = mx4_scale(sc[u]);
                uint4 raw[8 * sizeof(T) / 16];
                T *v = reinterpret_cast<T *>(raw);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float2 f = values2(w[u] >> (8 * k));
                    v[2 * k] = narrow<T>(f.x * s), v[2 * k + 1] = narrow<T>(f.y * s);
                }
                if constexpr (VEC) {
#pragma unroll
                    for (uint32_t k = 0; k < 8 * sizeof(T) / 16; k++) reinterpret_cast<uint4 *>(o + u * MX4_COLS)[k] = raw[k];
                } else {
#pragma unroll
                    for (int k = 0; k < 8; k++) o[u * MX4_COLS + k] = v[k];
                }
            }
        }
}

// CTAs of eight rows, by stretches of 1024 columns; eight of them an SM at most, which go on to further rows.
dim3 row_grid(uint64_t rows, uint32_t nk, int sms) {
    const uint32_t parts = (nk + QUANT_TILES - 1) / QUANT_TILES, y = parts < 1024 ? parts : 1024;
    const uint64_t want = (rows + MX4_QUANT_THREADS / 32 - 1) / (MX4_QUANT_THREADS / 32), most = ((uint64_t)sms * 8 + y - 1) / y;
    return dim3((uint32_t)(want < most ? want : most), y);
}

template <typename T>
cudaError_t quantize_as(const Mx4QuantArgs &a, int sms, cudaStream_t s) {
    const dim3 grid = row_grid(a.n_rows, a.nk, sms);
    if (a.vec) mx4_quantize_kernel<T, true><<<grid, MX4_QUANT_THREADS, 0, s>>>(a);
    else mx4_quantize_kernel<T, false><<<grid, MX4_QUANT_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t dequantize_as(const Mx4ReadArgs &a, int sms, cudaStream_t s) {
    const dim3 grid = row_grid(a.n_rows, a.nk, sms);
    if (a.vec) mx4_dequantize_kernel<T, true><<<grid, MX4_QUANT_THREADS, 0, s>>>(a);
    else mx4_dequantize_kernel<T, false><<<grid, MX4_QUANT_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t mx4_quantize_launch(const Mx4QuantArgs &a, int32_t type, int sms, cudaStream_t s) {
    return type == SG_F32 ? quantize_as<float>(a, sms, s) : type == SG_F16 ? quantize_as<__half>(a, sms, s) : quantize_as<__nv_bfloat16>(a, sms, s);
}

cudaError_t mx4_dequantize_launch(const Mx4ReadArgs &a, int32_t type, int sms, cudaStream_t s) {
    return type == SG_F32 ? dequantize_as<float>(a, sms, s) : type == SG_F16 ? dequantize_as<__half>(a, sms, s) : dequantize_as<__nv_bfloat16>(a, sms, s);
}

}  // namespace sg
