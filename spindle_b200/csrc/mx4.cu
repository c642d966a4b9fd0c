// mx4.cu — rows into microscaled 4-bit tiles (mx4.cuh) and back.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mx4.cuh"
#include "tiled_block.cuh"

namespace sg {
using namespace tiled;

namespace {

template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight values of a row from column c on.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    if constexpr (VEC) {
        constexpr int N = 16 / sizeof(T);
        uint4 w[8 / N];
#pragma unroll
        for (int i = 0; i < 8 / N; i++) w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
        const T *t = reinterpret_cast<const T *>(w);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = widen(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = widen(p[i]);
    }
}

// Eight codes, the first in the lowest bits.
__device__ __forceinline__ uint32_t codes8(const float (&y)[8]) {
    uint32_t w;
    asm("{\n .reg .b8 a, b, c, d;\n"
        " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        " mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(w)
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    return w;
}

// Four lanes have the 32 values of a block: each gets its eight codes, all its scale byte.
__device__ __forceinline__ uint32_t quantize8(const float (&v)[8], uint32_t &scale) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);  // an infinity or a NaN: the largest
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // the exponent of the largest, one more from 1.75 times a power of two on, less 2
    const int e = max((int)((top + 0x200000u) >> 23) - 2, 0);
    const bool bad = top >= 0x7F800000u;
    scale = bad ? 255u : (uint32_t)e;
    const float f = __uint_as_float((uint32_t)(254 - e) << 23);  // 2^(127 - e), e at most 253
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = bad ? 0.0f : v[i] * f;
    return codes8(y);
}

// Where a quantized row goes: its tiles along the columns and its place in them.
struct Dest {
    uint8_t *tile;
    uint32_t row;
};

// A warp takes a row's 256 columns of a tile: four lanes a block of 32.  What bounds it: reading x (and, where a token goes
// to several experts, writing its copies; it is read and quantized once for all of them).
template <typename T, bool VEC>
__global__ void __launch_bounds__(MX4_QUANT_THREADS) mx4_quantize_kernel(const __grid_constant__ Mx4QuantArgs a) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, chunk = lane >> 2;
    const uint64_t items = a.n_rows * a.nk, step = (uint64_t)gridDim.x * (MX4_QUANT_THREADS / 32);
    const uint32_t tile_bytes = mx4_tile_bytes(1u << a.tile_shift), mask = (1u << a.tile_shift) - 1;
    for (uint64_t at = (uint64_t)blockIdx.x * (MX4_QUANT_THREADS / 32) + warp; at < items; at += step) {
        const uint64_t i = at / a.nk;
        const uint32_t kt = (uint32_t)(at - i * a.nk), col = kt * MX4_COLS + lane * 8;
        const T *src = static_cast<const T *>(a.x);
        bool there = col < a.cols;
        if (a.n_used) src += i * a.ld;
        else {
            const uint64_t e = i / a.tile_rows, r = i - e * a.tile_rows;
            src += e * a.ld_expert + r * a.ld;
            there = there && r < a.rows;
        }
        float v[8] = {};
        if (there) load8<T, VEC>(src + col, v);
        uint32_t scale;
        const uint32_t w = quantize8(v, scale);
        // the scale bytes of four blocks make a word
        uint32_t s4 = (there ? scale : 0u) << (8 * (chunk & 3));
        s4 |= __shfl_xor_sync(0xffffffffu, s4, 4);
        s4 |= __shfl_xor_sync(0xffffffffu, s4, 8);
        auto put = [&](uint64_t row) {
            uint8_t *t = a.out + ((row >> a.tile_shift) * a.nk + kt) * tile_bytes;
            const uint32_t r = (uint32_t)row & mask;
            *reinterpret_cast<uint32_t *>(t + mx4_code_at(r, chunk) + 4 * (lane & 3)) = w;
            if ((lane & 15) == 0) *reinterpret_cast<uint32_t *>(t + (mask + 1) * 128 + mx4_scale_at(r, chunk)) = s4;
        };
        if (!a.n_used) put(i);
        else if (a.order) {
            const int32_t pair = __ldg(a.order + i);
            if (pair >= 0) {
                const int32_t e = __ldg(a.ids + pair);
                put(((uint64_t)__ldg(a.tiles + e) << a.tile_shift) + (i - __ldg(a.first + e)));
            }
        } else {
            for (uint32_t j = 0; j < a.n_used; j++) {
                const uint64_t pair = i * a.n_used + j;
                const int32_t p = __ldg(a.place + pair);
                if (p < 0) continue;
                const int32_t e = __ldg(a.ids + pair);
                put(((uint64_t)__ldg(a.tiles + e) << a.tile_shift) + (p - __ldg(a.first + e)));
            }
        }
    }
    grid_launch_dependents();
}

// The value of a code's 4 bits.
__device__ __forceinline__ float code_value(uint32_t c) {
    const uint32_t m = c & 7;
    // 0 and 0.5 below the first exponent, then 1 + the last bit's half
    const float v = m < 2 ? 0.5f * m : __uint_as_float((126u + (m >> 1)) << 23 | (m & 1) << 22);
    return c & 8 ? -v : v;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(MX4_QUANT_THREADS) mx4_dequantize_kernel(const __grid_constant__ Mx4ReadArgs a) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, chunk = lane >> 2;
    const uint64_t items = a.n_rows * a.nk, step = (uint64_t)gridDim.x * (MX4_QUANT_THREADS / 32);
    for (uint64_t at = (uint64_t)blockIdx.x * (MX4_QUANT_THREADS / 32) + warp; at < items; at += step) {
        const uint64_t i = at / a.nk, e = i / a.rows, r = i - e * a.rows, row = e * a.tile_rows + r;
        const uint32_t kt = (uint32_t)(at - i * a.nk), col = kt * MX4_COLS + lane * 8, in = (uint32_t)row % MX4_ROWS;
        if (col >= a.cols) continue;
        const uint8_t *t = a.data + (row / MX4_ROWS * a.nk + kt) * MX4_TILE;
        const uint32_t w = __ldg(reinterpret_cast<const uint32_t *>(t + mx4_code_at(in, chunk) + 4 * (lane & 3)));
        const float s = mx4_scale(__ldg(t + MX4_ROWS * 128 + mx4_scale_at(in, chunk)));
        T v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = narrow<T>(code_value(w >> (4 * k) & 15) * s);
        T *o = static_cast<T *>(a.out) + e * a.ld_expert + r * a.ld + col;
        if constexpr (VEC) {
#pragma unroll
            for (uint32_t k = 0; k < 8 * sizeof(T) / 16; k++) reinterpret_cast<uint4 *>(o)[k] = reinterpret_cast<const uint4 *>(v)[k];
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) o[k] = v[k];
        }
    }
}

uint32_t row_grid(uint64_t items, int sms) {
    const uint64_t want = (items + MX4_QUANT_THREADS / 32 - 1) / (MX4_QUANT_THREADS / 32);
    return (uint32_t)(want < (uint64_t)sms * 16 ? want : (uint64_t)sms * 16);
}

template <typename T>
cudaError_t quantize_as(const Mx4QuantArgs &a, int sms, cudaStream_t s) {
    const uint32_t grid = row_grid(a.n_rows * a.nk, sms);
    if (a.vec) mx4_quantize_kernel<T, true><<<grid, MX4_QUANT_THREADS, 0, s>>>(a);
    else mx4_quantize_kernel<T, false><<<grid, MX4_QUANT_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t dequantize_as(const Mx4ReadArgs &a, int sms, cudaStream_t s) {
    const uint32_t grid = row_grid(a.n_rows * a.nk, sms);
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
