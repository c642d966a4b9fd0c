// kv4.cuh — the paged KV cache held in 4 bits: layout, and the launch
// interfaces of the plan, append, read and attention kernels.
//
// The cache is n_blocks blocks of `page` positions.  For one KV head a block is
// page / 16 tiles of 16 positions, TILE = 20 * D bytes each, one after the
// other; the heads of a block follow each other.  With D = head_dim and G =
// D / 32 groups of 32 values (a value is m + s * c: c a code of 4 bits, s and m
// f16), a tile holds
//   K codes   [16 positions][D / 2 bytes]
//   V codes   [8 pairs of positions][D bytes]
//   K scales  [8 pairs][G][2] f16        K minima  [16 positions][G] f16
//   V scales  [8 pairs][G][2] f16        V minima  [8 pairs][G][2] f16
// so that one bulk copy brings everything a warp needs of 16 positions, and each
// lane's part of an m16n8k16 operand is whole aligned words:
//   K: the word kv4_word(j, g, 4) of a position holds the values d = 32 g + 8 j + n
//      in its nibbles n = 0..7 (lane j of a quad has all groups side by side);
//   V: the word kv4_word(j, g, 8) of a pair holds d = 32 g + 4 j + n in the
//      nibbles n = 0..3 of its low half for the even position and of its high
//      half for the odd one (the two halves of an f16x2 register after a mask).
#pragma once

#include "common.cuh"

namespace sg {

// Word index of (lane part j of J, group g) inside a position's or pair's codes;
// four groups of one j are 16 bytes.
__host__ __device__ constexpr uint32_t kv4_word(uint32_t j, uint32_t g, uint32_t J, uint32_t G) {
    return G < 4 ? j * G + g : ((g / 4) * J + j) * 4 + g % 4;
}

template <int D>
struct Kv4Tile {
    static constexpr uint32_t G = D / 32;
    static constexpr uint32_t KROW = D / 2, VROW = D;           // bytes of a position's K codes, of a pair's V codes
    static constexpr uint32_t VC = 8 * D, KS = 16 * D, KM = 17 * D, VS = 18 * D, VM = 19 * D, BYTES = 20 * D;
};

// The codes of a word as f16 pairs, c - OFF of the nibbles (0, 4), (1, 5), (2, 6), (3, 7): a nibble in the lowest
// mantissa bits of 1024, or four bits up in those of 64, less that number (the well-known way to turn small integers into
// floating point by their mantissa bits).  The masks and numbers are kept in registers
// that the compiler does not see through, so that mask and insertion are one instruction (which takes one immediate).
struct Kv4Codes {
    uint32_t k0, k1, m0, m1;
    __device__ __forceinline__ Kv4Codes() {
        asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(k0));
        asm volatile("mov.b32 %0, 0x00F000F0;" : "=r"(k1));
        asm volatile("mov.b32 %0, 0x64006400;" : "=r"(m0));
        asm volatile("mov.b32 %0, 0x54005400;" : "=r"(m1));
    }
    static __device__ __forceinline__ uint32_t put(uint32_t w, uint32_t k, uint32_t m) {
        uint32_t d;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(k), "r"(m));  // (w & k) | m
        return d;
    }
    static __device__ __forceinline__ uint32_t less(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    template <int OFF>
    __device__ __forceinline__ void get(uint32_t w, uint32_t (&c)[4]) const {
        const uint32_t o0 = OFF ? 0x64006400u + OFF * 0x00010001u : m0, o1 = OFF ? 0x54005400u + OFF * 0x00100010u : m1, h = w >> 8;
        c[0] = less(put(w, k0, m0), o0);
        c[1] = less(put(w, k1, m1), o1);
        c[2] = less(put(h, k0, m0), o0);
        c[3] = less(put(h, k1, m1), o1);
    }
};

// A result in f16.  It is a mean of values that are finite in f16, so its true value is, but the weights' sum is 1 only up
// to their rounding (2^-12 of it in the kernel for many rows): what that carries past the end of the range stays there.
__device__ __forceinline__ __half kv4_f16(float v) {
    return __float2half_rn(fabsf(v) > 65504.0f ? copysignf(65504.0f, v) : v);
}

struct Kv4Cache {
    uint8_t *data;
    uint32_t n_blocks, page_shift;  // page = 1 << page_shift positions
    uint32_t heads;
};

struct Kv4PlanArgs {
    const int32_t *ctx, *add;
    int32_t *tables;
    uint64_t ld_tables;
    int32_t *ring;
    const int32_t *cursor;
    int32_t *cu, *seq, *pos, *slots, *info;
    uint32_t n_req, max_tok, width, page_shift, n_blocks;
    bool vec;  // pos and slots allow 16-byte stores
    bool lengths;  // this launch writes cu, seq and info
};

struct Kv4RowArgs {
    Kv4Cache c;
    const void *k, *v;                 // append: the rows
    uint64_t k_tok, k_head, v_tok, v_head;  // strides in elements
    void *k_out, *v_out;               // read: [n_tok][heads][D]
    const int32_t *slots;
    int32_t *nonfinite;
    uint32_t lanes;  // tokens * heads * D / 8: a lane per sixteen values of K or V
};

struct Kv4AttnArgs {
    Kv4Cache c;
    const void *q;
    void *out;
    float *lse;
    uint64_t q_tok, q_head, o_tok, o_head;  // strides in elements
    const int32_t *cu, *seq, *tables;
    uint64_t ld_tables;
    uint32_t width, n_req, n_tok, n_heads, group, window, max_new;
    float scale;
    uint8_t *scratch;
    uint64_t block_bytes;  // of one block, all heads
    bool vec_q, vec_out;  // the rows allow 16-byte accesses
    bool first, last;     // this launch's requests are the first ones, the last ones
    uint32_t head0, n_kv; // and its KV heads
};

constexpr int KV4_PLAN_THREADS = 1024;
__global__ void kv4_plan_kernel(const __grid_constant__ Kv4PlanArgs a);

typedef void (*kv4_row_fn)(const Kv4RowArgs);
// type: SG_F32, SG_F16 or SG_BF16; vec: rows and strides allow 16-byte loads
kv4_row_fn kv4_append_kernel_for(int32_t type, uint32_t d, bool vec);
kv4_row_fn kv4_read_kernel_for(int32_t type, uint32_t d);
constexpr int KV4_ROW_THREADS = 256;

// Attention scratch: partial results of requests whose positions are spread over
// several CTAs, and their arrival counters (zero between calls).
constexpr uint64_t KV4_SCRATCH_BYTES = 16ull << 20;
// The tensor-core kernel for many rows a head, and whether it is the faster one.
cudaError_t kv4_prefill_launch(const Kv4AttnArgs &a, int32_t type, uint32_t d, cudaStream_t s);
bool kv4_prefill_pays(const Kv4AttnArgs &a, int32_t type, uint32_t d, int sms);
sg_status kv4_attention_launch(const Kv4AttnArgs &a, int32_t type, uint32_t d, int sms, cudaStream_t s, cudaError_t *err);

}  // namespace sg
