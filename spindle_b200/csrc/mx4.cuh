// mx4.cuh — microscaled 4-bit matrices: layout, and the launch interfaces of the
// kernels on them and of the sorting of tokens by expert.
//
// A matrix holds 32 values along a row as c * 2^(s - 127): s one byte, c of 4 bits
// (sign, and one of 0 0.5 1 1.5 2 3 4 6), the numbers that tcgen05's kind::mxf4
// multiplies as they are.  It is stored as tiles of 128 rows by 256 columns, the tiles
// of a stretch of rows one after the other along the columns; a tile is
//   codes   [128 rows][8 chunks of 32 values, 16 bytes each], chunk c of row r at
//           place c ^ (r & 7): the 128-byte swizzle of a K-major operand in shared memory;
//   scales  [2 halves of 128 columns][32][4][4]: the byte of row r, chunk 4 h + j at
//           512 h + 16 (r % 32) + 4 (r / 32) + j: a block of 32 rows by 16 bytes that
//           tcgen05.cp spreads over TMEM as the tensor cores take scales.
// So one bulk copy of 17408 contiguous bytes brings a stage of an operand, without a
// tensor map.  Rows past the last are zeros in a matrix; columns past the last are too
// (codes 0, scale byte 0).  Quantized activations have the same form with 32, 128, 192 or
// 256 rows a tile (codes of that many rows, then the scales; of more than 128 rows a half's are
// two such blocks, the second of rows 128 on).
#pragma once

#include "common.cuh"

namespace sg {

constexpr uint32_t MX4_ROWS = 128, MX4_COLS = 256;             // of a tile
constexpr uint32_t MX4_SCALES = 1024;                          // bytes of a tile's scales, of up to 128 rows
__host__ __device__ constexpr uint32_t mx4_scale_bytes(uint32_t rows) { return rows > 128 ? 2 * MX4_SCALES : MX4_SCALES; }
__host__ __device__ constexpr uint32_t mx4_tile_bytes(uint32_t rows) { return rows * 128 + mx4_scale_bytes(rows); }
constexpr uint32_t MX4_TILE = mx4_tile_bytes(MX4_ROWS);

// In a tile: the byte of a row's chunk of 32 codes, and of its scale (after the codes).
__host__ __device__ __forceinline__ uint32_t mx4_code_at(uint32_t row, uint32_t chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }
// (half: bytes of a half of the columns, 512 for up to 128 rows)
__host__ __device__ __forceinline__ uint32_t mx4_scale_at(uint32_t row, uint32_t chunk, uint32_t half = 512) {
    return (chunk >> 2) * half + (row >> 7) * 512 + (row & 31) * 16 + ((row >> 5 & 3) << 2) + (chunk & 3);
}

// 2^(s - 127) of a scale byte; 255 is NaN.
__device__ __forceinline__ float mx4_scale(uint32_t s) {
    return __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7FC00000u : s << 23);
}

// Rows of x, quantized into tiles.
struct Mx4QuantArgs {
    const void *x;
    uint64_t ld, ld_expert;        // in elements
    uint8_t *out;
    uint32_t cols, nk;             // nk: tiles along the columns
    uint32_t x_rows;               // rows of a tile
    uint64_t n_rows;               // rows that are read; of a matrix: all rows of its tiles
    // a matrix of several experts (n_used 0): rows each, and rows of its tiles each
    uint32_t rows, tile_rows;
    // rows that go to sorted places (n_used > 0): with order, row i is sorted place i; without, it goes to the
    // places of the pairs i * n_used + 0..
    uint32_t n_used;
    const int32_t *ids, *place, *order, *first, *tiles;
    uint32_t n_pairs, n_expert;    // what the host knows of them: nothing is read or written past these and out_rows
    uint64_t out_rows;             // rows of the tiles that out has room for
    bool vec;                      // x allows 16-byte loads
    bool early;                    // the next launch may begin at once: it waits for this one before it reads what is written here
};
constexpr uint32_t MX4_QUANT_THREADS = 256;
cudaError_t mx4_quantize_launch(const Mx4QuantArgs &a, int32_t type, int sms, cudaStream_t s);

struct Mx4ReadArgs {
    const uint8_t *data;
    void *out;
    uint64_t ld, ld_expert;
    uint32_t rows, cols, nk, tile_rows;
    uint64_t n_rows;               // experts * rows
    bool vec;
};
cudaError_t mx4_dequantize_launch(const Mx4ReadArgs &a, int32_t type, int sms, cudaStream_t s);

// out = x w^T (or silu(x w^T) * (x up^T)) on quantized operands.
struct Mx4GemmArgs {
    const uint8_t *w, *up, *x;
    void *out;
    uint64_t ldo, expert_bytes;
    int32_t type;                  // of out
    uint32_t feats, nk;            // rows of w, tiles along its columns
    uint32_t feat_tiles;
    uint64_t n_tok;                // rows of x, where they are one matrix
    const int32_t *first;          // experts: the first sorted place of each (n_expert + 1), at most n_places
    uint32_t n_expert, n_places;
    bool vec, pairs;               // out's rows allow 16-byte stores; 16-bit rows that allow 4-byte ones
};
cudaError_t mx4_many_launch(const Mx4GemmArgs &a, uint32_t x_rows, uint64_t token_tiles, int sms, cudaStream_t s);
cudaError_t mx4_few_launch(const Mx4GemmArgs &a, uint32_t x_rows, uint64_t token_tiles, int sms, cudaStream_t s);

// The choice of experts and the sorting of its pairs.
constexpr uint32_t MOE_SORT_MAX_EXPERTS = 1024, MOE_SORT_MAX_USED = 16;
constexpr uint32_t MOE_SORT_GROUP = 64;   // tokens whose pairs are ranked at a time
constexpr uint32_t MOE_SORT_JOIN = 4;     // stretches that make a row of counts, and whose pairs a CTA places
struct MoeSortArgs {
    const void *logits;            // null: ids are given
    uint64_t ld;
    uint32_t n_tok, n_expert, n_used;
    uint32_t stretch, stretches;   // tokens a CTA chooses for, and how many such
    int32_t norm;
    float prune;
    int32_t *ids;
    float *weights;
    int32_t *first, *order, *place;
    int32_t *tiles;                // [4][n_expert + 1]: the same for tiles of 32, 128, 192 and 256 rows
    int32_t *counts;               // [a row for MOE_SORT_JOIN stretches][counts_ld]
    uint32_t counts_ld;            // n_expert, up to the next multiple of four
};
cudaError_t moe_sort_launch(const MoeSortArgs &a, int32_t type, cudaStream_t s);

struct MoeCombineArgs {
    const void *y;
    uint64_t ldy, ldo;
    void *out;
    const int32_t *place;
    const float *weights;
    uint64_t n_tok;
    uint32_t n_used, dim, n_places;
    bool vec;
};
cudaError_t moe_combine_launch(const MoeCombineArgs &a, int32_t type, int32_t out_type, int sms, cudaStream_t s);

}  // namespace sg
