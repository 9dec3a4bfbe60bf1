// Where a weight of four bits (q4.cuh) keeps what, for the kernels that pack it and multiply with it.
//
// Rows of W come in tiles of 16, columns in blocks of 128, both filled up with zeros. A block of a tile is 1,024 bytes of codes, two
// pieces of 64 columns: lane 4 g + t of a warp owns 16 bytes of each, the words (row g: columns 8 t.., 32 + 8 t..), (row g + 8:
// the same), that is, the A operand of four m16n8k16 products in one load. Scales and zeros: [tile][block][row g][group of the
// block][row g, row g + 8], 16 bits each. A gated product's rows alternate by tiles: 16 gate rows, the 16 up rows of the same
// outputs. Eight tiles' codes and scales of a block in one run of bytes, one copy for the tcgen05 kernel, was tried and costs the
// product of few rows 15 to 35 % (8B gate and up 19 -> 26 us): its warps then read 1,024 bytes here and there.
#pragma once
#include "q4.cuh"

namespace {

constexpr int Q4W_BLOCK = 128;                                       // columns

__host__ __device__ constexpr int q4w_meta_bytes(int group) { return 4096 / group; }                  // of a tile's block
__device__ __forceinline__ size_t q4w_word_at(int row, int k8, int blocks) {          // the word of columns 8 k8 .. of a packed row
    return ((((size_t)(row >> 4) * blocks + (k8 >> 4)) * 2 + ((k8 >> 3) & 1)) * 32 + (row & 7) * 4 + (k8 & 3)) * 4 + ((row >> 3) & 1) * 2 + ((k8 >> 2) & 1);
}
__device__ __forceinline__ size_t q4w_meta_at(int row, int k8, int blocks, int group) {
    return ((((size_t)(row >> 4) * blocks + (k8 >> 4)) * 8 + (row & 7)) * (Q4W_BLOCK / group) + (8 * k8 % Q4W_BLOCK) / group) * 2 + ((row >> 3) & 1);
}
static inline int q4w_tiles(int rows, int half) { return half ? (half + 15) / 16 * 2 : (rows + 15) / 16; }

}  // namespace
