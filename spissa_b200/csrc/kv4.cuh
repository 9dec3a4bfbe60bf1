// Where a four-bit cache keeps what: see kv4_kernels.cu for the layout's reasons.
#pragma once
#include "q4.cuh"

namespace {

constexpr int KV4_PAGE = 64;
constexpr int KV4_MAX_HD = 128;

__host__ __device__ constexpr int kv4_k_meta(int hd) { return KV4_PAGE * hd / 2; }
__host__ __device__ constexpr int kv4_v_codes(int hd) { return KV4_PAGE * (hd / 2 + hd / 16); }
__host__ __device__ constexpr int kv4_v_meta(int hd) { return KV4_PAGE * (hd + hd / 16); }
__host__ __device__ constexpr int kv4_tile_bytes(int hd) { return KV4_PAGE * (hd + hd / 8); }

// The row of a position's key among its page's: the low three bits b2 b1 b0 become b1 b0 b2, so that row r of a score
// fragment, whose rows 2 t and 2 t + 1 are the columns 2 t and 2 t + 1 of the next product's operand, is position t or 4 + t.
__host__ __device__ constexpr int kv4_key_slot(int pos) { return (pos & ~7) | ((pos & 3) << 1) | ((pos >> 2) & 1); }

__device__ __forceinline__ int kv4_k_at(int pos, int t, int group, int hd) { return kv4_key_slot(pos) * (hd / 2) + (t * (hd / 32) + group) * 4; }
__device__ __forceinline__ int kv4_v_at(int pos, int g, int group, int hd) {
    const int at = (g * (hd / 32) + group) * 2;
    return pos * (hd / 2) + (hd == 128 ? at ^ ((pos & 2) << 4) : at);
}

}  // namespace
