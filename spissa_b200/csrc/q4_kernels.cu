// Weights of four bits (q4.cuh): packing, unpacking.
//
// Layout. Rows of W come in tiles of 16, columns in blocks of 64, both filled up with zeros. A block of a tile is 512 bytes:
// lane 4 g + t of a warp owns 16 of them, the words (row g: columns 8 t.., 32 + 8 t..), (row g + 8: the same), that
// is, the A operand of four m16n8k16 products in one load. Scales and zeros: [tile][group of columns][16 rows], 16 bits each.
// A gated product's rows alternate by tiles: 16 gate rows, the 16 up rows of the same outputs.
#include "q4.cuh"

SP_API const char* sp_q4_last_error() { return sp_error_text; }
SP_DEFINE_RANGE_API(q4)

namespace {

// Where a row of the packed weight comes from (or goes to): plain, or gate and up rows of ``half`` outputs, in the source
// one after the other, ``block`` gate rows and then the same outputs' up rows (block 0: all gate rows, then all up rows).
struct RowMap { int half, block; };
__device__ __forceinline__ int source_row(int packed, int rows, const RowMap& m) {      // -1: filled up with zeros
    if (m.half == 0) return packed < rows ? packed : -1;
    const int o = (packed >> 5) * 16 + (packed & 15), up = (packed >> 4) & 1;
    if (o >= m.half) return -1;
    return m.block ? (o / m.block) * 2 * m.block + up * m.block + o % m.block : up * m.half + o;
}

__device__ __forceinline__ size_t word_at(int row, int k8, int kblocks) {            // the word of columns 8 k8 .. of a packed row
    const int kb = k8 >> 3, t = k8 & 3, h = (k8 >> 2) & 1;
    return (((size_t)(row >> 4) * kblocks + kb) * 32 + (row & 7) * 4 + t) * 4 + ((row >> 3) & 1) * 2 + h;
}

// A thread packs eight columns of a row; 4, 8 or 16 neighbouring threads share a group.
__global__ void pack_kernel(const void* w, int dt, long long ldw, uint32_t* codes, uint16_t* meta, int rows, int K, int kblocks,
                            int group, RowMap map) {
    const int row = blockIdx.x, k8 = blockIdx.y * blockDim.x + threadIdx.x;
    const int src = source_row(row, rows, map);
    const bool in = src >= 0 && 8 * k8 < K;
    float x[8], lo = 0.0f, hi = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = in ? sp_ld_dt(w, dt, (size_t)src * ldw + 8 * k8 + i) : 0.0f;
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        bad |= q4_bad(x[i]);
    }
    int any = bad;
    for (int o = 1; o < group / 8; o *= 2) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        any |= __shfl_xor_sync(0xffffffffu, any, o);
    }
    const Q4Scale g = q4_group(lo, hi, any != 0);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) word |= (uint32_t)q4_code(x[i], g) << (4 * (i / 2 + 4 * (i & 1)));
    if (k8 >= kblocks * 8) return;
    codes[word_at(row, k8, kblocks)] = word;
    if ((8 * k8) % group == 0) meta[((size_t)(row >> 4) * (kblocks * 64 / group) + 8 * k8 / group) * 16 + (row & 15)] = (uint16_t)q4_meta(g);
}

template <typename T>
__global__ void unpack_kernel(const uint32_t* codes, const uint16_t* meta, T* out, int rows, int K, int kblocks, int group, RowMap map) {
    const int row = blockIdx.x, k8 = blockIdx.y * blockDim.x + threadIdx.x;
    const int dst = source_row(row, rows, map);
    if (dst < 0 || 8 * k8 >= K) return;
    const uint32_t word = codes[word_at(row, k8, kblocks)];
    const uint32_t m = meta[((size_t)(row >> 4) * (kblocks * 64 / group) + 8 * k8 / group) * 16 + (row & 15)];
    T* to = out + (size_t)dst * K + 8 * k8;
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        sp_st2(to, i, q4_value((word >> (2 * i)) & 15, m), q4_value((word >> (2 * i + 16)) & 15, m));
}

int check_sizes(const char* what, int rows, int K, int group, int half, int block) {
    if (rows <= 0 || K <= 0 || K % 32) SP_FAIL("%s: rows of a multiple of 32 columns, got %d x %d", what, rows, K);
    if (group != 32 && group != 64 && group != 128) SP_FAIL("%s: groups of 32, 64 or 128, got %d", what, group);
    if (K % group) SP_FAIL("%s: %d columns are no multiple of the group of %d", what, K, group);
    if (half < 0 || (half && rows != 2 * half)) SP_FAIL("%s: gate and up have %d rows each, the weight %d", what, half, rows);
    if (block < 0 || (block && half % block)) SP_FAIL("%s: %d outputs do not come in blocks of %d", what, half, block);
    return 0;
}

}  // namespace

// Rows of the packed weight (a multiple of 16): each half filled up for itself.
SP_API int sp_q4_packed_rows(int rows, int half) { return half ? (half + 15) / 16 * 32 : (rows + 15) / 16 * 16; }

SP_API int sp_q4_pack(const void* w, int dt, long long ldw, void* codes, void* meta, int rows, int K, int group, int half, cudaStream_t stream) {
    if (check_sizes("q4_pack", rows, K, group, half, 0)) return 1;
    if ((uintptr_t)codes & 15) SP_FAIL("q4_pack: the codes must start on a 16-byte boundary");
    const int packed = sp_q4_packed_rows(rows, half), kblocks = (K + 63) / 64;
    pack_kernel<<<dim3(packed, (kblocks * 8 + 127) / 128), 128, 0, stream>>>(w, dt, ldw, (uint32_t*)codes, (uint16_t*)meta, rows, K,
                                                                             kblocks, group, RowMap{half, 0});
    SP_CHECK_LAUNCH("q4_pack");
    return 0;
}

// out [rows, K] (contiguous) = the numbers that the packed weight stands for; ``half``, ``block``: gate and up rows in blocks.
SP_API int sp_q4_unpack(const void* codes, const void* meta, void* out, int dt, int rows, int K, int group, int half, int block, cudaStream_t stream) {
    if (check_sizes("q4_unpack", rows, K, group, half, block)) return 1;
    if ((uintptr_t)out & 15) SP_FAIL("q4_unpack: the output must start on a 16-byte boundary");
    const int packed = sp_q4_packed_rows(rows, half), kblocks = (K + 63) / 64;
    const dim3 grid(packed, (kblocks * 8 + 127) / 128);
    if (dt == SP_DT_F32) unpack_kernel<<<grid, 128, 0, stream>>>((const uint32_t*)codes, (const uint16_t*)meta, (float*)out, rows, K, kblocks, group, RowMap{half, block});
    else unpack_kernel<<<grid, 128, 0, stream>>>((const uint32_t*)codes, (const uint16_t*)meta, (__nv_bfloat16*)out, rows, K, kblocks, group, RowMap{half, block});
    SP_CHECK_LAUNCH("q4_unpack");
    return 0;
}
