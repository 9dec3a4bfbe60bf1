// Weights of four bits (q4.cuh): packing, unpacking, and the product for up to 16 tokens.
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

// ---------------------------------------------------------------- the product for a few tokens
// out[M, N] = x[M, K] · Ŵ[N, K]ᵀ, M <= 16, bound by streaming the codes once.
//
// A CTA owns two tiles of 16 rows (gated: 16 gate rows and the up rows of the same outputs); its warps, and the CTAs of a cluster,
// share the blocks of K. Per block of 64 a lane loads 16 bytes of codes per tile and 32 of x per eight tokens, and four
// mma.sync m16n8k16 multiply the codes less their zero (c − z, exact in bfloat16) with x as the columns. A
// group's sum is scaled in 32 bits and added to the row's: no rounding but the sums' own. float32 rows are taken apart into
// three bfloat16 parts, 8 bits of the mantissa each, and each part is multiplied: the same sums, exactly x.
// Partial sums are added in the order of the warps, then of the CTAs, so a row's result depends neither on timing nor on M.
enum { MODE_STORE = 0, MODE_ACCUMULATE = 1, MODE_SILU_MUL = 2 };
constexpr int WARPS = 8;

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld_once(const uint4* p) {           // codes: read once, not kept in L1
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// The bfloat16 pairs of eight neighbouring entries of a row of x, in one part or in three.
__device__ __forceinline__ void x_pairs(const __nv_bfloat16* p, bool ok, uint32_t (&out)[1][4]) {
    const uint4 v = ok ? *(const uint4*)p : make_uint4(0, 0, 0, 0);
    out[0][0] = v.x; out[0][1] = v.y; out[0][2] = v.z; out[0][3] = v.w;
}
__device__ __forceinline__ void x_pairs(const float* p, bool ok, uint32_t (&out)[3][4]) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (ok) {
        *(float4*)v = *(const float4*)p;
        *(float4*)(v + 4) = *(const float4*)(p + 4);
    }
#pragma unroll
    for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t a = __float_as_uint(v[2 * i]), b = __float_as_uint(v[2 * i + 1]);
            out[part][i] = __byte_perm(a, b, 0x7632);
            v[2 * i] -= __uint_as_float(a & 0xffff0000u);
            v[2 * i + 1] -= __uint_as_float(b & 0xffff0000u);
            if (v[2 * i] != v[2 * i]) v[2 * i] = 0.0f;               // an infinity is its first part
            if (v[2 * i + 1] != v[2 * i + 1]) v[2 * i + 1] = 0.0f;
        }
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_peer(const void* local, uint32_t rank) {
    uint32_t ra;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(ra) : "memory");
    return v;
}

struct Product {
    const uint4* codes;
    const uint16_t* meta;
    void* out;
    long long ldx, ldo;
    int out_dt, M, rows, tiles, kblocks, K, group, mode, half, cs;
    SpGate ga;
};

template <typename TX, int NT, bool G32>
__global__ void __launch_bounds__(WARPS * 32)
gemv_kernel(const TX* x, const Product p) {
    constexpr int PARTS = sizeof(TX) == 4 ? 3 : 1, RT = 2, UNROLL = NT * PARTS > 1 ? 2 : 4;
    __shared__ __align__(16) float4 red[WARPS][RT][NT][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = p.cs > 1 ? (int)cluster_rank() : 0, pair = blockIdx.x / p.cs;
    const int slices = WARPS * p.cs, slice = rank * WARPS + warp;
    const int kb0 = (int)((long long)p.kblocks * slice / slices), kb1 = (int)((long long)p.kblocks * (slice + 1) / slices);
    const int mgroups = p.kblocks * 64 / p.group, shift = p.group == 128 ? 1 : 0;

    const uint4* code[RT];
    const uint16_t* meta[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int tile = min(pair * RT + r, p.tiles - 1);            // an odd last tile is computed twice, stored once
        code[r] = p.codes + (size_t)tile * p.kblocks * 32 + lane;
        meta[r] = p.meta + (size_t)tile * mgroups * 16 + g;
    }
    const TX* row[NT];
    bool have[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        have[n] = n * 8 + g < p.M;
        row[n] = x + (size_t)(have[n] ? n * 8 + g : 0) * p.ldx + 8 * t;
    }
    float y[RT][NT][4];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) y[r][n][0] = y[r][n][1] = y[r][n][2] = y[r][n][3] = 0.0f;

    for (int kb = kb0; kb < kb1; kb += UNROLL) {
        uint4 w[UNROLL][RT];
        uint32_t m[UNROLL][RT][G32 ? 4 : 2];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int b = min(kb + u, kb1 - 1);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                w[u][r] = ld_once(code[r] + (size_t)b * 32);
                const uint16_t* at = meta[r] + (size_t)(G32 ? 2 * b : b >> shift) * 16;
                m[u][r][0] = __ldg(at);
                m[u][r][1] = __ldg(at + 8);
                if (G32) {
                    m[u][r][G32 ? 2 : 0] = __ldg(at + 16);
                    m[u][r][G32 ? 3 : 1] = __ldg(at + 24);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int b = kb + u;
            if (b >= kb1) break;
            uint32_t xb[NT][2][PARTS][4];                            // [half of the block]
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    x_pairs(row[n] + (size_t)b * 64 + 32 * h, have[n] && (h == 0 || b * 64 + 32 < p.K), xb[n][h]);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                float acc[NT][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t m0 = m[u][r][G32 ? 2 * h : 0], m1 = m[u][r][G32 ? 2 * h + 1 : 1];
                    if (h == 0 || G32)
#pragma unroll
                        for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
                    const uint32_t z0 = 0x43004300u | (m0 & 15u) * 0x10001u, z1 = 0x43004300u | (m1 & 15u) * 0x10001u;
                    const uint32_t w0 = h ? w[u][r].y : w[u][r].x, w1 = h ? w[u][r].w : w[u][r].z;
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const uint32_t a0 = bf2_sub(q4_pair(w0, 2 * s), z0), a1 = bf2_sub(q4_pair(w1, 2 * s), z1);
                        const uint32_t a2 = bf2_sub(q4_pair(w0, 2 * s + 1), z0), a3 = bf2_sub(q4_pair(w1, 2 * s + 1), z1);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int q = PARTS - 1; q >= 0; --q) mma_bf16(acc[n], a0, a1, a2, a3, xb[n][h][q][2 * s], xb[n][h][q][2 * s + 1]);
                    }
                    if (h == 1 || G32) {
                        const float s0 = q4_scale_of(m0), s1 = q4_scale_of(m1);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            y[r][n][0] = fmaf(s0, acc[n][0], y[r][n][0]);
                            y[r][n][1] = fmaf(s0, acc[n][1], y[r][n][1]);
                            y[r][n][2] = fmaf(s1, acc[n][2], y[r][n][2]);
                            y[r][n][3] = fmaf(s1, acc[n][3], y[r][n][3]);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) red[warp][r][n][lane] = make_float4(y[r][n][0], y[r][n][1], y[r][n][2], y[r][n][3]);
    __syncthreads();
    // the warps' sums, a thread per four values; then the cluster's
    const bool mine = threadIdx.x < NT * 32;
    const int n = threadIdx.x >> 5;
    float4 sum[RT];
    if (mine) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            sum[r] = red[0][r][n][lane];
#pragma unroll
            for (int o = 1; o < WARPS; ++o) {
                const float4 v = red[o][r][n][lane];
                sum[r].x += v.x; sum[r].y += v.y; sum[r].z += v.z; sum[r].w += v.w;
            }
            red[0][r][n][lane] = sum[r];
        }
    }
    if (p.cs > 1) {
        cluster_sync();
        if (rank == 0 && mine) {
            for (int o = 1; o < p.cs; ++o)
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const float4 v = ld_peer(&red[0][r][n][lane], o);
                    sum[r].x += v.x; sum[r].y += v.y; sum[r].z += v.z; sum[r].w += v.w;
                }
        }
        cluster_sync();                                              // nobody leaves before its sums are read
        if (rank != 0) return;
    }
    if (!mine) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int token = n * 8 + 2 * t + (e & 1), at = g + (e & 2 ? 8 : 0);
        if (token >= p.M) continue;
        const float a = e == 0 ? sum[0].x : e == 1 ? sum[0].y : e == 2 ? sum[0].z : sum[0].w;
        const float b = e == 0 ? sum[1].x : e == 1 ? sum[1].y : e == 2 ? sum[1].z : sum[1].w;
        if (p.mode == MODE_SILU_MUL) {
            const int o = pair * 16 + at;
            if (o < p.half) sp_st_dt(p.out, p.out_dt, (size_t)token * p.ldo + o, sp_gated(a, b, p.ga));
            continue;
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int o = (pair * RT + r) * 16 + at;
            if (o >= p.rows) continue;
            const size_t i = (size_t)token * p.ldo + o;
            if (p.mode == MODE_ACCUMULATE) ((float*)p.out)[i] += r ? b : a;
            else sp_st_dt(p.out, p.out_dt, i, r ? b : a);
        }
    }
}

template <typename TX>
cudaError_t launch_gemv(const TX* x, const Product& p, cudaStream_t stream) {
    const dim3 grid((p.tiles + 1) / 2 * p.cs), block(WARPS * 32);
    const bool two = p.M > 8, g32 = p.group == 32;
    if (two) return g32 ? sp_launch_cluster(gemv_kernel<TX, 2, true>, grid, block, 0, stream, p.cs, x, p)
                        : sp_launch_cluster(gemv_kernel<TX, 2, false>, grid, block, 0, stream, p.cs, x, p);
    return g32 ? sp_launch_cluster(gemv_kernel<TX, 1, true>, grid, block, 0, stream, p.cs, x, p)
               : sp_launch_cluster(gemv_kernel<TX, 1, false>, grid, block, 0, stream, p.cs, x, p);
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

// The product for 1 to 16 rows of x (bfloat16 or float32, 16-byte boundaries): mode 0 out = x·Ŵᵀ (bfloat16 or float32), 1 out
// (float32) += x·Ŵᵀ, 2 out [M, half] = act(gate)·up · mult.
SP_API int sp_q4_gemv(const void* x, int x_dt, const void* codes, const void* meta, void* out, int out_dt, int M, int rows, int K,
                      int group, int half, long long ldx, long long ldo, int mode, int act, float mult, cudaStream_t stream) {
    if (check_sizes("q4_gemv", rows, K, group, half, 0)) return 1;
    if (M <= 0 || M > 16) SP_FAIL("q4_gemv: built for 1 to 16 rows, got %d", M);
    if ((mode == MODE_SILU_MUL) != (half > 0) || mode < 0 || mode > MODE_SILU_MUL) SP_FAIL("q4_gemv: mode %d does not go with %d gate rows", mode, half);
    if (mode == MODE_SILU_MUL && act != SP_ACT_SILU && act != SP_ACT_GELU) SP_FAIL("q4_gemv: activation code %d is not built for gated rows", act);
    if (mode == MODE_ACCUMULATE && out_dt != SP_DT_F32) SP_FAIL("q4_gemv: accumulation needs a float32 output");
    if (((uintptr_t)x & 15) || (ldx * (x_dt == SP_DT_F32 ? 4 : 2)) % 16) SP_FAIL("q4_gemv: rows of x must start on 16-byte boundaries");
    if (((uintptr_t)codes & 15) || ((uintptr_t)meta & 1)) SP_FAIL("q4_gemv: codes must start on a 16-byte boundary");
    const int packed = sp_q4_packed_rows(rows, half), kblocks = (K + 63) / 64, tiles = packed / 16;
    Product p{(const uint4*)codes, (const uint16_t*)meta, out, ldx, ldo, out_dt, M, rows, tiles, kblocks, K, group, mode, half, 1, SpGate{act, mult}};
    const int sms = sp_sm_count() > 0 ? sp_sm_count() : 148, pairs = (tiles + 1) / 2;
    while (p.cs < 8 && pairs * p.cs < 3 * sms && kblocks >= 4 * WARPS * p.cs) p.cs *= 2;
    SP_CHECK_CALL("q4_gemv", x_dt == SP_DT_F32 ? launch_gemv((const float*)x, p, stream) : launch_gemv((const __nv_bfloat16*)x, p, stream));
    return 0;
}
