// Weights of four bits (q4.cuh): packing, unpacking, and the product for up to 16 tokens.
//
#include "q4w.cuh"

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

// Runs once for a weight. A thread packs eight columns of a row; 4, 8 or 16 neighbouring threads share a group.
__global__ void pack_kernel(const void* w, int dt, long long ldw, uint32_t* codes, uint16_t* meta, int rows, int K, int blocks,
                            int group, RowMap map) {
    const int row = blockIdx.x, k8 = blockIdx.y * blockDim.x + threadIdx.x;
    const int src = source_row(row, rows, map);
    const bool in = src >= 0 && 8 * k8 < K, kept = k8 < blocks * 16;
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
    if (!kept) return;
    codes[q4w_word_at(row, k8, blocks)] = word;
    if ((8 * k8) % group == 0) meta[q4w_meta_at(row, k8, blocks, group)] = (uint16_t)q4_meta(g);
}

// The numbers themselves, a warp a block of a tile at a time: its codes in two loads, eight neighbouring numbers in one store.
// c − z and its product with s are exact in bfloat16. 2 x 14336 x 4096: 50 us, 4.7 TB/s written; 4096 x 4096 7.5.
__device__ __forceinline__ void store_eight(__nv_bfloat16* to, const uint32_t (&v)[4]) { *(uint4*)to = make_uint4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store_eight(float* to, const uint32_t (&v)[4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
        *(float4*)(to + 4 * h) = make_float4(__uint_as_float(v[2 * h] << 16), __uint_as_float(v[2 * h] & 0xffff0000u),
                                             __uint_as_float(v[2 * h + 1] << 16), __uint_as_float(v[2 * h + 1] & 0xffff0000u));
}
template <typename T>
__global__ void __launch_bounds__(256)
unpack_kernel(const uint4* codes, const uint16_t* meta, T* out, int rows, int K, int blocks, int group, RowMap map) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, tile = blockIdx.x, block = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (block >= blocks) return;
    const uint4* from = codes + ((size_t)tile * blocks + block) * 64 + lane;
    const uint4 w[2] = {from[0], from[32]};
    const int per = Q4W_BLOCK / group;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int dst = source_row(tile * 16 + g + 8 * r, rows, map);
        if (dst < 0) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {                                // quarters of 32 columns
            const int k = block * Q4W_BLOCK + 32 * i + 8 * t;
            if (k >= K) break;
            const uint32_t m = meta[((((size_t)tile * blocks + block) * 8 + g) * per + 32 * i / group) * 2 + r];
            const uint32_t z = 0x43004300u | (m & 15u) * 0x10001u, s = (m & 0xfff0u) * 0x10001u;
            const uint4 c = w[i >> 1];
            const uint32_t word = r ? (i & 1 ? c.w : c.z) : (i & 1 ? c.y : c.x);
            uint32_t v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = bf2_mul(bf2_sub(q4_pair(word, j), z), s);
            store_eight(out + (size_t)dst * K + k, v);
        }
    }
}

// ---------------------------------------------------------------- the product for a few tokens
// out[M, N] = x[M, K] · Ŵ[N, K]ᵀ, M <= 16, bound by streaming the codes once; what stands in the way is instructions, so the
// number type is the one that takes the fewest to pull a code out of its word: the four bits in the lowest place of a half word
// ARE the float16 c · 2^-24, one place up 16 c · 2^-24, so w & 0x000f000f and w & 0x00f000f0, a multiplication that takes the zero
// off (q4_minus), are operands (c − z) 2^-9 of m16n8k16, and w >> 8 holds the next two pairs. (As e4m3 numbers a code is c · 2^-9 and
// takes half of that, but m16n8k32 on those runs at half the rate of two on float16 here.)
// Why c − z: tensor cores cut partial sums to 24 bits, and sums of x c are many times those of x (c − z), which are nothing where
// weights are zeros beside a large one of their group. (With z Σ x taken off
// afterwards a row of such zeros came to 2^-24 of the large one. us so / now: a row at 4096 x 14336 15.8 / 16.1, eight of gate and up of
// 14336 x 4096 19.0 / 20.3, sixteen at 4096 x 14336 23.6 / 23.6; float32 rows, which met 1024 + c less 1024 + z, 20.9 / 19.5.)
// x is multiplied by a power of two per row and block of 128 columns that brings the block's largest entry into 2^14 .. 2^15:
// exact for bfloat16 entries down to 2^-27 of the block's largest, off by 2^-35 of the largest below (every other pair of columns meets
// 16 (c − z), and x / 16; the others: 2^-39). float32 entries are two float16 numbers each, 22 bits, which end at the same places.
// (Blocks whose largest entry lies outside 2^-80 .. 2^100 overflow or vanish.) A group's sum is scaled in 32 bits. A row with
// an entry that is not finite gives NaN.
//
// x stands still: a warp owns a block of columns, whose x it holds in registers as the operands want it, and walks over
// tiles of 16 rows, fetching the next codes while it multiplies. So shared memory, whose 128 bytes a cycle the codes alone
// would half fill, takes one partial sum a tile and block; warps of a CTA and CTAs of a cluster share K, and at the end
// their sums are added in order: a row's result depends neither on timing nor on the other rows.
//
// Measured (us; 1, 8 and 16 bfloat16 rows, 8 float32 ones; weights in turns beyond L2): 4096 x 14336 16.1, 16.4, 23.6, 19.5; 4096 x 4096 7.2,
// 7.6, 10.0, 7.9; 2 x 14336 x 4096 in groups of 128 19.5, 20.3, 48.5, 25.3. Up to 3.1 TB/s of codes; over the launch 57 % of the issue
// slots and half of the arithmetic pipe are used: a start and an end of some microseconds, and 16 warps an SM, are the rest. From 9 bfloat16 rows on
// all but small weights go to the tcgen05 cores (q4_tc.cu).
enum { MODE_STORE = 0, MODE_ACCUMULATE = 1, MODE_SILU_MUL = 2 };

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float finite_or_nan(float v) { return fabsf(v) < INFINITY ? v : __int_as_float(0x7fc00000); }
__device__ __forceinline__ void load8(const __nv_bfloat16* p, bool ok, float (&v)[8]) {
    const uint4 w = ok ? *(const uint4*)p : make_uint4(0, 0, 0, 0);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = finite_or_nan(__uint_as_float(u[i] << 16)); v[2 * i + 1] = finite_or_nan(__uint_as_float(u[i] & 0xffff0000u)); }
}
__device__ __forceinline__ void load8(const float* p, bool ok, float (&v)[8]) {
    const float4 a = ok ? *(const float4*)p : make_float4(0.f, 0.f, 0.f, 0.f), b = ok ? *(const float4*)(p + 4) : a;
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = finite_or_nan(v[i]);
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t*)&h;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_peer(const float4* local, uint32_t rank) {
    uint32_t ra;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(ra) : "memory");
    return v;
}
__device__ __forceinline__ uint4 ld_once(const uint8_t* p) {         // codes: read once, not kept in L1
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
template <int WORDS> __device__ __forceinline__ void ld_words(const uint8_t* p, uint32_t (&m)[WORDS]) {
    if constexpr (WORDS == 4) {
        const uint4 v = __ldg((const uint4*)p);
        m[0] = v.x; m[1] = v.y; m[2] = v.z; m[3] = v.w;
    } else if constexpr (WORDS == 2) {
        const uint2 v = __ldg((const uint2*)p);
        m[0] = v.x; m[1] = v.y;
    } else {
        m[0] = __ldg((const uint32_t*)p);
    }
}

struct Product {
    const uint8_t* codes;
    const uint8_t* meta;
    void* out;
    long long ldx, ldo;
    int out_dt, M, rows, tiles, blocks, K, mode, half;
    int cs, ki, sets, tpc;         // CTAs of a cluster and warps of a CTA that share K, such sets of warps in a CTA, tiles of a CTA
    SpGate ga;
};

constexpr int MOST_WARPS = 16;

template <typename TX, int NT, int GROUP, int RT, int DEPTH>
__global__ void __launch_bounds__(MOST_WARPS * 32)
gemv_kernel(const TX* x, const Product p) {
    constexpr int PARTS = sizeof(TX) == 4 ? 2 : 1, GROUPS = Q4W_BLOCK / GROUP, META = 4 * GROUPS;        // META: bytes of a lane row's scales
    extern __shared__ __align__(16) float4 red[];                    // [tile][share][column group][lane]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warps = p.sets * p.ki;
    const int rank = p.cs > 1 ? (int)cluster_rank() : 0, set = warp / p.ki, share = warp % p.ki;
    const int cta_tile = (blockIdx.x / p.cs) * p.tpc, n_tiles = min(p.tpc, p.tiles - cta_tile);
    const int c0 = (int)((long long)p.blocks * rank / p.cs), c1 = (int)((long long)p.blocks * (rank + 1) / p.cs);      // the CTA's blocks

    for (int b = c0 + share; b == c0 + share || b < c1; b += p.ki) {
        const bool there = b < c1;                                   // (a CTA may have fewer blocks than shares: zeros)
        const uint8_t* code = p.codes + ((size_t)(cta_tile + set * RT) * p.blocks + b) * 1024 + lane * 16;
        const uint8_t* meta = p.meta + ((size_t)(cta_tile + set * RT) * p.blocks + b) * (8 * META) + g * META;
        uint4 w[DEPTH][RT][2];
        uint32_t m[DEPTH][RT][GROUPS];
        int asked = set * RT;
        auto ask = [&](int i) {
#pragma unroll
            for (int r = 0; r < RT; ++r)
                if (there && asked + r < n_tiles) {
                    w[i][r][0] = ld_once(code + (size_t)r * p.blocks * 1024);
                    w[i][r][1] = ld_once(code + (size_t)r * p.blocks * 1024 + 512);
                    ld_words<GROUPS>(meta + (size_t)r * p.blocks * (8 * META), m[i][r]);
                }
            asked += p.sets * RT;
            code += (size_t)p.sets * RT * p.blocks * 1024;
            meta += (size_t)p.sets * RT * p.blocks * (8 * META);
        };
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) ask(i);

        // x of this block: lane (row g, columns 32 q + 8 t ..), eight rows at a time
        uint4 xv[NT][4][PARTS];
        float2 by[NT];                                               // of rows 2 t and 2 t + 1
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int token = n * 8 + g;
            const TX* row = x + (size_t)min(token, p.M - 1) * p.ldx + (size_t)b * Q4W_BLOCK + 8 * t;
            float v[4][8], top = 0.0f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                load8(row + 32 * q, there && token < p.M && b * Q4W_BLOCK + 32 * q < p.K, v[q]);
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[q][e]));                        // (NaN is left out)
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int up = top > 0.0f ? min(94, max(-94, 141 - (int)(__float_as_uint(top) >> 23))) : 0;
            const float scale = __uint_as_float((uint32_t)(127 + up) << 23), unit = __uint_as_float((uint32_t)(136 - up) << 23);
            by[n] = make_float2(__shfl_sync(0xffffffffu, unit, 8 * t), __shfl_sync(0xffffffffu, unit, 8 * t + 4));
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t h[PARTS][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float lo = v[q][2 * j] * scale, hi = v[q][2 * j + 1] * scale, f = j & 1 ? 0.0625f : 1.0f;
                    h[0][j] = half2_of(lo * f, hi * f);
                    if (PARTS == 2) {
                        const float2 first = __half22float2(*(const __half2*)&h[0][j]);
                        h[PARTS - 1][j] = half2_of(lo * f - first.x, hi * f - first.y);
                    }
                }
#pragma unroll
                for (int part = 0; part < PARTS; ++part) xv[n][q][part] = make_uint4(h[part][0], h[part][1], h[part][2], h[part][3]);
            }
        }

        for (int j0 = set * RT; j0 < n_tiles; j0 += DEPTH * RT * p.sets) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const int j = j0 + d * RT * p.sets;
                if (j >= n_tiles) break;
                float4 y[RT][NT];
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int n = 0; n < NT; ++n) y[r][n] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (there) {
                    float acc[RT][NT][4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (q % (GROUP / 32) == 0)
#pragma unroll
                            for (int r = 0; r < RT; ++r)
#pragma unroll
                                for (int n = 0; n < NT; ++n) acc[r][n][0] = acc[r][n][1] = acc[r][n][2] = acc[r][n][3] = 0.0f;
#pragma unroll
                        for (int half = 0; half < 2; ++half)
#pragma unroll
                            for (int r = 0; r < RT; ++r) {
                                const uint4 c = w[d][r][q >> 1];
                                const uint32_t r0 = (q & 1 ? c.y : c.x) >> (8 * half), r1 = (q & 1 ? c.w : c.z) >> (8 * half);
                                uint32_t a0 = r0 & 0x000f000fu, a1 = r1 & 0x000f000fu, a2 = r0 & 0x00f000f0u, a3 = r1 & 0x00f000f0u;
                                const uint32_t mm = m[d][r][q / (GROUP / 32)], z0 = (mm & 15u) * 0x10001u, z1 = ((mm >> 16) & 15u) * 0x10001u;
                                const uint32_t n0 = q4_zero(z0), n1 = q4_zero(z1), n2 = q4_zero(z0 << 4), n3 = q4_zero(z1 << 4);
                                a0 = q4_minus(a0, n0);
                                a1 = q4_minus(a1, n1);
                                a2 = q4_minus(a2, n2);
                                a3 = q4_minus(a3, n3);
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int part = PARTS - 1; part >= 0; --part) {
                                        const uint4 v = xv[n][q][part];
                                        mma_f16(acc[r][n], a0, a1, a2, a3, half ? v.z : v.x, half ? v.w : v.y);
                                    }
                            }
                        if ((q + 1) % (GROUP / 32) == 0) {
                            const int i = q / (GROUP / 32);
#pragma unroll
                            for (int r = 0; r < RT; ++r) {
                                const uint32_t mm = m[d][r][i];
                                const float s0 = __uint_as_float((mm << 16) & 0xfff00000u), s1 = __uint_as_float(mm & 0xfff00000u);
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    y[r][n].x = fmaf(s0, acc[r][n][0], y[r][n].x);
                                    y[r][n].y = fmaf(s0, acc[r][n][1], y[r][n].y);
                                    y[r][n].z = fmaf(s1, acc[r][n][2], y[r][n].z);
                                    y[r][n].w = fmaf(s1, acc[r][n][3], y[r][n].w);
                                }
                            }
                        }
                    }
                }
                ask(d);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    if (j + r >= n_tiles) break;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float4* to = red + (((j + r) * p.ki + share) * NT + n) * 32 + lane;
                        float4 v = make_float4(y[r][n].x * by[n].x, y[r][n].y * by[n].y, y[r][n].z * by[n].x, y[r][n].w * by[n].y);
                        if (b >= c0 + p.ki) { const float4 o = *to; v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w; }
                        *to = v;
                    }
                }
            }
        }
    }

    // the sums of all shares of K, in their order; a warp takes a tile's (gated: a pair of tiles') eight rows of x at a time
    if (p.cs > 1) cluster_sync();
    else __syncthreads();
    const int step = p.mode == MODE_SILU_MUL ? 2 : 1;
    for (int i = warp * p.cs + rank; i < n_tiles / step * NT; i += warps * p.cs) {
        const int n = i % NT, at = i / NT * step;
        float4 sum[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            sum[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r >= step) break;
            for (int o = 0; o < p.cs; ++o) {
#pragma unroll 4
                for (int k = 0; k < p.ki; ++k) {
                    const float4* from = red + (((at + r) * p.ki + k) * NT + n) * 32 + lane;
                    const float4 v = p.cs > 1 ? ld_peer(from, o) : *from;
                    sum[r].x += v.x; sum[r].y += v.y; sum[r].z += v.z; sum[r].w += v.w;
                }
            }
        }
        const float a[4] = {sum[0].x, sum[0].y, sum[0].z, sum[0].w}, u[4] = {sum[1].x, sum[1].y, sum[1].z, sum[1].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int token = n * 8 + 2 * t + (e & 1), o = (cta_tile + at) / step * 16 + g + (e & 2 ? 8 : 0);
            if (token >= p.M || o >= (step == 2 ? p.half : p.rows)) continue;
            const size_t to = (size_t)token * p.ldo + o;
            if (step == 2) sp_st_dt(p.out, p.out_dt, to, sp_gated(a[e], u[e], p.ga));
            else if (p.mode == MODE_ACCUMULATE) ((float*)p.out)[to] += a[e];
            else sp_st_dt(p.out, p.out_dt, to, a[e]);
        }
    }
    if (p.cs > 1) cluster_sync();                                    // nobody leaves before its sums are read
}

constexpr int SMEM_LIMIT = 200 * 1024;

// How a product is divided: CTAs of a cluster and warps of a CTA that share K, sets of such warps, tiles of a CTA. A warp's time
// goes with the tiles it multiplies, 0.5 us each at 8 rows; a further block of columns costs it about one and a half, a
// cluster's exchange two. 8 rows of x (us, as chosen / the next best): 4,096 x 4,096 7.1 / 7.5, 4,096 x 14,336 16.2 / 17.2,
// 2,048 x 8,192 8.9 / 9.0, gated 2 x 14,336 x 4,096 19.5 / 20.5.
// (Clusters of 4 and 8 do not find room on every SM and took two rounds: 4,096 x 14,336 40 us.) ``sum_bytes``: a tile's and share's partial sums.
void divide(Product& p, int sum_bytes) {
    const int sms = sp_sm_count() > 0 ? sp_sm_count() : 148;
    double best = 0;
    Product c = p;
    for (c.cs = 1; c.cs <= 2 && c.cs <= p.blocks; ++c.cs) {
        const int mine = (p.blocks + c.cs - 1) / c.cs, phases = (mine + MOST_WARPS - 1) / MOST_WARPS;
        c.ki = (mine + phases - 1) / phases;
        const int clusters = sms / c.cs;
        c.tpc = (p.tiles + clusters - 1) / clusters;
        if (p.mode == MODE_SILU_MUL) c.tpc += c.tpc & 1;
        const int fits = SMEM_LIMIT / (c.ki * sum_bytes) & ~1;
        int rounds = 1;
        if (c.tpc > fits) { rounds = (c.tpc + fits - 1) / fits; c.tpc = fits; }
        c.sets = MOST_WARPS / c.ki < c.tpc ? MOST_WARPS / c.ki : c.tpc;
        const double cost = rounds * ((double)((c.tpc + c.sets - 1) / c.sets) * phases + 1.5 * phases + (c.cs > 1 ? 2.0 : 0.0) + 4.0);
        if (best == 0 || cost < best) { best = cost; p = c; }
    }
}

template <typename TX, int NT, int GROUP>
int launch_gemv(const TX* x, Product p, cudaStream_t stream) {
    constexpr int RT = 1, DEPTH = sizeof(TX) == 4 ? 2 : 3;          // (two tiles at a time: 18.5 us instead of 19.5 where K is short, slower elsewhere)
    static SpPerDevice configured;
    if (!configured.done()) {
        cudaError_t e = cudaFuncSetAttribute(gemv_kernel<TX, NT, GROUP, RT, DEPTH>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT);
        if (e != cudaSuccess) SP_FAIL("q4_gemv: cannot reserve %d bytes of shared memory: %s", SMEM_LIMIT, cudaGetErrorString(e));
        configured.mark();
    }
    divide(p, NT * 512);
    const dim3 grid((p.tiles + p.tpc - 1) / p.tpc * p.cs);
    SP_CHECK_CALL("q4_gemv", sp_launch_cluster(gemv_kernel<TX, NT, GROUP, RT, DEPTH>, grid, dim3(p.sets * p.ki * 32), (size_t)(p.tpc * p.ki * NT * 512), stream, p.cs, x, p));
    return 0;
}

template <typename TX>
int launch_gemv(const void* xp, const Product& p, int group, cudaStream_t stream) {
    const TX* x = (const TX*)xp;
    if (p.M > 8) return group == 32 ? launch_gemv<TX, 2, 32>(x, p, stream) : group == 64 ? launch_gemv<TX, 2, 64>(x, p, stream) : launch_gemv<TX, 2, 128>(x, p, stream);
    return group == 32 ? launch_gemv<TX, 1, 32>(x, p, stream) : group == 64 ? launch_gemv<TX, 1, 64>(x, p, stream) : launch_gemv<TX, 1, 128>(x, p, stream);
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

SP_API int sp_q4_pack(const void* w, int dt, long long ldw, void* codes, void* meta, int rows, int K, int group, int half, cudaStream_t stream) {
    if (check_sizes("q4_pack", rows, K, group, half, 0)) return 1;
    if ((uintptr_t)codes & 15) SP_FAIL("q4_pack: the codes must start on a 16-byte boundary");
    const int packed = q4w_tiles(rows, half) * 16, blocks = (K + Q4W_BLOCK - 1) / Q4W_BLOCK;
    pack_kernel<<<dim3(packed, (blocks * 16 + 127) / 128), blocks < 8 ? (blocks * 16 + 31) / 32 * 32 : 128, 0, stream>>>(w, dt, ldw, (uint32_t*)codes, (uint16_t*)meta, rows, K,
                                                                             blocks, group, RowMap{half, 0});
    SP_CHECK_LAUNCH("q4_pack");
    return 0;
}

// out [rows, K] (contiguous) = the numbers that the packed weight stands for; ``half``, ``block``: gate and up rows in blocks.
SP_API int sp_q4_unpack(const void* codes, const void* meta, void* out, int dt, int rows, int K, int group, int half, int block, cudaStream_t stream) {
    if (check_sizes("q4_unpack", rows, K, group, half, block)) return 1;
    if ((uintptr_t)out & 15) SP_FAIL("q4_unpack: the output must start on a 16-byte boundary");
    const int packed = q4w_tiles(rows, half) * 16, blocks = (K + Q4W_BLOCK - 1) / Q4W_BLOCK;
    const dim3 grid(packed / 16, (blocks + 7) / 8), block_dim(blocks < 8 ? blocks * 32 : 256);
    const RowMap map{half, block};
    if (dt == SP_DT_F32) unpack_kernel<<<grid, block_dim, 0, stream>>>((const uint4*)codes, (const uint16_t*)meta, (float*)out, rows, K, blocks, group, map);
    else unpack_kernel<<<grid, block_dim, 0, stream>>>((const uint4*)codes, (const uint16_t*)meta, (__nv_bfloat16*)out, rows, K, blocks, group, map);
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
    if (((uintptr_t)codes & 15) || ((uintptr_t)meta & 15)) SP_FAIL("q4_gemv: codes and scales must start on 16-byte boundaries");
    const int packed = q4w_tiles(rows, half) * 16, blocks = (K + Q4W_BLOCK - 1) / Q4W_BLOCK;
    const Product p{(const uint8_t*)codes, (const uint8_t*)meta, out, ldx, ldo, out_dt, M, rows, packed / 16, blocks, K, mode, half, 1, 1, 1, 1, SpGate{act, mult}};
    return x_dt == SP_DT_F32 ? launch_gemv<float>(x, p, group, stream) : launch_gemv<__nv_bfloat16>(x, p, group, stream);
}
