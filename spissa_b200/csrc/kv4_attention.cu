// Attention over a cache of four bits (kv4_kernels.cu states the layout, q4.cuh the format): one token of each sequence, or a
// few, over all the keys that they see, the keys split over CTAs and joined.
//
// score = scale · q · k̂, softmax in 32 bits, out = Σ p v̂; query head h reads kv head h / (heads / kv heads); a token at position p
// sees keys p − window + 1 .. p.
//
// The cache is read once per kv head and 8 NT columns, a column being a query head of a token. Codes are used as they lie: the
// four bits in the lowest place of a half word ARE the float16 c · 2^-24, one place up 16 c · 2^-24, so an AND and a multiplication
// that takes the zero off (q4_minus) make an operand (c − z) 2^-9 of mma.sync m16n8k16, with 16 keys (scores) or 16 columns of the values
// (output) as its rows and the query columns as its columns: nothing is wasted on padding up to eight heads. Scales are applied to
// what is small:
//   score  Σ_groups s Σ q' (c − z), q' = q times a power of two that brings a head's largest entry to 2^14: exact for bfloat16 entries
//          down to 2^-27 of the largest, off by 2^-35 of the largest below; float32 as two such numbers, 22 bits;
//   output Σ_keys (p s) (c − z): p s as a float16 number (off by 2^-11 of itself; float32: two, the second times 2^11, 2^-22), so that
//          the scale s of a key's group of values costs no rounding of the values.
// The operands are c − z: tensor cores cut partial sums to 24 bits, and sums of codes are many times those of c − z, which are nothing where
// keys or values are zeros beside a large one of their group. (With z Σ q' and z Σ p s taken off at the end a value of zero came to 2^-24 of
// 15 s a page, and a channel of large keys to errors of the scores.) With float32 queries a page's sums are added in 32 bits; 2,000 to
// 30,000 keys are then 2.4e-7 off 64 bits, a plain evaluation in 32 bits 5 to 9e-7.
// Two references, both moved in powers of two. A column's scores have one that follows the largest in steps: it moves only when a score
// passes it by more than 2^8. And p s is multiplied by a power of two of its own for EVERY column and group of 32 columns of the values,
// lowered (with the group's sums) when a product would pass float16: its largest then lies in 2^8 .. 2^9, so that p s is off by no
// less than 2^-33 of the group's largest (float32: 2^-44), whatever other groups, heads or keys of little weight hold. When the scores'
// reference rises by a factor, these rise with it, and the sums stay as they are. (One reference for the largest scale of any group and key
// lost whole groups behind one large value; it took 50.5 us at 64 sequences of 2,048 keys where this takes 53.1, 46.5 / 48.4 for 40 tokens
// behind 6,000, 221 / 251 for 2,000 float32 tokens of three prompts.)
//
// A page of a kv head is one run of bytes and arrives by one bulk copy in a ring; four warps take 16 of its keys each and keep
// sums of their own, joined at the end in the order of the warps, then of the chunks: results do not depend on timing.
// A key or value that is not finite reaches the columns that see it and no others.
//
// Measured (32 heads on 8 of 128, bfloat16): 64 sequences of up to 2,048 keys 53 us for 122 MB of pages, 2.3 TB/s; 3 of about 50,000 76;
// 40 tokens behind 6,000 48; one sequence of 2,048 with heads of 64 11. Some 530 instructions a warp for 16 keys and eight columns; no
// pipe is full (issue slots 60 %, the arithmetic pipe 53 % at 64 sequences): latency at 16 warps an SM, a start and an end are the rest;
// more CTAs an SM (five of eight columns, three of sixteen) gain nothing.
#include "kv4.cuh"
#include "async_copy.cuh"
#include <cuda_fp16.h>

SP_API const char* sp_kv4_attention_last_error() { return sp_error_text; }
SP_DEFINE_RANGE_API(kv4_attention)

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int WARPS = 4;
constexpr int STAGES = 4;
constexpr float STEP = 8.0f;                // how far a score may pass the reference, log2
constexpr int MOST_NORM = 120;              // the largest power of two that p s is multiplied by, log2

struct Args {
    const void* q;                 // [T][nh * hd]
    void* out;                     // the same shape
    const uint8_t* pool;
    const int* seq_start;          // [n_seqs + 1]; null: one token each
    const int* positions;          // [T]
    const int* seq_row;
    const int* page_table;
    const float* sink;             // [nh] or null
    float* part;                   // [T * nh][n_chunks][hd], then [T * nh][n_chunks] (reference, sum); unused with one chunk
    int* status;
    int max_pages, nh, nkv, window, chunk_pages, n_chunks, T, n_seqs;
    float scale;
    SpRange rg;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {          // of an 8 x 8 matrix of half words spread over the warp
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
// N words from shared memory, and N half words (as words of two)
template <int N> __device__ __forceinline__ void lds_words(uint32_t at, uint32_t (&w)[N]) {
    if constexpr (N == 4) asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
    else if constexpr (N == 2) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
    else
#pragma unroll
        for (int i = 0; i < N; ++i) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[i]) : "r"(at + 4 * i));
}
template <int N> __device__ __forceinline__ void lds_halves(uint32_t at, uint32_t (&w)[(N + 1) / 2]) {
    if constexpr (N == 4) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
    else if constexpr (N == 2) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at));
    else {
#pragma unroll
        for (int i = 0; i < (N + 1) / 2; ++i) w[i] = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            uint16_t h;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(at + 2 * i));
            w[i / 2] |= (uint32_t)h << (16 * (i & 1));
        }
    }
}
__device__ __forceinline__ float finite_or_nan(float v) { return fabsf(v) < INFINITY ? v : __int_as_float(0x7fc00000); }
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 w = *(const uint4*)p;
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = finite_or_nan(__uint_as_float(u[i] << 16)); v[2 * i + 1] = finite_or_nan(__uint_as_float(u[i] & 0xffff0000u)); }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = finite_or_nan(v[i]);
}

// scale (group i of a row's half words) and zero as numbers; the zero from the last place of 2^23
__device__ __forceinline__ float scale_at(const uint32_t* m, int i) {
    return __uint_as_float(i & 1 ? m[i >> 1] & 0xfff00000u : (m[i >> 1] << 16) & 0xfff00000u);
}
// powers of two
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ float log2_of(float v) { return (float)((int)(__float_as_uint(v) >> 23) - 127); }      // rounded down, v > 0
// over a fragment's rows; what is not a number is left out
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
// two at a time
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

template <typename TQ, int NG, int NT>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 ? 4 : 2)
attend_kernel(const Args a) {
    constexpr int HD = 32 * NG, PARTS = sizeof(TQ) == 4 ? 2 : 1, COLS = 8 * NT, TILE = kv4_tile_bytes(HD), MW = (NG + 1) / 2;
    // groups of columns whose p s are formed before one vote whether they fit (64 sequences of 2,048 keys: 54.6 us with one, 52.3 with
    // two, 53.1 with all four; float32, registers: 69.9 with one, 71.9 with two)
    constexpr int AT_ONCE = PARTS == 2 ? 1 : 2;
    constexpr bool Q_HELD = NT == 1 && PARTS == 1;                   // the queries' operands in registers, else in shared memory
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES];
    __shared__ int failed, fetched;
    __shared__ float ref_s[WARPS][COLS], sum_s[WARPS][COLS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int seq = blockIdx.z, kvh = blockIdx.y % a.nkv, tile = blockIdx.y / a.nkv, chunk = blockIdx.x, G = a.nh / a.nkv;
    const int tok0 = a.seq_start ? a.seq_start[seq] : seq, n_tok = a.seq_start ? a.seq_start[seq + 1] - tok0 : 1;
    const int col0 = tile * COLS, n_cols = min(COLS, n_tok * G - col0);
    if (n_cols <= 0) return;
    const int first_pos = a.positions[tok0 + col0 / G], last_pos = a.positions[tok0 + (col0 + n_cols - 1) / G];        // of the tile's tokens
    const int lowest = a.window ? max(0, first_pos + 1 - a.window) : 0;
    // the last chunk takes what there is: a sequence may be longer than the split was made for
    const int page0 = lowest / KV4_PAGE + chunk * a.chunk_pages, page_end = last_pos / KV4_PAGE + 1;
    const int n_pages = max(0, (chunk + 1 == a.n_chunks ? page_end : min(page0 + a.chunk_pages, page_end)) - page0), row = sp_checked_row(a.seq_row[seq], a.rg);
    const int* table = a.page_table + (size_t)row * a.max_pages;
    constexpr int ROW = HD + 8;                                      // of the joined sums: neighbouring columns' rows lie in other banks
    float* acc = (float*)smem;                                       // [warp][column][ROW]
    const uint32_t ring = smem_u32(smem), q_at = ring + STAGES * TILE;

    if (threadIdx.x == 0) {
        failed = fetched = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    // the first warp's lanes hold the numbers of 32 pages
    int held = 0;
    auto hold = [&](int i) { if (i + lane < n_pages) held = sp_checked_page(table[sp_checked_entry(page0 + i + lane, a.max_pages, a.rg)], a.rg); };
    auto fetch = [&](int i, int page) {                              // one thread
        const int s = i % STAGES;
        mbar_expect_tx(smem_u32(&full[s]), TILE);
        fetched = i + 1;
        bulk_copy_g2s(ring + s * TILE, a.pool + ((size_t)page * a.nkv + kvh) * TILE, TILE, smem_u32(&full[s]));
    };
    if (warp == 0) {
        hold(0);
#pragma unroll
        for (int i = 0; i < STAGES; ++i) {
            const int page = __shfl_sync(0xffffffffu, held, i);
            if (lane == 0 && i < n_pages) fetch(i, page);
        }
    }

    // The queries: lane (column g, dims 32 i + 8 t ..). Columns that are not there are zeros and see nothing.
    uint32_t qh[Q_HELD ? NG : 1][4];
    float unit[NT][2];                                               // of columns 2 t and 2 t + 1
    int pos[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int c = col0 + n * 8 + g, tok = min(c / G, n_tok - 1);
        const bool there = n * 8 + g < n_cols;
        const TQ* from = (const TQ*)a.q + ((size_t)(tok0 + tok) * a.nh + kvh * G + c % G) * HD + 8 * t;
        float v[NG][8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            load8(from + 32 * i, v[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (!there) v[i][e] = 0.0f;
                top = fmaxf(top, fabsf(v[i][e]));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int up = top > 0.0f ? min(94, max(-94, 141 - (int)(__float_as_uint(top) >> 23))) : 0;
        const float by = __uint_as_float((uint32_t)(127 + up) << 23), back = __uint_as_float((uint32_t)(136 - up) << 23) * a.scale * LOG2E;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            uint32_t h[PARTS][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float lo = v[i][2 * j] * by, hi = v[i][2 * j + 1] * by, f = j & 1 ? 0.0625f : 1.0f;
                h[0][j] = half2_of(lo * f, hi * f);
                if (PARTS == 2) {
                    const float2 first = __half22float2(*(const __half2*)&h[0][j]);
                    h[PARTS - 1][j] = half2_of(lo * f - first.x, hi * f - first.y);
                }
            }
            if (Q_HELD) {
#pragma unroll
                for (int j = 0; j < 4; ++j) qh[Q_HELD ? i : 0][j] = h[0][j];
            } else if (warp == 0) {
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(q_at + (uint32_t)(((n * NG + i) * PARTS + part) * 32 + lane) * 16), "r"(h[part][0]), "r"(h[part][1]), "r"(h[part][2]), "r"(h[part][3]) : "memory");
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            unit[n][e] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * e);
            const int ce = n * 8 + 2 * t + e;
            pos[n][e] = ce < n_cols ? a.positions[tok0 + (col0 + ce) / G] : -1;
        }
    }
    if (!Q_HELD) __syncthreads();

    // ref: the score (log2, rounded up) that a column's probabilities are relative to; limit: how far a raw score may go under it. O holds
    // the sums times a power of two, norm, for every column and group of the values' columns
    float O[NT][NG][2][4], norm[NT][NG][2], sum[NT][2], ref[NT][2], limit[NT][2];
    uint32_t poison[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        poison[n] = 0;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            norm[n][i][0] = norm[n][i][1] = two_to(MOST_NORM);
#pragma unroll
            for (int h = 0; h < 2; ++h) O[n][i][h][0] = O[n][i][h][1] = O[n][i][h][2] = O[n][i][h][3] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) { sum[n][e] = ref[n][e] = 0.0f; limit[n][e] = -INFINITY; }
    }

    for (int it = 0; it < n_pages; ++it) {
        // the stage that every warp had done with a page ago gets the next page
        if (warp == 0 && it > 0 && it - 1 + STAGES < n_pages) {
            const int i = it - 1 + STAGES;
            if (i % 32 == 0) hold(i);
            const int page = __shfl_sync(0xffffffffu, held, i % 32);
            if (lane == 0 && mbar_wait_flag(smem_u32(&empty[(it - 1) % STAGES]), ((it - 1) / STAGES) & 1, a.status, 171, &failed)) fetch(i, page);
        }
        __syncwarp();
        mbar_wait_flag(smem_u32(&full[it % STAGES]), (it / STAGES) & 1, a.status, 172, &failed);
        const int page_pos = (page0 + it) * KV4_PAGE;
        const uint32_t at = ring + (it % STAGES) * TILE;
        const int r0 = warp * 16 + g;                            // rows of the page's keys as they lie: this lane's are r0 and r0 + 8
        const int p0 = warp * 16 + (g & 1) * 4 + (g >> 1), key = page_pos + p0;        // their positions: this and 8 on
        float x[NT][4];
        uint32_t m0[MW], m1[MW];                                     // the values' scales of this lane's two keys
        // scores of 16 keys: rows g and g + 8, columns 2 t and 2 t + 1
#pragma unroll
        for (int n = 0; n < NT; ++n) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.0f;
        uint32_t k0[NG], k1[NG], km0[MW], km1[MW];
        lds_words<NG>(at + r0 * (HD / 2) + t * (NG * 4), k0);
        lds_words<NG>(at + (r0 + 8) * (HD / 2) + t * (NG * 4), k1);
        lds_halves<NG>(at + kv4_k_meta(HD) + r0 * (NG * 2), km0);
        lds_halves<NG>(at + kv4_k_meta(HD) + (r0 + 8) * (NG * 2), km1);
        lds_halves<NG>(at + kv4_v_meta(HD) + p0 * (NG * 2), m0);
        lds_halves<NG>(at + kv4_v_meta(HD) + (p0 + 8) * (NG * 2), m1);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const float s0 = scale_at(km0, i), s1 = scale_at(km1, i);
            const uint32_t u0 = k0[i], u1 = k1[i], w0 = u0 >> 8, w1 = u1 >> 8;
            uint32_t c[8] = {u0 & 0x000f000fu, u1 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x00f000f0u, w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u};
            const uint32_t y0 = __byte_perm(km0[i >> 1], 0, i & 1 ? 0x3232 : 0x1010) & 0x000f000fu, y1 = __byte_perm(km1[i >> 1], 0, i & 1 ? 0x3232 : 0x1010) & 0x000f000fu;
#pragma unroll
            for (int k = 0; k < 8; ++k) c[k] = q4_minus(c[k], q4_zero((k & 1 ? y1 : y0) << (k & 2 ? 4 : 0)));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int part = PARTS - 1; part >= 0; --part) {
                    uint4 qv;
                    if (Q_HELD) qv = make_uint4(qh[Q_HELD ? i : 0][0], qh[Q_HELD ? i : 0][1], qh[Q_HELD ? i : 0][2], qh[Q_HELD ? i : 0][3]);
                    else qv = lds16(q_at + (uint32_t)(((n * NG + i) * PARTS + part) * 32 + lane) * 16);
                    mma_f16(acc, c[0], c[1], c[2], c[3], qv.x, qv.y);
                    mma_f16(acc, c[4], c[5], c[6], c[7], qv.z, qv.w);
                }
                float (&y)[4] = x[n];
                const float2 u = fma2(make_float2(s0, s0), make_float2(acc[0], acc[1]), make_float2(y[0], y[1]));
                const float2 w = fma2(make_float2(s1, s1), make_float2(acc[2], acc[3]), make_float2(y[2], y[3]));
                y[0] = u.x; y[1] = u.y; y[2] = w.x; y[3] = w.y;
            }
        }
        if (page_pos + KV4_PAGE - 1 > first_pos || (a.window && page_pos < last_pos + 1 - a.window)) {       // not all of it is seen by all
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int p = pos[n][e & 1], k = key + (e & 2) * 4;
                    if (k > p || (a.window && k <= p - a.window)) x[n][e] = -INFINITY;
                }
#pragma unroll
            for (int i = 0; i < MW; ++i) {                       // what nobody sees may be anything
                if (key > last_pos || key < lowest) m0[i] = 0;
                if (key + 8 > last_pos || key + 8 < lowest) m1[i] = 0;
            }
        }
        // does a score pass its column's reference by too much?
        bool moves = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) moves |= x[n][e] > limit[n][e & 1];
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float big = column_max(fmaxf(x[n][e], x[n][2 + e]));
                    if (!(big > limit[n][e])) continue;
                    const float top = ceilf(big * unit[n][e]), up = limit[n][e] != -INFINITY ? top - ref[n][e] : 0.0f;
                    limit[n][e] = (top + STEP) / unit[n][e];
                    ref[n][e] = top;
                    sum[n][e] *= ex2(-up);
                    // the sums of the values stay: their power of two rises by as much as the probabilities fall, as far as it goes
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const float was = log2_of(norm[n][i][e]), now = fminf(was + up, MOST_NORM), f = ex2(now - was - up);
                        norm[n][i][e] = two_to((int)now);
#pragma unroll
                        for (int h = 0; h < 2; ++h) { O[n][i][h][e] *= f; O[n][i][h][2 + e] *= f; }
                    }
                }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[n][e] = ex2(fmaf(x[n][e], unit[n][e & 1], -ref[n][e & 1]));
            sum[n][0] += x[n][0] + x[n][2];
            sum[n][1] += x[n][1] + x[n][3];
        }
        // the output of 16 keys
        uint32_t v[4][MW], mz[4][MW];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int p = warp * 16 + 4 * k + t, sw = HD == 128 ? (p & 2) << 4 : 0;
            lds_halves<NG>(at + kv4_v_codes(HD) + p * (HD / 2) + ((g * NG * 2) ^ sw), v[k]);
            lds_halves<NG>(at + kv4_v_meta(HD) + p * (NG * 2), mz[k]);
        }
#pragma unroll
        for (int i0 = 0; i0 < NG; i0 += AT_ONCE) {
            // p s as float16 numbers
            uint32_t h0[AT_ONCE][NT], h1[AT_ONCE][NT], over = 0;
            auto weigh = [&](int i, int n, uint32_t& h0, uint32_t& h1, float s0, float s1) {
                const float2 by = make_float2(norm[n][i][0], norm[n][i][1]);
                const float2 p = mul2(mul2(make_float2(x[n][0], x[n][1]), make_float2(s0, s0)), by), w = mul2(mul2(make_float2(x[n][2], x[n][3]), make_float2(s1, s1)), by);
                h0 = half2_of(p.x, p.y);
                h1 = half2_of(w.x, w.y);
            };
#pragma unroll
            for (int i = i0; i < NG && i < i0 + AT_ONCE; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    weigh(i, n, h0[i - i0][n], h1[i - i0][n], scale_at(m0, i), scale_at(m1, i));
                    over = __vimax3_u16x2(over, h0[i - i0][n], h1[i - i0][n]);
                }
            if (__any_sync(0xffffffffu, ((over + 0x04000400u) & 0x80008000u) != 0)) {        // beyond float16, or not a number
#pragma unroll
                for (int i = i0; i < NG && i < i0 + AT_ONCE; ++i) {
                    // scales that are not numbers: noted for the columns that see their keys, and taken as zero
                    float s0 = scale_at(m0, i), s1 = scale_at(m1, i);
                    const bool bad0 = !(s0 < INFINITY), bad1 = !(s1 < INFINITY);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int p = pos[n][e], from = a.window ? p - a.window : -1;
                            if ((bad0 && key <= p && key > from) || (bad1 && key + 8 <= p && key + 8 > from)) poison[n] |= 1u << (2 * i + e);
                        }
                    if (bad0) { s0 = 0.0f; m0[i >> 1] &= i & 1 ? 0xffffu : 0xffff0000u; }
                    if (bad1) { s1 = 0.0f; m1[i >> 1] &= i & 1 ? 0xffffu : 0xffff0000u; }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float big = column_max(fmaxf(x[n][e] * s0, x[n][2 + e] * s1));
                            if (!(big * norm[n][i][e] > 32768.0f)) continue;
                            const float now = two_to(8 - (int)log2_of(big)), f = ex2(log2_of(now) - log2_of(norm[n][i][e]));        // big · now in 2^8 .. 2^9
                            norm[n][i][e] = now;
#pragma unroll
                            for (int h = 0; h < 2; ++h) { O[n][i][h][e] *= f; O[n][i][h][2 + e] *= f; }
                        }
                        weigh(i, n, h0[i - i0][n], h1[i - i0][n], s0, s1);
                    }
                }
            }
#pragma unroll
            for (int i = i0; i < NG && i < i0 + AT_ONCE; ++i) {
                const int half = i & 1 ? 0x7632 : 0x5410;
                // keys t, 4 + t and 8 + t, 12 + t side by side
                const uint32_t u0 = __byte_perm(v[0][i >> 1], v[1][i >> 1], half), u1 = __byte_perm(v[2][i >> 1], v[3][i >> 1], half);
                const uint32_t w0 = u0 >> 8, w1 = u1 >> 8;
                uint32_t c[8] = {u0 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x000f000fu, u1 & 0x00f000f0u, w0 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x000f000fu, w1 & 0x00f000f0u};
                const uint32_t y0 = __byte_perm(mz[0][i >> 1], mz[1][i >> 1], half) & 0x000f000fu, y1 = __byte_perm(mz[2][i >> 1], mz[3][i >> 1], half) & 0x000f000fu;
#pragma unroll
                for (int k = 0; k < 8; ++k) c[k] = q4_minus(c[k], q4_zero((k & 2 ? y1 : y0) << (k & 1 ? 4 : 0)));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint32_t b0 = transposed(h0[i - i0][n]), b1 = transposed(h1[i - i0][n]);
                    if (PARTS == 2) {
                        // what is left of p s, times 2^11; sums of a page of their own, added in 32 bits: the tensor cores' own additions cut
                        const float2 by = make_float2(norm[n][i][0], norm[n][i][1]);
                        auto rest = [&](float p, float q, float s, uint32_t h) {
                            const float2 f = __half22float2(*(const __half2*)&h), r = mul2(mul2(make_float2(p, q), make_float2(s, s)), by);
                            const float2 d = mul2(fma2(f, make_float2(-1.0f, -1.0f), r), make_float2(2048.0f, 2048.0f));
                            return transposed(half2_of(d.x, d.y));
                        };
                        const uint32_t l0 = rest(x[n][0], x[n][1], scale_at(m0, i), h0[i - i0][n]), l1 = rest(x[n][2], x[n][3], scale_at(m1, i), h1[i - i0][n]);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float o[4] = {0.f, 0.f, 0.f, 0.f}, l[4] = {0.f, 0.f, 0.f, 0.f};
                            mma_f16(l, c[4 * h], c[4 * h + 1], c[4 * h + 2], c[4 * h + 3], l0, l1);
                            mma_f16(o, c[4 * h], c[4 * h + 1], c[4 * h + 2], c[4 * h + 3], b0, b1);
#pragma unroll
                            for (int e = 0; e < 4; e += 2) {
                                const float2 up = make_float2(4.8828125e-4f, 4.8828125e-4f), one = make_float2(1.0f, 1.0f);
                                const float2 t = fma2(fma2(make_float2(l[e], l[e + 1]), up, make_float2(o[e], o[e + 1])), one, make_float2(O[n][i][h][e], O[n][i][h][e + 1]));
                                O[n][i][h][e] = t.x;
                                O[n][i][h][e + 1] = t.y;
                            }
                        }
                        continue;
                    }
                    mma_f16(O[n][i][0], c[0], c[1], c[2], c[3], b0, b1);
                    mma_f16(O[n][i][1], c[4], c[5], c[6], c[7], b0, b1);
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&empty[it % STAGES]));
    }

    // each warp's sums over its lanes, its columns' numbers in shared memory (where the pages were); then the warps', in their order
    __syncthreads();
    if (failed) {                                                    // a wait ran out: copies may still be on their way into this CTA's memory
        if (threadIdx.x == 0)
            for (int i = max(0, fetched - STAGES); i < fetched; ++i) mbar_wait(smem_u32(&full[i % STAGES]), (i / STAGES) & 1, nullptr, 0);
        __syncthreads();
        return;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int o = 4; o < 32; o *= 2) {
#pragma unroll
            for (int e = 0; e < 2; ++e) sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], o);
            poison[n] |= __shfl_xor_sync(0xffffffffu, poison[n], o);
        }
        if (g == 0)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                ref_s[warp][n * 8 + 2 * t + e] = limit[n][e] == -INFINITY && sum[n][e] == 0.0f ? -INFINITY : ref[n][e];
                sum_s[warp][n * 8 + 2 * t + e] = sum[n][e];
            }
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float back = __uint_as_float((254u << 23) - __float_as_uint(norm[n][i][e]));
                    float2 v = make_float2(O[n][i][h][e] * (back * 512.0f), O[n][i][h][2 + e] * (back * 32.0f));
                    if (poison[n] >> (2 * i + e) & 1) v.x = v.y = __int_as_float(0x7fc00000);
                    *(float2*)(acc + (warp * COLS + n * 8 + 2 * t + e) * ROW + 32 * i + 4 * g + 2 * h) = v;
                }
    }
    __syncthreads();
    for (int c = warp; c < n_cols; c += WARPS) {
        float big = ref_s[0][c], total = 0.0f, f[WARPS];
#pragma unroll
        for (int k = 1; k < WARPS; ++k) big = fmaxf(big, ref_s[k][c]);
#pragma unroll
        for (int k = 0; k < WARPS; ++k) {
            f[k] = ref_s[k][c] == -INFINITY ? 0.0f : ex2(ref_s[k][c] - big);
            total += ref_s[k][c] == -INFINITY ? 0.0f : sum_s[k][c] * f[k];
        }
        float v[NG];
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            v[i] = 0.0f;
#pragma unroll
            for (int k = 0; k < WARPS; ++k)
                if (ref_s[k][c] != -INFINITY) v[i] = fmaf(f[k], acc[(k * COLS + c) * ROW + 32 * i + lane], v[i]);
        }
        const int head = kvh * G + (col0 + c) % G;
        const size_t out_row = (size_t)(tok0 + (col0 + c) / G) * a.nh + head;
        if (a.n_chunks > 1) {
            float* part = a.part + (out_row * a.n_chunks + chunk) * HD;
#pragma unroll
            for (int i = 0; i < NG; ++i) part[32 * i + lane] = v[i];
            if (lane == 0) ((float2*)(a.part + (size_t)a.T * a.nh * a.n_chunks * HD))[out_row * a.n_chunks + chunk] = make_float2(big, total);
            continue;
        }
        float down = 1.0f;
        if (a.sink) {
            const float y = a.sink[head] * LOG2E, most = fmaxf(big, y);
            down = big == -INFINITY ? 0.0f : ex2(big - most);
            total = total * down + ex2(y - most);
        }
#pragma unroll
        for (int i = 0; i < NG; ++i)                                 // (no key seen: zeros)
            sp_st((TQ*)a.out, out_row * HD + 32 * i + lane, big == -INFINITY ? 0.0f : v[i] * down / total);
    }
}

// The chunks' sums of a row (a token's head), in their order: a warp a row.
template <typename TQ>
__global__ void __launch_bounds__(128)
join_kernel(const Args a, int hd) {
    sp_wait_for_predecessor();
    const int lane = threadIdx.x & 31;
    const size_t rows = (size_t)a.T * a.nh, row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= rows || (a.seq_start && row >= (size_t)a.seq_start[a.n_seqs] * a.nh)) return;        // rows behind the last sequence stay as they are
    const float* part = a.part + row * a.n_chunks * hd;
    const float2* heads = (const float2*)(a.part + rows * a.n_chunks * hd) + row * a.n_chunks;
    float big = -INFINITY;
    for (int c = lane; c < a.n_chunks; c += 32) big = fmaxf(big, sp_ld_written(heads + c).x);
    big = sp_warp_max(big);
    float sum = 0.0f;
    for (int c = lane; c < a.n_chunks; c += 32) {
        const float2 h = sp_ld_written(heads + c);
        if (h.x != -INFINITY) sum += h.y * ex2(h.x - big);
    }
    float f = 1.0f, total = sp_warp_sum(sum);
    if (a.sink) {
        const float y = a.sink[row % a.nh] * LOG2E, most = fmaxf(big, y);
        f = big == -INFINITY ? 0.0f : ex2(big - most);
        total = total * f + ex2(y - most);
    }
    float v[KV4_MAX_HD / 32] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = 0; c0 < a.n_chunks; c0 += 32) {
        const float2 h = c0 + lane < a.n_chunks ? sp_ld_written(heads + c0 + lane) : make_float2(-INFINITY, 0.0f);
        const float mine = h.x == -INFINITY ? -1.0f : ex2(h.x - big);
        for (int c = 0; c < min(32, a.n_chunks - c0); ++c) {
            const float w = __shfl_sync(0xffffffffu, mine, c);
            if (w < 0.0f) continue;                                  // a chunk without a key that the row sees (one of weight zero counts where it is NaN)
#pragma unroll
            for (int k = 0; k < KV4_MAX_HD / 32; ++k)
                if (32 * k < hd) v[k] = fmaf(w, sp_ld_written(part + (size_t)(c0 + c) * hd + 32 * k + lane), v[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < KV4_MAX_HD / 32; ++k)
        if (32 * k < hd) sp_st((TQ*)a.out, row * hd + 32 * k + lane, big == -INFINITY ? 0.0f : v[k] * f / total);
}

template <typename TQ, int NG, int NT>
int launch(const Args& a, int n_seqs, int tiles, cudaStream_t stream) {
    constexpr int HD = 32 * NG, PARTS = sizeof(TQ) == 4 ? 2 : 1, RING = STAGES * kv4_tile_bytes(HD), SUMS = WARPS * 8 * NT * (HD + 8) * 4;
    constexpr int HELD = RING + (NT == 1 && PARTS == 1 ? 0 : NT * NG * PARTS * 512), SMEM = HELD > SUMS ? HELD : SUMS;
    static SpPerDevice configured;
    if (!configured.done()) {
        cudaError_t e = cudaFuncSetAttribute(attend_kernel<TQ, NG, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) SP_FAIL("kv4_attention: cannot reserve %d bytes of shared memory: %s", SMEM, cudaGetErrorString(e));
        configured.mark();
    }
    attend_kernel<TQ, NG, NT><<<dim3(a.n_chunks, a.nkv * tiles, n_seqs), WARPS * 32, SMEM, stream>>>(a);
    SP_CHECK_LAUNCH("kv4_attention");
    if (a.n_chunks > 1)
        SP_CHECK_CALL("kv4_attention", sp_launch_dependent(join_kernel<TQ>, dim3((unsigned)(((size_t)a.T * a.nh + 3) / 4)), dim3(128), 0, stream, a, 32 * NG));
    return 0;
}

template <typename TQ, int NG>
int launch(const Args& a, int n_seqs, int nt, int max_new, cudaStream_t stream) {
    const int G = a.nh / a.nkv, tiles = (max_new * G + 8 * nt - 1) / (8 * nt);
    if ((long long)a.nkv * tiles > 65535 || n_seqs > 65535) SP_FAIL("kv4_attention: %d sequences of %d tokens, %d kv heads", n_seqs, max_new, a.nkv);
    if (nt == 2) return launch<TQ, NG, 2>(a, n_seqs, tiles, stream);
    return launch<TQ, NG, 1>(a, n_seqs, tiles, stream);
}

template <typename TQ>
int launch(const Args& a, int n_seqs, int nt, int max_new, int hd, cudaStream_t stream) {
    switch (hd) {
        case 32: return launch<TQ, 1>(a, n_seqs, nt, max_new, stream);
        case 64: return launch<TQ, 2>(a, n_seqs, nt, max_new, stream);
        case 96: return launch<TQ, 3>(a, n_seqs, nt, max_new, stream);
        default: return launch<TQ, 4>(a, n_seqs, nt, max_new, stream);
    }
}

}  // namespace

// Floats of scratch that a call needs.
SP_API long long sp_kv4_attend_scratch(int T, int nh, int hd, int n_chunks) { return n_chunks > 1 ? (long long)T * nh * n_chunks * (hd + 2) : 0; }

// out [T, nh·hd] for queries q of the same shape and type (bfloat16 or float32). ``seq_start`` [n_seqs + 1], null: one token a
// sequence. ``max_new``: the most tokens of a sequence. ``nt``: 8 nt columns a CTA (1 or 2). ``chunk_pages``, ``n_chunks``:
// the split of the keys, from the first that a CTA's tokens see.
SP_API int sp_kv4_attend(const void* q, void* out, int dt, const void* pool, const int* seq_start, const int* positions, const int* seq_row,
                         const int* page_table, int max_pages, int page_size, int T, int n_seqs, int max_new, int nh, int nkv, int hd,
                         int window, float scale, const float* sink, int nt, int chunk_pages, int n_chunks, float* scratch,
                         long long scratch_floats, int* status, cudaStream_t stream) {
    if (T <= 0 || n_seqs <= 0) return 0;
    if (hd <= 0 || hd % 32 || hd > KV4_MAX_HD) SP_FAIL("kv4_attention: head sizes 32, 64, 96 and 128, got %d", hd);
    if (page_size != KV4_PAGE) SP_FAIL("kv4_attention: pages of %d positions, got %d", KV4_PAGE, page_size);
    if (nkv <= 0 || nh <= 0 || nh % nkv) SP_FAIL("kv4_attention: %d heads are no multiple of %d kv heads", nh, nkv);
    if (nt != 1 && nt != 2) SP_FAIL("kv4_attention: 8 or 16 columns a CTA, got 8 x %d", nt);
    if (window < 0 || max_new <= 0 || (!seq_start && (max_new != 1 || T != n_seqs))) SP_FAIL("kv4_attention: window %d, %d tokens of %d sequences, at most %d of one", window, T, n_seqs, max_new);
    if (chunk_pages <= 0 || n_chunks <= 0 || n_chunks > 65535) SP_FAIL("kv4_attention: %d chunks of %d pages", n_chunks, chunk_pages);
    if (!(scale > 0.0f) || scale > 1e30f) SP_FAIL("kv4_attention: a positive scale is wanted, got %g", scale);
    if (((uintptr_t)q & 15) || ((uintptr_t)pool & 15)) SP_FAIL("kv4_attention: queries and pages must start on 16-byte boundaries");
    if (sp_kv4_attend_scratch(T, nh, hd, n_chunks) > scratch_floats) SP_FAIL("kv4_attention: %lld floats of scratch are needed, got %lld", sp_kv4_attend_scratch(T, nh, hd, n_chunks), scratch_floats);
    const Args a{q, out, (const uint8_t*)pool, seq_start, positions, seq_row, page_table, sink, scratch, status,
                 max_pages, nh, nkv, window, chunk_pages, n_chunks, T, n_seqs, scale, sp_range_host};
    return dt == SP_DT_F32 ? launch<float>(a, n_seqs, nt, max_new, hd, stream) : launch<__nv_bfloat16>(a, n_seqs, nt, max_new, hd, stream);
}
