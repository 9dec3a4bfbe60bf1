// The product of four-bit weights (q4.cuh, layout in q4w.cuh) with some dozens to some hundreds of bfloat16 rows on the
// 5th-generation tensor cores: out[M, N] = x[M, K] · Ŵ[N, K]ᵀ.
//
// A CTA owns 128 packed rows of W (eight tiles of 16; gated: 64 outputs, gate and up tiles in turns), up to 256 rows of x and a piece
// of K; the pieces' CTAs form a cluster. Per 128 columns of K (a stage):
//   warp 0     one thread fetches the eight tiles' codes, their scales and x, 2 x 64 columns, each by TMA (as 16 bulk copies of a
//              tile's bytes, of one thread or of 16: 2 x 8192 x 2048 with 17 rows of x 24.9 and 21.8 us);
//   warps 2-17 a thread owns a row of W and 64 of its columns: the codes out of shared memory, (128 + c) − (128 + z) times s in
//              bfloat16 pairs, which is exact, into TENSOR memory, where the A operand may lie: W's numbers pass through no
//              shared memory and need no swizzle;
//   warp 1     one thread issues tcgen05.mma (A from tensor memory, B = x from shared memory, M 128, N = rows of x, K 16).
// So W is read from memory in four bits and the products are those of bfloat16 weights. Epilogue as in tc_mid.cu: the accumulator
// goes to shared memory as [row of x][128], the pieces of K are added in their order through distributed shared memory, a warp a
// row of x. More than 256 rows of x are cut into equal parts, each of which takes the codes apart again.
// Measured, us, against unpacking the weight and the bfloat16 product (fused / unpacked; M rows of x, four weights in turns):
//   M                   17           64           128          256          512          1024
//   2 x 8192 x 2048     12.2/25.6    13.8/28.4    16.9/32.1    25.3/33.3    49.2/44.7    96.0/68.1    (gate and up)
//   2 x 14336 x 4096    32.3/98.8    35.6/99.3    49.1/103     73.2/111     139/150      250/228
//   4096 x 4096          9.7/17.6    10.8/19.9    12.1/21.3    16.7/24.6    21.0/29.4    30.9/36.6
//   4096 x 14336        18.2/44.0    19.1/46.8    20.9/52.0    30.9/61.2    48.1/80.4    88.9/107
//   2048 x 2048          7.6/10.0     8.7/11.0     9.6/12.8    12.8/13.6    13.0/15.5    15.5/20.2
//   6144 x 4096         12.1/21.0    13.0/22.7    14.4/27.1    20.2/29.5    30.9/38.9    57.7/60.0
// What bounds it: at few rows a stage takes 0.37 us an SM, of which 0.27 is the products of 32 rows of x (64 cycles each with A in
// tensor memory, whether of 16 or of 64 rows) and 0.25 the instructions that take the codes apart, side by side but in one
// another's way; from 128 rows on x's way from L2 to every CTA (11 TB/s), and the start and epilogue, 5 us and 15 ns a row of x. What helped on the
// way (2 x 14336 x 4096, 17 rows): one TMA copy for the eight tiles' codes, 74 -> 52 us; elect.sync in place of a lane's number, so
// that a product is issued from uniform registers (100 cycles each before), and one wait a stage there, 52 -> 35; the working
// warps in two halves that take stages in turns, 35 -> 32.
// Every mbarrier wait is bounded and records a code in ``status``; no load uses cluster multicast.
#include "tcgen05.cuh"
#include "q4w.cuh"
#include <string.h>

SP_API const char* sp_q4_tc_last_error() { return sp_error_text; }
SP_DEFINE_RANGE_API(q4_tc)

namespace {

constexpr int BW = 128, TILES = 8;          // packed rows of a CTA, tiles of 16
constexpr int MAX_NT = 256, MAX_STAGES = 12, MAX_SLOTS = 4, MAX_PIECES = 8;
constexpr int WORK_WARPS = 16;
constexpr int THREADS = 64 + 32 * WORK_WARPS;
constexpr int SMEM_LIMIT = 220 * 1024, SMEM_HALF = 112 * 1024;      // of an SM's one CTA, of one of two
constexpr int A_COLS = 64;                  // tensor-memory columns of a slot of A
enum { MODE_STORE = 0, MODE_ACCUMULATE = 1, MODE_SILU_MUL = 2 };

struct Args {
    void* out;
    long long ldo;
    int* status;
    int out_dt, M, rows, half, tiles, blocks, mode, nt, pieces, stages, slots;      // stages of x and codes in shared memory, slots of A in tensor memory
    uint32_t tmem_cols, d_cols;             // d_cols: where A's slots begin
    int wide;                               // whether four outputs go in one store
    SpGate ga;
};

// bytes of a stage's codes and scales; x's tiles begin on 1,024-byte boundaries
__host__ __device__ constexpr uint32_t stage_codes(int group) { return (uint32_t)(TILES * (1024 + q4w_meta_bytes(group)) + 1023) & ~1023u; }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}
// 128-byte swizzle within 1,024 bytes: rows of 128 bytes, their 16-byte pieces exchanged by the row's number. The eight rows g of a
// place t then lie in eight different pieces, and a thread that reads a row of W meets no other in its banks.
__device__ __forceinline__ uint32_t swizzle128(uint32_t at) { return at ^ ((at >> 3) & 0x70u); }

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}

// one lane of a warp; the compiler then knows that the branch is one thread's, and keeps what it passes on in uniform registers
__device__ __forceinline__ bool elected() {
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is != 0;
}
// a wait that finds its phase over costs one instruction
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, int* status, int code, volatile int* flag) {
    return mbar_try_wait(bar, parity) || mbar_wait_flag(bar, parity, status, code, flag);
}

template <int GROUP>
__global__ void __launch_bounds__(THREADS, 2)
q4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ CUtensorMap map_meta,
             const Args a) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[MAX_STAGES], bar_empty[MAX_STAGES], bar_a[MAX_SLOTS], bar_used[MAX_SLOTS], bar_acc;
    __shared__ uint32_t tmem_slot;
    __shared__ int failed, asked;                                    // a wait ran out; stages that copies were asked for
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row_tile = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
    const int tok0 = blockIdx.y * a.nt, count = min(a.nt, a.M - tok0);
    const int per = (a.blocks + a.pieces - 1) / a.pieces, b0 = piece * per, b1 = min(a.blocks, b0 + per);      // the host makes every piece non-empty
    const uint32_t x_bytes = (uint32_t)a.nt * 256, stage_bytes = x_bytes + stage_codes(GROUP);
    const uint32_t stage_bytes_in = x_bytes + TILES * (1024 + q4w_meta_bytes(GROUP));      // tiles behind the last come as zeros

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        for (int s = 0; s < a.slots; ++s) {
            mbar_init(smem_u32(&bar_a[s]), WORK_WARPS / 2);
            mbar_init(smem_u32(&bar_used[s]), 1);
        }
        mbar_init(smem_u32(&bar_acc), 1);
        failed = asked = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(a.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        if (elected()) {
            int s = 0;
            uint32_t ph = 1;
            for (int b = b0; b < b1; ++b) {
                if (!wait_for(smem_u32(&bar_empty[s]), ph, a.status, 181, &failed)) break;
                const uint32_t to = base + (uint32_t)s * stage_bytes, bar = smem_u32(&bar_full[s]);
                asked = b - b0 + 1;
                mbar_expect_tx(bar, stage_bytes_in);
                tma_load_4d(to + x_bytes, &map_codes, 0, 0, b, row_tile * TILES, bar);
                tma_load_3d(to + x_bytes + TILES * 1024, &map_meta, 0, b, row_tile * TILES, bar);
                tma_load_2d(to, &map_x, b * Q4W_BLOCK, tok0, bar);
                tma_load_2d(to + x_bytes / 2, &map_x, b * Q4W_BLOCK + 64, tok0, bar);
                if (++s == a.stages) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        if (elected()) {
            const uint32_t idesc = umma_idesc_bf16(BW, a.nt);
            int s = 0, slot = 0;
            uint32_t slot_ph = 0;
            for (int b = b0; b < b1; ++b) {
                if (!wait_for(smem_u32(&bar_a[slot]), slot_ph, a.status, 182, &failed)) break;
                tc_fence_after();                                    // (x is there too: those who took the codes apart have waited for it)
                const uint32_t x_at = base + (uint32_t)s * stage_bytes, a_at = tmem + a.d_cols + slot * A_COLS;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint64_t dx = umma_desc_sw128(x_at + h * (x_bytes / 2));
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc_mma_bf16_ts(tmem, a_at + h * 32 + k * 8, dx + 2 * k, idesc, (b != b0 || h != 0 || k != 0) ? 1u : 0u);
                }
                tc_commit(smem_u32(&bar_empty[s]));
                tc_commit(smem_u32(&bar_used[slot]));
                if (++s == a.stages) s = 0;
                if (++slot == a.slots) { slot = 0; slot_ph ^= 1u; }
            }
            tc_commit(smem_u32(&bar_acc));                           // also after a failed wait: the epilogue must not hang
        }
    } else {
        // Eight warps a stage, the two halves of the sixteen in turns: a stage's way through a warp (a wait, loads, stores to tensor
        // memory and their wait) is longer than its instructions. An even number of slots, no more than stages: a slot is one half's
        // only, and who finds it used knows that all stages before it were full, so the wait for a stage passes over no phase
        // although the stage's last use may have been the other half's.
        const int ew = warp - 2, q = warp & 3, turn = ew >> 3, h = (ew >> 2) & 1, row = q * 32 + lane;       // this thread's row of W, half of a stage
        const int g = row & 7, hi = (row >> 3) & 1, tile = row >> 4;
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        int s = turn, slot = turn;
        uint32_t ph = 0, slot_ph = 1;
        for (int b = b0 + turn; b < b1; b += 2) {
            if (!wait_for(smem_u32(&bar_used[slot]), slot_ph, a.status, 185, &failed)) break;            // what the slot held has been multiplied
            if (!wait_for(smem_u32(&bar_full[s]), ph, a.status, 183, &failed)) break;
            tc_fence_after();
            const uint32_t at = base + (uint32_t)s * stage_bytes + x_bytes, codes = at + tile * 1024 + hi * 8;
            const uint32_t meta = at + TILES * 1024 + tile * q4w_meta_bytes(GROUP) + g * (512 / GROUP) + hi * 2;
            uint32_t w[4][2];                                        // place t: columns 8 t.., 32 + 8 t..
            uint16_t m[2];
#pragma unroll
            for (int part = 0; part < 2; ++part) asm volatile("ld.shared.u16 %0, [%1];" : "=h"(m[part]) : "r"(meta + (64 * h + 32 * part) / GROUP * 4));
#pragma unroll
            for (int t = 0; t < 4; ++t)
                asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[t][0]), "=r"(w[t][1])
                             : "r"(codes + swizzle128((uint32_t)(h * 512 + (g * 4 + t) * 16))));
#pragma unroll
            for (int part = 0; part < 2; ++part) {                   // 32 columns
                uint32_t v[16];
                const uint32_t z = 0x43004300u | (m[part] & 15u) * 0x10001u, sc = (m[part] & 0xfff0u) * 0x10001u;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[4 * t + j] = bf2_mul(bf2_sub(q4_pair(w[t][part], j), z), sc);
                tc_st_32x16(tmem + lanes + a.d_cols + slot * A_COLS + h * 32 + part * 16, v);
            }
            tc_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bar_a[slot]));
            if ((s += 2) >= a.stages) { s -= a.stages; ph ^= 1u; }
            if ((slot += 2) >= a.slots) { slot = turn; slot_ph ^= 1u; }
        }
        wait_for(smem_u32(&bar_acc), 0, a.status, 184, &failed);
        tc_fence_after();
        // the accumulator into shared memory (the stages are free by now), [row of x][128 rows of W]
        asm volatile("bar.sync 1, 512;" ::: "memory");
#pragma unroll 1
        for (int c0 = (ew >> 2) * 32; c0 < count; c0 += 128) {
            uint32_t r[32];
            tc_ld_32x32(tmem + lanes + (uint32_t)c0, r);
            tc_ld_wait();
            const uint32_t to = base + (uint32_t)((c0 * BW + row) * 4);
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (c0 + j < count) asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + (uint32_t)(j * BW * 4)), "r"(r[j]) : "memory");
        }
    }
    // The tensor memory goes back before the CTAs of a cluster wait for one another: a CTA that held it there could keep it from one of
    // its own cluster on the same SM, or from a cluster of another stream that holds what this one's other CTAs wait for.
    tc_fence_before();
    __syncthreads();
    if (failed && threadIdx.x == 0)                                  // copies may still be on their way into this CTA's memory
        for (int i = max(0, asked - a.stages); i < asked; ++i) mbar_wait(smem_u32(&bar_full[i % a.stages]), (uint32_t)(i / a.stages) & 1u, nullptr, 0);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
    }
    __syncwarp();
    // every CTA of the cluster has left its piece in its shared memory
    if (a.pieces > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");

    if (warp >= 2 && !failed && !(a.status && *(volatile int*)a.status != 0)) {
        const bool gated = a.mode == MODE_SILU_MUL;
        const int share = (count + a.pieces - 1) / a.pieces, j0 = piece * share, j1 = min(count, j0 + share);
        const int n_out = gated ? a.half : a.rows, o = gated ? row_tile * 64 + 4 * (lane & 15) : row_tile * BW + 4 * lane;
        const int r0 = gated ? (lane & 15) / 4 * 32 + (lane & 3) * 4 : 4 * lane;       // where this lane's four (gate) rows lie
        for (int j = j0 + warp - 2; j < j1; j += WORK_WARPS) {
            if (gated && lane >= 16) continue;
            float v[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
            for (int p = 0; p < a.pieces; ++p) {
                uint32_t from = base + (uint32_t)((j * BW + r0) * 4);
                if (a.pieces > 1) asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(from), "r"(p));
                const float4 x = ld_cluster4(from);
                v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
                if (gated) {
                    const float4 y = ld_cluster4(from + 64);
                    u[0] += y.x; u[1] += y.y; u[2] += y.z; u[3] += y.w;
                }
            }
            if (gated)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = sp_gated(v[e], u[e], a.ga);
            const size_t to = (size_t)(tok0 + j) * a.ldo + o;
            if (a.wide && o + 4 <= n_out) {
                if (a.out_dt == SP_DT_F32) {
                    float4* dst = (float4*)((float*)a.out + to);
                    if (a.mode == MODE_ACCUMULATE) { const float4 old = *dst; v[0] += old.x; v[1] += old.y; v[2] += old.z; v[3] += old.w; }
                    *dst = make_float4(v[0], v[1], v[2], v[3]);
                } else {
                    const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), up = __floats2bfloat162_rn(v[2], v[3]);
                    *(uint2*)((__nv_bfloat16*)a.out + to) = make_uint2(*(const uint32_t*)&lo, *(const uint32_t*)&up);
                }
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (o + e >= n_out) break;
                if (a.mode == MODE_ACCUMULATE) ((float*)a.out)[to + e] += v[e];
                else sp_st_dt(a.out, a.out_dt, to + e, v[e]);
            }
        }
    }
    __syncwarp();
    // nobody leaves (and frees its shared memory) before every CTA has read what it needs
    if (a.pieces > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encode(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* ptr, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
           CUtensorMapSwizzle swizzle) {
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            SP_FAIL("q4_tc: the driver does not offer cuTensorMapEncodeTiled");
        fn = (EncodeTiledFn)p;
    }
    cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, type, rank, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) SP_FAIL("q4_tc: cuTensorMapEncodeTiled failed with code %d", (int)r);
    return 0;
}

struct Plan { int nt, token_tiles, pieces, resident, stages, slots, smem; uint32_t tmem_cols, d_cols; };

bool fill_plan(Plan& p, int M, int blocks, int group) {
    p.token_tiles = (M + MAX_NT - 1) / MAX_NT;
    p.nt = ((M + p.token_tiles - 1) / p.token_tiles + 15) / 16 * 16;
    const int mine = (blocks + p.pieces - 1) / p.pieces;
    if ((p.pieces - 1) * mine >= blocks) return false;                // no empty piece
    const int stage = p.nt * 256 + (int)stage_codes(group), held = p.nt * BW * 4;
    const int limit = p.resident == 2 ? SMEM_HALF : SMEM_LIMIT, cols = 512 / p.resident;
    p.d_cols = (p.nt + 31) / 32 * 32;
    p.slots = (cols - (int)p.d_cols) / A_COLS;
    p.slots = p.slots >= MAX_SLOTS ? MAX_SLOTS : p.slots & ~1;
    p.stages = (limit - 1024) / stage;
    if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
    if (p.stages > mine) p.stages = mine;
    if (p.slots > p.stages) p.slots = 2;
    const int ring = p.stages * stage;
    p.smem = (ring > held ? ring : held) + 1024;
    p.tmem_cols = cols;
    return p.stages >= (mine < 2 ? mine : 2) && p.slots >= 2 && p.smem <= limit;
}

// The pieces of K, and whether two CTAs share an SM (where there are more CTAs than SMs, and room for rings of three stages), by an
// estimate of the time, ns: a CTA takes a start and an epilogue that goes with its rows of x, a stage the taking apart of its codes
// (365), its products (2.55 a row of x) or its way from L2, which gives all SMs together some 11 KB a ns; clusters of 4 and 8 do not
// find room on every SM.
Plan plan_of(int M, int tiles, int blocks, int group, double* estimate) {
    const int row_tiles = (tiles + TILES - 1) / TILES, sms = sp_sm_count() > 0 ? sp_sm_count() : 148;
    Plan best{};
    double best_t = 0;
    for (int resident = 1; resident <= 2; ++resident)
        for (int pieces = 1; pieces <= MAX_PIECES; pieces *= 2) {
            Plan p{0, 0, pieces, resident, 0, 0, 0, 0, 0};
            const int room = pieces <= 2 ? sms : pieces == 4 ? sms * 136 / 148 : sms * 120 / 148;
            if (!fill_plan(p, M, blocks, group)) continue;
            const int ctas = row_tiles * pieces * p.token_tiles;
            if (resident == 2 && (ctas <= room || p.stages < 3)) continue;
            const int at_once = resident * room;
            double stage = resident * (2.55 * p.nt > 365.0 ? 2.55 * p.nt : 365.0), waves = (double)ctas / at_once;
            const double fetch = (ctas < at_once ? ctas : at_once) * ((double)p.nt * 256 + stage_codes(group)) / 11000.0;
            if (stage < fetch) stage = fetch;
            waves = waves <= 1 ? 1 : pieces == 1 ? waves + 0.3 : (ctas + at_once - 1) / at_once;      // single CTAs of two waves run side by side
            const double t = waves * (5000.0 + (blocks + pieces - 1) / pieces * stage + 15.0 * p.nt + (pieces > 1 ? 300.0 + 100.0 * pieces : 0.0));
            if (!best.nt || t < best_t) { best = p; best_t = t; }
        }
    if (estimate) *estimate = best_t;
    return best;
}

struct Maps { CUtensorMap x, codes, meta; };

template <int GROUP>
int launch(const Maps& m, const Args& a, const Plan& p, int row_tiles, cudaStream_t stream) {
    static SpPerDevice configured;
    if (!configured.done()) {
        cudaError_t e = cudaFuncSetAttribute(q4_tc_kernel<GROUP>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT);
        if (e != cudaSuccess) SP_FAIL("q4_tc: cannot reserve %d bytes of shared memory: %s", SMEM_LIMIT, cudaGetErrorString(e));
        configured.mark();
    }
    SP_CHECK_CALL("q4_tc", sp_launch_cluster(q4_tc_kernel<GROUP>, dim3(row_tiles * p.pieces, p.token_tiles), dim3(THREADS), (size_t)p.smem, stream, p.pieces, m.x, m.codes, m.meta, a));
    return 0;
}

}  // namespace

// The estimated time of a product with M rows of x, ns; 0 where no division fits.
SP_API double sp_q4_tc_estimate(int M, int rows, int K, int group, int half) {
    double t = 0;
    return M > 0 && plan_of(M, q4w_tiles(rows, half), (K + Q4W_BLOCK - 1) / Q4W_BLOCK, group, &t).nt ? t : 0;
}

// Modes as sp_q4_gemv (q4_kernels.cu); x bfloat16 with rows on 16-byte boundaries, M up to 1,024.
SP_API int sp_q4_tc(const void* x, const void* codes, const void* meta, void* out, int out_dt, int M, int rows, int K, int group, int half,
                    long long ldx, long long ldo, int mode, int act, float mult, int* status, cudaStream_t stream) {
    if (M <= 0 || M > 1024) SP_FAIL("q4_tc: built for 1 to 1,024 rows, got %d", M);
    if (rows <= 0 || K <= 0 || K % 32 || (group != 32 && group != 64 && group != 128) || K % group) SP_FAIL("q4_tc: a weight of %d x %d in groups of %d", rows, K, group);
    if ((mode == MODE_SILU_MUL) != (half > 0) || mode < 0 || mode > MODE_SILU_MUL || (half && rows != 2 * half)) SP_FAIL("q4_tc: mode %d does not go with %d gate rows", mode, half);
    if (mode == MODE_SILU_MUL && act != SP_ACT_SILU && act != SP_ACT_GELU) SP_FAIL("q4_tc: activation code %d is not built for gated rows", act);
    if (mode == MODE_ACCUMULATE && out_dt != SP_DT_F32) SP_FAIL("q4_tc: accumulation needs a float32 output");
    if (((uintptr_t)x & 15) || ldx % 8) SP_FAIL("q4_tc: rows of x must start on 16-byte boundaries");
    if (((uintptr_t)codes & 15) || ((uintptr_t)meta & 15)) SP_FAIL("q4_tc: codes and scales must start on 16-byte boundaries");
    const int tiles = q4w_tiles(rows, half), blocks = (K + Q4W_BLOCK - 1) / Q4W_BLOCK;
    const Plan p = plan_of(M, tiles, blocks, group, nullptr);
    if (!p.nt) SP_FAIL("q4_tc: no division of %d x %d x %d fits", M, rows, K);
    Args a{out, ldo, status, out_dt, M, rows, half, tiles, blocks, mode, p.nt, p.pieces, p.stages, p.slots,
           p.tmem_cols, p.d_cols, ldo % 4 == 0 && ((uintptr_t)out & 15) == 0, SpGate{act, mult}};
    Maps m;
    const cuuint64_t meta_bytes = q4w_meta_bytes(group);
    const cuuint64_t x_dims[2] = {(cuuint64_t)K, (cuuint64_t)M}, x_strides[1] = {(cuuint64_t)ldx * 2};
    const cuuint64_t c_dims[4] = {32, 8, (cuuint64_t)blocks, (cuuint64_t)tiles}, c_strides[3] = {128, 1024, (cuuint64_t)blocks * 1024};
    const cuuint64_t m_dims[3] = {meta_bytes / 4, (cuuint64_t)blocks, (cuuint64_t)tiles}, m_strides[2] = {meta_bytes, blocks * meta_bytes};
    const cuuint32_t x_box[2] = {64, (cuuint32_t)p.nt}, c_box[4] = {32, 8, 1, TILES}, m_box[3] = {(cuuint32_t)meta_bytes / 4, 1, TILES};
    if (encode(&m.x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, x_dims, x_strides, x_box, CU_TENSOR_MAP_SWIZZLE_128B)) return 1;
    if (encode(&m.codes, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, codes, c_dims, c_strides, c_box, CU_TENSOR_MAP_SWIZZLE_128B)) return 1;
    if (encode(&m.meta, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, meta, m_dims, m_strides, m_box, CU_TENSOR_MAP_SWIZZLE_NONE)) return 1;
    const int row_tiles = (tiles + TILES - 1) / TILES;
    return group == 32 ? launch<32>(m, a, p, row_tiles, stream) : group == 64 ? launch<64>(m, a, p, row_tiles, stream) : launch<128>(m, a, p, row_tiles, stream);
}
