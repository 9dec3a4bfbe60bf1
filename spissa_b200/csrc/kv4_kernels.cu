// A cache of four bits (q4.cuh, groups of 32 along the head): storing into its pages and reading them back.
//
// A page of a kv head (64 positions) is one run of bytes: key codes [64][hd / 2], key scales [64][hd / 32] of 16 bits, value
// codes, value scales, so that a reader fetches it in one copy. The places of a row's bytes follow the tensor-core fragments
// that read them (kv4_attention.cu):
//   keys    row ``key_slot``; lane t (of 4) of a fragment row owns the words of columns 32 i + 8 t .. + 7 of all groups i,
//           side by side (word t · groups + i), numbers in the order of q4_pair;
//   values  row = position; lane row g (of 8) owns the columns 32 i + 4 g .. + 3 of all groups, side by side (half word
//           g · groups + i, number e in its nibble e); with heads of 128 the two halves of the row change places at every other
//           pair of rows, so that the four rows that a half warp reads together lie in different banks.
#include "kv4.cuh"

SP_API const char* sp_kv4_last_error() { return sp_error_text; }
SP_DEFINE_RANGE_API(kv4)

namespace {

struct Place {                 // where the step's tokens live
    const int* token_seq;
    const int* positions;
    const int* seq_row;
    const int* page_table;
    int max_pages;
    SpRange rg;
};

// The page of a token's position, or -1 where the debug build finds an index out of bounds.
__device__ __forceinline__ int page_of(const Place& p, int t, int pos) {
    const int row = p.seq_row[p.token_seq[t]], entry = pos / KV4_PAGE;
    if (!sp_index_ok(row, p.rg.n_rows, p.rg, 402) || !sp_index_ok(entry, p.max_pages, p.rg, 403)) return -1;
    const int page = p.page_table[(size_t)row * p.max_pages + entry];
    return sp_index_ok(page, p.rg.n_pages, p.rg, 401) ? page : -1;
}

__device__ __forceinline__ void write_quad(float* to, float4 v) { *(float4*)to = v; }
__device__ __forceinline__ void write_quad(__nv_bfloat16* to, float4 v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *(uint2*)to = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
}

constexpr int STORE_TOKENS = 4;             // of a block at most

// threads that a q head of so many units takes: 2^this
__host__ __device__ __forceinline__ int store_shift(int units) { return units <= 4 ? 2 : units <= 8 ? 3 : units <= 16 ? 4 : 5; }

// The angles are formed and their sine and cosine taken in 64 bits, keys are rotated in 64 bits and rounded to 32 once: at position
// 100,000 an angle in 32 bits is off by up to 0.004, and a key's code is a comparison that an error of the rotation may turn.
// 2,000 tokens of 32 + 2 x 8 heads of 128: 26.2 us for 68 MB with rows from memory (without rotation 23.6), 19.6 with rows that L2 holds
// (17.3); 8 tokens 3.6. Bound by latency: a block's sines, rows
// in, a group's bounds by shuffles, codes out, at four blocks an SM. Eight columns a thread, more blocks an SM, rows prefetched
// while the sines are formed: within 7 % either way.
template <typename TQ, int NG>
__global__ void __launch_bounds__(256)
store_kernel(const float* qkv, TQ* q_out, uint8_t* pool, Place place, const float* inv_freq, int T, int per_block, int nh, int nkv, int rd, int write_kv) {
    constexpr int HD = 32 * NG, PER_HEAD = HD / 4, TILE = kv4_tile_bytes(HD);
    __shared__ double2 turns[STORE_TOKENS][HD / 2];                  // cos, sin
    __shared__ __align__(16) float cos32[STORE_TOKENS][HD / 2], sin32[STORE_TOKENS][HD / 2];      // the same rounded, for q
    __shared__ int places[STORE_TOKENS][2];                          // page (or -1), place in it
    const int t0 = blockIdx.x * per_block, n_t = min(per_block, T - t0), half = rd >> 1;
    for (int i = threadIdx.x; i < n_t * half; i += blockDim.x) {
        const int k = i / half, j = i - k * half;
        double s, c;
        sincos((double)place.positions[t0 + k] * (double)inv_freq[j], &s, &c);
        turns[k][j] = make_double2(c, s);
        cos32[k][j] = (float)c;
        sin32[k][j] = (float)s;
    }
    if (threadIdx.x < n_t) {
        const int pos = place.positions[t0 + threadIdx.x];
        places[threadIdx.x][0] = write_kv ? page_of(place, t0 + threadIdx.x, pos) : -1;
        places[threadIdx.x][1] = pos % KV4_PAGE;
    }
    __syncthreads();
    // q: a thread turns four columns and their partners, or copies four that stay; a head takes 2^shift threads
    const int pairs = rd >> 3, units = pairs + ((HD - rd) >> 2), shift = store_shift(units), stride = gridDim.y * blockDim.x;
    for (int k = 0; k < n_t; ++k) {
        const float* x = qkv + (size_t)(t0 + k) * (nh + 2 * nkv) * HD;
        TQ* to = q_out + (size_t)(t0 + k) * nh * HD;
        for (int u0 = blockIdx.y * blockDim.x + threadIdx.x; u0 < nh << shift; u0 += 2 * stride) {       // two units a turn, the second's columns on their way
            float4 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int u = u0 + i * stride, un = u & ((1 << shift) - 1);
                if (u >= nh << shift || un >= units) continue;
                const float* from = x + (u >> shift) * HD + (un < pairs ? 4 * un : rd + 4 * (un - pairs));
                a[i] = *(const float4*)from;
                if (un < pairs) b[i] = *(const float4*)(from + half);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int u = u0 + i * stride, un = u & ((1 << shift) - 1);
                if (u >= nh << shift || un >= units) continue;
                TQ* at = to + (u >> shift) * HD + (un < pairs ? 4 * un : rd + 4 * (un - pairs));
                if (un < pairs) {
                    const float4 c = *(const float4*)&cos32[k][4 * un], s = *(const float4*)&sin32[k][4 * un];
                    write_quad(at, make_float4(c.x * a[i].x - s.x * b[i].x, c.y * a[i].y - s.y * b[i].y, c.z * a[i].z - s.z * b[i].z, c.w * a[i].w - s.w * b[i].w));
                    write_quad(at + half, make_float4(c.x * b[i].x + s.x * a[i].x, c.y * b[i].y + s.y * a[i].y, c.z * b[i].z + s.z * a[i].z, c.w * b[i].w + s.w * a[i].w));
                } else {
                    write_quad(at, a[i]);
                }
            }
        }
    }
    if (!write_kv) return;
    // keys and values: a thread four columns, eight neighbouring threads a group; from the other end of the token's blocks
    const int quads = 2 * nkv * PER_HEAD;
    for (int k = 0; k < n_t; ++k) {
        const int page = places[k][0], slot = places[k][1];
        const float* x = qkv + ((size_t)(t0 + k) * (nh + 2 * nkv) + nh) * HD;
        // Whole warps go through the loop together: eight lanes share a group (quads come in eights).
        for (int u0 = ((gridDim.y - 1 - blockIdx.y) * blockDim.x + threadIdx.x) & ~31; u0 < quads; u0 += 2 * stride) {
            float4 vs[2], os[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int u = u0 + i * stride + (threadIdx.x & 31), head = u / PER_HEAD, d = (u - head * PER_HEAD) * 4;
                vs[i] = os[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (u < quads) {
                    vs[i] = *(const float4*)(x + 4 * u);
                    if (head < nkv && d < rd) os[i] = *(const float4*)(x + 4 * u + (d < half ? half : -half));
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int u = u0 + i * stride + (threadIdx.x & 31);
                const bool in = u < quads;
                if (!__any_sync(0xffffffffu, in)) break;
                const int head = u / PER_HEAD, d = (u - head * PER_HEAD) * 4;
                const bool is_v = head >= nkv, first = d < half;
                float4 v = vs[i];
                if (in && !is_v && d < rd) {
                    const int at = first ? d : d - half;
                    float* a = &v.x;
                    const float* b = &os[i].x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const double2 w = turns[k][at + e];
                        a[e] = (float)((double)a[e] * w.x + (double)b[e] * (first ? -w.y : w.y));
                    }
                }
                float lo = fminf(fminf(fminf(v.x, v.y), fminf(v.z, v.w)), 0.0f), hi = fmaxf(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)), 0.0f);
                const bool bad = q4_bad(v.x) || q4_bad(v.y) || q4_bad(v.z) || q4_bad(v.w);
#pragma unroll
                for (int s = 1; s < 8; s *= 2) {
                    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, s));
                    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, s));
                }
                const Q4Scale g = q4_group(lo, hi, (__ballot_sync(0xffffffffu, bad) >> (threadIdx.x & 24) & 255u) != 0);
                const int c0 = q4_code(v.x, g), c1 = q4_code(v.y, g), c2 = q4_code(v.z, g), c3 = q4_code(v.w, g);
                const int p8 = (d >> 2) & 7, group = d >> 5;
                // a key's word holds eight columns: two threads'
                uint32_t word = ((uint32_t)c0 | (uint32_t)c1 << 16 | (uint32_t)c2 << 4 | (uint32_t)c3 << 20) << (8 * (p8 & 1));
                word |= __shfl_xor_sync(0xffffffffu, word, 1);
                if (!in || page < 0) continue;
                uint8_t* tile = pool + ((size_t)page * nkv + (is_v ? head - nkv : head)) * TILE;
                if (is_v) *(uint16_t*)(tile + kv4_v_codes(HD) + kv4_v_at(slot, p8, group, HD)) = (uint16_t)(c0 | c1 << 4 | c2 << 8 | c3 << 12);
                else if (!(p8 & 1)) *(uint32_t*)(tile + kv4_k_at(slot, p8 >> 1, group, HD)) = word;
                if (p8 == 0) *(uint16_t*)(tile + (is_v ? kv4_v_meta(HD) : kv4_k_meta(HD)) + ((is_v ? slot : kv4_key_slot(slot)) * NG + group) * 2) = (uint16_t)q4_meta(g);
            }
        }
    }
}

template <typename TQ>
void launch_store(int hd, dim3 grid, cudaStream_t stream, const float* qkv, TQ* q_out, uint8_t* pool, const Place& place, const float* inv_freq, int T,
                  int per_block, int nh, int nkv, int rd, int write_kv) {
    switch (hd) {
        case 32: store_kernel<TQ, 1><<<grid, 256, 0, stream>>>(qkv, q_out, pool, place, inv_freq, T, per_block, nh, nkv, rd, write_kv); break;
        case 64: store_kernel<TQ, 2><<<grid, 256, 0, stream>>>(qkv, q_out, pool, place, inv_freq, T, per_block, nh, nkv, rd, write_kv); break;
        case 96: store_kernel<TQ, 3><<<grid, 256, 0, stream>>>(qkv, q_out, pool, place, inv_freq, T, per_block, nh, nkv, rd, write_kv); break;
        default: store_kernel<TQ, 4><<<grid, 256, 0, stream>>>(qkv, q_out, pool, place, inv_freq, T, per_block, nh, nkv, rd, write_kv); break;
    }
}

// Four neighbouring columns of a position's key or value.
__device__ __forceinline__ float4 read_quad(const uint8_t* tile, int slot, int d, int hd, bool is_v) {
    const int p8 = (d >> 2) & 7, group = d >> 5, groups = hd >> 5;
    if (is_v) {
        const uint32_t w = *(const uint16_t*)(tile + kv4_v_codes(hd) + kv4_v_at(slot, p8, group, hd));
        const uint32_t m = *(const uint16_t*)(tile + kv4_v_meta(hd) + (slot * groups + group) * 2);
        return make_float4(q4_value(w & 15, m), q4_value((w >> 4) & 15, m), q4_value((w >> 8) & 15, m), q4_value(w >> 12, m));
    }
    const uint32_t w = *(const uint32_t*)(tile + kv4_k_at(slot, p8 >> 1, group, hd)) >> (8 * (p8 & 1));
    const uint32_t m = *(const uint16_t*)(tile + kv4_k_meta(hd) + (kv4_key_slot(slot) * groups + group) * 2);
    return make_float4(q4_value(w & 15, m), q4_value((w >> 16) & 15, m), q4_value((w >> 4) & 15, m), q4_value((w >> 20) & 15, m));
}

// 2,000 tokens of 8 kv heads of 128: 8.7 us, two and four bytes a read.
template <typename T>
__global__ void __launch_bounds__(256)
load_kernel(const uint8_t* pool, T* k_out, T* v_out, Place place, int nkv, int hd) {
    const int t = blockIdx.x, pos = place.positions[t], page = page_of(place, t, pos), per_head = hd >> 2;
    if (page < 0) return;
    for (int u = blockIdx.y * blockDim.x + threadIdx.x; u < 2 * nkv * per_head; u += gridDim.y * blockDim.x) {
        const int row = u / per_head, d = (u - row * per_head) * 4, head = row < nkv ? row : row - nkv;
        const uint8_t* tile = pool + ((size_t)page * nkv + head) * kv4_tile_bytes(hd);
        write_quad((row < nkv ? k_out : v_out) + ((size_t)t * nkv + head) * hd + d, read_quad(tile, pos % KV4_PAGE, d, hd, row >= nkv));
    }
}

// Pages of the step's sequences, one block each and kv head, one after another into pools of their own; ``table`` [seqs][max_pages]
// says where each went. Positions behind a sequence's end become zeros: a page's rest holds what the memory held. Pages that lie
// wholly before every query's window are left out.
template <typename T>
__global__ void __launch_bounds__(256)
unpack_pages_kernel(const uint8_t* pool, T* k_out, T* v_out, int* table, const int* seq_len, const int* seq_start, const int* positions, int window,
                    const int* seq_row, const int* page_table, int max_pages, int n_out, int nkv, int hd, SpRange rg) {
    __shared__ int before;
    const int entry = blockIdx.x, head = blockIdx.y, b = blockIdx.z, len = seq_len[b];
    if (entry * KV4_PAGE >= len) {
        if (head == 0 && threadIdx.x == 0) table[(size_t)b * max_pages + entry] = 0;
        return;
    }
    if (threadIdx.x == 0) before = 0;
    __syncthreads();
    int mine = 0;
    for (int i = threadIdx.x; i < b; i += blockDim.x) mine += (seq_len[i] + KV4_PAGE - 1) / KV4_PAGE;
    if (mine) atomicAdd(&before, mine);
    __syncthreads();
    const int out = before + entry, row = sp_checked_row(seq_row[b], rg);
    if (head == 0 && threadIdx.x == 0) table[(size_t)b * max_pages + entry] = out < n_out ? out : 0;
    if (out >= n_out || seq_start[b + 1] == seq_start[b]) return;    // (the host counted fewer pages than the lengths say; no queries)
    if (window && (entry + 1) * KV4_PAGE <= positions[seq_start[b]] + 1 - window) return;      // the first query's
    const int page = sp_checked_page(page_table[(size_t)row * max_pages + entry], rg);
    const uint8_t* tile = pool + ((size_t)page * nkv + head) * kv4_tile_bytes(hd);
    const int per_head = hd >> 2;
    for (int u = threadIdx.x; u < 2 * KV4_PAGE * per_head; u += blockDim.x) {
        const int r = u / per_head, d = (u - r * per_head) * 4, slot = r % KV4_PAGE;
        const bool is_v = r >= KV4_PAGE;
        const float4 v = entry * KV4_PAGE + slot < len ? read_quad(tile, slot, d, hd, is_v) : make_float4(0.f, 0.f, 0.f, 0.f);
        write_quad((is_v ? v_out : k_out) + (((size_t)out * nkv + head) * KV4_PAGE + slot) * hd + d, v);
    }
}

int check_heads(const char* what, int nkv, int hd, int page_size) {
    if (hd <= 0 || hd % 32 || hd > KV4_MAX_HD) SP_FAIL("%s: head sizes 32, 64, 96 and 128, got %d", what, hd);
    if (nkv <= 0) SP_FAIL("%s: %d kv heads", what, nkv);
    if (page_size != KV4_PAGE) SP_FAIL("%s: pages of %d positions, got %d", what, KV4_PAGE, page_size);
    return 0;
}

}  // namespace

SP_API int sp_kv4_tile_bytes(int hd) { return hd > 0 && hd % 32 == 0 && hd <= KV4_MAX_HD ? kv4_tile_bytes(hd) : 0; }

SP_API int sp_kv4_store(const void* qkv, void* q_out, int q_dt, void* pool, const int* token_seq, const int* positions, const int* seq_row,
                        const int* page_table, int max_pages, int page_size, const float* inv_freq, int T, int nh, int nkv, int hd,
                        int rd, int write_kv, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (check_heads("kv4_store", nkv, hd, page_size)) return 1;
    if (nh < 0 || (nh && !q_out)) SP_FAIL("kv4_store: %d query heads need a place to go", nh);
    if (rd < 0 || rd > hd || rd % 8) SP_FAIL("kv4_store: rotated sizes are multiples of 8 up to the head size, got %d of %d", rd, hd);
    if (rd && !inv_freq) SP_FAIL("kv4_store: rotation needs the frequencies");
    if (write_kv && (!pool || !page_table || max_pages <= 0)) SP_FAIL("kv4_store: writing needs the pages and their table");
    if (((uintptr_t)qkv & 15) || ((uintptr_t)q_out & 15) || ((uintptr_t)pool & 15)) SP_FAIL("kv4_store: rows, q and pages must start on 16-byte boundaries");
    const Place place{token_seq, positions, seq_row, page_table, max_pages, sp_range_host};
    const int units = (nh << store_shift(rd / 8 + (hd - rd) / 4)) + (write_kv ? 2 * nkv * (hd / 4) : 0), sms = sp_sm_count() > 0 ? sp_sm_count() : 148;
    // a few tokens: a token's heads over several blocks; many: several tokens to a block, whose angles are formed side by side
    int per_block = T / (16 * sms), parts = (units + 255) / 256;
    per_block = per_block < 1 ? 1 : per_block > STORE_TOKENS ? STORE_TOKENS : per_block;
    const int blocks = (T + per_block - 1) / per_block;
    if (blocks * parts > 6 * sms) parts = blocks >= 6 * sms ? 1 : (6 * sms + blocks - 1) / blocks;
    const dim3 grid(blocks, parts < 1 ? 1 : parts);
    if (q_dt == SP_DT_F32) launch_store(hd, grid, stream, (const float*)qkv, (float*)q_out, (uint8_t*)pool, place, inv_freq, T, per_block, nh, nkv, rd, write_kv);
    else launch_store(hd, grid, stream, (const float*)qkv, (__nv_bfloat16*)q_out, (uint8_t*)pool, place, inv_freq, T, per_block, nh, nkv, rd, write_kv);
    SP_CHECK_LAUNCH("kv4_store");
    return 0;
}

SP_API int sp_kv4_load(const void* pool, void* k_out, void* v_out, int dt, const int* token_seq, const int* positions, const int* seq_row,
                       const int* page_table, int max_pages, int page_size, int T, int nkv, int hd, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (check_heads("kv4_load", nkv, hd, page_size)) return 1;
    if (((uintptr_t)k_out & 15) || ((uintptr_t)v_out & 15) || ((uintptr_t)pool & 15)) SP_FAIL("kv4_load: pages and rows must start on 16-byte boundaries");
    const Place place{token_seq, positions, seq_row, page_table, max_pages, sp_range_host};
    const int parts = (2 * nkv * (hd / 4) + 255) / 256;
    const dim3 grid(T, parts);
    if (dt == SP_DT_F32) load_kernel<<<grid, 256, 0, stream>>>((const uint8_t*)pool, (float*)k_out, (float*)v_out, place, nkv, hd);
    else load_kernel<<<grid, 256, 0, stream>>>((const uint8_t*)pool, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, place, nkv, hd);
    SP_CHECK_LAUNCH("kv4_load");
    return 0;
}

// k_out, v_out [n_out][nkv][64][hd]; ``table`` [n_seqs][max_pages] gets the pages' numbers there.
SP_API int sp_kv4_unpack_pages(const void* pool, void* k_out, void* v_out, int dt, int* table, const int* seq_len, const int* seq_start,
                               const int* positions, int window, const int* seq_row, const int* page_table, int max_pages, int page_size, int n_seqs, int n_out, int nkv,
                               int hd, cudaStream_t stream) {
    if (n_seqs <= 0 || n_out <= 0) return 0;
    if (check_heads("kv4_unpack_pages", nkv, hd, page_size)) return 1;
    if (nkv > 65535 || n_seqs > 65535) SP_FAIL("kv4_unpack_pages: %d kv heads, %d sequences", nkv, n_seqs);
    if (((uintptr_t)k_out & 15) || ((uintptr_t)v_out & 15) || ((uintptr_t)pool & 15)) SP_FAIL("kv4_unpack_pages: pools must start on 16-byte boundaries");
    const dim3 grid(max_pages, nkv, n_seqs);
    if (dt == SP_DT_F32)
        unpack_pages_kernel<<<grid, 256, 0, stream>>>((const uint8_t*)pool, (float*)k_out, (float*)v_out, table, seq_len, seq_start, positions, window, seq_row, page_table, max_pages, n_out, nkv, hd, sp_range_host);
    else
        unpack_pages_kernel<<<grid, 256, 0, stream>>>((const uint8_t*)pool, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, table, seq_len, seq_start, positions, window, seq_row, page_table, max_pages, n_out, nkv, hd, sp_range_host);
    SP_CHECK_LAUNCH("kv4_unpack_pages");
    return 0;
}
