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

// A thread owns four neighbouring columns of a head; eight neighbouring threads a group. The angles are formed and their sine
// and cosine taken in 64 bits, keys are rotated in 64 bits and rounded to 32 once: at position 100,000 an angle in 32 bits is
// off by up to 0.004, and a key's code is a comparison that an error of the rotation may turn.
template <typename TQ>
__global__ void __launch_bounds__(256)
store_kernel(const float* qkv, TQ* q_out, uint8_t* pool, Place place, const float* inv_freq, int nh, int nkv, int hd, int rd, int write_kv) {
    __shared__ double2 turn[KV4_MAX_HD / 2];
    const int t = blockIdx.x, pos = place.positions[t], half = rd >> 1;
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
        double s, c;
        sincos((double)pos * (double)inv_freq[i], &s, &c);
        turn[i] = make_double2(c, s);
    }
    __syncthreads();
    const int page = write_kv ? page_of(place, t, pos) : -1;
    const int per_head = hd >> 2, quads = (nh + (write_kv ? 2 * nkv : 0)) * per_head, groups = hd >> 5;
    const float* x = qkv + (size_t)t * (nh + 2 * nkv) * hd;
    // whole warps go through the loop together: eight lanes share a group (quads come in eights)
    for (int u0 = (blockIdx.y * blockDim.x + threadIdx.x) & ~31; u0 < quads; u0 += gridDim.y * blockDim.x) {
        const int u = u0 + (threadIdx.x & 31);
        const bool in = u < quads;
        const int head = in ? u / per_head : 0, d = in ? (u - head * per_head) * 4 : 0;
        const bool is_q = head < nh, is_v = head >= nh + nkv, rotates = in && !is_v && d < rd;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f), o = v;
        if (in) v = *(const float4*)(x + (size_t)head * hd + d);
        if (rotates) {
            const bool first = d < half;
            o = *(const float4*)(x + (size_t)head * hd + (first ? d + half : d - half));
            const double2* tr = turn + (first ? d : d - half);
            float* a = &v.x;
            const float* b = &o.x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double c = tr[e].x, s = first ? -tr[e].y : tr[e].y;
                a[e] = is_q ? (float)c * a[e] + (float)s * b[e] : (float)((double)a[e] * c + (double)b[e] * s);
            }
        }
        if (in && is_q) {
            TQ* to = q_out + ((size_t)t * nh + head) * hd + d;
            sp_st2(to, 0, v.x, v.y);
            sp_st2(to, 2, v.z, v.w);
        }
        if (!__any_sync(0xffffffffu, in && !is_q)) continue;
        float lo = fminf(fminf(fminf(v.x, v.y), fminf(v.z, v.w)), 0.0f), hi = fmaxf(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)), 0.0f);
        int bad = q4_bad(v.x) || q4_bad(v.y) || q4_bad(v.z) || q4_bad(v.w);
#pragma unroll
        for (int s = 1; s < 8; s *= 2) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, s));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, s));
            bad |= __shfl_xor_sync(0xffffffffu, bad, s);
        }
        const Q4Scale g = q4_group(lo, hi, bad != 0);
        const int c0 = q4_code(v.x, g), c1 = q4_code(v.y, g), c2 = q4_code(v.z, g), c3 = q4_code(v.w, g);
        const int p8 = (d >> 2) & 7, group = d >> 5, slot = pos % KV4_PAGE;
        // a key's word holds eight columns: two threads'
        uint32_t word = ((uint32_t)c0 | (uint32_t)c1 << 16 | (uint32_t)c2 << 4 | (uint32_t)c3 << 20) << (8 * (p8 & 1));
        word |= __shfl_xor_sync(0xffffffffu, word, 1);
        if (!in || is_q || page < 0) continue;
        uint8_t* tile = pool + ((size_t)page * nkv + (is_v ? head - nh - nkv : head - nh)) * kv4_tile_bytes(hd);
        if (is_v) {
            *(uint16_t*)(tile + kv4_v_codes(hd) + kv4_v_at(slot, p8, group, hd)) = (uint16_t)(c0 | c1 << 4 | c2 << 8 | c3 << 12);
        } else if (!(p8 & 1)) {
            *(uint32_t*)(tile + kv4_k_at(slot, p8 >> 1, group, hd)) = word;
        }
        if (p8 == 0) *(uint16_t*)(tile + (is_v ? kv4_v_meta(hd) : kv4_k_meta(hd)) + ((is_v ? slot : kv4_key_slot(slot)) * groups + group) * 2) = (uint16_t)q4_meta(g);
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

template <typename T>
__device__ __forceinline__ void write_quad(T* to, float4 v) {
    sp_st2(to, 0, v.x, v.y);
    sp_st2(to, 2, v.z, v.w);
}

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
    if (out >= n_out) return;                                        // (the host counted fewer pages than the lengths say)
    if (head == 0 && threadIdx.x == 0) table[(size_t)b * max_pages + entry] = out;
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
    if (((uintptr_t)qkv & 15) || ((uintptr_t)q_out & 7) || ((uintptr_t)pool & 15)) SP_FAIL("kv4_store: rows and pages must start on 16-byte boundaries, q on 8");
    const Place place{token_seq, positions, seq_row, page_table, max_pages, sp_range_host};
    const int quads = (nh + 2 * nkv) * (hd / 4), sms = sp_sm_count() > 0 ? sp_sm_count() : 148;
    int parts = (quads + 255) / 256;                                // a few tokens: a token's heads over several blocks
    if (T * parts > 4 * sms) parts = T >= 4 * sms ? 1 : (4 * sms + T - 1) / T;
    const dim3 grid(T, parts);
    if (q_dt == SP_DT_F32) store_kernel<<<grid, 256, 0, stream>>>((const float*)qkv, (float*)q_out, (uint8_t*)pool, place, inv_freq, nh, nkv, hd, rd, write_kv);
    else store_kernel<<<grid, 256, 0, stream>>>((const float*)qkv, (__nv_bfloat16*)q_out, (uint8_t*)pool, place, inv_freq, nh, nkv, hd, rd, write_kv);
    SP_CHECK_LAUNCH("kv4_store");
    return 0;
}

SP_API int sp_kv4_load(const void* pool, void* k_out, void* v_out, int dt, const int* token_seq, const int* positions, const int* seq_row,
                       const int* page_table, int max_pages, int page_size, int T, int nkv, int hd, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (check_heads("kv4_load", nkv, hd, page_size)) return 1;
    if (((uintptr_t)k_out & 7) || ((uintptr_t)v_out & 7) || ((uintptr_t)pool & 15)) SP_FAIL("kv4_load: pages must start on 16-byte boundaries, rows on 8");
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
