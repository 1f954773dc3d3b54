// The paged cache in 8 bits: e4m3 codes (e4m3.cuh) in pages of 64 positions, a block of one scale being the page's positions of one KV head; keys and values
// have scales of their own.
//
// Writing: the last T = cu[b + 1] - cu[b] of the L = kv_lens[b] positions of every sequence get the given rows. In a page whose positions from f on are
// new, the scale becomes s' = max(s, scale(new rows)), with f = 0 that of the new rows alone, and the codes before f move: rn(c s / s'), exact unless they fall
// below 2^-6 s'. What lies behind the last new position stays as it was. So the codes do not depend on how the rows before came in, but for those below
// 2^-6 of the scale. One block of threads writes a page's head, keys or values, which keeps its new rows in registers between their maximum and their codes.
//
// Attention over the cache (attention8.cu) asks for pages before it waits for the kernel ahead, but for those that hold one of its own new tokens. With at most one
// new row a sequence these are all that is written here, so it may come up beside this kernel; with more, the tokens that attend may be fewer than those that are
// written, so nothing starts until all stores have reached all (eight runs of up to 1,024 rows 10.2 -> 10.7 us, five rows of 64 sequences 5.4 -> 5.7; five rows of eight with their attention 35.4 -> 37.0).
//
// Bound by launch and three dependent reads (lengths, the page, its rows and old scale), so that blocks are small enough to come up at once where they are many:
// one token of 64 sequences takes 3.6 us, eight runs of up to 1,024 rows 10.7 (8 heads of 128; 7.3 MB, 1.1 us at the rate of a copy).
//
// Widening, for kernels that read bfloat16: the pages that a step's tokens see become pages of bfloat16 in a pool of their own, page j of sequence b at
// b x (pages a sequence) + j, with its block table. A code times a power of two is exact in bfloat16. Positions that nobody sees become zeros.
#include "e4m3.cuh"

namespace {

constexpr int PAGE = 64, THREADS = 256;

struct Rows {
    const void* at;
    long long token, head;               // pitches, in elements
};

// blockIdx.x: sequence x page from the one with its first new position; blockIdx.y: head, keys or values. NT threads, J eights of new rows each.
template <typename T, bool VEC, int NT, int J>
__global__ void __launch_bounds__(NT) cache_write8_kernel(unsigned char* k_codes, unsigned char* v_codes, float* k_scales, float* v_scales, Rows k, Rows v,
                                                               const int* table, int table_stride, int slots, int columns, const int* seq_slots, const int* cu,
                                                               const int* kv_lens, int n, int nkv, int D, int pages, int touched, bool beside) {
    __shared__ float scratch[33];
    const int b = blockIdx.x / touched, kvh = blockIdx.y >> 1, is_v = blockIdx.y & 1;
    pdl_wait();
    if (beside) pdl_launch_dependents();
    const int begin = __ldcg(cu + b), T_new = __ldcg(cu + b + 1) - begin, L = __ldcg(kv_lens + b), slot = __ldcg(seq_slots + b);
    const int start = L - T_new, logical = start / PAGE + blockIdx.x % touched, base = logical * PAGE;
    // What does not fit (a length below the run's, a slot or page that does not exist) is not written.
    if (T_new <= 0 || start < 0 || base >= L || begin < 0 || begin + T_new > n || slot < 0 || slot >= slots || logical >= columns) return;
    const int page = __ldcg(table + (size_t)slot * table_stride + logical);
    if (page < 0 || page >= pages) return;
    const int first = max(start - base, 0), rows = min(L - base, PAGE) - first;
    const Rows src = is_v ? v : k;
    const T* from = (const T*)src.at + (long long)(begin + base + first - start) * src.token + (long long)kvh * src.head;
    const size_t block = (size_t)page * nkv + kvh;
    unsigned char* codes = (is_v ? v_codes : k_codes) + block * PAGE * D;
    float* scale = (is_v ? v_scales : k_scales) + block;
    const float before = first > 0 ? __ldcg(scale) : 0.f;
    const int per_row = D / 8, more_rows = NT / per_row, more_pieces = NT % per_row;
    Eight<T> x[J];
    int r = threadIdx.x / per_row, piece = threadIdx.x % per_row;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        x[j].clear();
        if (r < rows) x[j].template load<VEC>(from + r * src.token + piece * 8);
        r += more_rows;
        piece += more_pieces;
        if (piece >= per_row) { piece -= per_row; ++r; }
    }
    bool finite;
    const float m = largest(x, finite);
    const float after = fmaxf(power_of_two(e4m3_scale_power(block_max(m, scratch))), before), inverse = 1.f / after;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int e = threadIdx.x + j * NT;
        if (e < rows * per_row) *reinterpret_cast<uint2*>(codes + (size_t)first * D + (size_t)e * 8) = codes_of(x[j], inverse, finite);
    }
    if (after != before && first > 0) {
        const float by = before / after;
        const auto moved = [by](unsigned w) {
            const float2 a = e4m3_float2((unsigned short)w), c = e4m3_float2((unsigned short)(w >> 16));
            return e4m3_codes(a.x, a.y, c.x, c.y, by);
        };
        uint4* old = reinterpret_cast<uint4*>(codes);
        constexpr int W = 4;
        for (int e0 = threadIdx.x; e0 < first * D / 16; e0 += W * NT) {
            uint4 w[W];
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (e0 + j * NT < first * D / 16) w[j] = __ldcg(old + e0 + j * NT);
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (e0 + j * NT < first * D / 16) old[e0 + j * NT] = make_uint4(moved(w[j].x), moved(w[j].y), moved(w[j].z), moved(w[j].w));
        }
    }
    if (threadIdx.x == 0 && after != before) *scale = after;
    if (!beside) __threadfence();
}

// blockIdx: page, head, sequence.
__global__ void __launch_bounds__(THREADS) cache_widen8_kernel(bf16* k_out, bf16* v_out, int* table_out, int* slots_out, int* lens_out, int* cu_out, const unsigned char* k, const unsigned char* v,
                                                               const float* k_scales, const float* v_scales, const int* table, int table_stride, int slots,
                                                               int columns, const int* seq_slots, const int* cu, const int* kv_lens, int n, int nkv, int D, int pages,
                                                               int per_seq, int window) {
    const int j = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    pdl_enter();
    // Readers stay within the table and the n rows of queries, whatever they were given.
    const int begin = min(max(__ldcg(cu + b), 0), n), end = min(max(__ldcg(cu + b + 1), 0), n), T_new = end - begin;
    const int L = min(max(__ldcg(kv_lens + b), 0), per_seq * PAGE), slot = __ldcg(seq_slots + b);
    if (kvh == 0 && threadIdx.x == 0) {
        table_out[(size_t)b * per_seq + j] = b * per_seq + j;
        if (j == 0) {
            slots_out[b] = b;
            lens_out[b] = L;
            cu_out[b] = begin;
            if (b == gridDim.z - 1) cu_out[b + 1] = end;
        }
    }
    const int first = window > 0 ? max(0, L - T_new - window + 1) : 0;
    if (T_new <= 0 || j * PAGE >= L || j < first / PAGE / 2 * 2) return;              // the readers walk the pages in pairs
    const int page = slot >= 0 && slot < slots && j < columns && (j + 1) * PAGE > first ? __ldcg(table + (size_t)slot * table_stride + j) : -1;
    const bool there = page >= 0 && page < pages;
    const size_t from = ((size_t)page * nkv + kvh) * PAGE * D, to = (((size_t)b * per_seq + j) * nkv + kvh) * PAGE * D;
    const float sk = there ? __ldcg(k_scales + (size_t)page * nkv + kvh) : 0.f, sv = there ? __ldcg(v_scales + (size_t)page * nkv + kvh) : 0.f;
    const int pieces = PAGE * D / 16;
    for (int e = threadIdx.x; e < 2 * pieces; e += THREADS) {
        const bool is_v = e >= pieces;
        const int piece = is_v ? e - pieces : e, key = j * PAGE + piece * 16 / D;
        const float s = is_v ? sv : sk;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (there && key >= first && key < L) w = __ldcg(reinterpret_cast<const uint4*>((is_v ? v : k) + from) + piece);
        const unsigned c[4] = {w.x, w.y, w.z, w.w};
        unsigned o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 lo = e4m3_float2((unsigned short)c[i]), hi = e4m3_float2((unsigned short)(c[i] >> 16));
            const __nv_bfloat162 x = __floats2bfloat162_rn(lo.x * s, lo.y * s), y = __floats2bfloat162_rn(hi.x * s, hi.y * s);
            o[2 * i] = *reinterpret_cast<const unsigned*>(&x);
            o[2 * i + 1] = *reinterpret_cast<const unsigned*>(&y);
        }
        uint4* dst = reinterpret_cast<uint4*>((is_v ? v_out : k_out) + to) + 2 * piece;
        dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
        dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
}

}  // namespace

// k and v: [n, nkv, D] rows of `dtype` with the given pitches of tokens and heads (in elements); pools [pages, nkv, 64, D] and scales [pages, nkv]; the page of
// sequence b's positions from 64 i on is table[seq_slots[b], i] ([slots, columns], rows table_stride apart). max_new: the most new positions of a sequence.
extern "C" int ti_cache_write8_table(void* k_codes, void* v_codes, float* k_scales, float* v_scales, const void* k, long long k_token, long long k_head, const void* v,
                                     long long v_token, long long v_head, const int* table, int table_stride, int slots, const int* seq_slots, const int* cu,
                                     const int* kv_lens, int B, int n, int nkv, int D, int page_size, int pages, int max_new, int dtype, int columns, cudaStream_t stream) {
    if (B == 0 || n == 0 || max_new == 0) return 0;
    TI_REQUIRE(B > 0 && n > 0 && max_new > 0 && nkv > 0 && pages > 0 && slots > 0 && columns > 0 && table_stride >= 0, "cache_write8: %d sequences, %d tokens", B, n);
    if (page_size != PAGE || D <= 0 || D > 256 || D % 16 != 0 || nkv > 32767) {
        ti_fail("cache_write8 takes pages of %d and heads of a multiple of 16 up to 256; got pages of %d, %d heads of %d", PAGE, page_size, nkv, D);
        return 2;
    }
    TI_REQUIRE(aligned16(k_codes) && aligned16(v_codes), "cache_write8: pages must be 16-byte aligned");
    const long long touched = ((long long)max_new + PAGE - 2) / PAGE + 1;
    TI_REQUIRE(touched * B < 1LL << 31, "cache_write8: %d sequences of up to %d new positions are too many", B, max_new);
    const int size = dtype == TI_F32 ? 4 : 2;
    TI_REQUIRE((uintptr_t)k % size == 0 && (uintptr_t)v % size == 0, "cache_write8: a misaligned address");
    const bool vec = aligned16(k) && aligned16(v) && (k_token * size | k_head * size | v_token * size | v_head * size) % 16 == 0;
    const Rows kr = {k, k_token, k_head}, vr = {v, v_token, v_head};
    // Where all new rows of a page are few, two warps: all pages then come up at once (one token of 64 sequences, 8 heads of 128: 3.8 us,
    // with eight warps 8.8).
    const bool few = (long long)max_new * D <= 64 * 2 * 8;
    TI_DISPATCH_DTYPE(dtype, auto* kernel = few ? (vec ? cache_write8_kernel<T, true, 64, 2> : cache_write8_kernel<T, false, 64, 2>) :
                                            D <= 128 ? (vec ? cache_write8_kernel<T, true, THREADS, 4> : cache_write8_kernel<T, false, THREADS, 4>) :
                                                       (vec ? cache_write8_kernel<T, true, THREADS, 8> : cache_write8_kernel<T, false, THREADS, 8>);
                      ti_launch(kernel, dim3((unsigned)(touched * B), 2 * nkv), dim3(few ? 64 : THREADS), 0, stream, (unsigned char*)k_codes, (unsigned char*)v_codes,
                                k_scales, v_scales, kr, vr, table, table_stride, slots, columns, seq_slots, cu, kv_lens, n, nkv, D, pages, (int)touched, max_new == 1));
    return ti_check_launch("cache_write8");
}

// The same where a row of the table has as many columns as its pitch.
extern "C" int ti_cache_write8(void* k_codes, void* v_codes, float* k_scales, float* v_scales, const void* k, long long k_token, long long k_head, const void* v,
                               long long v_token, long long v_head, const int* table, int table_stride, int slots, const int* seq_slots, const int* cu,
                               const int* kv_lens, int B, int n, int nkv, int D, int page_size, int pages, int max_new, int dtype, cudaStream_t stream) {
    return ti_cache_write8_table(k_codes, v_codes, k_scales, v_scales, k, k_token, k_head, v, v_token, v_head, table, table_stride, slots, seq_slots, cu, kv_lens, B, n, nkv, D,
                                 page_size, pages, max_new, dtype, table_stride, stream);
}

// For attention8.cu: pools k_out, v_out [B * per_seq, nkv, 64, D] bfloat16, table_out [B, per_seq], slots_out [B], lens_out [B], cu_out [B + 1].
int cache_widen8(void* k_out, void* v_out, int* table_out, int* slots_out, int* lens_out, int* cu_out, const void* k, const void* v, const float* k_scales, const float* v_scales,
                 const int* table, int table_stride, int slots, int columns, const int* seq_slots, const int* cu, const int* kv_lens, int B, int n, int nkv, int D, int pages, int per_seq,
                 int window, cudaStream_t stream) {
    ti_launch(cache_widen8_kernel, dim3(per_seq, nkv, B), dim3(THREADS), 0, stream, (bf16*)k_out, (bf16*)v_out, table_out, slots_out, lens_out, cu_out, (const unsigned char*)k,
              (const unsigned char*)v, k_scales, v_scales, table, table_stride, slots, columns, seq_slots, cu, kv_lens, n, nkv, D, pages, per_seq, window);
    return ti_check_launch("cache_widen8");
}
