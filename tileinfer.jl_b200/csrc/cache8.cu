// The paged cache in 8 bits: e4m3 codes (e4m3.cuh) in pages of 64 positions, a block of one scale being the page's positions of one KV head; keys and values
// have scales of their own.
//
// Writing: the last T = cu[b + 1] - cu[b] of the L = kv_lens[b] positions of every sequence get the given rows. In a page whose positions from f on are
// new, the scale becomes s' = max(s, scale(new rows)), with f = 0 that of the new rows alone, and the codes before f move: rn(c s / s'), exact unless they fall
// below 2^-6 s'. What lies behind the last new position stays as it was. So the codes do not depend on how the rows before came in, but for those below
// 2^-6 of the scale. One block of threads writes a page's head, keys or values, which keeps its new rows in registers between their maximum and their codes.
//
// Bound by launch and three dependent reads (lengths, the page, its rows and old scale); a prompt by its bytes.
#include "e4m3.cuh"

namespace {

constexpr int PAGE = 64, THREADS = 256;

struct Rows {
    const void* at;
    long long token, head;               // pitches, in elements
};

// blockIdx.x: sequence x page from the one with its first new position; blockIdx.y: head, keys or values.
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) cache_write8_kernel(unsigned char* k_codes, unsigned char* v_codes, float* k_scales, float* v_scales, Rows k, Rows v,
                                                               const int* table, int table_stride, int slots, const int* seq_slots, const int* cu,
                                                               const int* kv_lens, int n, int nkv, int D, int pages, int touched) {
    __shared__ float scratch[33];
    const int b = blockIdx.x / touched, kvh = blockIdx.y >> 1, is_v = blockIdx.y & 1;
    pdl_enter();
    const int begin = __ldcg(cu + b), T_new = __ldcg(cu + b + 1) - begin, L = __ldcg(kv_lens + b), slot = __ldcg(seq_slots + b);
    const int start = L - T_new, logical = start / PAGE + blockIdx.x % touched, base = logical * PAGE;
    // What does not fit (a length below the run's, a slot or page that does not exist) is not written.
    if (T_new <= 0 || start < 0 || base >= L || begin < 0 || begin + T_new > n || slot < 0 || slot >= slots || logical >= table_stride) return;
    const int page = __ldcg(table + (size_t)slot * table_stride + logical);
    if (page < 0 || page >= pages) return;
    const int first = max(start - base, 0), rows = min(L - base, PAGE) - first;
    const Rows src = is_v ? v : k;
    const T* from = (const T*)src.at + (long long)(begin + base + first - start) * src.token + (long long)kvh * src.head;
    const size_t block = (size_t)page * nkv + kvh;
    unsigned char* codes = (is_v ? v_codes : k_codes) + block * PAGE * D;
    float* scale = (is_v ? v_scales : k_scales) + block;
    const float before = first > 0 ? __ldcg(scale) : 0.f;
    const int per_row = D / 8;
    float x[8][8];
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int e = threadIdx.x + j * THREADS, r = e / per_row;
        if (r < rows) {
            load8<T, VEC>(x[j], from + r * src.token + (e - r * per_row) * 8);
            m = fmaxf(m, largest8(x[j]));
        }
    }
    const float after = fmaxf(power_of_two(e4m3_scale_power(block_max(m, scratch))), before), inverse = 1.f / after;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int e = threadIdx.x + j * THREADS, r = e / per_row;
        if (r < rows) *reinterpret_cast<uint2*>(codes + (size_t)first * D + (size_t)e * 8) = codes8(x[j], inverse);
    }
    if (after == before) return;
    if (first > 0) {
        const float by = before / after;
        for (int e = threadIdx.x; e < first * D / 4; e += THREADS) {
            unsigned* at = reinterpret_cast<unsigned*>(codes) + e;
            const unsigned w = __ldcg(at);
            const float2 a = e4m3_float2((unsigned short)w), c = e4m3_float2((unsigned short)(w >> 16));
            *at = e4m3_codes(a.x, a.y, c.x, c.y, by);
        }
    }
    if (threadIdx.x == 0) *scale = after;
}

}  // namespace

// k and v: [n, nkv, D] rows of `dtype` with the given pitches of tokens and heads (in elements); pools [pages, nkv, 64, D] and scales [pages, nkv]; the page of
// sequence b's positions from 64 i on is table[seq_slots[b], i] ([slots, table_stride]). max_new: the most new positions of a sequence.
extern "C" int ti_cache_write8(void* k_codes, void* v_codes, float* k_scales, float* v_scales, const void* k, long long k_token, long long k_head, const void* v,
                               long long v_token, long long v_head, const int* table, int table_stride, int slots, const int* seq_slots, const int* cu,
                               const int* kv_lens, int B, int n, int nkv, int D, int page_size, int pages, int max_new, int dtype, cudaStream_t stream) {
    if (B == 0 || n == 0 || max_new == 0) return 0;
    TI_REQUIRE(B > 0 && n > 0 && max_new > 0 && nkv > 0 && pages > 0 && slots > 0 && table_stride > 0, "cache_write8: %d sequences, %d tokens", B, n);
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
    TI_DISPATCH_DTYPE(dtype, ti_launch(vec ? cache_write8_kernel<T, true> : cache_write8_kernel<T, false>, dim3((unsigned)(touched * B), 2 * nkv), dim3(THREADS), 0,
                                       stream, (unsigned char*)k_codes, (unsigned char*)v_codes, k_scales, v_scales, kr, vr, table, table_stride, slots,
                                       seq_slots, cu, kv_lens, n, nkv, D, pages, (int)touched));
    return ti_check_launch("cache_write8");
}
