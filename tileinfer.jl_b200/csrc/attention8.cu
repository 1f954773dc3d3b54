// Attention over the paged cache in 8 bits (cache8.cu), bfloat16 queries and results: one warp a token's head, one key after another.
//
//   out[i, h] = sum_j softmax_j(scale q[i, h] . sk[page of j] ck[j]) sv[page of j] cv[j], over the visible j.
#include "e4m3.cuh"

namespace {

constexpr int PAGE = 64;

__global__ void __launch_bounds__(32) attention8_kernel(bf16* out, const bf16* q, const unsigned char* k, const unsigned char* v, const float* k_scales,
                                                        const float* v_scales, const int* table, int table_stride, const int* seq_slots, const int* cu,
                                                        const int* kv_lens, float scale_log2e, int nq, int nkv, int D, int window) {
    const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x, kvh = h / (nq / nkv);
    pdl_enter();
    const int begin = __ldcg(cu + b), T = __ldcg(cu + b + 1) - begin, L = __ldcg(kv_lens + b);
    if ((int)blockIdx.x >= T) return;
    const int i = blockIdx.x, last = L - T + i, first = window > 0 ? max(0, last - window + 1) : 0;
    const bf16* qr = q + ((size_t)(begin + i) * nq + h) * D;
    float qv[8], o[8] = {}, m = -INFINITY, l = 0.f;
    for (int c = 0; c < 8; ++c) qv[c] = lane + 32 * c < D ? to_f32(__ldcg(qr + lane + 32 * c)) : 0.f;
    for (int j = first; j <= last; ++j) {
        const size_t block = (size_t)__ldcg(table + (size_t)seq_slots[b] * table_stride + j / PAGE) * nkv + kvh;
        const unsigned char *kr = k + (block * PAGE + j % PAGE) * D, *vr = v + (block * PAGE + j % PAGE) * D;
        float s = 0.f;
        for (int c = 0; c < 8; ++c)
            if (lane + 32 * c < D) s += qv[c] * e4m3_float2(kr[lane + 32 * c]).x;
        s = warp_sum(s) * scale_log2e * k_scales[block];
        const float top = fmaxf(m, s), old = exp2f(m - top), p = exp2f(s - top);
        m = top;
        l = l * old + p;
        for (int c = 0; c < 8; ++c)
            if (lane + 32 * c < D) o[c] = o[c] * old + p * v_scales[block] * e4m3_float2(vr[lane + 32 * c]).x;
    }
    for (int c = 0; c < 8; ++c)
        if (lane + 32 * c < D) out[((size_t)(begin + i) * nq + h) * D + lane + 32 * c] = __float2bfloat16_rn(l == 0.f ? 0.f : o[c] / l);
}

}  // namespace

extern "C" long long ti_attention8_workspace(int B, int max_new, int nq, int nkv, int D, int max_len) { return 0; }

extern "C" int ti_attention8(void* out, const void* q, const void* k, const void* v, const float* k_scales, const float* v_scales, const int* table,
                             int table_stride, const int* seq_slots, const int* cu, const int* kv_lens, void* ws, long long ws_bytes, int* status, float scale,
                             int B, int n, int nq, int nkv, int D, int page_size, int max_new, int max_len, int pages, int window, cudaStream_t stream) {
    if (B == 0 || n == 0 || max_new == 0) return 0;
    TI_REQUIRE(scale > 0.f, "attention8: scale must be positive");
    if (page_size != PAGE || D > 256 || D % 16 != 0 || nq % nkv != 0 || B > 65535 || nq > 65535) {
        ti_fail("attention8 takes pages of %d and heads of a multiple of 16 up to 256; got pages of %d, %d / %d heads of %d", PAGE, page_size, nq, nkv, D);
        return 2;
    }
    ti_launch(attention8_kernel, dim3(max_new, nq, B), dim3(32), 0, stream, (bf16*)out, (const bf16*)q, (const unsigned char*)k, (const unsigned char*)v, k_scales,
              v_scales, table, table_stride, seq_slots, cu, kv_lens, scale * 1.4426950408889634f, nq, nkv, D, window);
    return ti_check_launch("attention8");
}
