// Products of e4m3 codes with a scale for every 128 of k (e4m3.cuh): one warp a result.
//
//   y[t, o] = sum_g sx[g, t] sw[g, o / 128] sum_{k in g} cx[t, k] cw[o, k]
#include "e4m3.cuh"
#include "linear4.cuh"

namespace {

__global__ void __launch_bounds__(256) linear8_kernel(void* y, long long ldy, const unsigned char* x, long long ldx, const float* x_scales, const unsigned char* w,
                                                      const float* scales, int n, int out, int K, int epilogue, XieluParams act) {
    const int t = blockIdx.y, o = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    pdl_enter();
    if (o >= out) return;
    float sum = 0.f;
    for (int g = 0; g * E4M3_BLOCK < K; ++g) {
        float part = 0.f;
        const int k = g * E4M3_BLOCK + lane * 4;
        if (k < K) {
            const unsigned a = __ldcg(reinterpret_cast<const unsigned*>(x + (long long)t * ldx + k)), b = __ldcg(reinterpret_cast<const unsigned*>(w + (long long)o * K + k));
            const float2 a0 = e4m3_float2((unsigned short)a), a1 = e4m3_float2((unsigned short)(a >> 16));
            const float2 b0 = e4m3_float2((unsigned short)b), b1 = e4m3_float2((unsigned short)(b >> 16));
            part = a0.x * b0.x + a0.y * b0.y + a1.x * b1.x + a1.y * b1.y;
        }
        sum += warp_sum(part) * __ldcg(x_scales + (long long)g * n + t) * __ldcg(scales + (long long)g * ((out + 127) / 128) + o / 128);
    }
    if (lane == 0) store_result(y, ldy, t, o, sum, epilogue, act, epilogue == L4_EPI_F32_OUT);
}

}  // namespace

extern "C" int ti_quantize8(void* codes, void* scales, const void* x, long long ldx, int dtype, int n, int k, int rows, cudaStream_t stream);

extern "C" long long ti_linear8_workspace(int n, int out, int K, int given) { return given ? 0 : (long long)n * K + 16 + 4LL * n * ((K + 127) / 128); }

extern "C" int ti_linear8(void* y, long long ldy, const void* x, long long ldx, const float* x_scales, const void* codes, const float* scales, int n, int out,
                          int K, int epilogue, float alpha_p, float alpha_n, float beta, float eps, void* ws, long long ws_bytes, int* status, cudaStream_t stream) {
    if (n == 0 || out == 0) return 0;
    TI_REQUIRE(n > 0 && out > 0 && K > 0 && K % 16 == 0 && n <= 65535, "linear8: %d tokens x %d x %d", n, out, K);
    TI_REQUIRE(linear4_epilogue_known(epilogue), "linear8: unknown epilogue %d", epilogue);
    TI_REQUIRE(aligned16(codes) && (x_scales == nullptr || (aligned16(x) && (n == 1 || ldx % 16 == 0))), "linear8: rows of codes must be 16-byte aligned");
    if (x_scales == nullptr) {
        unsigned char* c = (unsigned char*)ws;
        float* s = (float*)(c + ((long long)n * K + 15) / 16 * 16);
        if (int rc = ti_quantize8(c, s, x, ldx, TI_BF16, n, K, 1, stream)) return rc;
        x = c; ldx = K; x_scales = s;
    }
    ti_launch(linear8_kernel, dim3((out + 7) / 8, n), dim3(256), 0, stream, y, ldy, (const unsigned char*)x, ldx, x_scales, (const unsigned char*)codes, scales, n, out,
              K, epilogue, XieluParams{alpha_p, alpha_n, beta, eps});
    return ti_check_launch("linear8");
}
