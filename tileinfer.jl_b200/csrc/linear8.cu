// Products of e4m3 codes with a scale for every 128 of k: which kernel takes one.
#include "linear8.cuh"

extern "C" int ti_quantize8(void* codes, void* scales, const void* x, long long ldx, int dtype, int n, int k, int rows, cudaStream_t stream);

extern "C" int ti_xielu(void* out, const void* in, long long count, float alpha_p, float alpha_n, float beta, float eps, int dtype, cudaStream_t stream);
extern "C" int ti_gelu(void* out, const void* in, long long count, int kind, int dtype, cudaStream_t stream);

static long long up16(long long bytes) { return (bytes + 15) / 16 * 16; }

// Weight rows in the lanes, 64 tokens at once (linear8_mid.cu), or tokens in the lanes on SM pairs (linear8_many.cu): the shorter by estimates in microseconds. The
// one takes half of one for every 128 x 64 x 128 that an SM gets, the other 0.65 for every step of 256 of k of a pair's tiles, rounds of which are whole.
// Microseconds in turn: 64 tokens of 21,504 x 4,096 26 / 38, 256 78 / 39; 128 of 4,096 x 21,504 36 / 57, 256 70 / 57; 256 of 4,096 x 4,096 16 / 15.5.
static bool takes_many(int n, int out, int K) {
    const double groups = (K + 127) / 128, units = (double)((out + 127) / 128) * ((n + 63) / 64) * groups;
    const long long tiles = (long long)((out + 127) / 128) * ((n + 255) / 256), pairs = ti_sm_count() / 2, rounds = (tiles + pairs - 1) / pairs;
    return 3.0 + rounds * (1.0 + 0.65 * ((groups + 1) / 2)) < 5.0 + 0.5 * units / ti_sm_count();
}

// Tokens that come as bfloat16 are quantised by every block that needs them where they are few, else by a launch of its own ahead. Microseconds ahead / in the
// blocks: eight tokens of 1,024 x 1,024 4.9 / 3.8, 4,096 x 4,096 9.1 / 7.5, 14,336 x 4,096 16.1 / 16.3, 21,504 x 4,096 21.3 / 25.7; four of that 21.0 / 21.4.
static bool quantized_ahead(int n, int out, int K) { return !linear8_takes_few(n, out, K) || (n > 4 && (long long)out * K > 70000000); }

// Whether an activation is a launch of its own over the rounded sums, which is what it acts on in any case: beyond 32 tokens, where a product's few warps would
// take longer over it. Microseconds with xIELU in the product / apart: 21,504 x 4,096, 16 tokens 25.0 / 24.9, 64 33.8 / 29.5, 2,048 381 / 277.
extern "C" int ti_linear8_apart(int n, int out, long long ldy, int epilogue) {
    return n > 32 && ldy == out && (epilogue == L4_EPI_XIELU || epilogue == TI_EPI_GELU_ERF || epilogue == TI_EPI_GELU_TANH);
}

// xIELU in place, eight values a thread in packed arithmetic of 16 bits, which rounds as xielu_value does where the factors are bfloat16 numbers (a model's are):
// 2,048 x 21,504 take 77 us, in 32-bit 123 (exponentials; 27 us are its bytes).
__global__ void __launch_bounds__(256) linear8_xielu_kernel(bf16* y, size_t eights, const XieluParams params) {
    const XieluPacked act = xielu_pack(params);
    pdl_enter();
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < eights; i += (size_t)gridDim.x * 256) {
        uint4* at = reinterpret_cast<uint4*>(y) + i;
        const uint4 v = __ldcg(at);
        unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            unsigned lo, hi;
            xielu_bf16_pair(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u), act, lo, hi);
            w[j] = lo | hi << 16;
        }
        *at = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
static bool is_bf16(float f) { return __bfloat162float(__float2bfloat16(f)) == f; }
static int xielu_apart(void* y, long long count, float alpha_p, float alpha_n, float beta, float eps, cudaStream_t stream) {
    if (!(is_bf16(alpha_p) && is_bf16(alpha_n) && is_bf16(beta)) || count % 8 != 0 || !aligned16(y)) return ti_xielu(y, y, count, alpha_p, alpha_n, beta, eps, TI_BF16, stream);
    long long blocks = (count / 8 + 255) / 256;
    if (blocks > ti_sm_count() * 32) blocks = ti_sm_count() * 32;
    ti_launch(linear8_xielu_kernel, dim3((int)blocks), dim3(256), 0, stream, (bf16*)y, (size_t)(count / 8), XieluParams{alpha_p, alpha_n, beta, eps});
    return ti_check_launch("linear8_xielu");
}

// Bytes of the work space: the tokens' codes and scales, where they are made ahead.
extern "C" long long ti_linear8_workspace(int n, int out, int K, int given) {
    if (n <= 0 || out <= 0 || K <= 0 || given || !quantized_ahead(n, out, K)) return 0;
    return up16((long long)n * K) + up16(4LL * n * ((K + E4M3_BLOCK - 1) / E4M3_BLOCK));
}

extern "C" int ti_linear8(void* y, long long ldy, const void* x, long long ldx, const float* x_scales, const void* codes, const float* scales, int n, int out,
                          int K, int epilogue, float alpha_p, float alpha_n, float beta, float eps, void* ws, long long ws_bytes, int* status, cudaStream_t stream) {
    if (n == 0 || out == 0) return 0;
    TI_REQUIRE(n > 0 && out > 0 && K > 0 && K % 16 == 0, "linear8: %d tokens x %d x %d", n, out, K);
    TI_REQUIRE(linear4_epilogue_known(epilogue), "linear8: unknown epilogue %d", epilogue);
    TI_REQUIRE(aligned16(codes) && (x_scales == nullptr || (aligned16(x) && (n == 1 || ldx % 16 == 0))), "linear8: rows of codes must be 16-byte aligned");
    TI_REQUIRE((uintptr_t)x % 2 == 0 && (uintptr_t)y % 2 == 0, "linear8: a misaligned address");
    TI_REQUIRE(status != nullptr, "linear8: status word missing");
    const long long need = ti_linear8_workspace(n, out, K, x_scales != nullptr);
    TI_REQUIRE(need == 0 || (ws != nullptr && aligned16(ws) && ws_bytes >= need), "linear8: work space of %lld bytes, %lld needed", ws_bytes, need);
    if (need) {
        unsigned char* made = (unsigned char*)ws;
        float* made_scales = (float*)(made + up16((long long)n * K));
        if (int rc = ti_quantize8(made, made_scales, x, ldx, TI_BF16, n, K, 1, stream)) return rc;
        x = made; ldx = K; x_scales = made_scales;
    }
    const bool apart = ti_linear8_apart(n, out, ldy, epilogue);
    const Linear8 a = {y, ldy, x, ldx, x_scales, (const unsigned char*)codes, scales, n, out, K, apart ? L4_EPI_NONE : epilogue, XieluParams{alpha_p, alpha_n, beta, eps}, status};
    if (linear8_takes_few(n, out, K)) return linear8_few(a, stream);
    const int rc = takes_many(n, out, K) ? linear8_many(a, stream) : linear8_mid(a, stream);
    if (rc || !apart) return rc;
    const long long count = (long long)n * out;
    return epilogue == L4_EPI_XIELU ? xielu_apart(y, count, alpha_p, alpha_n, beta, eps, stream) : ti_gelu(y, y, count, epilogue - TI_EPI_GELU_ERF, TI_BF16, stream);
}
