// Codes of e4m3 (e4m3.cuh) from a matrix x [n, k]: a scale for every 128 columns of each row (a product's inputs), or of 128 rows (its weights).
//
//   scales[g, i] = the smallest power of two s with |x| <= 448 s over the block;  codes = rn(x / s).
//
// Bound by reading x and writing the codes once (3 bytes an element of bfloat16): a block's elements stay in registers between its maximum and its codes, as they
// were read. Instructions would be the bound otherwise, so sizes are compared as integers (two of bfloat16 at once) and what is not finite, which they show,
// is dealt with only where it is. 4,096 x 21,504 of bfloat16 in 128 x 128 blocks 43.7 us (6.0 TB/s; 40.2 while kernels behind started beside it), 2,048 x 4,096 by rows 6.6 us (3.8 TB/s: a launch and one wave).
// Scales lie [k / 128, rows]: a block of threads makes sixteen rows' next to one another.
#include "e4m3.cuh"

namespace {

// Rows on their own: sixteen lanes a row's group, four groups of sixteen rows a block of 256 threads.
constexpr int Q_ROWS = 16, Q_GROUPS = 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize8_rows_kernel(unsigned char* codes, float* scales, const T* x, long long ldx, int n, int k, int groups) {
    const int row = blockIdx.y * Q_ROWS + (threadIdx.x >> 4), part = threadIdx.x & 15, g0 = blockIdx.x * Q_GROUPS;
    pdl_enter();
    Eight<T> v[Q_GROUPS];
#pragma unroll
    for (int g = 0; g < Q_GROUPS; ++g) {
        const int col = (g0 + g) * E4M3_BLOCK + part * 8;
        v[g].clear();
        if (row < n && col < k) v[g].template load<VEC>(x + (long long)row * ldx + col);
    }
#pragma unroll
    for (int g = 0; g < Q_GROUPS; ++g) {
        const int col = (g0 + g) * E4M3_BLOCK + part * 8;
        bool finite;
        const Eight<T> one[1] = {v[g]};
        float m = largest(one, finite);
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const int power = e4m3_scale_power(m);
        if (row < n && col < k) *reinterpret_cast<uint2*>(codes + (long long)row * k + col) = codes_of(v[g], power_of_two(-power), finite);
        if (row < n && part == 0 && g0 + g < groups) scales[(long long)(g0 + g) * n + row] = power_of_two(power);
    }
}

// Blocks of 128 x 128: 256 threads hold one, 64 elements each. The products ask for weights before they wait for the kernel before them, so this one lets nothing
// start beside it and every thread's stores reach all before it ends.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize8_blocks_kernel(unsigned char* codes, float* scales, const T* x, long long ldx, int n, int k, int row_blocks) {
    __shared__ float scratch[33];
    const int g = blockIdx.x, row0 = blockIdx.y * E4M3_BLOCK + (threadIdx.x >> 4), col = g * E4M3_BLOCK + (threadIdx.x & 15) * 8;
    pdl_wait();
    Eight<T> v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j].clear();
        if (row0 + 16 * j < n && col < k) v[j].template load<VEC>(x + (long long)(row0 + 16 * j) * ldx + col);
    }
    bool finite;
    const float m = largest(v, finite);
    const int power = e4m3_scale_power(block_max(m, scratch));
    const float inverse = power_of_two(-power);
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (row0 + 16 * j < n && col < k) *reinterpret_cast<uint2*>(codes + (long long)(row0 + 16 * j) * k + col) = codes_of(v[j], inverse, finite);
    if (threadIdx.x == 0) scales[(long long)g * row_blocks + blockIdx.y] = power_of_two(power);
    __threadfence();
}

template <typename T> int launch(unsigned char* codes, float* scales, const T* x, long long ldx, int n, int k, int rows, cudaStream_t stream) {
    const bool vec = aligned16(x) && (n == 1 || ldx * (long long)sizeof(T) % 16 == 0);
    const int groups = (k + E4M3_BLOCK - 1) / E4M3_BLOCK;
    if (rows == 1) {
        const dim3 grid((groups + Q_GROUPS - 1) / Q_GROUPS, (n + Q_ROWS - 1) / Q_ROWS);
        TI_REQUIRE(grid.y <= 65535, "quantize8: %d rows, each with scales of its own, are too many", n);
        auto* kernel = vec ? quantize8_rows_kernel<T, true> : quantize8_rows_kernel<T, false>;
        static bool configured[2] = {};
        if (!configured[vec]) {
            // A product's blocks come up beside this kernel's and keep the split of the SMs that they find; without this those of 4,096 x 21,504 waited until the
            // SMs were free (5 tokens 34 us instead of 21).
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
            if (e != cudaSuccess) return ti_fail("quantize8: %s", cudaGetErrorString(e));
            configured[vec] = true;
        }
        ti_launch(kernel, grid, dim3(256), 0, stream, codes, scales, x, ldx, n, k, groups);
    } else {
        const int row_blocks = (n + E4M3_BLOCK - 1) / E4M3_BLOCK;
        TI_REQUIRE(row_blocks <= 65535, "quantize8: %d rows are too many", n);
        ti_launch(vec ? quantize8_blocks_kernel<T, true> : quantize8_blocks_kernel<T, false>, dim3(groups, row_blocks), dim3(256), 0, stream, codes, scales, x, ldx,
                  n, k, row_blocks);
    }
    return ti_check_launch("quantize8");
}

}  // namespace

// codes [n, k] (dense), scales [ceil(k / 128), ceil(n / rows)]; x [n, k] in rows of pitch ldx. rows 1 or 128; k a multiple of 16.
extern "C" int ti_quantize8(void* codes, void* scales, const void* x, long long ldx, int dtype, int n, int k, int rows, cudaStream_t stream) {
    if (n == 0 || k == 0) return 0;
    TI_REQUIRE(n > 0 && k > 0 && k % 16 == 0 && (rows == 1 || rows == E4M3_BLOCK), "quantize8: %d x %d in blocks of %d rows", n, k, rows);
    TI_REQUIRE(aligned16(codes), "quantize8: codes must be 16-byte aligned");
    TI_REQUIRE((uintptr_t)x % (dtype == TI_F32 ? 4 : 2) == 0 && (uintptr_t)scales % 4 == 0, "quantize8: a misaligned address");
    TI_DISPATCH_DTYPE(dtype, return launch<T>((unsigned char*)codes, (float*)scales, (const T*)x, ldx, n, k, rows, stream));
}
