// Numbers of 8 bits: e4m3 codes (sign, 4 exponent bits of bias 7, 3 mantissa bits; largest 448, no infinity, 0x7F and 0xFF NaN) with a 32-bit scale per block.
// A block's scale is the smallest power of two s >= 2^-100 with max |x| <= 448 s over the block's finite x, so that x / s is exact: a code depends on x and s
// alone, and a larger scale later moves a code exactly unless it falls below 2^-6 s. What is not finite has the code of NaN.
#pragma once
#include "common.cuh"

#define E4M3_BLOCK 128                   // columns (and, of weights, rows) that share a scale in a matrix

// The scale of blocks whose largest finite |x| is `largest` >= 0: 448 = 1.75 x 2^8.
__device__ __forceinline__ int e4m3_scale_power(float largest) {
    const unsigned bits = __float_as_uint(largest);
    const int power = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return power < -100 ? -100 : power;
}
__device__ __forceinline__ float power_of_two(int p) { return __uint_as_float((unsigned)(p + 127) << 23); }       // -126 <= p <= 127
// |x|, 0 for what is not finite.
__device__ __forceinline__ float finite_size(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;
}
// Two codes, the first in the lower byte.
__device__ __forceinline__ unsigned e4m3_pair(float lo, float hi) {
    unsigned short c;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(hi), "f"(lo));
    return c;
}
__device__ __forceinline__ float or_nan(float x) { return fabsf(x) < INFINITY ? x : __uint_as_float(0x7FFFFFFFu); }
// Four codes, the first in the lowest byte. `inverse` is 1 / scale, exact.
__device__ __forceinline__ unsigned e4m3_codes(float a, float b, float c, float d, float inverse) {
    return e4m3_pair(or_nan(a * inverse), or_nan(b * inverse)) | e4m3_pair(or_nan(c * inverse), or_nan(d * inverse)) << 16;
}
// Two codes as two numbers of 16 bits (exact).
__device__ __forceinline__ unsigned e4m3_half2(unsigned short pair) {
    unsigned h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(pair));
    return h;
}
__device__ __forceinline__ float2 e4m3_float2(unsigned short pair) {
    const unsigned h = e4m3_half2(pair);
    float2 f;
    asm("{.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}
// Eight elements as 32-bit numbers: the largest size and the codes.
__device__ __forceinline__ float largest8(const float (&v)[8]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_size(v[i]));
    return m;
}
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float inverse) {
    return make_uint2(e4m3_codes(v[0], v[1], v[2], v[3], inverse), e4m3_codes(v[4], v[5], v[6], v[7], inverse));
}
// Eight elements as they lie in memory; bits of sizes grow with the sizes.
template <typename T> struct Eight;
template <> struct Eight<bf16> {
    unsigned w[4];
    template <bool VEC> __device__ __forceinline__ void load(const bf16* p) {
        if (VEC) {
            const uint4 u = __ldcg(reinterpret_cast<const uint4*>(p));
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
        } else {
            const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __ldcg(h + 2 * i) | (unsigned)__ldcg(h + 2 * i + 1) << 16;
        }
    }
    __device__ __forceinline__ void clear() { w[0] = w[1] = w[2] = w[3] = 0; }
    __device__ __forceinline__ float operator[](int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16); }
    // The largest size of two lanes of 16 bits, and then of one number.
    __device__ __forceinline__ unsigned sizes(unsigned m) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
        return m;
    }
    static __device__ __forceinline__ unsigned size(unsigned m) { return max(m << 16, m & 0xFFFF0000u); }
};
template <> struct Eight<float> {
    unsigned w[8];
    template <bool VEC> __device__ __forceinline__ void load(const float* p) {
        const unsigned* u = reinterpret_cast<const unsigned*>(p);
        if (VEC) {
            const uint4 a = __ldcg(reinterpret_cast<const uint4*>(u)), b = __ldcg(reinterpret_cast<const uint4*>(u + 4));
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __ldcg(u + i);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0;
    }
    __device__ __forceinline__ float operator[](int i) const { return __uint_as_float(w[i]); }
    __device__ __forceinline__ unsigned sizes(unsigned m) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
        return m;
    }
    static __device__ __forceinline__ unsigned size(unsigned m) { return m; }
};
// The largest finite size of N eights, and whether all are finite.
template <typename T, int N> __device__ __forceinline__ float largest(const Eight<T> (&e)[N], bool& finite) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) m = e[j].sizes(m);
    float f = __uint_as_float(Eight<T>::size(m));
    finite = f < INFINITY;
    if (!finite) {
        f = 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) f = fmaxf(f, finite_size(e[j][i]));
    }
    return f;
}
template <typename T> __device__ __forceinline__ uint2 codes_of(const Eight<T>& e, float inverse, bool finite) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e[i];
    if (!finite) return codes8(v, inverse);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inverse;
    return make_uint2(e4m3_pair(v[0], v[1]) | (unsigned)e4m3_pair(v[2], v[3]) << 16, e4m3_pair(v[4], v[5]) | (unsigned)e4m3_pair(v[6], v[7]) << 16);
}
