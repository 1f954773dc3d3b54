// Shared by the products with 4-bit weights: widening of codes, epilogues.
#pragma once
#include "common.cuh"

#define L4_EPI_NONE 0
#define L4_EPI_XIELU 1
#define L4_EPI_F32_OUT 2

// Two of a word's codes as bfloat16 pairs, less the zero: 0x4300 | c is 128 + c in bfloat16 (its step is 1 there), and taking 128 + zero off is exact.
// (Written as the three instructions that it takes: from the operators the compiler makes five.)
__device__ __forceinline__ unsigned widen_pair(unsigned w, unsigned shift, unsigned base) {
    unsigned v;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w >> shift), "r"(0x000F000Fu), "r"(0x43004300u));
    asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(base));
    return v;
}

__device__ __forceinline__ void store_result(void* y, long long ldy, int token, int row, float s, int epilogue, const XieluParams& act, bool y32) {
    if (epilogue == L4_EPI_F32_OUT || (y32 && epilogue == L4_EPI_NONE)) {
        ((float*)y)[(size_t)token * ldy + row] = s;
        return;
    }
    if (y32) {
        ((float*)y)[(size_t)token * ldy + row] = epilogue == L4_EPI_XIELU ? xielu_value<float>(s, act) : gelu_epilogue(s, epilogue);
        return;
    }
    float v = rnd<bf16>(s);
    if (epilogue == L4_EPI_XIELU) v = xielu_value<bf16>(v, act);
    if (epilogue >= TI_EPI_GELU_ERF) v = gelu_epilogue(v, epilogue);
    ((bf16*)y)[(size_t)token * ldy + row] = __float2bfloat16_rn(v);
}

inline bool linear4_epilogue_known(int e) {
    return e == L4_EPI_NONE || e == L4_EPI_XIELU || e == L4_EPI_F32_OUT || (e >= TI_EPI_GELU_ERF && e <= TI_EPI_LAST);
}

// Whether runs of equal length end inside of an item of `steps` units, whose parts a second kernel then joins.
inline bool linear4_cuts_items(long long units, long long steps) {
    const long long runs = units < ti_sm_count() ? units : ti_sm_count();
    return units % runs != 0 || units / runs % steps != 0;
}

// linear4_wide.cu
extern "C" int ti_linear4_shared(int n, int out, int K);
int linear4_wide(void* y, long long ldy, const void* x, long long ldx, const void* codes, const void* scales, const void* zeros, int n, int out, int K,
                 int group, int epilogue, XieluParams act, void* parts, int* status, cudaStream_t stream);
