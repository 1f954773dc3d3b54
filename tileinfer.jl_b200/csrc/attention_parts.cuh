// Attention whose work is shared out by the sequences' lengths: the units of work, 64-key tiles of all (sequence, KV head, slab of rows), are numbered in that
// order and taken by every block in equal runs (even_runs.cuh); rows whose tiles lie in several runs are left as parts in 32-bit (maximum, sum,
// unnormalised output), which a second kernel joins.
#pragma once
#include "even_runs.cuh"

#define AF_PAGE 64

namespace {

struct FewShape {
    int T, L, first, t0, tiles, slabs;                       // new tokens, length, first visible key, first tile, tiles, slabs of rows
};
// What is given for a batch may be wrong: ranges stay within the rows that there are, runs within the most new tokens that were said (the units' number was checked with them),
// lengths within the positions that a sequence's row of the table has pages for.
struct FewLimits {
    int rows, most_new, positions;
    __device__ __forceinline__ int run(int T) const { return min(T, most_new); }
    __device__ __forceinline__ int row(int at) const { return min(max(at, 0), rows); }
    __device__ __forceinline__ int length(int len) const { return min(max(len, 0), positions); }
};
__device__ __forceinline__ FewShape few_shape(int T, int L, int window, int group, int M) {
    FewShape s;
    s.T = T; s.L = L;
    s.first = window > 0 ? max(0, L - T - window + 1) : 0;
    s.t0 = s.first / AF_PAGE;
    s.tiles = T > 0 && L > 0 ? (L + AF_PAGE - 1) / AF_PAGE - s.t0 : 0;
    s.slabs = (T * group + M - 1) / M;
    return s;
}
// Below 2^-126: 0.
__device__ __forceinline__ float power2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// sum + part 2^x, x <= 0 and f = 2^x: in two steps where f would have lost bits or be zero (scales of 8-bit pages that lie far apart).
__device__ __forceinline__ float add_times(float sum, float part, float x, float f) {
    if (x > -100.f) return fmaf(part, f, sum);
    const float half = exp2f(0.5f * x);
    return sum + part * half * half;
}

// The parts of the rows that several blocks share, joined in ascending order: AF_JOIN_WARPS / WPR rows a block, WPR warps a row, four elements a lane,
// every WPRth part a warp. Rows of items that one block did are done; rows without keys get zeros. What bounds it is one dependent load after another
// with the kernel before gone: so where the parts lie is worked out before that kernel ends, and maxima, sums and outputs of eight parts are asked
// for together.
#define AF_JOIN_WARPS 4
template <int WPR>
__global__ void __launch_bounds__(32 * AF_JOIN_WARPS) attention_few_join_kernel(bf16* out, const int* cu, const int* kv_lens, const float* ws_o,
                                                                                const float* ws_ml, int B, int nq, int nkv, int D, int M, int window,
                                                                                int blocks, FewLimits limits) {
    __shared__ unsigned s_sum[AF_JOIN_WARPS][2];
    __shared__ float4 s_o[WPR > 1 ? WPR : 1][32];
    __shared__ float2 s_ml[WPR];
    const int b = blockIdx.z, kvh = blockIdx.y, group = nq / nkv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned before = 0, U = 0;
    for (int c = threadIdx.x; c < B; c += 32 * AF_JOIN_WARPS) {
        const FewShape s = few_shape(limits.run(limits.row(__ldcg(cu + c + 1)) - limits.row(__ldcg(cu + c))), limits.length(__ldcg(kv_lens + c)), window, group, M);
        U += s.tiles * s.slabs * nkv;
        if (c < b) before += s.tiles * s.slabs * nkv;
    }
    U = __reduce_add_sync(0xffffffffu, U);
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) { s_sum[warp][0] = before; s_sum[warp][1] = U; }
    __syncthreads();
    before = U = 0;
#pragma unroll
    for (int w = 0; w < AF_JOIN_WARPS; ++w) { before += s_sum[w][0]; U += s_sum[w][1]; }
    const int first_token = limits.row(__ldcg(cu + b)), T = limits.run(limits.row(__ldcg(cu + b + 1)) - first_token), row = blockIdx.x * (AF_JOIN_WARPS / WPR) + warp / WPR, mine = warp % WPR;
    const FewShape s = few_shape(T, limits.length(__ldcg(kv_lens + b)), window, group, M);
    const int i = row / group, slab = row / M, in = row - slab * M;
    const Runs runs(U, max(min((unsigned)blocks, U), 1u));
    const unsigned u0 = before + (unsigned)((kvh * s.slabs + slab) * s.tiles);
    const bool empty = s.tiles == 0, real = row < T * group;
    const unsigned c0 = real && !empty ? runs.owner(u0) : 0, c1 = real && !empty ? runs.owner(u0 + s.tiles - 1) : 0;
    pdl_enter();
    if (!real || (!empty && c0 == c1)) return;               // with WPR > 1 the block's one row: all leave
    bf16* dst = out + ((size_t)(first_token + i) * nq + (size_t)kvh * group + (row - i * group)) * D;
    const int parts = empty ? 0 : (int)(c1 - c0 + 1);
    // A run that begins before the item holds its part in the second slot: the first part alone may.
    const size_t first = empty ? 0 : (size_t)runs.slot(c0, u0) * M + in, others = (size_t)2 * c0 * M + in;
    auto at = [&](int c) { return c == 0 ? first : others + (size_t)2 * c * M; };
    const float2* ml = reinterpret_cast<const float2*>(ws_ml);
    for (int d0 = 0; d0 < D; d0 += 128) {
        const int d = d0 + 4 * lane;
        const bool on = d < D;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f, mm = -INFINITY;
        for (int p = mine; p < parts; p += 8 * WPR) {
            float4 v[8];
            const int pl = p + lane * WPR;
            const float2 x = lane < 8 && pl < parts ? __ldcg(ml + at(pl)) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v[k] = on && p + k * WPR < parts ? __ldcg(reinterpret_cast<const float4*>(ws_o + at(p + k * WPR) * D + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
            const float top = fmaxf(mm, warp_max(x.x)), base = top == -INFINITY ? 0.f : top;
            const float old = exp2f(mm - base), f = exp2f(x.x - base);
            sum = add_times(warp_sum(add_times(0.f, x.y, x.x - base, f)), sum, mm - base, old);
            mm = top;
            acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float w = __shfl_sync(0xffffffffu, f, k);
                acc.x = fmaf(v[k].x, w, acc.x); acc.y = fmaf(v[k].y, w, acc.y); acc.z = fmaf(v[k].z, w, acc.z); acc.w = fmaf(v[k].w, w, acc.w);
            }
        }
        if (WPR > 1) {
            if (d0 > 0) __syncthreads();
            s_o[mine][lane] = acc;
            if (lane == 0) s_ml[mine] = make_float2(mm, sum);
            __syncthreads();
            if (mine > 0) continue;
            mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < WPR; ++w) mm = fmaxf(mm, s_ml[w].x);
            const float base = mm == -INFINITY ? 0.f : mm;
            acc = make_float4(0.f, 0.f, 0.f, 0.f);
            sum = 0.f;
#pragma unroll
            for (int w = 0; w < WPR; ++w) {
                const float f = exp2f(s_ml[w].x - base);
                const float4 v = s_o[w][lane];
                sum = add_times(sum, s_ml[w].y, s_ml[w].x - base, f);
                acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
            }
        }
        if (sum == 0.f) { acc = make_float4(0.f, 0.f, 0.f, 0.f); sum = 1.f; }            // nothing was visible; a NaN sum stays one
        const float inv = 1.f / sum;
        if (on) {
            reinterpret_cast<__nv_bfloat162*>(dst + d)[0] = __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
            reinterpret_cast<__nv_bfloat162*>(dst + d)[1] = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
        }
    }
}


// Joins what `blocks` blocks have left of the rows of slabs of M.
inline void join_parts(bf16* out, const int* cu, const int* kv_lens, const float* ws_o, const float* ws_ml, int B, int nq, int nkv, int D, int M, int max_new,
                       int window, int blocks, FewLimits limits, cudaStream_t stream) {
    const int rows = max_new * (nq / nkv);
    // More than eight parts an item: four warps a row (59.9 us in place of 62.3 at 37 parts; at two parts 90 in place of 70).
    const bool deep = 8LL * B * nkv * ((rows + M - 1) / M) < blocks;
    ti_launch(deep ? attention_few_join_kernel<4> : attention_few_join_kernel<1>, dim3(deep ? rows : (rows + AF_JOIN_WARPS - 1) / AF_JOIN_WARPS, nkv, B),
              dim3(32 * AF_JOIN_WARPS), 0, stream, out, cu, kv_lens, ws_o, ws_ml, B, nq, nkv, D, M, window, blocks, limits);
}

}  // namespace
