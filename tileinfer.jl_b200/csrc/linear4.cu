// Products with weights of 4 bits for steps of few tokens (a draft's): y[n, out] = x[n, in] · W[out, in]ᵀ with
//   W[o, k] = (code[o, k] - zero[k / group, o]) * scale[k / group, o],
// codes 0 to 15 (eight consecutive k in a 32-bit word: the even ones in its low half, the odd ones in its high half, four bits each in
// ascending order), a scale of x's type per row and group of 32, 64 or 128 k, and a zero per row and group (8 for all without a table).
//
// Exactness: code - zero is a whole number of at most 15 and exact in bfloat16. A group's products x (code - zero) are summed in 32-bit,
// the sum is multiplied by the group's scale in 32-bit, and the groups' sums are added in 32-bit; the result is rounded once. Nothing is
// rounded to fewer bits before that (a weight (code - zero) * scale rounded to bfloat16 would cost as much again as the output's rounding).
#include "common.cuh"
#include "mma_util.cuh"

#define L4_EPI_NONE 0
#define L4_EPI_XIELU 1
#define L4_EPI_F32_OUT 2

// Two of a word's codes as bfloat16 pairs, less the zero: 0x4300 | c is 128 + c in bfloat16 (its step is 1 there), and taking 128 + zero off is exact.
__device__ __forceinline__ unsigned widen_pair(unsigned w, unsigned shift, __nv_bfloat162 base) {
    const unsigned c = ((w >> shift) & 0x000F000Fu) | 0x43004300u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&c), base);
    return *reinterpret_cast<const unsigned*>(&v);
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

// ------------------------------------------------------------------------------ bfloat16, up to 16 tokens at once
// Bound by reading the codes once. The rows are shared out evenly among the resident blocks (in fours), the k of a block's rows among its
// warps in stretches of 256: a warp keeps its stretch's tokens in registers as MMA operands and streams [16 rows, 256 k] pieces (2 KB, a
// 128-byte line of every row) through a ring of its own in shared memory, so no barrier stands in the loop; the warps' sums are added once per
// pass over the rows. A word of codes feeds two MMAs as the rows' operand; the k of the two operands are permuted alike, and so that an MMA's
// sixteen k lie in one group: thread t of a quad takes group / 32 consecutive words of the group at a time.
#define L4_WARPS 8
#define L4_MT 5                      // tiles of 16 rows a pass
#define L4_STAGES 5
#define L4_KC 256                    // k of a stretch

template <int GROUP> struct L4Piece {
    static constexpr int GROUPS = L4_KC / GROUP;             // groups of a stretch
    static constexpr int CODES = 16 * L4_KC / 2;             // bytes
    static constexpr int SCALES = GROUPS * 32, ZEROS = GROUPS * 16;
    static constexpr int BYTES = CODES + SCALES + ZEROS;
};

__device__ __forceinline__ void cp_async4(unsigned dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src));
}

// The place of 16-byte piece p of row r: the rows that one phase of a 4-, 8- or 16-byte read covers fall into different banks.
__device__ __forceinline__ int l4_place(int r, int p) { return p ^ (((r & 1) << 2) | (r & 2) | ((r & 4) >> 2)); }

template <int NT, int GROUP>
__global__ void __launch_bounds__(L4_WARPS * 32, 2) linear4_kernel(const unsigned* __restrict__ codes, const bf16* __restrict__ scales,
                                                                   const unsigned char* __restrict__ zeros, const bf16* x, long long ldx, void* y,
                                                                   long long ldy, int n, int out, int K, int passes, bool x_wide, bool s_wide,
                                                                   int epilogue, XieluParams act, bool y32) {
    typedef L4Piece<GROUP> P;
    constexpr int WORDS = GROUP / 32;                        // consecutive words a thread takes
    extern __shared__ __align__(128) unsigned char l4_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = l4_smem + (size_t)warp * L4_STAGES * P::BYTES;
    const int token0 = blockIdx.y * 8 * NT;
    const int stretches = (K + L4_KC - 1) / L4_KC, groups = K / GROUP;
    const int mine = warp < stretches ? (stretches - warp + L4_WARPS - 1) / L4_WARPS : 0;
    const int fours = (out + 3) >> 2;
    bool waited = false;

    for (int pass = 0; pass < passes; ++pass) {
        const long long share = (long long)pass * gridDim.x + blockIdx.x, shares = (long long)passes * gridDim.x;
        const int r0 = 4 * (int)(fours * share / shares), r1 = min(out, 4 * (int)(fours * (share + 1) / shares));
        const int tiles = (r1 - r0 + 15) >> 4;
        // The pieces in the order of their use: the tiles of a stretch, stretch after stretch; each into the ring's next place.
        int next_s = 0, next_m = 0, next_at = 0, at = 0;
        auto issue = [&]() {
            if (next_s < mine) {
                unsigned char* dst = ring + next_at;
                const int stretch = warp + next_s * L4_WARPS, base = r0 + 16 * next_m;
                next_at = next_at == (L4_STAGES - 1) * P::BYTES ? 0 : next_at + P::BYTES;
                if (++next_m == tiles) { next_m = 0; ++next_s; }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int r = u * 4 + (lane >> 3), p = lane & 7, word = stretch * (L4_KC / 8) + 4 * p;
                    if (base + r < r1 && word * 8 < K)
                        cp_async16(smem_u32(dst + r * 128 + l4_place(r, p) * 16), codes + (size_t)(base + r) * (K >> 3) + word);
                }
                const int group0 = stretch * P::GROUPS;
                if (s_wide) {
                    for (int e = lane; e < P::GROUPS * 8; e += 32) {
                        const int grp = min(group0 + (e >> 3), groups - 1), r = base + 2 * (e & 7);
                        if (r < r1) cp_async4(smem_u32(dst + P::CODES + e * 4), scales + (size_t)grp * out + r);
                    }
                    if (zeros != nullptr)
                        for (int e = lane; e < P::GROUPS * 4; e += 32) {
                            const int grp = min(group0 + (e >> 2), groups - 1), r = base + 4 * (e & 3);
                            if (r < r1) cp_async4(smem_u32(dst + P::CODES + P::SCALES + e * 4), zeros + (size_t)grp * out + r);
                        }
                } else {
                    for (int e = lane; e < P::GROUPS * 16; e += 32) {
                        const int grp = min(group0 + (e >> 4), groups - 1), r = base + (e & 15);
                        if (r < r1) {
                            reinterpret_cast<bf16*>(dst + P::CODES)[e] = scales[(size_t)grp * out + r];
                            if (zeros != nullptr) dst[P::CODES + P::SCALES + e] = zeros[(size_t)grp * out + r];
                        }
                    }
                }
            }
            cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < L4_STAGES - 1; ++i) issue();
        if (!waited) { pdl_enter(); waited = true; }         // codes and scales are no result of a step: only the tokens are waited for

        float acc[L4_MT][NT][4];
#pragma unroll
        for (int m = 0; m < L4_MT; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;

        for (int s = 0; s < mine; ++s) {
            // The stretch's tokens: word w of the thread's words holds k = 8 w to 8 w + 7 of token g (+ 8 j).
            uint4 xv[NT][8];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int token = token0 + g + 8 * j;
#pragma unroll
                for (int w = 0; w < 8; ++w) {
                    const int word = (w / WORDS) * (GROUP / 8) + t * WORDS + w % WORDS, k = (warp + s * L4_WARPS) * L4_KC + 8 * word;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (token < n && k < K) {
                        const bf16* src = x + (size_t)token * ldx + k;
                        if (x_wide) v = __ldcg(reinterpret_cast<const uint4*>(src));
                        else {
                            unsigned short e[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) e[i] = __bfloat16_as_ushort(__ldcg(src + i));
                            v = make_uint4(e[0] | (unsigned)e[1] << 16, e[2] | (unsigned)e[3] << 16, e[4] | (unsigned)e[5] << 16,
                                           e[6] | (unsigned)e[7] << 16);
                        }
                    }
                    xv[j][w] = v;
                }
            }
#pragma unroll
            for (int m = 0; m < L4_MT; ++m) {
                if (m >= tiles) break;
                cp_async_wait<L4_STAGES - 2>();
                __syncwarp();
                issue();                                     // into the place of the piece before, which every lane has read
                const unsigned char* src = ring + at;
                at = at == (L4_STAGES - 1) * P::BYTES ? 0 : at + P::BYTES;
                const bf16* sc = reinterpret_cast<const bf16*>(src + P::CODES);
#pragma unroll
                for (int q = 0; q < P::GROUPS; ++q) {
                    float part[NT][4];
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int c = 0; c < 4; ++c) part[j][c] = 0.f;
                    unsigned lo[WORDS], hi[WORDS];
                    {
                        // This group's words of rows g and g + 8: GROUP / 2 bytes a row from byte q * GROUP / 2, thread t's from t * 4 WORDS on.
                        const int byte = q * (GROUP / 2) + t * 4 * WORDS, p = byte >> 4, in = byte & 15;
                        const unsigned* a = reinterpret_cast<const unsigned*>(src + g * 128 + l4_place(g, p) * 16 + in);
                        const unsigned* b = reinterpret_cast<const unsigned*>(src + (g + 8) * 128 + l4_place(g, p) * 16 + in);
                        if (WORDS == 4) {
                            const uint4 va = *reinterpret_cast<const uint4*>(a), vb = *reinterpret_cast<const uint4*>(b);
                            lo[0] = va.x; lo[1 % WORDS] = va.y; lo[2 % WORDS] = va.z; lo[3 % WORDS] = va.w;
                            hi[0] = vb.x; hi[1 % WORDS] = vb.y; hi[2 % WORDS] = vb.z; hi[3 % WORDS] = vb.w;
                        } else if (WORDS == 2) {
                            const uint2 va = *reinterpret_cast<const uint2*>(a), vb = *reinterpret_cast<const uint2*>(b);
                            lo[0] = va.x; lo[1 % WORDS] = va.y;
                            hi[0] = vb.x; hi[1 % WORDS] = vb.y;
                        } else { lo[0] = *a; hi[0] = *b; }
                    }
                    __nv_bfloat162 base_lo = __floats2bfloat162_rn(136.f, 136.f), base_hi = base_lo;
                    if (zeros != nullptr) {
                        base_lo = __float2bfloat162_rn(128.f + (float)src[P::CODES + P::SCALES + q * 16 + g]);
                        base_hi = __float2bfloat162_rn(128.f + (float)src[P::CODES + P::SCALES + q * 16 + g + 8]);
                    }
#pragma unroll
                    for (int w = 0; w < WORDS; ++w) {
                        const unsigned a[2][4] = {{widen_pair(lo[w], 0, base_lo), widen_pair(hi[w], 0, base_hi), widen_pair(lo[w], 4, base_lo),
                                                   widen_pair(hi[w], 4, base_hi)},
                                                  {widen_pair(lo[w], 8, base_lo), widen_pair(hi[w], 8, base_hi), widen_pair(lo[w], 12, base_lo),
                                                   widen_pair(hi[w], 12, base_hi)}};
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            mma16816(part[j], a[0], xv[j][q * WORDS + w].x, xv[j][q * WORDS + w].y);
                            mma16816(part[j], a[1], xv[j][q * WORDS + w].z, xv[j][q * WORDS + w].w);
                        }
                    }
                    const float s_lo = to_f32(sc[q * 16 + g]), s_hi = to_f32(sc[q * 16 + g + 8]);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        acc[m][j][0] = fmaf(s_lo, part[j][0], acc[m][j][0]);
                        acc[m][j][1] = fmaf(s_lo, part[j][1], acc[m][j][1]);
                        acc[m][j][2] = fmaf(s_hi, part[j][2], acc[m][j][2]);
                        acc[m][j][3] = fmaf(s_hi, part[j][3], acc[m][j][3]);
                    }
                }
            }
        }
        // The warps' sums in ascending order of the warps, through the ring's memory.
        cp_async_wait<0>();
        __syncthreads();
        float* red = reinterpret_cast<float*>(l4_smem);      // [warp][tile][j][lane][4]
#pragma unroll
        for (int m = 0; m < L4_MT; ++m)
            if (m < tiles)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    *reinterpret_cast<float4*>(red + ((((size_t)warp * L4_MT + m) * NT + j) * 32 + lane) * 4) =
                        make_float4(acc[m][j][0], acc[m][j][1], acc[m][j][2], acc[m][j][3]);
        __syncthreads();
        const int used = min(L4_WARPS, stretches);
        for (int e = threadIdx.x; e < tiles * NT * 128; e += L4_WARPS * 32) {
            const int l = (e & 127) >> 2, c = e & 3, j = (e >> 7) % NT, m = (e >> 7) / NT;
            const int row = r0 + 16 * m + (l >> 2) + ((c & 2) ? 8 : 0), token = token0 + 8 * j + 2 * (l & 3) + (c & 1);
            if (row >= r1 || token >= n) continue;
            float sum = 0.f;
            for (int w = 0; w < used; ++w) sum += red[((((size_t)w * L4_MT + m) * NT + j) * 32 + l) * 4 + c];
            store_result(y, ldy, token, row, sum, epilogue, act, y32);
        }
        __syncthreads();                                     // the ring is filled again
    }
}

template <int NT, int GROUP>
static int launch_linear4(const void* codes, const void* scales, const void* zeros, const void* x, long long ldx, void* y, long long ldy, int n,
                          int out, int K, int epilogue, XieluParams act, bool y32, cudaStream_t stream) {
    typedef L4Piece<GROUP> P;
    constexpr size_t ring = (size_t)L4_WARPS * L4_STAGES * P::BYTES, red = (size_t)L4_WARPS * L4_MT * NT * 128 * sizeof(float);
    constexpr size_t smem = ring > red ? ring : red;
    static_assert(smem <= 113 * 1024, "two blocks per SM");
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(linear4_kernel<NT, GROUP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return ti_fail("linear4: %s", cudaGetErrorString(e));
        configured = true;
    }
    const int fours = (out + 3) / 4, slots = 2 * ti_sm_count();
    const int blocks = fours < slots ? fours : slots;
    const int passes = (fours + blocks * (4 * L4_MT) - 1) / (blocks * (4 * L4_MT));
    const bool x_wide = aligned16(x) && ldx % 8 == 0;
    const bool s_wide = out % 4 == 0 && (uintptr_t)scales % 4 == 0 && (uintptr_t)zeros % 4 == 0;
    ti_launch(linear4_kernel<NT, GROUP>, dim3(blocks, (n + 8 * NT - 1) / (8 * NT)), dim3(L4_WARPS * 32), smem, stream, (const unsigned*)codes,
              (const bf16*)scales, (const unsigned char*)zeros, (const bf16*)x, ldx, y, ldy, n, out, K, passes, x_wide, s_wide, epilogue, act, y32);
    return ti_check_launch("linear4");
}

// ------------------------------------------------------------------------------ 32-bit
// Multiply-adds in 32-bit throughout. A block takes 4 rows, its warps' lanes take words of k in turn (a lane's word lies in one group), and
// every (row, token) sum is added up over the lanes and then the warps in a fixed order that depends on K alone, so a token's result does not
// depend on the step it is in.
#define L4F_WARPS 4
#define L4F_ROWS 4
#define L4F_TOKENS 8

__global__ void __launch_bounds__(L4F_WARPS * 32) linear4_f32_kernel(const unsigned* __restrict__ codes, const float* __restrict__ scales,
                                                                     const unsigned char* __restrict__ zeros, const float* x, long long ldx, float* y,
                                                                     long long ldy, int n, int out, int K, int group, bool x_wide, int epilogue,
                                                                     XieluParams act) {
    __shared__ float red[L4F_WARPS][L4F_ROWS][L4F_TOKENS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = blockIdx.x * L4F_ROWS, token0 = blockIdx.y * L4F_TOKENS, words = K >> 3;
    pdl_enter();
    float acc[L4F_ROWS][L4F_TOKENS];
#pragma unroll
    for (int r = 0; r < L4F_ROWS; ++r)
#pragma unroll
        for (int j = 0; j < L4F_TOKENS; ++j) acc[r][j] = 0.f;
    for (int w = threadIdx.x; w < words; w += L4F_WARPS * 32) {
        const int grp = 8 * w / group;
        float c[L4F_ROWS][8], s[L4F_ROWS];
#pragma unroll
        for (int r = 0; r < L4F_ROWS; ++r) {
            const int row = min(row0 + r, out - 1);
            const unsigned v = codes[(size_t)row * words + w];
            s[r] = scales[(size_t)grp * out + row];
            // 0x4B000000 | c is 2^23 + c
            const float base = 8388608.f + (zeros != nullptr ? (float)zeros[(size_t)grp * out + row] : 8.f);
#pragma unroll
            for (int i = 0; i < 8; ++i) c[r][i] = __uint_as_float(((v >> (4 * (i >> 1) + 16 * (i & 1))) & 15u) | 0x4B000000u) - base;
        }
#pragma unroll
        for (int j = 0; j < L4F_TOKENS; ++j) {
            if (token0 + j >= n) break;
            const float* src = x + (size_t)(token0 + j) * ldx + 8 * w;
            float xv[8];
            if (x_wide) {
                const float4 a = __ldcg(reinterpret_cast<const float4*>(src)), b = __ldcg(reinterpret_cast<const float4*>(src) + 1);
                xv[0] = a.x; xv[1] = a.y; xv[2] = a.z; xv[3] = a.w; xv[4] = b.x; xv[5] = b.y; xv[6] = b.z; xv[7] = b.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) xv[i] = __ldcg(src + i);
            }
#pragma unroll
            for (int r = 0; r < L4F_ROWS; ++r) {
                float p = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) p = fmaf(c[r][i], xv[i], p);
                acc[r][j] = fmaf(s[r], p, acc[r][j]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < L4F_ROWS; ++r)
#pragma unroll
        for (int j = 0; j < L4F_TOKENS; ++j) {
            const float v = warp_sum(acc[r][j]);
            if (lane == 0) red[warp][r][j] = v;
        }
    __syncthreads();
    if (threadIdx.x < L4F_ROWS * L4F_TOKENS) {
        const int r = threadIdx.x / L4F_TOKENS, j = threadIdx.x % L4F_TOKENS;
        if (row0 + r < out && token0 + j < n) {
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < L4F_WARPS; ++w) sum += red[w][r][j];
            store_result(y, ldy, token0 + j, row0 + r, sum, epilogue, act, true);
        }
    }
}

// codes [out, K / 8] words, scales [K / group, out] of x's type, zeros [K / group, out] bytes or null; y [n, ldy] of x's type, or 32-bit sums
// that are not rounded (epilogue 2).
extern "C" int ti_linear4(void* y, long long ldy, const void* x, long long ldx, const void* codes, const void* scales, const void* zeros, int n,
                          int out, int K, int group, int epilogue, float alpha_p, float alpha_n, float beta, float eps, int dtype,
                          cudaStream_t stream) {
    if (n == 0 || out == 0) return 0;
    TI_REQUIRE(n > 0 && out > 0 && K > 0, "linear4: %d tokens, %d x %d", n, out, K);
    TI_REQUIRE(group == 32 || group == 64 || group == 128, "linear4: groups of %d (32, 64 or 128)", group);
    TI_REQUIRE(K % group == 0, "linear4: %d inputs are not whole groups of %d", K, group);
    TI_REQUIRE(aligned16(codes), "linear4: the codes must be 16-byte aligned");
    TI_REQUIRE(dtype == TI_F32 || dtype == TI_BF16, "linear4: unknown element type code %d", dtype);
    TI_REQUIRE(epilogue == L4_EPI_NONE || epilogue == L4_EPI_XIELU || epilogue == L4_EPI_F32_OUT || (epilogue >= TI_EPI_GELU_ERF && epilogue <= TI_EPI_LAST),
               "linear4: unknown epilogue %d", epilogue);
    const XieluParams act{alpha_p, alpha_n, beta, eps};
    if (dtype == TI_F32) {
        TI_REQUIRE((n + L4F_TOKENS - 1) / L4F_TOKENS <= 65535, "linear4: %d tokens in one launch", n);
        const bool x_wide = aligned16(x) && ldx % 4 == 0;
        ti_launch(linear4_f32_kernel, dim3((out + L4F_ROWS - 1) / L4F_ROWS, (n + L4F_TOKENS - 1) / L4F_TOKENS), dim3(L4F_WARPS * 32), 0, stream,
                  (const unsigned*)codes, (const float*)scales, (const unsigned char*)zeros, (const float*)x, ldx, (float*)y, ldy, n, out, K, group,
                  x_wide, epilogue, act);
        return ti_check_launch("linear4");
    }
    TI_REQUIRE((n + 7) / 8 <= 65535, "linear4: %d tokens in one launch", n);
#define L4_CASE(nt, grp) return launch_linear4<nt, grp>(codes, scales, zeros, x, ldx, y, ldy, n, out, K, epilogue, act, epilogue == L4_EPI_F32_OUT, stream)
    if (n <= 8) {
        if (group == 32) L4_CASE(1, 32);
        if (group == 64) L4_CASE(1, 64);
        L4_CASE(1, 128);
    }
    if (group == 32) L4_CASE(2, 32);
    if (group == 64) L4_CASE(2, 64);
    L4_CASE(2, 128);
#undef L4_CASE
}

// ------------------------------------------------------------------------------ the codes of a matrix
// A group's scale and codes from its weights: without zeros scale = max |w| / 7 and code = 8 + round(w / scale) (1 to 15); with zeros
// scale = (max - min) / 15 over the group and 0, zero = round(-min / scale) and code = zero + round(w / scale), 0 to 15. The scale is rounded to
// its type first, and the codes go by the rounded one. One warp a group; runs once per matrix. The products read codes before they wait for the
// kernel before them, so this one lets nothing start beside it and every thread's stores reach all before it ends.
template <typename T, typename S>
__global__ void quantize4_kernel(const T* w, long long ldw, unsigned* codes, S* scales, unsigned char* zeros, int out, int K, int group) {
    const int lane = threadIdx.x & 31, groups = K / group, per = group / 32;
    const long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    pdl_wait();
    if (item >= (long long)out * groups) return;
    const int row = (int)(item / groups), grp = (int)(item % groups);
    const T* src = w + (size_t)row * ldw + (size_t)grp * group;
    float v[4], top = 0.f, low = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = i < per ? to_f32(src[lane + 32 * i]) : 0.f;
        top = fmaxf(top, v[i]);
        low = fminf(low, v[i]);
    }
    top = warp_max(top);
    low = -warp_max(-low);
    float scale = zeros != nullptr ? __fdiv_rn(top - low, 15.f) : __fdiv_rn(fmaxf(top, -low), 7.f);
    scale = to_f32(from_f32<S>(scale));
    const float zero = zeros == nullptr ? 8.f : scale > 0.f ? fminf(15.f, rintf(__fdiv_rn(-low, scale))) : 0.f;
    if (lane == 0) {
        scales[(size_t)grp * out + row] = from_f32<S>(scale);
        if (zeros != nullptr) zeros[(size_t)grp * out + row] = (unsigned char)zero;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i >= per) break;
        const float c = scale > 0.f ? fminf(15.f, fmaxf(zeros == nullptr ? 1.f : 0.f, zero + rintf(__fdiv_rn(v[i], scale)))) : zero;
        unsigned word = (unsigned)c << (4 * ((lane & 7) >> 1) + 16 * (lane & 1));
        word |= __shfl_xor_sync(0xffffffffu, word, 1);
        word |= __shfl_xor_sync(0xffffffffu, word, 2);
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        if ((lane & 7) == 0) codes[(size_t)row * (K >> 3) + (size_t)grp * (group >> 3) + 4 * i + (lane >> 3)] = word;
    }
    __threadfence();
}

extern "C" int ti_quantize4(const void* w, long long ldw, int w_dtype, void* codes, void* scales, int s_dtype, void* zeros, int out, int K, int group,
                            cudaStream_t stream) {
    if (out == 0) return 0;
    TI_REQUIRE(out > 0 && K > 0, "quantize4: %d x %d", out, K);
    TI_REQUIRE(group == 32 || group == 64 || group == 128, "quantize4: groups of %d (32, 64 or 128)", group);
    TI_REQUIRE(K % group == 0, "quantize4: %d inputs are not whole groups of %d", K, group);
    TI_REQUIRE((s_dtype == TI_F32 || s_dtype == TI_BF16) && (w_dtype == TI_F32 || w_dtype == TI_BF16), "quantize4: unknown element type code");
    const long long items = (long long)out * (K / group), blocks = (items + 7) / 8;
    TI_REQUIRE(blocks <= 0x7fffffffLL, "quantize4: %d x %d is too large for one launch", out, K);
#define Q4_CASE(T, S) \
    ti_launch(quantize4_kernel<T, S>, dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)w, ldw, (unsigned*)codes, (S*)scales, (unsigned char*)zeros, out, K, group)
    if (w_dtype == TI_F32 && s_dtype == TI_F32) Q4_CASE(float, float);
    else if (w_dtype == TI_F32) Q4_CASE(float, bf16);
    else if (s_dtype == TI_F32) Q4_CASE(bf16, float);
    else Q4_CASE(bf16, bf16);
#undef Q4_CASE
    return ti_check_launch("quantize4");
}
