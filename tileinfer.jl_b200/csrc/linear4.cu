// Products with weights of 4 bits for steps of few tokens (a draft's): y[n, out] = x[n, in] · W[out, in]ᵀ with
//   W[o, k] = (code[o, k] - zero[k / group, o]) * scale[k / group, o],
// codes 0 to 15 (eight consecutive k in a 32-bit word: the even ones in its low half, the odd ones in its high half, four bits each in
// ascending order), a scale of x's type per row and group of 32, 64 or 128 k, and a zero of 0 to 128 per row and group (8 for all without a table).
//
// Exactness: code - zero is a whole number from -128 to 15 and exact in bfloat16, and so is 128 + zero, by way of which it is made (beyond 128 it would
// not be). A group's products x (code - zero) are summed in 32-bit,
// the sum is multiplied by the group's scale in 32-bit, and the groups' sums are added in 32-bit; the result is rounded once. Nothing is
// rounded to fewer bits before that (a weight (code - zero) * scale rounded to bfloat16 would cost as much again as the output's rounding).
#include "linear4.cuh"
#include "mma_util.cuh"

// ------------------------------------------------------------------------------ bfloat16, eight tokens at once
// Bound by reading the codes once (and by the eleven instructions that widen a word of them, seven on a pipe of half rate). The rows are shared out evenly among the resident blocks (in fours), the k of a block's rows among its
// warps in stretches of 256: a warp keeps its stretch's tokens in registers as MMA operands and streams [16 rows, 256 k] pieces (2 KB, a
// 128-byte line of every row) through a ring of its own in shared memory, so no barrier stands in the loop; the warps' sums are added once per
// pass over the rows. A word of codes feeds two MMAs as the rows' operand; the k of the two operands are permuted alike, and so that an MMA's
// sixteen k lie in one group: thread t of a quad takes group / 32 consecutive words of the group at a time.
// One token of 21,504 x 4,096 (45 MB): 14.4 us, of which widening alone is 8; of 4,096 x 4,096 5.6 us.
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

template <int GROUP>
__global__ void __launch_bounds__(L4_WARPS * 32, 2) linear4_kernel(const unsigned* __restrict__ codes, const bf16* __restrict__ scales,
                                                                   const unsigned char* __restrict__ zeros, const bf16* x, long long ldx, void* y,
                                                                   long long ldy, int n, int out, int K, int passes, bool x_wide, bool s_wide,
                                                                   int epilogue, XieluParams act, bool y32) {
    typedef L4Piece<GROUP> P;
    constexpr int WORDS = GROUP / 32;                        // consecutive words a thread takes
    constexpr int S_EACH = (P::GROUPS * 8 + 31) / 32, Z_EACH = (P::GROUPS * 4 + 31) / 32;
    extern __shared__ __align__(128) unsigned char l4_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = l4_smem + (size_t)warp * L4_STAGES * P::BYTES;
    const int token0 = blockIdx.y * 8;
    const int stretches = (K + L4_KC - 1) / L4_KC, groups = K / GROUP;
    const int mine = warp < stretches ? (stretches - warp + L4_WARPS - 1) / L4_WARPS : 0;
    const int fours = (out + 3) >> 2;
    // Rows lane / 8 + 4 u of a piece: u turns one bit of the place of a 16-byte piece.
    const int place0 = l4_place(lane >> 3, lane & 7) * 16, place1 = l4_place((lane >> 3) + 4, lane & 7) * 16;
    const int read_at = g * 128 + l4_place(g, (t * WORDS) >> 2) * 16 + ((t * WORDS) & 3) * 4;
    bool waited = false;

#pragma unroll 1
    for (int pass = 0; pass < passes; ++pass) {
        const long long share = (long long)pass * gridDim.x + blockIdx.x, shares = (long long)passes * gridDim.x;
        const int r0 = 4 * (int)(fours * share / shares), r1 = min(out, 4 * (int)(fours * (share + 1) / shares));
        const int tiles = (r1 - r0 + 15) >> 4;
        // The pieces in the order of their use: the tiles of a stretch, stretch after stretch; each into the ring's next place. Addresses move
        // on by sums: `code` is this lane's first row and 16 bytes of the next piece, `scale` and `zero` its part of the scales and zeros.
        int next_m = 0, left = mine, next_at = 0, at = 0, next_word = warp * (L4_KC / 8) + 4 * (lane & 7), rows_left = r1 - r0 - (lane >> 3);
        const unsigned* code = codes + (size_t)(r0 + (lane >> 3)) * (K >> 3) + next_word;
        auto table_at = [&](auto* table, int e, int per, int wide) {                     // entry e of a stretch's `per` entries a group
            return table + (size_t)min((mine - left) * L4_WARPS * P::GROUPS + warp * P::GROUPS + e / per, groups - 1) * out + r0 + wide * (e % per);
        };
        const bf16* scale[S_EACH];
        const unsigned char* zero[Z_EACH];
        auto seek = [&] {
            if (!s_wide) return;
#pragma unroll
            for (int k = 0; k < S_EACH; ++k) scale[k] = table_at(scales, lane + 32 * k, 8, 2);
            if (zeros == nullptr) return;
#pragma unroll
            for (int k = 0; k < Z_EACH; ++k) zero[k] = table_at(zeros, lane + 32 * k, 4, 4);
        };
        auto issue = [&]() {
            if (left > 0) {
                unsigned char* dst = ring + next_at;
                const unsigned to = smem_u32(dst) + (lane >> 3) * 128;
                const bool inside = next_word * 8 < K;
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (inside && 4 * u < rows_left) cp_async16(to + u * 512 + ((u & 1) ? place1 : place0), code + (size_t)(4 * u) * (K >> 3));
                if (s_wide) {
#pragma unroll
                    for (int k = 0; k < S_EACH; ++k) {
                        const int e = lane + 32 * k;
                        if (e < P::GROUPS * 8 && 16 * next_m + 2 * (e & 7) < r1 - r0) cp_async4(smem_u32(dst + P::CODES + e * 4), scale[k] + 16 * next_m);
                    }
                    if (zeros != nullptr) {
#pragma unroll
                        for (int k = 0; k < Z_EACH; ++k) {
                            const int e = lane + 32 * k;
                            if (e < P::GROUPS * 4 && 16 * next_m + 4 * (e & 3) < r1 - r0)
                                cp_async4(smem_u32(dst + P::CODES + P::SCALES + e * 4), zero[k] + 16 * next_m);
                        }
                    }
                } else {
                    for (int e = lane; e < P::GROUPS * 16; e += 32) {
                        const bf16* from = table_at(scales, e, 16, 1) + 16 * next_m;
                        if (16 * next_m + (e & 15) < r1 - r0) {
                            reinterpret_cast<bf16*>(dst + P::CODES)[e] = *from;
                            if (zeros != nullptr) dst[P::CODES + P::SCALES + e] = *(table_at(zeros, e, 16, 1) + 16 * next_m);
                        }
                    }
                }
                next_at = next_at == (L4_STAGES - 1) * P::BYTES ? 0 : next_at + P::BYTES;
                code += (size_t)16 * (K >> 3);
                rows_left -= 16;
                if (++next_m == tiles) {
                    next_m = 0;
                    --left;
                    next_word += L4_WARPS * (L4_KC / 8);
                    code += L4_WARPS * (L4_KC / 8) - (size_t)(16 * tiles) * (K >> 3);
                    rows_left += 16 * tiles;
                    seek();
                }
            }
            cp_async_commit();
        };
        seek();
#pragma unroll
        for (int i = 0; i < L4_STAGES - 1; ++i) issue();
        if (!waited) { pdl_enter(); waited = true; }         // codes and scales are no result of a step: only the tokens are waited for

        float acc[L4_MT][4];
#pragma unroll
        for (int m = 0; m < L4_MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][i] = 0.f;

        for (int s = 0; s < mine; ++s) {
            // The stretch's tokens: word w of the thread's words holds eight k of token g.
            uint4 xv[8];
            {
                const int token = token0 + g;
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
                    xv[w] = v;
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
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
                    unsigned lo[WORDS], hi[WORDS];
                    {
                        // This group's words of rows g and g + 8: GROUP / 2 bytes a row from byte q * GROUP / 2, thread t's from t * 4 WORDS on.
                        const unsigned* a = reinterpret_cast<const unsigned*>(src + (read_at ^ (q * (GROUP / 32) * 16)));
                        const unsigned* b = a + 8 * 32;
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
                    unsigned base_lo = 0x43084308u, base_hi = base_lo;                   // 128 + zero, twice
                    if (zeros != nullptr) {
                        base_lo = src[P::CODES + P::SCALES + q * 16 + g] * 0x00010001u + 0x43004300u;
                        base_hi = src[P::CODES + P::SCALES + q * 16 + g + 8] * 0x00010001u + 0x43004300u;
                    }
#pragma unroll
                    for (int w = 0; w < WORDS; ++w) {
                        const unsigned a[2][4] = {{widen_pair(lo[w], 0, base_lo), widen_pair(hi[w], 0, base_hi), widen_pair(lo[w], 4, base_lo),
                                                   widen_pair(hi[w], 4, base_hi)},
                                                  {widen_pair(lo[w], 8, base_lo), widen_pair(hi[w], 8, base_hi), widen_pair(lo[w], 12, base_lo),
                                                   widen_pair(hi[w], 12, base_hi)}};
                        mma16816(part, a[0], xv[q * WORDS + w].x, xv[q * WORDS + w].y);
                        mma16816(part, a[1], xv[q * WORDS + w].z, xv[q * WORDS + w].w);
                    }
                    const float s_lo = to_f32(sc[q * 16 + g]), s_hi = to_f32(sc[q * 16 + g + 8]);
                    acc[m][0] = fmaf(s_lo, part[0], acc[m][0]);
                    acc[m][1] = fmaf(s_lo, part[1], acc[m][1]);
                    acc[m][2] = fmaf(s_hi, part[2], acc[m][2]);
                    acc[m][3] = fmaf(s_hi, part[3], acc[m][3]);
                }
            }
        }
        // The warps' sums in ascending order of the warps, through the ring's memory.
        cp_async_wait<0>();
        __syncthreads();
        float* red = reinterpret_cast<float*>(l4_smem);      // [warp][tile][lane][4]
#pragma unroll
        for (int m = 0; m < L4_MT; ++m)
            if (m < tiles)
                *reinterpret_cast<float4*>(red + (((size_t)warp * L4_MT + m) * 32 + lane) * 4) = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
        __syncthreads();
        const int used = min(L4_WARPS, stretches);
        for (int e = threadIdx.x; e < tiles * 128; e += L4_WARPS * 32) {
            const int l = (e & 127) >> 2, c = e & 3, m = e >> 7;
            const int row = r0 + 16 * m + (l >> 2) + ((c & 2) ? 8 : 0), token = token0 + 2 * (l & 3) + (c & 1);
            if (row >= r1 || token >= n) continue;
            float sum = 0.f;
            for (int w = 0; w < used; ++w) sum += red[(((size_t)w * L4_MT + m) * 32 + l) * 4 + c];
            store_result(y, ldy, token, row, sum, epilogue, act, y32);
        }
        __syncthreads();                                     // the ring is filled again
    }
}

// Blocks and passes over a block's rows, of the fours of rows that `out` makes.
static void linear4_grid(int out, int& blocks, int& passes) {
    const int fours = (out + 3) / 4, slots = 2 * ti_sm_count();
    blocks = fours < slots ? fours : slots;
    passes = (fours + blocks * (4 * L4_MT) - 1) / (blocks * (4 * L4_MT));
}

template <int GROUP>
static int launch_linear4(const void* codes, const void* scales, const void* zeros, const void* x, long long ldx, void* y, long long ldy, int n,
                          int out, int K, int epilogue, XieluParams act, bool y32, cudaStream_t stream) {
    typedef L4Piece<GROUP> P;
    constexpr size_t ring = (size_t)L4_WARPS * L4_STAGES * P::BYTES, red = (size_t)L4_WARPS * L4_MT * 128 * sizeof(float);
    constexpr size_t smem = ring > red ? ring : red;
    static_assert(smem <= 113 * 1024, "two blocks per SM");
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(linear4_kernel<GROUP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return ti_fail("linear4: %s", cudaGetErrorString(e));
        configured = true;
    }
    int blocks, passes;
    linear4_grid(out, blocks, passes);
    const bool x_wide = aligned16(x) && ldx % 8 == 0;
    const bool s_wide = out % 4 == 0 && (uintptr_t)scales % 4 == 0 && (uintptr_t)zeros % 4 == 0;
    ti_launch(linear4_kernel<GROUP>, dim3(blocks, (n + 7) / 8), dim3(L4_WARPS * 32), smem, stream, (const unsigned*)codes,
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

// Which of the two bfloat16 kernels: eight tokens at a time, each time over all codes, or up to 32 tokens through shared memory (linear4_wide.cu), whose
// blocks take equal runs of units and need a second kernel to join shared tiles. The one that an estimate of its microseconds says is the faster. The
// estimates are fitted to 738 measured shapes (1 to 64 tokens, 100 to 131,072 rows, 128 to 28,672 k); on those and 160 others, what is chosen takes 1.4 %
// more than the better of the two on average, and more than a tenth more in one of twenty.
//   Eights: the rounds of blocks, each with a start, a time per k and tile of 16 rows that a block takes one after the other, its tokens read once a
//   pass (twice as dear where two blocks share an SM), an end per pass, and, where rows are no whole fours, scales by loads that every piece waits for.
//   Shared memory: a start, the units an SM takes, wider stages from 17 tokens on, and for runs that cut items the join and its parts.
// us, eights / shared memory: 1 token x 21,504 x 4,096 14.6 / 17.1, x 28,672 x 4,096 22.4 / 20.4, x 8,192 x 8,192 13.1 / 13.9, x 10,240 x 8,192 17.3 / 16.1,
// x 12,856 x 8,000 18.2 / 19.8, x 131,072 x 4,096 83.6 / 68.1; 8 tokens x 1,024 x 6,144 10.2 / 6.7, x 4,096 x 4,096 6.7 / 7.7, x 4,096 x 8,192 12.1 / 9.9; 16 x
// 1,024 x 512 5.5 / 4.4, x 512 x 512 2.7 / 4.3; 32 x 320 x 2,048 6.3 / 6.4, x 256 x 2,048 4.1 / 6.3; 48 x 1,024 x 256 13.7 / 4.7; 7 x 27,221 x 224 17.1 / 3.8.
extern "C" int ti_linear4_shared(int n, int out, int K) {
    if (n <= 0 || out <= 0 || K <= 0) return 0;
    const int sms = ti_sm_count(), tokens = n <= 8 ? 8 : n <= 16 ? 16 : 32;
    const long long steps = (K + L4_KC - 1) / L4_KC, row_tiles = (out + 255) / 256;
    int blocks, passes;
    linear4_grid(out, blocks, passes);
    const long long resident = (long long)blocks * ((n + 7) / 8), rounds = (resident + 2 * sms - 1) / (2 * sms);
    const long long share = ((out + 3) / 4 + (long long)passes * blocks - 1) / ((long long)passes * blocks);
    const double tiles = (double)passes * ((share + 3) / 4), k = steps * L4_KC / 1000.0, dense = resident > sms ? 2 : 1;
    const double eighths = (n < 8 ? n : 8) / 8.0;
    double eights = 1.9 + 3.5 * (passes - 1) + k * (0.46 * tiles + passes * dense * (0.17 + 0.2 * eighths * eighths));
    if (out % 4 != 0) eights += 0.6 * ((steps + L4_WARPS - 1) / L4_WARPS) * tiles;
    eights *= rounds;

    const long long units = row_tiles * ((n + tokens - 1) / tokens) * steps;
    double shared = 2.4 + 1.45 * units / sms + (tokens == 32 ? 1.55 : 0.0);
    if (linear4_cuts_items(units, steps)) {
        const double parts = sms / (double)row_tiles;
        shared += 1.4 + 0.095 * (steps < parts ? steps : parts);
    }
    return shared < eights;
}

// codes [out, K / 8] words, scales [K / group, out] of x's type, zeros [K / group, out] bytes or null; y [n, ldy] of x's type, or 32-bit sums
// that are not rounded (epilogue 2). `parts`: ti_linear4_parts(n, out, K) bytes (null where that is 0); `status`: the word of bounded waits.
extern "C" int ti_linear4(void* y, long long ldy, const void* x, long long ldx, const void* codes, const void* scales, const void* zeros, int n,
                          int out, int K, int group, int epilogue, float alpha_p, float alpha_n, float beta, float eps, int dtype, void* parts,
                          int* status, cudaStream_t stream) {
    if (n == 0 || out == 0) return 0;
    TI_REQUIRE(n > 0 && out > 0 && K > 0, "linear4: %d tokens, %d x %d", n, out, K);
    TI_REQUIRE(group == 32 || group == 64 || group == 128, "linear4: groups of %d (32, 64 or 128)", group);
    TI_REQUIRE(K % group == 0, "linear4: %d inputs are not whole groups of %d", K, group);
    TI_REQUIRE(aligned16(codes), "linear4: the codes must be 16-byte aligned");
    TI_REQUIRE(dtype == TI_F32 || dtype == TI_BF16, "linear4: unknown element type code %d", dtype);
    TI_REQUIRE(linear4_epilogue_known(epilogue), "linear4: unknown epilogue %d", epilogue);
    const XieluParams act{alpha_p, alpha_n, beta, eps};
    if (dtype == TI_F32) {
        TI_REQUIRE((n + L4F_TOKENS - 1) / L4F_TOKENS <= 65535, "linear4: %d tokens in one launch", n);
        const bool x_wide = aligned16(x) && ldx % 4 == 0;
        ti_launch(linear4_f32_kernel, dim3((out + L4F_ROWS - 1) / L4F_ROWS, (n + L4F_TOKENS - 1) / L4F_TOKENS), dim3(L4F_WARPS * 32), 0, stream,
                  (const unsigned*)codes, (const float*)scales, (const unsigned char*)zeros, (const float*)x, ldx, (float*)y, ldy, n, out, K, group,
                  x_wide, epilogue, act);
        return ti_check_launch("linear4");
    }
    if (n == 1) ldx = K;                                     // a single row's pitch means nothing
    // Rows of x that TMA does not take (unaligned ones, ones that overlap) go eight tokens at a time, too.
    if (ti_linear4_shared(n, out, K) && aligned16(x) && ldx % 8 == 0 && ldx >= K)
        return linear4_wide(y, ldy, x, ldx, codes, scales, zeros, n, out, K, group, epilogue, act, parts, status, stream);
    TI_REQUIRE((n + 7) / 8 <= 65535, "linear4: %d tokens in one launch", n);
    const bool y32 = epilogue == L4_EPI_F32_OUT;
    if (group == 32) return launch_linear4<32>(codes, scales, zeros, x, ldx, y, ldy, n, out, K, epilogue, act, y32, stream);
    if (group == 64) return launch_linear4<64>(codes, scales, zeros, x, ldx, y, ldy, n, out, K, epilogue, act, y32, stream);
    return launch_linear4<128>(codes, scales, zeros, x, ldx, y, ldy, n, out, K, epilogue, act, y32, stream);
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
