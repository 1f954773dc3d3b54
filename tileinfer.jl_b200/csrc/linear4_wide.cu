// Products with weights of 4 bits whose tokens come through shared memory, up to 32 at once: see linear4.cu for what is computed.
//
// A stage holds [256 rows, 256 k] of codes, the tokens of these k (both by TMA, in swizzled rows of 128 bytes) and the rows' scales and zeros; one warp
// asks for them (a thread of a computing warp that did so held up its warp and then all), sixteen take 16 rows each and go through the stages on their
// own: no barrier of the block stands in the loop. A lane's word of codes (8 consecutive k of a row) feeds two MMAs as the rows' operand, 32 consecutive k at a
// time, so an MMA's k lie in one group; the k of both operands are permuted alike. Rows and tokens stand in the MMAs in bit-reversed order, which
// spreads every phase of a swizzled read over all banks.
//
// What bounds it: reading the codes once (up to 16 tokens: 131,072 x 4,096 without the arithmetic takes 51 us for 8 tokens, with it 70), then mma.sync: 8 cycles a
// scheduler for 16 rows x 16 k x 8 tokens, 10 beside other instructions, and 26 for the codes' eleven instructions a word, seven of them on a pipe of half
// rate. 131,072 x 4,096: 70 us for 8 tokens, 82 for 16, 118 for 32, 222 for 64. Other forms took longer: weights widened into tensor memory as tcgen05.mma's operand with a
// group's sum read back from there (165 us for 16, 245 for 64), the same with codes as float16 of 2^-24 (five instructions a word, tokens brought to
// float16 by a kernel ahead: 108 and 419), float16 with mma.sync (66 us for 8 tokens, but 137 for 32 and a launch more on small weights), e4m3
// (its operands are widened again by 20 cycles an MMA), eight warps of 32 rows (the tokens read half as often: 137 for 32), 64 tokens at once (271).
//
// The units of work, [256 rows, 256 k], are numbered along k, then over the rows (and the tokens in thirty-twos), and every SM takes an equal run of them
// (even_runs.cuh). Parts of a tile that several blocks share go to the work space; a second kernel adds them in the blocks' order.
#include "linear4.cuh"
#include "even_runs.cuh"
#include "mma_util.cuh"
#include "tcgen05.cuh"
#include "tensor_map.h"

namespace {
using namespace tc;

constexpr int KC = 256, ROWS = 256, CODES = ROWS * KC / 2;

// Tokens in eights (NT); sixteen computing warps of 16 rows, and the one that asks.
template <int NT, int GROUP> struct Shape {
    static constexpr int N = 8 * NT, WARPS = ROWS / 16, THREADS = 32 * (WARPS + 1), GROUPS = KC / GROUP;
    static constexpr int X = N * KC * 2;
    // Per group the 16-byte pieces of memory that hold its scales (zeros), wherever they begin: the place of the first in its piece is what its address says.
    static constexpr int S_ROW = 2 * ROWS + 16, Z_ROW = ROWS + 16, SCALES = GROUPS * (S_ROW + Z_ROW);
    static constexpr int BYTES = (CODES + X + SCALES + 1023) / 1024 * 1024;
    // A warp's results on their way out, sixteen tokens of 16 rows at a time (24 apart: no two lanes of a write meet in a bank).
    static constexpr int OUT_ROW = 24, OUT_EIGHTS = NT < 2 ? NT : 2, OUT = OUT_EIGHTS * 8 * OUT_ROW * 4, OUTS = WARPS * OUT;
    static constexpr int FIT = (226 * 1024 - OUTS) / BYTES, STAGES = FIT > 5 ? 5 : FIT;
};

struct Args {
    const bf16* scales;
    const unsigned char* zeros;
    void* y;
    long long ldy;
    float* parts;                                            // [slot][N tokens][256 rows]
    int* status;
    int n, out, groups, steps, chunks;                       // steps of 256 k; chunks of N tokens
    unsigned units;
    int epilogue;
    XieluParams act;
    bool y32;
};

// Both addresses and the size are multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(unsigned dst, uintptr_t src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// MMAs that the compiler may move (their results are functions of their operands), so that the next words' loads and widening stand between them.
__device__ __forceinline__ void mma_more(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ int reversed3(int g) { return ((g & 1) << 2) | (g & 2) | ((g & 4) >> 2); }

template <int NT, int GROUP>
__global__ void __launch_bounds__(Shape<NT, GROUP>::THREADS, 1) linear4_wide_kernel(const __grid_constant__ CUtensorMap map_codes,
                                                                                    const __grid_constant__ CUtensorMap map_x, const Args p) {
    typedef Shape<NT, GROUP> S;
    constexpr int N = S::N;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* tiles = smem_dyn + ((1024u - (smem_addr(smem_dyn) & 1023u)) & 1023u);
    const unsigned stages = smem_addr(tiles);
    __shared__ __align__(8) unsigned long long bars[2 * S::STAGES];
    const unsigned full0 = smem_addr(bars), empty0 = full0 + 8 * S::STAGES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = reversed3(lane >> 2), t = lane & 3;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, S::WARPS); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const unsigned steps = p.steps;
    const Runs runs(p.units, gridDim.x);
    const unsigned lo = runs.low(blockIdx.x), hi = runs.low(blockIdx.x + 1);
    // Item = 256 rows x a chunk of tokens; the chunks of one stretch of rows follow one another, so its codes are read from memory once.
    pdl_launch_dependents();
    if (warp == S::WARPS) {
        // ---------------------------------------------------------------- asking: a lane a copy
        // A group's scales and zeros come as the 16-byte pieces that hold them: whole ones, none beyond the last with a byte of the tables.
        const int q = lane & 7;                              // lanes 0 to 7: codes and tokens, 8 to 15: scales, 16 to 23: zeros of group q
        const bool is_scale = (lane >> 3) == 1 && q < S::GROUPS, is_zero = (lane >> 3) == 2 && q < S::GROUPS && p.zeros != nullptr;
        const unsigned char* table = is_zero ? p.zeros : reinterpret_cast<const unsigned char*>(p.scales);
        const unsigned width = is_zero ? 1 : 2, most = is_zero ? S::Z_ROW : S::S_ROW;
        const unsigned to = CODES + S::X + (is_zero ? S::GROUPS * S::S_ROW + q * S::Z_ROW : q * S::S_ROW);
        const uintptr_t end = ((uintptr_t)table + (size_t)p.groups * p.out * width + 15) & ~(uintptr_t)15;
        unsigned item = lo / steps, phase = 0;
        int step = lo - item * steps, slot = 0;
        int row = item / p.chunks * ROWS, token = item % p.chunks * N;
        bool waited = false;
        for (unsigned u = lo; u < hi; ++u) {
            const unsigned bar = full0 + 8 * slot, dst = stages + slot * S::BYTES;
            if (u >= lo + S::STAGES && !__all_sync(0xffffffffu, mbar_wait(empty0 + 8 * slot, phase ^ 1, p.status, 17))) break;
            unsigned bytes = 0;
            uintptr_t from = 0;
            if ((is_scale || is_zero) && step * S::GROUPS + q < p.groups) {
                from = ((uintptr_t)table + ((size_t)(step * S::GROUPS + q) * p.out + row) * width) & ~(uintptr_t)15;
                bytes = end - from < most ? (unsigned)(end - from) : most;
            }
            const unsigned all = __reduce_add_sync(0xffffffffu, bytes);
            if (lane == 0) mbar_expect_tx(bar, CODES + N * KC * 2 + all);
            __syncwarp();
            if (lane == 0) tma_load_2d(dst, &map_codes, step * (KC / 4), row, bar);
            if (bytes) bulk_load(dst + to, from, bytes, bar);
            // Weights are no result of a step: the first stages' are asked for before the wait for the kernel before.
            if (waited && lane >= 1 && lane <= KC / 64)
                tma_load_2d(dst + CODES + (lane - 1) * (S::X / 4), &map_x, step * KC + (lane - 1) * 64, token, bar);
            if (!waited && (u + 1 == hi || u + 1 == lo + S::STAGES)) {
                pdl_wait();
                waited = true;
                if (lane >= 1 && lane <= KC / 64) {
                    unsigned at = lo / steps;
                    int s = lo - at * steps;
                    for (unsigned v = lo; v <= u; ++v) {
                        tma_load_2d(stages + (v - lo) * S::BYTES + CODES + (lane - 1) * (S::X / 4), &map_x, s * KC + (lane - 1) * 64, at % p.chunks * N, full0 + 8 * (v - lo));
                        if (++s == (int)steps) { s = 0; ++at; }
                    }
                }
            }
            if (++slot == S::STAGES) { slot = 0; phase ^= 1; }
            if (++step == (int)steps) {
                step = 0;
                ++item;
                row = item / p.chunks * ROWS;
                token = item % p.chunks * N;
            }
        }
        if (*reinterpret_cast<volatile int*>(p.status) != 0) drain_after_timeout();      // a wait ran out: let what is in flight land
        return;
    }
    pdl_wait();                                              // y may still be read by the kernel before

    float acc[NT][4];
    auto clear = [&] {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[j][c] = 0.f;
    };
    clear();
    unsigned item = lo / steps;
    int step = lo - item * steps, stage = 0, row0 = item / p.chunks * ROWS;
    unsigned phase = 0;
    bool ok = true;
    // A lane's places in a stage at its first 32 k: the swizzle turns bits 4 to 6 by the row's lowest three (bit-reversed order: g).
    const unsigned code_at = (warp * 16 + g) * 128 + (g << 4) + 4 * t, x_at = CODES + g * 128 + ((t ^ g) << 4);
    for (unsigned u = lo; u < hi; ++u) {
        ok = __all_sync(0xffffffffu, mbar_wait(full0 + 8 * stage, phase, p.status, 16));
        if (!ok) break;
        const unsigned char* src = tiles + stage * S::BYTES;
        const int here = min(S::GROUPS, p.groups - step * S::GROUPS);
        // Where the step's scales and zeros begin in their first pieces: low bits of addresses, moving on by a row of the tables a group.
        unsigned s_low = (unsigned)(uintptr_t)p.scales + 2u * ((unsigned)(step * S::GROUPS) * (unsigned)p.out + (unsigned)row0);
        unsigned z_low = (unsigned)(uintptr_t)p.zeros + (unsigned)(step * S::GROUPS) * (unsigned)p.out + (unsigned)row0;
        const unsigned char *scales = src + CODES + S::X + 2 * (warp * 16 + g), *zeros = src + CODES + S::X + S::GROUPS * S::S_ROW + warp * 16 + g;
        unsigned chunk = 0;                                  // 32 k: a 16-byte piece of a row of codes, four of a row of tokens
        // The groups of a step side by side: 131,072 x 4,096 and 8 tokens 79 us in turn, 72 so; 16 tokens 94 and 86.
#pragma unroll
        for (int q = 0; q < S::GROUPS; ++q) {
            if (q >= here) break;
            float part[NT][4];
            unsigned base[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const unsigned z = p.zeros != nullptr ? zeros[(z_low & 15) + 8 * h] : 8u;
                base[h] = z * 0x00010001u + 0x43004300u;     // 128 + zero, twice
            }
            auto block = [&](bool first) {
                const unsigned char *rows = src + (code_at ^ (chunk << 4)), *x = src + (x_at ^ ((chunk & 1) << 6)) + (chunk >> 1) * (S::X / 4);
                uint4 b[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j) b[j] = *reinterpret_cast<const uint4*>(x + j * 1024);
                const unsigned lo_w = *reinterpret_cast<const unsigned*>(rows), hi_w = *reinterpret_cast<const unsigned*>(rows + 1024);
                const unsigned a0[4] = {widen_pair(lo_w, 0, base[0]), widen_pair(hi_w, 0, base[1]), widen_pair(lo_w, 4, base[0]), widen_pair(hi_w, 4, base[1])};
                const unsigned a1[4] = {widen_pair(lo_w, 8, base[0]), widen_pair(hi_w, 8, base[1]), widen_pair(lo_w, 12, base[0]), widen_pair(hi_w, 12, base[1])};
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if (first) mma_first(part[j], a0, b[j].x, b[j].y);
                    else mma_more(part[j], a0, b[j].x, b[j].y);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) mma_more(part[j], a1, b[j].z, b[j].w);
                ++chunk;
            };
            block(true);
#pragma unroll
            for (int i = 1; i < GROUP / 32; ++i) block(false);
            const float s_lo = to_f32(*reinterpret_cast<const bf16*>(scales + (s_low & 15))), s_hi = to_f32(*reinterpret_cast<const bf16*>(scales + (s_low & 15) + 16));
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                acc[j][0] = fmaf(s_lo, part[j][0], acc[j][0]);
                acc[j][1] = fmaf(s_lo, part[j][1], acc[j][1]);
                acc[j][2] = fmaf(s_hi, part[j][2], acc[j][2]);
                acc[j][3] = fmaf(s_hi, part[j][3], acc[j][3]);
            }
            scales += S::S_ROW; zeros += S::Z_ROW;
            s_low += 2u * (unsigned)p.out; z_low += (unsigned)p.out;
        }
        fence_async_smem();                                  // the stage's next copies are another proxy's than these reads
        __syncwarp();
        if (lane == 0) mbar_arrive(empty0 + 8 * stage);
        if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
        if (step + 1 == (int)steps || u + 1 == hi) {              // the item's end, or this run's
            const unsigned u0 = item * steps;
            const bool whole = u0 >= lo && u0 + steps <= hi;
            const int token0 = item % p.chunks * N;
            float* part = p.parts + (size_t)runs.slot(blockIdx.x, u0) * N * ROWS;
            if (!whole) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        // A thread's columns 2 t and 2 t + 1 are tokens in bit-reversed order, its rows g and g + 8.
                        const int r = warp * 16 + g + ((c & 2) ? 8 : 0), token = 8 * j + reversed3(2 * t + (c & 1));
                        if (token0 + token < p.n && row0 + r < p.out) part[(size_t)token * ROWS + r] = acc[j][c];
                    }
            } else {
                // Through shared memory to a loop: the code of all epilogues once per sixteen tokens, not once per result (131,072 x 4,096, 64 tokens: 274 us
                // with it unrolled, 244 so).
                float* mine = reinterpret_cast<float*>(tiles + S::STAGES * S::BYTES + warp * S::OUT);
                const int row = warp * 16 + (lane & 15), tokens = min(N, p.n - token0);
#pragma unroll
                for (int j0 = 0; j0 < NT; j0 += S::OUT_EIGHTS) {
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < S::OUT_EIGHTS; ++j)
#pragma unroll
                        for (int c = 0; c < 4; ++c) mine[(8 * j + reversed3(2 * t + (c & 1))) * S::OUT_ROW + g + ((c & 2) ? 8 : 0)] = acc[j0 + j][c];
                    __syncwarp();
                    const int first = 8 * j0, last = min(first + 8 * S::OUT_EIGHTS, tokens);
                    if (row0 + row >= p.out) continue;
#pragma unroll 1
                    for (int e = first + (lane >> 4); e < last; e += 2)
                        store_result(p.y, p.ldy, token0 + e, row0 + row, mine[(e - first) * S::OUT_ROW + (lane & 15)], p.epilogue, p.act, p.y32);
                }
            }
            clear();
        }
        if (++step == (int)steps) { step = 0; ++item; row0 = item / p.chunks * ROWS; }
    }
}

// The parts of 256 rows that several blocks share, in the blocks' order: blocks of (128 rows, two tokens), a thread a row: small enough to stand beside
// a product's block (2,048 x 9,216 and 8 tokens 8 us; in blocks of 512 threads, which find no registers beside it, 10.7).
constexpr int JOIN_TOKENS = 2, JOIN_ROWS = 128;
__global__ void __launch_bounds__(JOIN_ROWS) linear4_join_kernel(const Args p, int N, int G, bool by_cuts) {
    const int r = (blockIdx.x & 1) * JOIN_ROWS + threadIdx.x, which = blockIdx.x >> 1;
    const Runs runs(p.units, G);
    // The items, or, where those are more, the cuts between runs (131,072 x 4,096 and 64 tokens 251 us, 222 by cuts): a cut's item is that cut's if no cut
    // before lies in it.
    unsigned tile = which, chunk = blockIdx.z;
    if (by_cuts) {
        const unsigned cut = runs.low(which + 1) / p.steps;
        tile = cut / p.chunks;
        chunk = cut - tile * p.chunks;
    }
    const unsigned u0 = (tile * p.chunks + chunk) * p.steps, c0 = runs.owner(u0), c1 = runs.owner(u0 + p.steps - 1);
    const int row = tile * ROWS + r, token0 = chunk * N, token = token0 + blockIdx.y * JOIN_TOKENS;
    pdl_enter();
    if (c0 == c1 || (by_cuts && c0 != (unsigned)which) || row >= p.out || token >= p.n) return;
    const float* part = p.parts + (size_t)(token - token0) * ROWS + r;
    float s0 = 0.f, s1 = 0.f;
    for (unsigned c = c0; c <= c1; c += 6) {
        float a[6], b[6];
#pragma unroll
        for (int k = 0; k < 6; ++k) {
            const bool ok = c + k <= c1;
            const float* src = part + (size_t)runs.slot(ok ? c + k : c1, u0) * N * ROWS;
            a[k] = ok && token < p.n ? __ldcg(src) : 0.f;
            b[k] = ok && token + 1 < p.n ? __ldcg(src + ROWS) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 6; ++k) { s0 += a[k]; s1 += b[k]; }
    }
    if (token < p.n) store_result(p.y, p.ldy, token, row, s0, p.epilogue, p.act, p.y32);
    if (token + 1 < p.n) store_result(p.y, p.ldy, token + 1, row, s1, p.epilogue, p.act, p.y32);
}

int tokens_at_once(int n) { return n <= 8 ? 8 : n <= 16 ? 16 : 32; }

template <int NT, int GROUP> int launch(const CUtensorMap& codes, const CUtensorMap& x, const Args& a, cudaStream_t stream) {
    typedef Shape<NT, GROUP> S;
    constexpr size_t smem = (size_t)S::STAGES * S::BYTES + S::OUTS + 1024;
    static_assert(S::STAGES >= 3, "stages");
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(linear4_wide_kernel<NT, GROUP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return ti_fail("linear4_wide: %s", cudaGetErrorString(e));
        configured = true;
    }
    const int blocks = (int)a.units < ti_sm_count() ? (int)a.units : ti_sm_count();
    ti_launch(linear4_wide_kernel<NT, GROUP>, dim3(blocks), dim3(S::THREADS), smem, stream, codes, x, a);
    if (int rc = ti_check_launch("linear4_wide")) return rc;
    if (!linear4_cuts_items(a.units, a.steps)) return 0;     // every run ends with an item: no parts
    const int tiles = (a.out + ROWS - 1) / ROWS;
    const bool by_cuts = (long long)tiles * a.chunks > blocks - 1 || a.chunks > 65535;
    ti_launch(linear4_join_kernel, dim3(2 * (by_cuts ? blocks - 1 : tiles), ((a.n < 8 * NT ? a.n : 8 * NT) + JOIN_TOKENS - 1) / JOIN_TOKENS, by_cuts ? 1 : a.chunks),
              dim3(JOIN_ROWS), 0, stream, a, 8 * NT, blocks, by_cuts);
    return ti_check_launch("linear4_join");
}

}  // namespace

// Bytes of the work space for parts: 0 where the product takes none.
extern "C" long long ti_linear4_parts(int n, int out, int K) {
    return ti_linear4_shared(n, out, K) ? 2LL * ti_sm_count() * tokens_at_once(n) * ROWS * 4 : 0;
}

// Kernels of a product whose rows TMA takes: two where it goes through shared memory and leaves parts to join.
extern "C" int ti_linear4_kernels(int n, int out, int K) {
    if (!ti_linear4_shared(n, out, K)) return 1;
    const long long steps = (K + KC - 1) / KC, N = tokens_at_once(n);
    return linear4_cuts_items((long long)((out + ROWS - 1) / ROWS) * ((n + N - 1) / N) * steps, steps) ? 2 : 1;
}

int linear4_wide(void* y, long long ldy, const void* x, long long ldx, const void* codes, const void* scales, const void* zeros, int n, int out, int K,
                 int group, int epilogue, XieluParams act, void* parts, int* status, cudaStream_t stream) {
    TI_REQUIRE(parts != nullptr && status != nullptr, "linear4: work space missing");
    TI_REQUIRE(aligned16(parts), "linear4: the work space must be 16-byte aligned");
    const int N = tokens_at_once(n);
    CUtensorMap map_codes, map_x;
    {   // The codes as [out, K / 4] numbers of 16 bits, moved as they are.
        const unsigned long long dims[2] = {(unsigned long long)K / 4, (unsigned long long)out}, strides[1] = {(unsigned long long)K / 2};
        const unsigned box[2] = {KC / 4, ROWS};
        if (int rc = ti_tensor_map_bf16(&map_codes, codes, 2, dims, strides, box, true)) return rc;
        const unsigned long long x_dims[2] = {(unsigned long long)K, (unsigned long long)n}, x_strides[1] = {(unsigned long long)ldx * 2};
        const unsigned x_box[2] = {64, (unsigned)N};
        if (int rc = ti_tensor_map_bf16(&map_x, x, 2, x_dims, x_strides, x_box, true)) return rc;
    }
    Args a;
    a.scales = (const bf16*)scales; a.zeros = (const unsigned char*)zeros;
    a.y = y; a.ldy = ldy; a.parts = (float*)parts; a.status = status;
    a.n = n; a.out = out; a.groups = K / group; a.steps = (K + KC - 1) / KC; a.chunks = (n + N - 1) / N;
    const long long units = (long long)((out + ROWS - 1) / ROWS) * a.chunks * a.steps;
    TI_REQUIRE(units < (1LL << 31), "linear4: %d tokens x %d x %d are too many units of work", n, out, K);
    a.units = (unsigned)units;
    a.epilogue = epilogue; a.act = act; a.y32 = epilogue == L4_EPI_F32_OUT;
#define L4_GROUPS(nt)                                                  \
    if (group == 32) return launch<nt, 32>(map_codes, map_x, a, stream); \
    if (group == 64) return launch<nt, 64>(map_codes, map_x, a, stream); \
    return launch<nt, 128>(map_codes, map_x, a, stream);
    if (N == 8) { L4_GROUPS(1) }
    if (N == 16) { L4_GROUPS(2) }
    L4_GROUPS(4)
#undef L4_GROUPS
}
