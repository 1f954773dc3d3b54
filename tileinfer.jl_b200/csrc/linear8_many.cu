// Products of e4m3 codes for prompts: tiles of 256 tokens x 128 weight rows on SM pairs.
//
//   y[t, o] = sum_g sx[g, t] sw[g, o / 128] sum_{k in g} cx[t, k] cw[o, k]
//
// tcgen05.mma.cta_group::2 takes the tokens as rows: each block of a pair stages its own 128 tokens and half of the 128 weight rows, and its tensor memory
// receives its 128 tokens' sums. A step is two groups of 128 of k (48 KB a block); a group's sums stand in an accumulator of their own, and eight warps (two a
// quarter of the lanes, 64 columns each) add them, times sx sw, to 32-bit sums in registers: a thread has a token, so that sx sw is one number a group.
//
// Bound by the hand-overs: the tensor cores need 256 cycles a group and are busy for half of the time. By the clock, read in every warp of a block with one group
// a step, the issuing warp took 620 cycles a group (waits 100; the next step's question, four MMAs and a commit 350; its loop), the adding warps 650. What had
// taken the longest: a factor multiplied as soon as it was asked for (the adding warps waited for its loads; now a warp of its own brings factors), and waits for
// barriers that were over long since, 300 cycles each beside the MMAs (now asked one step ahead). A commit frees the stage and gives the sums over at once.
// 256 tokens of 4,096 x 21,504 69.6 -> 55.0 us, 2,048 of 21,504 x 4,096 221 -> 197 us (1,830 TFLOP/s; 230 us in a long loop, where the power limit lowers the clock). Tiles of 256 x 256 took the same time for the same work,
// one group a step 59.3 us, sixteen adding warps 63.5.
//
// Block 0 of the pair issues the MMAs; its `full` barriers count the bytes of both blocks' loads; commits arrive on both blocks' barriers; the partner's
// warps arrive on block 0's accumulator barriers. All waits are bounded.
#include "linear8.cuh"
#include "packed_f32.cuh"

namespace {
using namespace tc;

constexpr int BM = 128, BN = 128, KB = 128, HALF = BN / 2, EPI_WARPS = 8, THREADS = 96 + 32 * EPI_WARPS;
constexpr int A_BYTES = BM * KB, B_BYTES = BN / 2 * KB, STEP = 2, STAGE = STEP * (A_BYTES + B_BYTES);
constexpr int STAGES = 4, SLOTS = 2;                         // of operands; of sums: a step's
constexpr int AHEAD = STAGES - SLOTS;                        // steps whose factors are brought before their products are there
constexpr int OUT_COLS = 16, OUT = 32 * OUT_COLS * 4;        // a warp's results on their way out
constexpr int BYTES = STAGES * STAGE + EPI_WARPS * OUT + 1024;
static_assert(BYTES + STAGES * STEP * BM * 4 <= 226 * 1024 && SLOTS * STEP * BN <= 512, "shared and tensor memory");

struct Args {
    Linear8 p;
    int groups, steps, row_blocks, token_tiles, tiles;              // row_blocks: of 128 weight rows, as scales have them
};

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned in_block0(unsigned addr) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void arrive_block0(unsigned cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Into this block's shared memory; the bytes are counted on block 0's barrier.
__device__ __forceinline__ void load_pair(unsigned dst, const CUtensorMap* map, int x, int y, unsigned bar_cluster) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar_cluster) : "memory");
}
__device__ __forceinline__ void mma_pair(unsigned tmem_d, unsigned long long desc_a, unsigned long long desc_b, unsigned idesc, unsigned accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// One arrival on the barrier at this offset in both blocks when every MMA issued so far has completed.
__device__ __forceinline__ void commit_pair(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((unsigned short)3) : "memory");
}
// kind::f8f6f4: 32-bit sums of e4m3, both operands K-major, 256 x 128.
constexpr unsigned IDESC = (1u << 4) | ((unsigned)(BN >> 3) << 17) | ((unsigned)(2 * BM >> 4) << 24);

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
linear8_many_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Args a) {
    const Linear8& p = a.p;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* tiles = smem_dyn + ((1024u - (smem_addr(smem_dyn) & 1023u)) & 1023u);
    __shared__ __align__(8) unsigned long long bars[2 * STAGES + SLOTS];
    __shared__ unsigned s_tmem;
    __shared__ float s_factor[STAGES][STEP][BM];
    // done: a stage has been read, its sums are complete and their factors there.
    const unsigned full0 = smem_addr(bars), done0 = full0 + 8 * STAGES, free0 = done0 + 8 * STAGES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(done0 + 8 * s, 2); }
        for (int s = 0; s < SLOTS; ++s) mbar_init(free0 + 8 * s, 2 * EPI_WARPS);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(SLOTS * STEP * BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                          // the partner's barriers exist before anything arrives on them
    tc_fence_after();
    pdl_enter();
    const unsigned tmem = s_tmem;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    bool ok = true;

    if (warp == 0) {
        // ---------------------------------------------------------------- copies, in both blocks, one thread
        int stage = 0;
        unsigned phase = 0;
        bool ready = true;                                   // every stage is free at first
        for (int tile = pair; lane == 0 && ok && tile < a.tiles; tile += pairs) {
            const int token = tile % a.token_tiles * (2 * BM) + rank * BM, row = tile / a.token_tiles * BN + rank * (BN / 2);
            for (int step = 0; step < a.steps; ++step) {
                if (!ready) ok = mbar_wait(done0 + 8 * stage, phase ^ 1, p.status, 24);
                if (!ok) break;
                const int next = stage + 1 == STAGES ? 0 : stage + 1;
                const unsigned next_phase = next == 0 ? phase ^ 1 : phase;
                ready = mbar_test(done0 + 8 * next, next_phase ^ 1, true);
                if (rank == 0) mbar_expect_tx(full0 + 8 * stage, 2 * STAGE);
                const unsigned bar = in_block0(full0 + 8 * stage), to = smem_addr(tiles + stage * STAGE);
#pragma unroll
                for (int i = 0; i < STEP; ++i) {             // beyond the last group: zeros
                    load_pair(to + i * A_BYTES, &map_x, (step * STEP + i) * (KB / 2), token, bar);
                    load_pair(to + STEP * A_BYTES + i * B_BYTES, &map_w, (step * STEP + i) * (KB / 2), row, bar);
                }
                stage = next;
                phase = next_phase;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMAs: block 0, one thread of a warp that walks along
        if (rank == 0) {
            int stage = 0, slot = 0;
            unsigned phase = 0, slot_phase = 0;
            const unsigned long long first = smem_desc_sw128(smem_addr(tiles));
            // One lane asks for the operands, another for the accumulator.
            const bool asks = lane < 2;
            bool ready = false;
            for (int tile = pair; ok && tile < a.tiles; tile += pairs)
                for (int step = 0; step < a.steps; ++step) {
                    ok = warp_wait_after(ready, lane ? free0 + 8 * slot : full0 + 8 * stage, lane ? slot_phase ^ 1 : phase, asks, p.status, 25);
                    if (!ok) break;
                    tc_fence_after();
                    const unsigned long long dx = first + (unsigned)(stage * (STAGE >> 4)), dw = dx + (STEP * A_BYTES >> 4);
                    const unsigned to = tmem + slot * (STEP * BN), done = done0 + 8 * stage;
                    if (++stage == STAGES) { stage = 0; phase ^= 1; }
                    if (++slot == SLOTS) { slot = 0; slot_phase ^= 1; }
                    ready = mbar_test(lane ? free0 + 8 * slot : full0 + 8 * stage, lane ? slot_phase ^ 1 : phase, asks);
                    if (elected()) {
#pragma unroll
                        for (int i = 0; i < STEP; ++i)
#pragma unroll
                            for (int k = 0; k < KB / 32; ++k) mma_pair(to + i * BN, dx + i * (A_BYTES >> 4) + 2 * k, dw + i * (B_BYTES >> 4) + 2 * k, IDESC, k > 0);
                        commit_pair(done);
                    }
                    __syncwarp();
                }
        }
    } else if (warp == 2) {
        // ---------------------------------------------------------------- the factors sx sw of the block's tokens, LOADS steps ahead in registers (multiplied when they
        // are wanted: a product at once would wait for its loads), then AHEAD in shared memory: a place is written again when the products AHEAD steps before are
        // there, for which the sums of STAGES steps before had to have been read
        constexpr int LOADS = 2, V = BM / 32;
        int next_tile = pair, next_step = 0, at[V];
        float sx[LOADS][STEP][V], sw[LOADS][STEP];
        const float *from = nullptr, *from_w = nullptr;
        auto ask = [&](float (&x)[STEP][V], float (&w)[STEP]) {
            if (next_tile >= a.tiles) return;
            if (next_step == 0) {
                const int token0 = next_tile % a.token_tiles * (2 * BM) + rank * BM + lane;
#pragma unroll
                for (int i = 0; i < V; ++i) at[i] = min(token0 + 32 * i, p.n - 1);
                from = p.x_scales;
                from_w = p.scales + next_tile / a.token_tiles;
            }
#pragma unroll
            for (int j = 0; j < STEP; ++j) {
                const bool there = next_step * STEP + j < a.groups;              // products beyond the last group are zeros
                w[j] = there ? __ldg(from_w) : 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) x[j][i] = there ? __ldcg(from + at[i]) : 0.f;
                if (!there) continue;
                from += p.n;
                from_w += a.row_blocks;
            }
            if (++next_step == a.steps) { next_step = 0; next_tile += pairs; }
        };
#pragma unroll
        for (int j = 0; j < LOADS; ++j) ask(sx[j], sw[j]);
        const long long all = (long long)((a.tiles - pair + pairs - 1) / pairs) * a.steps;
        int place = 0, behind = STAGES - AHEAD;
        unsigned phase = 1;
        bool ready = true;
        for (long long s0 = 0; ok && s0 < all; s0 += LOADS) {
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                if (s0 + j >= all) break;
                ok = warp_wait_after(ready, done0 + 8 * behind, phase, lane == 0, p.status, 30);
                if (!ok) break;
                if (++behind == STAGES) { behind = 0; phase ^= 1; }
                ready = mbar_test(done0 + 8 * behind, phase, lane == 0);
#pragma unroll
                for (int h = 0; h < STEP; ++h)
#pragma unroll
                    for (int i = 0; i < V; ++i) s_factor[place][h][lane + 32 * i] = sx[j][h][i] * sw[j][h];
                ask(sx[j], sw[j]);
                __syncwarp();
                if (lane == 0) mbar_arrive(done0 + 8 * place);
                if (++place == STAGES) place = 0;
            }
        }
    } else {
        // ---------------------------------------------------------------- sums: a thread a token, 64 weight rows
        const int half = (warp - 3) >> 2, quarter = warp & 3;
        const unsigned columns = tmem + ((unsigned)(quarter * 32) << 16) + half * HALF, release0 = in_block0(free0);
        float* out = reinterpret_cast<float*>(tiles + STAGES * STAGE) + (warp - 3) * (OUT / 4);
        const bool y32 = p.epilogue == L4_EPI_F32_OUT, quads = linear8_quads(p), singles = !quads || (p.epilogue != L4_EPI_NONE && !y32);
        // 32 bytes at a time straight from the registers.
        const bool direct = (p.epilogue == L4_EPI_NONE && ((uintptr_t)p.y & 31) == 0 && p.ldy % 16 == 0) || (y32 && ((uintptr_t)p.y & 31) == 0 && p.ldy % 8 == 0);
        int slot = 0, stage = 0;
        unsigned phase = 0;
        bool ready = false;
        for (int tile = pair; ok && tile < a.tiles; tile += pairs) {
            const int token0 = tile % a.token_tiles * (2 * BM) + rank * BM + quarter * 32, token = min(token0 + lane, p.n - 1);
            const int row0 = tile / a.token_tiles * BN + half * HALF;
            f32x2 acc[HALF / 2];
#pragma unroll
            for (int c = 0; c < HALF / 2; ++c) acc[c] = 0ull;
            for (int step = 0; step < a.steps; ++step) {
                ok = warp_wait_after(ready, done0 + 8 * stage, phase, lane == 0, p.status, 27);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < STEP; ++i) {
                    unsigned r[2][32];
                    tmem_ld32(columns + (slot * STEP + i) * BN, r[0]);
                    tmem_ld32(columns + (slot * STEP + i) * BN + 32, r[1]);
                    float f = s_factor[stage][i][quarter * 32 + lane];
                    tmem_ld_wait();
                    if (i == STEP - 1) {
                        tc_fence_before();
                        f = __shfl_sync(0xffffffffu, f, lane);               // every lane's factor has been read, too, when lane 0 gives step and factors back
                        if (lane == 0) arrive_block0(release0 + 8 * slot);
                        if (++slot == SLOTS) slot = 0;
                        if (++stage == STAGES) { stage = 0; phase ^= 1; }
                        ready = mbar_test(done0 + 8 * stage, phase, lane == 0);
                    }
                    const f32x2 ff = pack2(f, f);
#pragma unroll
                    for (int c = 0; c < HALF / 2; ++c)
                        acc[c] = fma2(pack2(__uint_as_float(r[c / 16][2 * c % 32]), __uint_as_float(r[c / 16][2 * c % 32 + 1])), ff, acc[c]);
                }
            }
            if (!ok) break;
            if (direct && row0 + HALF <= p.out) {
                if (token0 + lane >= p.n) continue;
                if (y32) {
                    float* to = (float*)p.y + (size_t)token * p.ldy + row0;
#pragma unroll
                    for (int c = 0; c < HALF / 2; c += 4)
                        asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(to + 2 * c), "l"(acc[c]), "l"(acc[c + 1]), "l"(acc[c + 2]), "l"(acc[c + 3]) : "memory");
                } else {
                    bf16* to = (bf16*)p.y + (size_t)token * p.ldy + row0;
#pragma unroll
                    for (int c = 0; c < HALF / 2; c += 8) {
                        unsigned v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            float lo, hi;
                            unpack2(acc[c + j], lo, hi);
                            const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
                            v[j] = *reinterpret_cast<const unsigned*>(&h);
                        }
                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + 2 * c), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                                     "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
                    }
                }
                continue;
            }
            // Others through shared memory, 16 columns at a time: [token][16-byte piece turned by the token], then four lanes a token; sixteen where four
            // neighbouring results cannot be written at once (1,914 tokens of 18,375 x 304: a lane's four one after another 165 us, next to one another 78).
#pragma unroll
            for (int c0 = 0; c0 < HALF; c0 += OUT_COLS) {
                __syncwarp();
#pragma unroll
                for (int j = 0; j < OUT_COLS / 4; ++j) {
                    float4 v;
                    unpack2(acc[c0 / 2 + 2 * j], v.x, v.y);
                    unpack2(acc[c0 / 2 + 2 * j + 1], v.z, v.w);
                    *reinterpret_cast<float4*>(out + lane * OUT_COLS + ((j ^ ((lane >> 1) & 3)) << 2)) = v;
                }
                __syncwarp();
                if (singles) {
                    const int column = lane & 15, o = row0 + c0 + column;
#pragma unroll 4
                    for (int t = lane >> 4; t < min(32, p.n - token0); t += 2)
                        if (o < p.out) store_result(p.y, p.ldy, token0 + t, o, out[t * OUT_COLS + (((column >> 2) ^ ((t >> 1) & 3)) << 2) + (column & 3)], p.epilogue, p.act, y32);
                    continue;
                }
                const int o = row0 + c0 + (lane & 3) * 4;
#pragma unroll 2
                for (int t = lane >> 2; t < min(32, p.n - token0); t += 8)
                    linear8_store(p, token0 + t, o, *reinterpret_cast<const float4*>(out + t * OUT_COLS + (((lane & 3) ^ ((t >> 1) & 3)) << 2)), quads, y32);
            }
        }
    }
    tc_fence_before();
    if (__syncthreads_or(!ok)) drain_after_timeout();        // a wait ran out: let what is in flight land
    cluster_sync();                                          // neither block leaves while the other may still touch it
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(SLOTS * STEP * BN) : "memory");
    }
}

}  // namespace

int linear8_many(const Linear8& p, cudaStream_t stream) {
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(linear8_many_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
        if (e != cudaSuccess) return ti_fail("linear8_many: %s", cudaGetErrorString(e));
        configured = true;
    }
    Args a;
    a.p = p;
    a.groups = (p.K + KB - 1) / KB;
    a.steps = (a.groups + STEP - 1) / STEP;
    a.row_blocks = (p.out + E4M3_BLOCK - 1) / E4M3_BLOCK;
    a.token_tiles = (p.n + 2 * BM - 1) / (2 * BM);
    const long long tiles = (long long)a.token_tiles * ((p.out + BN - 1) / BN);
    TI_REQUIRE(tiles < (1LL << 30), "linear8: %d tokens x %d rows are too many", p.n, p.out);
    a.tiles = (int)tiles;
    CUtensorMap map_w, map_x;
    if (int rc = linear8_map(&map_w, p.codes, p.out, p.K, p.K, BN / 2)) return rc;
    if (int rc = linear8_map(&map_x, p.x, p.n, p.K, p.n == 1 ? p.K : p.ldx, BM)) return rc;
    const int pairs = a.tiles < ti_sm_count() / 2 ? a.tiles : ti_sm_count() / 2;
    ti_launch(linear8_many_kernel, dim3(2 * pairs), dim3(THREADS), BYTES, stream, map_w, map_x, a);
    return ti_check_launch("linear8_many");
}
