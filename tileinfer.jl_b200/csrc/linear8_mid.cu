// Products of e4m3 codes for nine to some hundred tokens: the weight rows in the lanes of tcgen05.mma.
//
//   y[t, o] = sum_g sx[g, t] sw[g, o / 128] sum_{k in g} cx[t, k] cw[o, k]
//
// A block takes 128 weight rows (the lanes) by N tokens (the columns) and a stretch of k in groups of 128. A group's sum goes to an accumulator of its own in
// tensor memory, from where eight warps (two a quarter of the lanes, half of the columns each) add it, times sx sw, to 32-bit sums in registers. The blocks that
// share 128 rows stand in one cluster, each with its stretch of k; their sums meet in the cluster's shared memory and are added in rank order: one
// launch, no work space for parts.
//
// Bound by reading the weights, 16 KB of them a group: 16 tokens of 21,504 x 4,096 take 22.9 us with their quantisation, 64 take 26.0 (88 MB, 13.5 us at the rate of a
// copy; 18 us of it the weights' own stream, the rest launches, the fill and the cluster's sums). Four groups' factors are on their way at once: multiplied as they
// came, they cost a group the latency of its loads (26.1 and 28.2 us).
//
// Warp 0 asks for weights and tokens (TMA), warp 1 issues the MMAs, warps 2 to 9 add, warp 10 brings the factors sx sw. All waits are bounded.
#include "linear8.cuh"

namespace {
using namespace tc;

constexpr int ROWS = 128, KB = 128, W_BYTES = ROWS * KB, THREADS = 352, MAX_SPLIT = 8;

template <int N> struct Shape {
    static constexpr int ACCS = 4, COLS = ACCS * N, X_BYTES = N * KB, STAGE = W_BYTES + X_BYTES;
    static constexpr int STAGES = 104 * 1024 / STAGE;        // two blocks an SM
    // Factors of a group's tokens: a place is written again when the group STAGES + ACCS before has been added (its accumulator was given to a
    // group whose stage has been read since).
    static constexpr int PLACES = STAGES + ACCS;
    static constexpr int BYTES = STAGES * STAGE + 1024;
};

struct Args {
    Linear8 p;
    int groups, row_tiles, split;
};

template <int N>
__global__ void __launch_bounds__(THREADS, 2) linear8_mid_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Args a) {
    typedef Shape<N> S;
    const Linear8& p = a.p;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* tiles = smem_dyn + ((1024u - (smem_addr(smem_dyn) & 1023u)) & 1023u);
    __shared__ __align__(16) float s_factor[S::PLACES][N];
    __shared__ __align__(8) unsigned long long bars[2 * S::STAGES + 2 * S::ACCS + S::PLACES];
    __shared__ unsigned s_tmem;
    const unsigned full0 = smem_addr(bars), empty0 = full0 + 8 * S::STAGES, accf0 = empty0 + 8 * S::STAGES, acce0 = accf0 + 8 * S::ACCS, fac0 = acce0 + 8 * S::ACCS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % a.split, tile = blockIdx.x / a.split, token0 = blockIdx.y * N, tokens = min(N, p.n - token0);
    const int lo = (int)((long long)a.groups * rank / a.split), hi = (int)((long long)a.groups * (rank + 1) / a.split);
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(full0 + 8 * s, 2); mbar_init(empty0 + 8 * s, 1); }
        for (int s = 0; s < S::ACCS; ++s) { mbar_init(accf0 + 8 * s, 1); mbar_init(acce0 + 8 * s, 8); }
        for (int s = 0; s < S::PLACES; ++s) mbar_init(fac0 + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_addr(&s_tmem), S::COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = s_tmem;
    bool ok = true;

    if (warp == 0) {
        // ---------------------------------------------------------------- the weights, which no kernel of a step writes, at once; the tokens after the wait
        if (lane == 0) {
            const int ahead = min(S::STAGES, hi - lo);
            for (int i = 0; i < ahead; ++i) {
                mbar_expect_tx(full0 + 8 * i, S::STAGE);
                tma_load_2d(smem_addr(tiles + i * S::STAGE), &map_w, (lo + i) * (KB / 2), tile * ROWS, full0 + 8 * i);
            }
            pdl_wait();
            for (int i = 0; i < ahead; ++i) tma_load_2d(smem_addr(tiles + i * S::STAGE + W_BYTES), &map_x, (lo + i) * (KB / 2), token0, full0 + 8 * i);
            int stage = 0;
            unsigned phase = 0;
            for (int g = lo + ahead; g < hi; ++g) {
                ok = mbar_wait(empty0 + 8 * stage, phase, p.status, 18);
                if (!ok) break;
                const unsigned to = smem_addr(tiles + stage * S::STAGE), bar = full0 + 8 * stage;
                mbar_expect_tx(bar, S::STAGE);
                tma_load_2d(to, &map_w, g * (KB / 2), tile * ROWS, bar);
                tma_load_2d(to + W_BYTES, &map_x, g * (KB / 2), token0, bar);
                if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMAs: one thread of a warp that walks along
        int stage = 0, slot = 0;
        unsigned phase = 0, slot_phase = 0;
        const unsigned long long first = smem_desc_sw128(smem_addr(tiles));
        for (int g = lo; g < hi; ++g) {
            ok = __all_sync(0xffffffffu, mbar_wait(acce0 + 8 * slot, slot_phase ^ 1, p.status, 19) && mbar_wait(full0 + 8 * stage, phase, p.status, 20));
            if (!ok) break;
            tc_fence_after();
            const unsigned long long dw = first + (unsigned)(stage * (S::STAGE >> 4)), dx = dw + (W_BYTES >> 4);
            if (elected()) {
#pragma unroll
                for (int k = 0; k < KB / 32; ++k)            // 32 bytes further along the swizzled rows
                    umma_e4m3(tmem + slot * N, dw + 2 * k, dx + 2 * k, instr_desc_e4m3(N), k > 0);
                umma_commit(empty0 + 8 * stage);
                umma_commit(accf0 + 8 * slot);
            }
            __syncwarp();
            if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
            if (++slot == S::ACCS) { slot = 0; slot_phase ^= 1; }
        }
    } else if (warp < 10) {
        // ---------------------------------------------------------------- the groups' sums, scaled and added: a thread a weight row, half of the tokens
        constexpr int H = N / 2;
        const int first = warp < 6 ? 0 : H;
        float acc[H];
#pragma unroll
        for (int c = 0; c < H; ++c) acc[c] = 0.f;
        int slot = 0, place = 0;
        unsigned slot_phase = 0, place_phase = 0;
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
        for (int g = lo; g < hi; ++g) {
            ok = warp_wait(fac0 + 8 * place, place_phase, p.status, 21) && warp_wait(accf0 + 8 * slot, slot_phase, p.status, 22);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < H; c += 16) {
                unsigned r[16];
                tmem_ld16(tmem + lanes + slot * N + first + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const float4 f = *reinterpret_cast<const float4*>(&s_factor[place][first + c + j]);
                    acc[c + j] = fmaf(__uint_as_float(r[j]), f.x, acc[c + j]);
                    acc[c + j + 1] = fmaf(__uint_as_float(r[j + 1]), f.y, acc[c + j + 1]);
                    acc[c + j + 2] = fmaf(__uint_as_float(r[j + 2]), f.z, acc[c + j + 2]);
                    acc[c + j + 3] = fmaf(__uint_as_float(r[j + 3]), f.w, acc[c + j + 3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acce0 + 8 * slot);
            if (++slot == S::ACCS) { slot = 0; slot_phase ^= 1; }
            if (++place == S::PLACES) { place = 0; place_phase ^= 1; }
        }
        // Every MMA has read its stage and every stage's copies have landed: the sums go where the stages were, [token][row].
        float* sums = reinterpret_cast<float*>(tiles) + (warp & 3) * 32 + lane;
#pragma unroll
        for (int c = 0; c < H; ++c) sums[(first + c) * ROWS] = acc[c];
    } else {
        // ---------------------------------------------------------------- the factors, LOADS groups ahead, multiplied when they are wanted (a product at once would
        // wait for its loads)
        pdl_enter();
        constexpr int V = N / 32, LOADS = 4;
        int stage = 0, place = 0;
        unsigned phase = 0;
        float sx[LOADS][V], sw[LOADS];
        auto ask = [&](int g, float (&x)[V], float& w) {
            if (g >= hi) return;
            w = __ldg(p.scales + (long long)g * a.row_tiles + tile);
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = __ldcg(p.x_scales + (long long)g * p.n + min(token0 + lane + 32 * i, p.n - 1));
        };
#pragma unroll
        for (int j = 0; j < LOADS; ++j) ask(lo + j, sx[j], sw[j]);
        for (int g0 = lo; ok && g0 < hi; g0 += LOADS) {
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                if (g0 + j >= hi) break;
                ok = warp_wait(empty0 + 8 * stage, phase ^ 1, p.status, 23);
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < V; ++i) s_factor[place][lane + 32 * i] = sx[j][i] * sw[j];
                ask(g0 + j + LOADS, sx[j], sw[j]);
                __syncwarp();
                // The group's MMAs wait for this too: were they ahead, the stage could be emptied again before the wait above has seen it emptied once.
                if (lane == 0) { mbar_arrive(full0 + 8 * stage); mbar_arrive(fac0 + 8 * place); }
                if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
                if (++place == S::PLACES) place = 0;
            }
        }
    }
    pdl_wait();                                              // y may still be read by the kernel before
    if (__syncthreads_or(!ok)) drain_after_timeout();        // a wait ran out: let what is in flight land
    if (a.split > 1) cluster_meets();
    // Four rows of a token at a time; all ranks' sums are asked for together.
    const float* sums = reinterpret_cast<const float*>(tiles);
    const bool y32 = p.epilogue == L4_EPI_F32_OUT, whole = linear8_quads(p);
    for (int e = rank * THREADS + threadIdx.x; e < tokens * (ROWS / 4); e += a.split * THREADS) {
        float4 s;
        if (a.split == 1) s = reinterpret_cast<const float4*>(sums)[e];
        else {
            float4 v[MAX_SPLIT];
#pragma unroll
            for (int r = 0; r < MAX_SPLIT; ++r) v[r] = r < a.split ? rank_sums(sums + 4 * e, r) : make_float4(0.f, 0.f, 0.f, 0.f);
            s = v[0];
#pragma unroll
            for (int r = 1; r < MAX_SPLIT; ++r) { s.x += v[r].x; s.y += v[r].y; s.z += v[r].z; s.w += v[r].w; }
        }
        linear8_store(p, token0 + e / (ROWS / 4), tile * ROWS + e % (ROWS / 4) * 4, s, whole, y32);
    }
    tc_fence_before();
    if (a.split > 1) cluster_meets(); else __syncthreads();  // the others may still read this block's sums
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, S::COLS);
    }
}

template <int N> int launch(const Linear8& p, int split, cudaStream_t stream) {
    typedef Shape<N> S;
    static_assert(S::STAGES >= 3 && S::STAGES * S::STAGE >= N * ROWS * 4, "stages");
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(linear8_mid_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES);
        if (e != cudaSuccess) return ti_fail("linear8_mid: %s", cudaGetErrorString(e));
        configured = true;
    }
    Args a;
    a.p = p;
    a.groups = (p.K + KB - 1) / KB;
    a.row_tiles = (p.out + ROWS - 1) / ROWS;
    a.split = split;
    CUtensorMap map_w, map_x;
    if (int rc = linear8_map(&map_w, p.codes, p.out, p.K, p.K, ROWS)) return rc;
    if (int rc = linear8_map(&map_x, p.x, p.n, p.K, p.n == 1 ? p.K : p.ldx, N)) return rc;
    linear8_launch(linear8_mid_kernel<N>, dim3(a.row_tiles * split, (p.n + N - 1) / N), THREADS, S::BYTES, split, stream, map_w, map_x, a);
    return ti_check_launch("linear8_mid");
}

}  // namespace

int linear8_mid(const Linear8& p, cudaStream_t stream) {
    const int groups = (p.K + KB - 1) / KB, N = p.n <= 32 ? 32 : 64;
    const long long tiles = (long long)((p.out + ROWS - 1) / ROWS) * ((p.n + N - 1) / N);
    int split = 1;                                           // blocks of a cluster: powers of two, as in linear8_few.cu
    while (split < MAX_SPLIT && 2 * split <= groups && 2 * split * tiles <= 2 * ti_sm_count()) split *= 2;
    TI_REQUIRE((p.n + N - 1) / N <= 65535, "linear8: %d tokens are too many", p.n);
    return N == 32 ? launch<32>(p, split, stream) : launch<64>(p, split, stream);
}
