// Products of e4m3 codes for up to eight tokens: the weights stream through once, a warp on its own.
//
//   y[t, o] = sum_g sx[g, t] sw[g, o / 128] sum_{k in g} cx[t, k] cw[o, k]
//
// Both operands' codes are widened to 16 bits in registers, which is exact (one instruction for two), and multiplied by mma.sync with 32-bit sums. A block of
// up to eight warps takes sixteen rows a warp, and then further ones; where there are fewer rows than that keeps the device busy, the blocks of a cluster
// take a stretch of k each, and their sums meet in the cluster's shared memory, added in rank order: one launch, no work space. A warp copies its rows' groups
// (2 KB) to shared memory of its own, AHEAD of them in flight, and waits for no other warp. (With the codes kept in registers until they are used, a group took
// as long as its reads from memory do: a warp has six counters for what it waits for, and the reads ahead shared them with everything else.) The k of both
// operands are permuted alike, so that a lane's 32 consecutive codes of a row are its share of eight MMAs. The tokens' codes of the block's stretch
// of k lie in shared memory, made from bfloat16 (or copied, where they are given) while the first weights are coming. A row's 16-byte pieces are turned by the
// row (the token), so that the reads of a warp meet all banks.
//
// Bound by reading the weights: one token of 21,504 x 4,096 takes 18.1 us (88 MB, 4.9 TB/s; launch, first reads and the last blocks are some 5 us), of
// 4,096 x 21,504 17.6, of 131,072 x 4,096 87 (6.2 TB/s). A copy reads 6.5 TB/s.
#include "linear8.cuh"
#include "mma_util.cuh"

namespace {

constexpr int N = 8, KB = 128, WARPS = 8, AHEAD = 4, UNIT = 16 * KB, MAX_SPLIT = 8, MAX_SMEM = 113 * 1024;         // WARPS: of a block at most; two blocks an SM

struct Args {
    Linear8 p;
    int groups, row_tiles, row_blocks, split;                // row_blocks: of 128 rows, as scales have them
    bool vec;                                                // bfloat16 tokens in 16-byte pieces
};

// 16 bytes, or zeros.
__device__ __forceinline__ void copy16(unsigned dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0));
}
// Bytes of shared memory: the warps' rings, codes [groups][N][128], factors [groups][N], sums [N][rows].
int few_bytes(int groups, int warps) { return warps * AHEAD * UNIT + groups * N * (KB + 4) + N * 16 * warps * 4; }

template <bool GIVEN>
__global__ void __launch_bounds__(32 * WARPS, 2) linear8_few_kernel(const Args a) {
    const Linear8& p = a.p;
    extern __shared__ __align__(128) unsigned char smem_dyn[];
    const int threads = blockDim.x, ROWS = threads / 2;      // sixteen rows a warp
    unsigned char* smem = smem_dyn + threads / 32 * (AHEAD * UNIT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % a.split, stride = gridDim.x / a.split;
    const int lo = (int)((long long)a.groups * rank / a.split), hi = (int)((long long)a.groups * (rank + 1) / a.split), own = hi - lo;
    const int room = (a.groups + a.split - 1) / a.split;     // the longest stretch: the ranks' sums lie at the same place
    float* factors = reinterpret_cast<float*>(smem + room * N * KB);         // sx; sw is the tile's
    float* sums = factors + room * N;

    // What is read next. A tile's groups are numbered up to a multiple of AHEAD, so that every tile begins with the first set of registers. Rows beyond
    // the last read the last one's codes; nobody takes their sums.
    const int end = lo + (own + AHEAD - 1) / AHEAD * AHEAD;
    int next_tile = blockIdx.x / a.split, next_group = lo;
    const unsigned char* ring = smem_dyn + warp * (AHEAD * UNIT);
    const unsigned ring_to = smem_u32(ring) + (lane >> 3) * KB;
    const unsigned char* rows[4];                            // a lane copies the same piece of every fourth row
    float scale[AHEAD];                                      // of the groups on their way: a product with one asked for in its own group waits for the read
    int next_block = 0;
    auto enter = [&] {
        next_block = min(next_tile * ROWS + warp * 16, p.out - 1) / E4M3_BLOCK;
#pragma unroll
        for (int i = 0; i < 4; ++i) rows[i] = p.codes + (size_t)min(next_tile * ROWS + warp * 16 + 4 * i + (lane >> 3), p.out - 1) * p.K + (lane & 7) * 16;
    };
    enter();
    auto load = [&](int place) {
        if (next_tile < a.row_tiles) {
            const int k = next_group * KB;
            const bool there = k + (lane & 7) * 16 < p.K;
            if (next_group < hi) {
                scale[place] = __ldg(p.scales + (long long)next_group * a.row_blocks + next_block);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    copy16(ring_to + place * UNIT + 4 * i * KB + (((lane & 7) ^ ((4 * i + (lane >> 3)) & 7)) << 4), there ? rows[i] + k : p.codes, there);
            }
            if (++next_group == end) {
                next_group = lo;
                next_tile += stride;
                enter();
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(i);
    pdl_enter();

    // The tokens' codes and factors: eight lanes a token's group of codes, sixteen of bfloat16 numbers.
    if (GIVEN) {
        constexpr int BATCH = 6;
        for (int e0 = threadIdx.x; e0 < own * N * 8; e0 += BATCH * threads) {
            uint4 v[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int e = e0 + i * threads, token = (e >> 3) % N, k = (lo + (e >> 3) / N) * KB + (e & 7) * 16;
                v[i] = e < own * N * 8 && token < p.n && k < p.K ? __ldcg(reinterpret_cast<const uint4*>((const unsigned char*)p.x + (long long)token * p.ldx + k)) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int e = e0 + i * threads, token = (e >> 3) % N;
                if (e < own * N * 8) *reinterpret_cast<uint4*>(smem + (e >> 3) * KB + (((e & 7) ^ token) << 4)) = v[i];
            }
        }
        for (int e = threadIdx.x; e < own * N; e += threads) factors[e] = e % N < p.n ? __ldcg(p.x_scales + (long long)(lo + e / N) * p.n + e % N) : 0.f;
    } else {
        constexpr int BATCH = 4;
        const int piece = lane & 15, total = own * p.n;
        for (int first = 2 * warp; first < total; first += BATCH * (threads / 16)) {         // the same for a warp's two halves: they exchange maxima
            const int e0 = first + (lane >> 4);
            uint4 v[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int e = e0 + i * (threads / 16), token = e / own, k = (lo + e - token * own) * KB + piece * 8;
                v[i] = make_uint4(0, 0, 0, 0);
                if (e < total && k < p.K) {
                    const bf16* from = (const bf16*)p.x + (long long)token * p.ldx + k;
                    if (a.vec) v[i] = __ldcg(reinterpret_cast<const uint4*>(from));
                    else {
                        const unsigned short* h = reinterpret_cast<const unsigned short*>(from);
                        v[i] = make_uint4(__ldcg(h) | (unsigned)__ldcg(h + 1) << 16, __ldcg(h + 2) | (unsigned)__ldcg(h + 3) << 16,
                                          __ldcg(h + 4) | (unsigned)__ldcg(h + 5) << 16, __ldcg(h + 6) | (unsigned)__ldcg(h + 7) << 16);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int e = e0 + i * (threads / 16), token = e / own, group = e - token * own;
                Vec16<bf16> x;
                x.unpack(v[i]);
                float m = largest8(x.v);
#pragma unroll
                for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                const int power = e4m3_scale_power(m);
                if (e < total) {
                    *reinterpret_cast<uint2*>(smem + (group * N + token) * KB + (((piece >> 1) ^ (token & 7)) << 4) + (piece & 1) * 8) = codes8(x.v, power_of_two(-power));
                    if (piece == 0) factors[group * N + token] = power_of_two(power);
                }
            }
        }
        // Columns without a token: their sums are not taken, so that what lies there may be anything.
    }
    __syncthreads();

    const bool y32 = p.epilogue == L4_EPI_F32_OUT, quads = linear8_quads(p);
    const unsigned char* x_row = smem + g * KB;
    for (int tile = blockIdx.x / a.split; tile < a.row_tiles; tile += stride) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int g0 = lo; g0 < hi; g0 += AHEAD) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int group = g0 + i;
                if (group >= hi) {
                    load(i);
                    continue;
                }
                cp_async_wait<AHEAD - 1>();
                __syncwarp();
                const unsigned char* w = ring + i * UNIT + g * KB;
                const unsigned char* x = x_row + (group - lo) * (N * KB);
                const float sw = scale[i];
                float part[2][4] = {};                       // of the even and the odd pieces: two chains of MMAs
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 b = *reinterpret_cast<const uint4*>(x + (((2 * t + h) ^ g) << 4));
                    const uint4 wl = *reinterpret_cast<const uint4*>(w + (((2 * t + h) ^ g) << 4)), wh = *reinterpret_cast<const uint4*>(w + 8 * KB + (((2 * t + h) ^ g) << 4));
                    const unsigned lo_w[4] = {wl.x, wl.y, wl.z, wl.w}, hi_w[4] = {wh.x, wh.y, wh.z, wh.w}, xw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const unsigned f[4] = {e4m3_half2((unsigned short)lo_w[q]), e4m3_half2((unsigned short)hi_w[q]), e4m3_half2((unsigned short)(lo_w[q] >> 16)),
                                               e4m3_half2((unsigned short)(hi_w[q] >> 16))};
                        mma16816_f16(part[h], f, e4m3_half2((unsigned short)xw[q]), e4m3_half2((unsigned short)(xw[q] >> 16)));
                    }
                }
                __syncwarp();
                load(i);
                const float2 f = *reinterpret_cast<const float2*>(factors + (group - lo) * N + 2 * t);
                const float f0 = f.x * sw, f1 = f.y * sw;
                acc[0] = fmaf(part[0][0] + part[1][0], f0, acc[0]);
                acc[1] = fmaf(part[0][1] + part[1][1], f1, acc[1]);
                acc[2] = fmaf(part[0][2] + part[1][2], f0, acc[2]);
                acc[3] = fmaf(part[0][3] + part[1][3], f1, acc[3]);
            }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) sums[(2 * t + (c & 1)) * ROWS + warp * 16 + g + 8 * (c >> 1)] = acc[c];
        if (a.split == 1) {                                  // a warp writes its own rows, four of a token at a time
            __syncwarp();
            for (int e = lane; e < p.n * 4; e += 32)
                linear8_store(p, e >> 2, tile * ROWS + warp * 16 + (e & 3) * 4, *reinterpret_cast<const float4*>(sums + (e >> 2) * ROWS + warp * 16 + (e & 3) * 4), quads, y32);
            __syncwarp();
            continue;
        }
        cluster_meets();                                     // one tile a cluster
        for (int e = rank * threads + threadIdx.x; e < p.n * (ROWS / 4); e += a.split * threads) {
            float4 v[MAX_SPLIT];
#pragma unroll
            for (int r = 0; r < MAX_SPLIT; ++r) v[r] = r < a.split ? rank_sums(sums + 4 * e, r) : make_float4(0.f, 0.f, 0.f, 0.f);
            float4 s = v[0];
#pragma unroll
            for (int r = 1; r < MAX_SPLIT; ++r) { s.x += v[r].x; s.y += v[r].y; s.z += v[r].z; s.w += v[r].w; }
            linear8_store(p, e / (ROWS / 4), tile * ROWS + e % (ROWS / 4) * 4, s, quads, y32);
        }
        cluster_meets();                                     // the others may still read this block's sums
    }
}

template <bool GIVEN> int launch(const Linear8& p, int warps, int split, cudaStream_t stream) {
    Args a;
    a.p = p;
    a.groups = (p.K + KB - 1) / KB;
    a.row_tiles = (p.out + 16 * warps - 1) / (16 * warps);
    a.row_blocks = (p.out + E4M3_BLOCK - 1) / E4M3_BLOCK;
    a.split = split;
    a.vec = aligned16(p.x) && (p.n == 1 || p.ldx % 8 == 0);
    const int bytes = few_bytes((a.groups + split - 1) / split, warps);
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(linear8_few_kernel<GIVEN>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
        if (e != cudaSuccess) return ti_fail("linear8_few: %s", cudaGetErrorString(e));
        configured = true;
    }
    // Clusters take one tile each; single blocks go on to further ones, so that a block's tokens are made once.
    const int slots = 2 * ti_sm_count(), blocks = split > 1 || a.row_tiles < slots ? a.row_tiles * split : slots;
    linear8_launch(linear8_few_kernel<GIVEN>, dim3(blocks), 32 * warps, bytes, split, stream, a);
    return ti_check_launch("linear8_few");
}

// Blocks of the cluster that shares a product's rows; 0 where the tokens' codes do not fit. As many as two blocks an SM have room for: 4,096 x 4,096 takes
// 6.5 us with 8, 7.4 with 4, 10.2 with 2. Powers of two: clusters of 6 do not fill the device (6,144 x 4,096 8.2 us with 4, 13.0 with 6).
int few_split(int out, int K, int warps) {
    const int groups = (K + KB - 1) / KB, tiles = (out + 16 * warps - 1) / (16 * warps);
    int split = 1;
    while (split < MAX_SPLIT && 2 * split <= groups && (2LL * split * tiles <= 2 * ti_sm_count() || few_bytes((groups + split - 1) / split, warps) > MAX_SMEM)) split *= 2;
    return few_bytes((groups + split - 1) / split, warps) > MAX_SMEM ? 0 : split;
}
// Groups of sixteen rows that the busiest SM reads, where the tokens' codes fit.
long long few_load(int out, int K, int warps) {
    const int groups = (K + KB - 1) / KB, split = few_split(out, K, warps);
    const long long blocks = (long long)((out + 16 * warps - 1) / (16 * warps)) * split, sms = ti_sm_count();
    return (blocks + sms - 1) / sms * warps * ((groups + split - 1) / split);
}
// Warps of a block: eight, or the most that leave the busiest SM at least a fifth less to read (168 blocks of 128 rows leave 20 of 148 SMs two). Microseconds for
// one and eight tokens with 8, 7, 6, 5: 21,504 x 4,096 19.9 / 22.5, 19.7 / 22.7, 18.1 / 21.2, 18.3 / 21.8 (6 is taken); 6,144 x 4,096 7.7 / 9.0, 7.5 / 9.7, 7.2 / 9.4 (6),
// 9.7 / 14.1; 4,096 x 21,504 17.6 / 20.5 (8), 26.1 / 29.6, 22.1 / 25.8, 23.2 / 25.3.
// Rows of more than 44,032 columns, whose tokens' codes fit beside four to seven warps alone, are linear8_mid.cu's: one and eight tokens of 4,096 x 50,000 53.0 / 63.9 here,
// 40.3 / 42.1 there; 4,096 x 72,000 66.2 / 74.4, 52.5 / 53.6; 512 x 50,000 20.1 / 29.8, 25.3 / 25.9.
int few_warps(int out, int K) {
    if (few_split(out, K, WARPS) == 0) return WARPS;
    int w = WARPS;
    while (--w >= 4)
        if (few_load(out, K, w) * 5 <= few_load(out, K, WARPS) * 4) return w;
    return WARPS;
}

}  // namespace

bool linear8_takes_few(int n, int out, int K) { return n <= N && few_split(out, K, few_warps(out, K)) > 0; }

int linear8_few(const Linear8& p, cudaStream_t stream) {
    const int warps = few_warps(p.out, p.K), split = few_split(p.out, p.K, warps);
    return p.x_scales != nullptr ? launch<true>(p, warps, split, stream) : launch<false>(p, warps, split, stream);
}
