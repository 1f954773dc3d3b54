// Attention over the paged cache in 8 bits (cache8.cu), bfloat16 queries and results: one to some tens of new tokens of every sequence. The new tokens'
// keys and values are in the cache already; token i of a sequence's T stands at position L - T + i, and sees the keys up to itself (and, with a window, the
// window's last ones only).
//
//   out[i, h] = sum_j softmax_j(scale q[i, h] . sk[p(j)] ck[j]) sv[p(j)] cv[j], over the visible j; p(j) is j's page.
//
// Bound by reading the cache once, so the T x (query heads per KV head) rows that share a KV head are the rows of the MMA tiles (slabs of 16, 32 or
// 64), and the work is shared out by length (attention_parts.cuh). A page's head is one tile, 64 x D consecutive bytes of keys and as many of values, which
// come as two TMA copies of rows of 128 swizzled bytes, whatever D is. A warp asks for them and brings the scales; four others share a tile out as MT groups
// of 16 rows x 4 / MT groups of keys, each on its own.
//
// Codes are widened in registers to numbers of 16 bits, exactly (one instruction for two; values of four keys are first put side by side, one for two
// more). Queries are scaled by a power of two a row, so that they fit those numbers without loss. Keys' dimensions are permuted alike in both operands, so that a
// lane's share of four MMAs is 16 consecutive bytes; so are the keys, so that a warp's reads meet all banks.
//
// With z_j = (the score in base 2) + log2 sv[p(j)], the running maximum m is that of z: P = 2^(z - m + 7) <= 128 are the weights of the values' codes, rounded
// to 16 bits (2^-11) as the MMA's operand, and the denominator is the 32-bit sum of P / sv. So neither pages of very unequal scales nor a
// scale of 2^-100 (a page of zeros) cost anything but an addition to the exponent. Scores, sums and outputs stand in 32-bit.
//
// Keys and values beyond the sequence's end or before the first visible key may hold any codes: their scores are replaced and their values' codes are
// zero. A NaN code of a key that some rows see and others do not (a drafted token's own) reaches the rows that see it alone.
#include "attention_parts.cuh"
#include "e4m3.cuh"
#include "linear8.cuh"
#include "mma_util.cuh"

namespace {

constexpr int A8_THREADS = 160, A8_MAX_SEQS = 512;           // four warps that compute, one that asks
constexpr float P_POWER = 7.f;

// DP: D rounded up to 64, 128 or 256.
template <int DP> struct Smem8 {
    static constexpr int STAGES = DP <= 128 ? 4 : 3;
    // Queries of heads beyond 128 lie in shared memory (the outputs take the registers): [64 dimensions][4][lane].
    static constexpr int Q = DP > 128 ? DP / 64 * 4 * 32 * 16 : 0;
    // Stages, queries, then the warps' shares of `rows` rows of an item: [key group][row][DP].
    static __host__ __device__ int bytes(int D, int groups_of_keys, int rows) { return STAGES * 2 * AF_PAGE * D + Q + groups_of_keys * rows * DP * 4 + 1024; }
};

struct Args8 {
    bf16* out;
    const bf16* q;
    const unsigned char* v;                                  // for NaN codes that were taken out
    const float *k_scales, *v_scales;
    const int* table;
    int table_stride;
    const int *seq_slots, *cu, *kv_lens;
    float *ws_o, *ws_ml;
    int* status;
    float scale_log2e;
    int B, nq, nkv, D, window, rows, pages, n;               // rows: of an item, at most (the merge's room)
};

// Byte i of a tile of swizzled 128-byte rows.
__device__ __forceinline__ int tile_at(int i) { return (i & ~0x70) | ((i ^ (i >> 3)) & 0x70); }
// 0xFF in the places of NaN codes.
__device__ __forceinline__ unsigned nan_codes(unsigned w) { return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu); }
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <int DP, int MT, int BLOCKS>
__global__ void __launch_bounds__(A8_THREADS, BLOCKS) attention8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Args8 a) {
    constexpr int M = 16 * MT, WK = 4 / MT, KH = DP / 64, NT = DP / 8, STAGES = Smem8<DP>::STAGES;
    // Bytes of a key's values that a lane reads at once, and how often.
    constexpr int VB = DP == 64 ? 8 : 16, VH = DP == 256 ? 2 : 1;
    extern __shared__ __align__(128) unsigned char smem_dyn[];
    __shared__ unsigned s_units[A8_MAX_SEQS + 1], s_scan[A8_THREADS / 32];
    __shared__ int s_cu[A8_MAX_SEQS + 1], s_len[A8_MAX_SEQS], s_slot[A8_MAX_SEQS];
    __shared__ float s_ml[WK][M][2], s_scale[STAGES][2];
    __shared__ __align__(8) unsigned long long bars[2 * STAGES];
    unsigned char* ring = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    const int D = a.D, tile_bytes = AF_PAGE * D, B = a.B, nkv = a.nkv, group = a.nq / nkv;
    const unsigned full0 = smem_u32(bars), empty0 = full0 + 8 * STAGES;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { tc::mbar_init(full0 + 8 * s, 1); tc::mbar_init(empty0 + 8 * s, 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

    // Units before every sequence.
    unsigned carry = 0;
    for (int b0 = 0; b0 < B; b0 += A8_THREADS) {
        const int b = b0 + threadIdx.x;
        unsigned v = 0;
        if (b < B) {
            const int at = __ldcg(a.cu + b), end = __ldcg(a.cu + b + 1), len = __ldcg(a.kv_lens + b);
            s_slot[b] = __ldcg(a.seq_slots + b);
            s_cu[b] = at;
            if (b == B - 1) s_cu[B] = end;
            s_len[b] = len;
            const FewShape s = few_shape(end - at, len, a.window, group, M);
            v = (unsigned)(s.tiles * s.slabs * nkv);
        }
        const unsigned own = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        __syncthreads();
        if (lane == 31) s_scan[warp] = v;
        __syncthreads();
        unsigned before = carry;
        for (int w = 0; w < A8_THREADS / 32; ++w) {
            if (w < warp) before += s_scan[w];
            carry += s_scan[w];
        }
        if (b < B) s_units[b] = before + v - own;
    }
    if (threadIdx.x == 0) s_units[B] = carry;
    __syncthreads();
    const unsigned U = s_units[B], G = min(gridDim.x, U);
    if (blockIdx.x >= max(G, 1u)) return;                    // more blocks than units
    const Runs runs(U, max(G, 1u));
    const unsigned lo = runs.low(blockIdx.x), hi = runs.low(blockIdx.x + 1);

    struct Place {
        FewShape s;
        int b, kvh, slab, tile;                              // tile counts from the first visible one
    };
    auto locate = [&](unsigned u) {
        Place p;
        int x = 0, z = B;                                    // the last sequence with units before it <= u and units of its own
        while (z - x > 1) {
            const int mid = (x + z) >> 1;
            if (s_units[mid] <= u) x = mid; else z = mid;
        }
        p.b = x;
        p.s = few_shape(s_cu[x + 1] - s_cu[x], s_len[x], a.window, group, M);
        const int v = (int)(u - s_units[x]), item = v / p.s.tiles;
        p.tile = v - item * p.s.tiles;
        p.kvh = item / p.s.slabs;
        p.slab = item - p.kvh * p.s.slabs;
        return p;
    };

    if (warp == 4) {
        // ---------------------------------------------------------------- copies: lane 0, with a tile's page asked for one tile ahead
        bool ok = true, waited = false;
        unsigned u = lo, phase = 0;
        int stage = 0;
        Place at{};
        const int* pages = nullptr;
        int page = 0;
        auto enter = [&] {
            at = locate(u);
            pages = a.table + (size_t)s_slot[at.b] * a.table_stride + at.s.t0;
            page = __ldcg(pages + at.tile);
        };
        if (lane == 0 && u < hi) enter();
        while (lane == 0 && u < hi) {
            // Tiles with new keys were written by the kernel before this one; the others stand since earlier steps.
            if (!waited && (at.s.t0 + at.tile + 1) * AF_PAGE > at.s.L - at.s.T) { pdl_wait(); waited = true; }
            const bool there = page >= 0 && page < a.pages;  // a page that does not exist reads as zeros
            const int block = there ? page * nkv + at.kvh : -1;
            const float sk = there ? __ldcg(a.k_scales + block) : 1.f, sv = there ? __ldcg(a.v_scales + block) : 1.f;
            const bool last = at.tile + 1 == at.s.tiles;
            const int next_page = last ? 0 : __ldcg(pages + at.tile + 1);
            ok = tc::mbar_wait(empty0 + 8 * stage, phase ^ 1, a.status, 29);
            if (!ok) break;
            const unsigned bar = full0 + 8 * stage, to = smem_u32(ring) + stage * 2 * tile_bytes;
            s_scale[stage][0] = sk;
            s_scale[stage][1] = sv;
            tc::mbar_expect_tx(bar, 2 * tile_bytes);
            tc::tma_load_2d(to, &map_k, 0, block * (D / 2), bar);
            tc::tma_load_2d(to + tile_bytes, &map_v, 0, block * (D / 2), bar);
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
            ++u;
            if (last) {
                if (u < hi) enter();
            } else {
                ++at.tile;
                page = next_page;
            }
        }
        if (!ok) tc::drain_after_timeout();                  // a wait ran out: let what is in flight land
        __syncwarp();
        return;
    }

    pdl_enter();
    const int wr = warp % MT, wk = warp / MT;
    // Column n of eight scores is key n, with its bit 2 turned where n is odd: neighbouring columns' rows then lie in different halves of the banks.
    const int key_g = g ^ ((g & 1) << 2), key_t0 = 2 * t, key_t1 = (2 * t + 1) ^ 4;
    int stage = 0;
    unsigned phase = 0;
    bool ok = true;                                          // once a wait has run out, all that is left is to meet the other warps
    unsigned u = lo;
    uint4* sq = reinterpret_cast<uint4*>(ring + STAGES * 2 * tile_bytes) + lane;              // all warps write the same
    float* mg = reinterpret_cast<float*>(ring + STAGES * 2 * tile_bytes + Smem8<DP>::Q);
    while (u < hi) {
        // One segment: the tiles of one item that lie in this block's run.
        const Place at = locate(u);
        const FewShape& s = at.s;
        const unsigned seg_begin = u, seg_end = min(hi, u + (unsigned)(s.tiles - at.tile));
        const int rows = s.T * group, first_token = s_cu[at.b];
        int pos[2], low[2];
        unsigned qf[KH][4][4];
        float row_scale[2];
        {
            unsigned raw[2][KH][4][2];
            float top[2] = {0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = at.slab * M + wr * 16 + g + 8 * h, i = r / group;
                const bool real = r < rows;
                pos[h] = real ? s.L - s.T + i : -1;
                low[h] = a.window > 0 ? max(0, pos[h] - a.window + 1) : 0;
                const bf16* row = a.q + ((size_t)(first_token + i) * a.nq + (size_t)at.kvh * group + (r - i * group)) * D;
#pragma unroll
                for (int kh = 0; kh < KH; ++kh) {
                    const int d = (t + 4 * kh) * 16;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const unsigned w = real && d < D ? __ldcg(reinterpret_cast<const unsigned*>(row + d + 4 * j + 2 * e)) : 0u;
                            raw[h][kh][j][e] = w;
                            top[h] = fmaxf(top[h], fmaxf(finite_size(__uint_as_float(w << 16)), finite_size(__uint_as_float(w & 0xFFFF0000u))));
                        }
                }
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                const int power = max((int)(__float_as_uint(top[h]) >> 23) - 127, -100) - 14;        // the row's largest becomes 2^14 to 2^15
                row_scale[h] = power_of_two(power) * a.scale_log2e;
                const float inverse = power_of_two(-power);
#pragma unroll
                for (int kh = 0; kh < KH; ++kh)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const unsigned w = raw[h][kh][j][e];
                            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(qf[kh][j][2 * e + h]) : "f"(__uint_as_float(w & 0xFFFF0000u) * inverse), "f"(__uint_as_float(w << 16) * inverse));
                        }
            }
        }
        if (DP > 128) {
#pragma unroll
            for (int kh = 0; kh < KH; ++kh)
#pragma unroll
                for (int j = 0; j < 4; ++j) sq[(kh * 4 + j) * 32] = make_uint4(qf[kh][j][0], qf[kh][j][1], qf[kh][j][2], qf[kh][j][3]);
            __syncwarp();
        }
        float o[NT][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

        bool odd = false;
        int tile = s.t0 + at.tile;
        for (; u < seg_end; ++u, ++tile) {
            if (ok) ok = tc::warp_wait(full0 + 8 * stage, phase, a.status, 28);
            if (!ok) continue;
            const unsigned char* kt = ring + stage * 2 * tile_bytes;
            const unsigned char* vt = kt + tile_bytes;
            const float sk = s_scale[stage][0], sv = s_scale[stage][1];
            const int key_base = tile * AF_PAGE, share = wk * MT * 16;
            float sc[2 * MT][4];
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[i][j] = 0.f;
#pragma unroll
            for (int kh = 0; kh < KH; ++kh)
#pragma unroll
                for (int i = 0; i < 2 * MT; ++i) {
                    const int piece = t + 4 * kh;
                    const uint4 w4 = piece * 16 < D ? *reinterpret_cast<const uint4*>(kt + tile_at((share + 8 * i + key_g) * D + piece * 16)) : make_uint4(0, 0, 0, 0);
                    const unsigned w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (DP > 128) {
                            const uint4 x = sq[(kh * 4 + j) * 32];
                            const unsigned xf[4] = {x.x, x.y, x.z, x.w};
                            mma16816_f16(sc[i], xf, e4m3_half2((unsigned short)w[j]), e4m3_half2((unsigned short)(w[j] >> 16)));
                        } else mma16816_f16(sc[i], qf[kh][j], e4m3_half2((unsigned short)w[j]), e4m3_half2((unsigned short)(w[j] >> 16)));
                    }
                }
            // A tile at an edge has scores replaced: of keys that a row does not see.
            const bool edge = key_base + AF_PAGE > s.L - s.T + 1 || (a.window > 0 && key_base < s.L - a.window);
            if (edge) {
#pragma unroll
                for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int key = key_base + share + 8 * i + (j == 0 ? key_t0 : key_t1);
                        if (key > pos[0] || key < low[0]) sc[i][j] = -INFINITY;
                        if (key > pos[1] || key < low[1]) sc[i][2 + j] = -INFINITY;
                    }
            }
            float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) {
                mx0 = fmaxf(mx0, fmaxf(sc[i][0], sc[i][1]));
                mx1 = fmaxf(mx1, fmaxf(sc[i][2], sc[i][3]));
            }
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
            const float f0 = row_scale[0] * sk, f1 = row_scale[1] * sk, lv = __log2f(sv), inv = 1.f / sv;
            const float n0 = fmaxf(m0, fmaf(mx0, f0, lv)), n1 = fmaxf(m1, fmaf(mx1, f1, lv));
            const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
            if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {             // most tiles leave the maxima, and then the sums, as they are
                const float c0 = power2(m0 - b0), c1 = power2(m1 - b1);
                l0 *= c0; l1 *= c1;
#pragma unroll
                for (int i = 0; i < NT; ++i) { o[i][0] *= c0; o[i][1] *= c0; o[i][2] *= c1; o[i][3] *= c1; }
            }
            m0 = n0; m1 = n1;
            const float e0 = lv - b0 + P_POWER, e1 = lv - b1 + P_POWER;
            float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
            for (int nb = 0; nb < MT; ++nb) {
                unsigned pf[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float* x = sc[2 * nb + h];
                    x[0] = power2(fmaf(x[0], f0, e0)); x[1] = power2(fmaf(x[1], f0, e0));
                    x[2] = power2(fmaf(x[2], f1, e1)); x[3] = power2(fmaf(x[3], f1, e1));
                    sum0 += x[0] + x[1];
                    sum1 += x[2] + x[3];
                    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(pf[2 * h]) : "f"(x[1]), "f"(x[0]));
                    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(pf[2 * h + 1]) : "f"(x[3]), "f"(x[2]));
                }
                // A lane's four keys of the sixteen: 16 (8, twice 16) bytes of each.
                int row[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) row[e] = share + nb * 16 + 8 * (e >> 1) + (e & 1 ? key_t1 : key_t0);
#pragma unroll
                for (int vh = 0; vh < VH; ++vh) {
                    unsigned w[4][VB / 4];
                    const int byte = vh * 128 + g * VB;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (VB == 16) {
                            const uint4 v = byte < D ? *reinterpret_cast<const uint4*>(vt + tile_at(row[e] * D + byte)) : make_uint4(0, 0, 0, 0);
                            w[e][0] = v.x; w[e][1] = v.y; w[e][VB / 4 - 2] = v.z; w[e][VB / 4 - 1] = v.w;
                        } else {
                            const uint2 v = byte < D ? *reinterpret_cast<const uint2*>(vt + (tile_at((row[e] * D + byte) & ~15) | (byte & 8))) : make_uint2(0, 0);
                            w[e][0] = v.x; w[e][1] = v.y;
                        }
                    }
                    if (edge) {
                        // Values that nobody sees may have any code, and 0 x NaN is NaN; NaN codes that some rows see are added at the segment's end.
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key_base + row[e];
                            const bool seen = key < s.L && key >= s.first;
#pragma unroll
                            for (int j = 0; j < VB / 4; ++j) {
                                if (!seen) w[e][j] = 0;
                                else if (s.T > 1) {
                                    const unsigned bad = nan_codes(w[e][j]);
                                    odd |= bad != 0;
                                    w[e][j] &= ~bad;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < VB / 4; ++j) {
                        // Side by side: bytes of the keys at k = 2t and 2t + 1, and of those eight further on.
                        const unsigned a01 = __byte_perm(w[0][j], w[1][j], 0x5140), a23 = __byte_perm(w[0][j], w[1][j], 0x7362);
                        const unsigned b01 = __byte_perm(w[2][j], w[3][j], 0x5140), b23 = __byte_perm(w[2][j], w[3][j], 0x7362);
                        const int c = vh * 16 + 4 * j;
                        mma16816_f16(o[c], pf, e4m3_half2((unsigned short)a01), e4m3_half2((unsigned short)b01));
                        mma16816_f16(o[c + 1], pf, e4m3_half2((unsigned short)(a01 >> 16)), e4m3_half2((unsigned short)(b01 >> 16)));
                        mma16816_f16(o[c + 2], pf, e4m3_half2((unsigned short)a23), e4m3_half2((unsigned short)b23));
                        mma16816_f16(o[c + 3], pf, e4m3_half2((unsigned short)(a23 >> 16)), e4m3_half2((unsigned short)(b23 >> 16)));
                    }
                }
            }
            l0 = fmaf(sum0, inv, l0);
            l1 = fmaf(sum1, inv, l1);
            tc::fence_async_smem();                          // the stage's next copies are another proxy's than these reads
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(empty0 + 8 * stage);
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        // The dimension of column n of results c: VB consecutive ones a column.
        auto dim = [&](int c, int n) { return (c / 16) * 128 + n * VB + c % 16; };
        if (ok && __any_sync(0xffffffffu, odd)) {            // what this warp has taken out: NaN whatever its weight
            auto put_back = [&](int from, int to) {
                for (int key = max(from, (s.t0 + at.tile) * AF_PAGE); key < min(to, tile * AF_PAGE); ++key) {
                    if ((key % AF_PAGE) / (MT * 16) != wk) continue;
                    const int page = __ldcg(a.table + (size_t)s_slot[at.b] * a.table_stride + key / AF_PAGE);
                    if (page < 0 || page >= a.pages) continue;
                    const unsigned char* value = a.v + (((size_t)page * nkv + at.kvh) * AF_PAGE + key % AF_PAGE) * D;
                    const bool s0 = key <= pos[0] && key >= low[0], s1 = key <= pos[1] && key >= low[1];
#pragma unroll
                    for (int c = 0; c < NT; ++c)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int d = dim(c, 2 * t + e);
                            if (d < D && (__ldcg(value + d) & 0x7F) == 0x7F) {
                                if (s0) o[c][e] = __uint_as_float(0x7FFFFFFFu);
                                if (s1) o[c][2 + e] = __uint_as_float(0x7FFFFFFFu);
                            }
                        }
                }
            };
            put_back(s.L - s.T + 1, s.L);
            if (a.window > 0) put_back(s.first, min(s.L - a.window, s.L - s.T + 1));
        }
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);

        // The warps' shares of the keys joined: row r of key group k at [k][r], its 16-byte pieces turned by the row and the column, so that a write's
        // lanes meet all banks.
        const int here = min(M, rows - at.slab * M);
        auto piece_at = [&](int r, int piece) { return piece ^ ((((VB == 8 ? piece / 2 : piece % 32 / 4) >> 1) & 3) + 4 * (r & 1)); };
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = wr * 16 + g + 8 * h;
            if (r < here) {
                float* to = mg + (size_t)(wk * a.rows + r) * DP;
#pragma unroll
                for (int c = 0; c < NT; c += 4)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<float4*>(to + 4 * piece_at(r, dim(c, 2 * t + e) / 4)) = make_float4(o[c][2 * h + e], o[c + 1][2 * h + e], o[c + 2][2 * h + e], o[c + 3][2 * h + e]);
                if (t == 0) { s_ml[wk][r][0] = h ? m1 : m0; s_ml[wk][r][1] = h ? l1 : l0; }
            }
        }
        compute_sync();
        const bool whole = (int)(seg_end - seg_begin) == s.tiles;
        const size_t slot = (size_t)blockIdx.x * 2 + (seg_begin == lo ? 0 : 1);
        for (int e = threadIdx.x; e < here * (D / 4); e += 128) {
            const int r = e / (D / 4), piece = e - r * (D / 4);
            float mm = -INFINITY;
#pragma unroll
            for (int k = 0; k < WK; ++k) mm = fmaxf(mm, s_ml[k][r][0]);
            const float base = mm == -INFINITY ? 0.f : mm;
            float sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < WK; ++k) {
                const float f = power2(s_ml[k][r][0] - base);
                const float4 x = *reinterpret_cast<const float4*>(mg + (size_t)(k * a.rows + r) * DP + 4 * piece_at(r, piece));
                sum = fmaf(s_ml[k][r][1], f, sum);
                acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
            }
            if (whole) {
                const int row = at.slab * M + r, i = row / group;
                __nv_bfloat162* to = reinterpret_cast<__nv_bfloat162*>(a.out + ((size_t)(first_token + i) * a.nq + (size_t)at.kvh * group + (row - i * group)) * D + 4 * piece);
                if (sum == 0.f) { acc = make_float4(0.f, 0.f, 0.f, 0.f); sum = 1.f; }
                const float f = 1.f / sum;
                to[0] = __floats2bfloat162_rn(acc.x * f, acc.y * f);
                to[1] = __floats2bfloat162_rn(acc.z * f, acc.w * f);
            } else {
                *reinterpret_cast<float4*>(a.ws_o + (slot * M + r) * D + 4 * piece) = acc;
                if (piece == 0) { a.ws_ml[(slot * M + r) * 2] = mm; a.ws_ml[(slot * M + r) * 2 + 1] = sum; }
            }
        }
        compute_sync();
    }
}

int slab_rows(long long max_rows, int D) { return D > 128 || max_rows <= 16 ? 16 : max_rows <= 32 ? 32 : 64; }
int sm_blocks(int D) { return D > 128 ? 1 : 2; }

struct Call {
    Args8 a;
    CUtensorMap k, v;
    int max_new;
    cudaStream_t stream;
};

template <int DP, int MT, int BLOCKS> int launch(const Call& c) {
    constexpr int M = 16 * MT;
    const int bytes = Smem8<DP>::bytes(c.a.D, 4 / MT, c.a.rows);
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(attention8_kernel<DP, MT, BLOCKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem8<DP>::bytes(DP, 4 / MT, M));
        if (e != cudaSuccess) return ti_fail("attention8: %s", cudaGetErrorString(e));
        configured = true;
    }
    const int G = BLOCKS * ti_sm_count();
    ti_launch(attention8_kernel<DP, MT, BLOCKS>, dim3(G), dim3(A8_THREADS), bytes, c.stream, c.k, c.v, c.a);
    if (int rc = ti_check_launch("attention8")) return rc;
    join_parts(c.a.out, c.a.cu, c.a.kv_lens, c.a.ws_o, c.a.ws_ml, c.a.B, c.a.nq, c.a.nkv, c.a.D, M, c.max_new, c.a.window, G, c.stream);
    return ti_check_launch("attention8_join");
}
template <int DP> int launch_rows(const Call& c, long long max_rows) {
    const int M = slab_rows(max_rows, c.a.D);
    if constexpr (DP > 128) return launch<DP, 1, 1>(c);
    else return M == 16 ? launch<DP, 1, 2>(c) : M == 32 ? launch<DP, 2, 2>(c) : launch<DP, 4, 2>(c);
}

}  // namespace

// Bytes of the work space: two slots of rows a block.
extern "C" long long ti_attention8_workspace(int B, int max_new, int nq, int nkv, int D, int max_len) {
    if (B <= 0 || max_new <= 0 || nq <= 0 || nkv <= 0 || D <= 0) return 0;
    const long long rows = max_new * (long long)(nq / nkv), slots = 2LL * sm_blocks(D) * ti_sm_count();
    return slots * slab_rows(rows, D) * (D + 2) * 4;
}

// q [n, nq, D] and out [n, nq * D]; pools [pages, nkv, 64, D] with scales [pages, nkv]; the tokens of sequence b are cu[b] to cu[b + 1], at most max_new;
// kv_lens[b] its length with them, at most max_len; its pages are row seq_slots[b] of table. `status`: the word of bounded waits. Returns 2 for sizes
// outside what it takes.
extern "C" int ti_attention8(void* out, const void* q, const void* k, const void* v, const float* k_scales, const float* v_scales, const int* table,
                             int table_stride, const int* seq_slots, const int* cu, const int* kv_lens, void* ws, long long ws_bytes, int* status, float scale,
                             int B, int n, int nq, int nkv, int D, int page_size, int max_new, int max_len, int pages, int window, cudaStream_t stream) {
    if (B == 0 || n == 0 || max_new == 0) return 0;
    TI_REQUIRE(B > 0 && n > 0 && max_new > 0 && nq > 0 && nkv > 0 && D > 0 && window >= 0 && pages > 0, "attention8: %d sequences, %d new tokens, %d / %d heads of %d", B,
               max_new, nq, nkv, D);
    TI_REQUIRE(scale > 0.f, "attention8: scale must be positive");
    const long long rows = max_new * (long long)(nq / nkv), M = slab_rows(rows, D);
    if (page_size != AF_PAGE || D > 256 || D % 16 != 0 || nq % nkv != 0 || nkv > 65535 ||
        (rows + M - 1) / M * nkv * table_stride * (B < A8_MAX_SEQS ? B : A8_MAX_SEQS) >= 1LL << 31) {
        ti_fail("attention8 takes pages of %d, heads of a multiple of 16 up to 256 and fewer than 2^31 tiles of %d keys; got pages of %d, %d sequences of up to %d pages, %d new "
                "tokens, %d / %d heads of %d", AF_PAGE, AF_PAGE, page_size, B, table_stride, max_new, nq, nkv, D);
        return 2;
    }
    if ((long long)pages * nkv * (D / 2) > 0x7fffffffLL) {
        ti_fail("attention8: a pool of %d pages of %d heads has more than 2^31 rows", pages, nkv);
        return 2;
    }
    TI_REQUIRE(status != nullptr && aligned16(k) && aligned16(v), "attention8: pages must be 16-byte aligned");
    TI_REQUIRE(((uintptr_t)q | (uintptr_t)out) % 4 == 0, "attention8: queries and outputs must be 4-byte aligned (two elements are moved at a time)");
    const long long need = ti_attention8_workspace(B, max_new, nq, nkv, D, max_len);
    TI_REQUIRE(ws != nullptr && aligned16(ws) && ws_bytes >= need, "attention8: work space of %lld bytes, %lld needed", ws_bytes, need);
    Call c;
    c.max_new = max_new;
    c.stream = stream;
    // A page's head as rows of 64 numbers of 16 bits, moved as they are.
    const unsigned long long dims[2] = {64, (unsigned long long)pages * nkv * (D / 2)}, strides[1] = {128};
    const unsigned box[2] = {64, (unsigned)D / 2};
    if (int rc = ti_tensor_map_bf16(&c.k, k, 2, dims, strides, box, true)) return rc;
    if (int rc = ti_tensor_map_bf16(&c.v, v, 2, dims, strides, box, true)) return rc;
    const long long slots = 2LL * sm_blocks(D) * ti_sm_count();
    for (int b0 = 0; b0 < B; b0 += A8_MAX_SEQS) {            // the sequences in turns of as many as a launch takes
        c.a = Args8{(bf16*)out, (const bf16*)q, (const unsigned char*)v, k_scales, v_scales, table, table_stride, seq_slots + b0, cu + b0, kv_lens + b0, (float*)ws,
                    (float*)ws + slots * M * D, status, scale * 1.4426950408889634f, B - b0 < A8_MAX_SEQS ? B - b0 : A8_MAX_SEQS, nq, nkv, D, window, (int)(rows < M ? rows : M),
                    pages, n};
        if (int rc = D <= 64 ? launch_rows<64>(c, rows) : D <= 128 ? launch_rows<128>(c, rows) : launch_rows<256>(c, rows)) return rc;
    }
    return 0;
}
