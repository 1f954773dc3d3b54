// Attention of a few new tokens of every sequence over the paged cache, in bfloat16: the step that tests a drafted run. The new tokens'
// keys and values are in the cache already; token i of a sequence's T stands at position L - T + i, and sees the keys up to itself (and, with a
// window, the window's last ones only).
//
//   out[i, h] = sum_j softmax_j(scale q[i, h] k[j]) v[j], over the visible j.
//
// Bound by reading the cache once, so the T x (query heads per KV head) rows that share a KV head are the rows of the MMA tiles (slabs of 16,
// 32 or 64), and the work is shared out by length: the units, 64-key tiles of all (sequence, KV head, slab), are numbered in that order, and every
// resident block takes an equal run of them, whatever the sequences' lengths. A block that does a whole item writes its rows; the parts of an
// item that several blocks share are left in 32-bit (maximum, sum, unnormalised output) and joined by a second kernel in ascending order.
//
// Four warps share a tile out as MT groups of 16 rows x 4 / MT groups of keys. Scores, the running maximum and sum, and the output stand in
// 32-bit; P is rounded to bfloat16 as the operand of P V alone (its sum is not), O once: outputs are off by 2.1e-3 to 2.3e-3 of their size, where O's
// own rounding makes 1.7e-3. A tile's keys and values beyond the sequence's end or before the first visible key may hold anything: their scores are
// replaced and their values zeroed. An infinite or NaN value of a key that some rows see and others do not (a drafted token's own) reaches the rows
// that see it alone.
//
// 5 tokens after 65,531 (32 / 8 heads of 128, 268 MB) 53.5 us, 5.0 TB/s; 64 x 4 tokens after 1,024 61 us, 4.4 TB/s with the joins of two or three parts an
// item; 8 x 8 tokens after up to 32,768 (64 / 8 heads: slabs of 64 rows) 124 us, 1.44 of the bytes' time: the softmax's instructions beside the MMAs.
#include "even_runs.cuh"
#include "mma_util.cuh"
#include "tcgen05.cuh"
#include "tensor_map.h"

#define AF_PAGE 64
#define AF_THREADS 128
#define AF_MAX_SEQS 512                  // of one launch: their lengths, slots and units stand in shared memory

struct FewShape {
    int T, L, first, t0, tiles, slabs;                       // new tokens, length, first visible key, first tile, tiles, slabs of rows
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
template <int D> struct FewSmem {
    // Two tiles in flight a block, and as many blocks an SM as the registers let in: 65,536 keys of one sequence, 5 tokens, 32 / 8 heads of 128, took
    // 67.4 us with three stages and 62.3 with two, which leave room for the joining kernel beside it; heads of 32 took 35 us in two blocks and 27.6 in
    // three, heads of 128 62 in two and 66 in three (whose parts are more).
    static constexpr int STAGES = 2, BLOCKS = D <= 64 ? 3 : D <= 128 ? 2 : 1;
    static constexpr int TILE = AF_PAGE * D;
    // Heads of whole 64 elements come by TMA, as columns of [64 keys, 64 elements] in rows of 128 swizzled bytes; others by 16-byte copies.
    static constexpr bool TMA = D % 64 == 0;
    static constexpr size_t BYTES = (size_t)STAGES * 2 * TILE * sizeof(bf16) + (TMA ? 1024 : 0);
};
// The 16-byte piece c of key `row` in a tile, in elements.
template <int D> __device__ __forceinline__ int few_at(int row, int c) {
    if (FewSmem<D>::TMA) return (c >> 3) * (AF_PAGE * 64) + row * 64 + (((c & 7) ^ (row & 7)) << 3);
    return (row * (D / 8) + swz<D>(row, c)) * 8;
}
// Two bfloat16 numbers with 0 in the place of an infinity or NaN.
__device__ __forceinline__ unsigned finite_pair(unsigned pair) {
    return ((pair & 0x7F80u) == 0x7F80u ? 0u : pair & 0xFFFFu) | ((pair & 0x7F800000u) == 0x7F800000u ? 0u : pair & 0xFFFF0000u);
}
// Below 2^-126: 0.
__device__ __forceinline__ float power2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int D, int MT>
__global__ void __launch_bounds__(AF_THREADS, FewSmem<D>::BLOCKS) attention_few_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                                     const __grid_constant__ CUtensorMap map_v, bf16* out, const bf16* q,
                                                                                     const bf16* k_cache, const bf16* v_cache, const int* block_table, int table_stride, const int* seq_slots,
                                                                                     const int* cu, const int* kv_lens, float* ws_o, float* ws_ml, int* status, float scale_log2e, int B, int nq, int nkv, int window) {
    constexpr int M = 16 * MT, WK = 4 / MT, KS = D / 16, NT = D / 8, CPR = D / 8;
    typedef FewSmem<D> SM;
    extern __shared__ __align__(128) unsigned char af_smem[];
    __shared__ unsigned s_units[AF_MAX_SEQS + 1], s_scan[AF_THREADS / 32];
    __shared__ int s_cu[AF_MAX_SEQS + 1], s_len[AF_MAX_SEQS], s_slot[AF_MAX_SEQS];
    __shared__ float s_ml[WK][M][2];
    __shared__ __align__(8) unsigned long long s_full[SM::STAGES];
    bf16* ring = reinterpret_cast<bf16*>(af_smem + (SM::TMA ? (1024u - (smem_u32(af_smem) & 1023u)) & 1023u : 0u));
    if (SM::TMA && threadIdx.x == 0) {                       // the barriers below stand between this and the first use
        for (int s = 0; s < SM::STAGES; ++s) tc::mbar_init(smem_u32(s_full + s), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const int group = nq / nkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wr = warp % MT, wk = warp / MT;

    // Units before every sequence.
    unsigned carry = 0;
    for (int b0 = 0; b0 < B; b0 += AF_THREADS) {
        const int b = b0 + threadIdx.x;
        unsigned v = 0;
        if (b < B) {
            const int at = __ldcg(cu + b), end = __ldcg(cu + b + 1), len = __ldcg(kv_lens + b);
            s_slot[b] = __ldcg(seq_slots + b);
            s_cu[b] = at;
            if (b == B - 1) s_cu[B] = end;
            s_len[b] = len;
            const FewShape s = few_shape(end - at, len, window, group, M);
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
        for (int w = 0; w < AF_THREADS / 32; ++w) {
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
        int a = 0, z = B;                                    // the last sequence with units before it <= u and units of its own
        while (z - a > 1) {
            const int mid = (a + z) >> 1;
            if (s_units[mid] <= u) a = mid; else z = mid;
        }
        p.b = a;
        p.s = few_shape(s_cu[a + 1] - s_cu[a], s_len[a], window, group, M);
        const int v = (int)(u - s_units[a]), item = v / p.s.tiles;
        p.tile = v - item * p.s.tiles;
        p.kvh = item / p.s.slabs;
        p.slab = item - p.kvh * p.s.slabs;
        return p;
    };

    // What is asked for next: its place, and its page one tile ahead of its copies.
    bool waited = false;
    auto wait_once = [&] {
        if (!waited) { pdl_enter(); waited = true; }
    };
    unsigned next_u = lo;
    Place next{};
    int next_page = 0;
    const int* next_table = nullptr;
    auto enter = [&] {
        if (next_u < hi) {
            next = locate(next_u);
            next_table = block_table + (size_t)s_slot[next.b] * table_stride + next.s.t0;
            next_page = __ldcg(next_table + next.tile);
        }
    };
    enter();
    int fill = 0;
    auto issue = [&] {
        if (next_u < hi) {
            // Tiles with new keys were written by the kernel before this one; the others stand since earlier steps.
            if ((next.s.t0 + next.tile + 1) * AF_PAGE > next.s.L - next.s.T) wait_once();
            bf16* dst = ring + (size_t)fill * 2 * SM::TILE;
            if (SM::TMA) {
                if (threadIdx.x == 0) {
                    const unsigned bar = smem_u32(s_full + fill);
                    const int row = (next_page * nkv + next.kvh) * AF_PAGE;
                    tc::mbar_expect_tx(bar, 2 * SM::TILE * sizeof(bf16));
#pragma unroll
                    for (int c = 0; c < D / 64; ++c) {
                        tc::tma_load_2d(smem_u32(dst + c * (AF_PAGE * 64)), &map_k, c * 64, row, bar);
                        tc::tma_load_2d(smem_u32(dst + SM::TILE + c * (AF_PAGE * 64)), &map_v, c * 64, row, bar);
                    }
                }
            } else {
                const size_t base = ((size_t)next_page * nkv + next.kvh) * SM::TILE;
                for (int c = threadIdx.x; c < AF_PAGE * CPR; c += AF_THREADS) {
                    const int at = few_at<D>(c / CPR, c % CPR);
                    cp_async16(smem_u32(dst + at), k_cache + base + (size_t)c * 8);
                    cp_async16(smem_u32(dst + SM::TILE + at), v_cache + base + (size_t)c * 8);
                }
            }
            ++next_u;
            if (++next.tile == next.s.tiles) enter();
            else if (next_u < hi) next_page = __ldcg(next_table + next.tile);
        }
        fill = fill == SM::STAGES - 1 ? 0 : fill + 1;
        if (!SM::TMA) cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < SM::STAGES; ++s) issue();
    wait_once();

    int stage = 0;
    unsigned phase = 0;
    bool ok = true;
    unsigned u = lo;
    while (ok && u < hi) {
        // One segment: the tiles of one item that lie in this block's run.
        const Place at = locate(u);
        const FewShape& s = at.s;
        const unsigned seg_begin = u, seg_end = min(hi, u + (unsigned)(s.tiles - at.tile));
        const int rows = s.T * group, first_token = s_cu[at.b];
        int pos[2], low[2];
        const bf16* qrow[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = at.slab * M + wr * 16 + g + 8 * h, i = r / group;
            const bool real = r < rows;
            pos[h] = real ? s.L - s.T + i : -1;
            low[h] = window > 0 ? max(0, pos[h] - window + 1) : 0;
            qrow[h] = real ? q + ((size_t)(first_token + i) * nq + (size_t)at.kvh * group + (r - i * group)) * D : nullptr;
        }
        unsigned qf[KS][4];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = ks * 16 + 2 * t;
            qf[ks][0] = qrow[0] != nullptr ? __ldcg(reinterpret_cast<const unsigned*>(qrow[0] + d)) : 0u;
            qf[ks][1] = qrow[1] != nullptr ? __ldcg(reinterpret_cast<const unsigned*>(qrow[1] + d)) : 0u;
            qf[ks][2] = qrow[0] != nullptr ? __ldcg(reinterpret_cast<const unsigned*>(qrow[0] + d + 8)) : 0u;
            qf[ks][3] = qrow[1] != nullptr ? __ldcg(reinterpret_cast<const unsigned*>(qrow[1] + d + 8)) : 0u;
        }
        float o[NT][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

        bool odd = false;
        int tile = s.t0 + at.tile;
        for (; u < seg_end; ++u, ++tile) {
            if (SM::TMA) ok = tc::mbar_wait(smem_u32(s_full + stage), phase, status, 28);
            else {
                cp_async_wait<SM::STAGES - 1>();
                __syncthreads();
            }
            bf16* kt = ring + (size_t)stage * 2 * SM::TILE;
            bf16* vt = kt + SM::TILE;
            if (++stage == SM::STAGES) { stage = 0; phase ^= 1; }
            const int key_base = tile * AF_PAGE;
            if (key_base + AF_PAGE > s.L || key_base < s.first) {          // values that nobody sees may be infinite or NaN: 0 x those is NaN
                for (int c = threadIdx.x; c < AF_PAGE * CPR; c += AF_THREADS) {
                    const int row = c / CPR, key = key_base + row;
                    if (key >= s.L || key < s.first) *reinterpret_cast<uint4*>(vt + few_at<D>(row, c % CPR)) = make_uint4(0, 0, 0, 0);
                }
                if (SM::TMA) tc::fence_async_smem();
                __syncthreads();
            }
            // A tile at the run's or the window's edge holds keys that some rows see and others do not. 0 x infinity and 0 x NaN are NaN, so a warp takes such
            // values out of its share of the tile and adds them at the segment's end, to the rows that see them. (Warps of other rows take out the same.)
            const bool edge = key_base + AF_PAGE > s.L - s.T + 1 || (window > 0 && key_base < s.L - window);
            if (edge && s.T > 1) {
                const int share = key_base + wk * MT * 16;
                bool found = false;
                auto take_out = [&](int from, int to) {      // keys from `from` up to `to`, as far as they lie in the share
                    const int first = max(from - share, 0), count = (min(to - share, MT * 16) - first) * CPR;
                    for (int c = lane; c < count; c += 32) {
                        uint4* at16 = reinterpret_cast<uint4*>(vt + few_at<D>(wk * MT * 16 + first + c / CPR, c % CPR));
                        const uint4 v = *at16, f = make_uint4(finite_pair(v.x), finite_pair(v.y), finite_pair(v.z), finite_pair(v.w));
                        if ((v.x ^ f.x) | (v.y ^ f.y) | (v.z ^ f.z) | (v.w ^ f.w)) { *at16 = f; found = true; }
                    }
                };
                take_out(s.L - s.T + 1, s.L);
                if (window > 0) take_out(s.first, s.L - window);
                if (SM::TMA && found) tc::fence_async_smem();
                odd |= __any_sync(0xffffffffu, found);
                __syncwarp();
            }
            float sc[2 * MT][4];
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[i][j] = 0.f;
            const int mat = lane >> 3, r8 = lane & 7;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int nb = 0; nb < MT; ++nb) {
                    const int row = (wk * MT + nb) * 16 + (mat >> 1) * 8 + r8;
                    unsigned kb[4];
                    ldmatrix_x4(kb, smem_u32(kt + few_at<D>(row, 2 * ks + (mat & 1))));
                    mma16816(sc[2 * nb], qf[ks], kb[0], kb[1]);
                    mma16816(sc[2 * nb + 1], qf[ks], kb[2], kb[3]);
                }
            // Maxima of the unscaled scores (the scale, which is positive, is taken with the exponent); a tile at an edge has its scores replaced first.
            float mx0 = -INFINITY, mx1 = -INFINITY;
            const int key0 = key_base + wk * MT * 16 + 2 * t;
            if (edge) {
#pragma unroll
                for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int key = key0 + 8 * i + j;
                        if (key > pos[0] || key < low[0]) sc[i][j] = -INFINITY;
                        if (key > pos[1] || key < low[1]) sc[i][2 + j] = -INFINITY;
                    }
            }
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) {
                mx0 = fmaxf(mx0, fmaxf(sc[i][0], sc[i][1]));
                mx1 = fmaxf(mx1, fmaxf(sc[i][2], sc[i][3]));
            }
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
            const float n0 = fmaxf(m0, mx0 * scale_log2e), n1 = fmaxf(m1, mx1 * scale_log2e);
            const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
            if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {             // most tiles leave the maxima, and then the sums, as they are
                const float c0 = power2(m0 - b0), c1 = power2(m1 - b1);
                l0 *= c0; l1 *= c1;
#pragma unroll
                for (int i = 0; i < NT; ++i) { o[i][0] *= c0; o[i][1] *= c0; o[i][2] *= c1; o[i][3] *= c1; }
            }
            m0 = n0; m1 = n1;
#pragma unroll
            for (int nb = 0; nb < MT; ++nb) {
                unsigned pf[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float* x = sc[2 * nb + h];
                    x[0] = power2(fmaf(x[0], scale_log2e, -b0)); x[1] = power2(fmaf(x[1], scale_log2e, -b0));
                    x[2] = power2(fmaf(x[2], scale_log2e, -b1)); x[3] = power2(fmaf(x[3], scale_log2e, -b1));
                    l0 += x[0] + x[1];
                    l1 += x[2] + x[3];
                    pf[2 * h] = pack_bf16(x[0], x[1]);
                    pf[2 * h + 1] = pack_bf16(x[2], x[3]);
                }
                const int row = (wk * MT + nb) * 16 + (mat & 1) * 8 + r8;
#pragma unroll
                for (int c = 0; c < NT; c += 2) {
                    unsigned vb[4];
                    ldmatrix_x4_trans(vb, smem_u32(vt + few_at<D>(row, c + (mat >> 1))));
                    mma16816(o[c], pf, vb[0], vb[1]);
                    mma16816(o[c + 1], pf, vb[2], vb[3]);
                }
            }
            // The stage is filled again as soon as all have left it, before the next tile is waited for. A barrier alone does not keep the copies, which are
            // another proxy's, behind reads that a warp has asked for and not yet used: without the fence a few of a hundred thousand items met the
            // next but one tile's values.
            if (SM::TMA) tc::fence_async_smem();
            ok = __syncthreads_and(ok);
            if (!ok) break;
            if (u + 1 < seg_end) issue();
        }
        if (!ok) break;
        if (s.T > 1 && __syncthreads_or(odd)) {              // what was taken out (by any warp): infinite or NaN whatever its weight
            auto put_back = [&](int from, int to) {
                for (int key = max(from, (s.t0 + at.tile) * AF_PAGE); key < min(to, tile * AF_PAGE); ++key) {
                    if ((key % AF_PAGE) / (MT * 16) != wk) continue;
                    const int page = __ldcg(block_table + (size_t)s_slot[at.b] * table_stride + key / AF_PAGE);
                    const bf16* value = v_cache + (((size_t)page * nkv + at.kvh) * AF_PAGE + key % AF_PAGE) * D + 2 * t;
                    const bool s0 = key <= pos[0] && key >= low[0], s1 = key <= pos[1] && key >= low[1];
#pragma unroll
                    for (int c = 0; c < NT; ++c) {
                        const unsigned v = __ldcg(reinterpret_cast<const unsigned*>(value + 8 * c)), e = v ^ finite_pair(v);         // 0 for what stayed
                        const float e0 = __uint_as_float(e << 16), e1 = __uint_as_float(e & 0xFFFF0000u);
                        if (s0) { o[c][0] += e0; o[c][1] += e1; }
                        if (s1) { o[c][2] += e0; o[c][3] += e1; }
                    }
                }
            };
            put_back(s.L - s.T + 1, s.L);
            if (window > 0) put_back(s.first, min(s.L - window, s.L - s.T + 1));
        }
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);

        // The warps' shares of the keys joined, in the stage that the segment's last tile has left (it is filled again after that): row r of key group
        // k at [k][r], its columns turned by 8 r so that a quad's neighbours meet other banks.
        float* mg = reinterpret_cast<float*>(ring + (size_t)(stage == 0 ? SM::STAGES - 1 : stage - 1) * 2 * SM::TILE);
        {
            float* a = mg + (size_t)(wk * M + wr * 16 + g) * D;
            float* b = a + 8 * D;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int col = ((i + g) % NT) * 8 + 2 * t;
                *reinterpret_cast<float2*>(a + col) = make_float2(o[i][0], o[i][1]);
                *reinterpret_cast<float2*>(b + col) = make_float2(o[i][2], o[i][3]);
            }
            if (t == 0) {
                s_ml[wk][wr * 16 + g][0] = m0; s_ml[wk][wr * 16 + g][1] = l0;
                s_ml[wk][wr * 16 + g + 8][0] = m1; s_ml[wk][wr * 16 + g + 8][1] = l1;
            }
        }
        __syncthreads();
        const bool whole = (int)(seg_end - seg_begin) == s.tiles;
        const size_t slot = (size_t)blockIdx.x * 2 + (seg_begin == lo ? 0 : 1);
        const int here = min(M, rows - at.slab * M);
        for (int e = threadIdx.x; e < here * D; e += AF_THREADS) {
            const int r = e / D, d = e - r * D, col = (d + 8 * (r & 7)) % D;
            float mm = -INFINITY;
#pragma unroll
            for (int k = 0; k < WK; ++k) mm = fmaxf(mm, s_ml[k][r][0]);
            const float base = mm == -INFINITY ? 0.f : mm;
            float sum = 0.f, acc = 0.f;
#pragma unroll
            for (int k = 0; k < WK; ++k) {
                const float f = exp2f(s_ml[k][r][0] - base);
                sum += s_ml[k][r][1] * f;
                acc += mg[(size_t)(k * M + r) * D + col] * f;
            }
            if (whole) {
                const int row = at.slab * M + r, i = row / group;
                out[((size_t)(first_token + i) * nq + (size_t)at.kvh * group + (row - i * group)) * D + d] = __float2bfloat16_rn(sum == 0.f ? 0.f : acc / sum);
            } else {
                ws_o[(slot * M + r) * D + d] = acc;
                if (d == 0) { ws_ml[(slot * M + r) * 2] = mm; ws_ml[(slot * M + r) * 2 + 1] = sum; }
            }
        }
        if (SM::TMA) tc::fence_async_smem();
        __syncthreads();
        issue();
    }
    if (!SM::TMA) cp_async_wait<0>();
    if (!ok) tc::drain_after_timeout();                      // a wait ran out: let what is in flight land
}

// The parts of the rows that several blocks share, joined in ascending order: AF_JOIN_WARPS / WPR rows a block, WPR warps a row, four elements a lane,
// every WPRth part a warp. Rows of items that one block did are done; rows without keys get zeros. What bounds it is one dependent load after another
// with the kernel before gone: so where the parts lie is worked out before that kernel ends, and maxima, sums and outputs of eight parts are asked
// for together.
#define AF_JOIN_WARPS 4
template <int WPR>
__global__ void __launch_bounds__(32 * AF_JOIN_WARPS) attention_few_join_kernel(bf16* out, const int* cu, const int* kv_lens, const float* ws_o,
                                                                                const float* ws_ml, int B, int nq, int nkv, int D, int M, int window,
                                                                                int blocks) {
    __shared__ unsigned s_sum[AF_JOIN_WARPS][2];
    __shared__ float4 s_o[WPR > 1 ? WPR : 1][32];
    __shared__ float2 s_ml[WPR];
    const int b = blockIdx.z, kvh = blockIdx.y, group = nq / nkv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned before = 0, U = 0;
    for (int c = threadIdx.x; c < B; c += 32 * AF_JOIN_WARPS) {
        const FewShape s = few_shape(__ldcg(cu + c + 1) - __ldcg(cu + c), __ldcg(kv_lens + c), window, group, M);
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
    const int first_token = __ldcg(cu + b), T = __ldcg(cu + b + 1) - first_token, row = blockIdx.x * (AF_JOIN_WARPS / WPR) + warp / WPR, mine = warp % WPR;
    const FewShape s = few_shape(T, __ldcg(kv_lens + b), window, group, M);
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
            mm = top;
            sum = sum * old + warp_sum(x.y * f);
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
                sum = fmaf(s_ml[w].y, f, sum);
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

static int few_rows(int max_rows, int D) { return D > 128 || max_rows <= 16 ? 16 : max_rows <= 32 ? 32 : 64; }
static int few_blocks(int D) { return (D <= 64 ? 3 : D <= 128 ? 2 : 1) * ti_sm_count(); }

// Bytes of the work space: two slots of rows a block.
extern "C" long long ti_attention_few_workspace(int B, int max_new, int nq, int nkv, int D) {
    if (B <= 0 || max_new <= 0 || nq <= 0 || nkv <= 0 || D <= 0) return 0;
    const long long M = few_rows(max_new * (nq / nkv), D), slots = 2LL * few_blocks(D);
    return slots * M * (D + 2) * 4;
}

template <int D, int MT>
static int launch_few(bf16* out, const bf16* q, const bf16* k, const bf16* v, const int* table, int table_stride, const int* seq_slots, const int* cu,
                      const int* kv_lens, void* ws, int* status, float scale, int B, int nq, int nkv, int max_new, int pages, int window, cudaStream_t stream) {
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(attention_few_kernel<D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FewSmem<D>::BYTES);
        if (e != cudaSuccess) return ti_fail("attention_few: %s", cudaGetErrorString(e));
        configured = true;
    }
    constexpr int M = 16 * MT;
    const int G = few_blocks(D);
    float* ws_o = (float*)ws;
    float* ws_ml = ws_o + (size_t)2 * G * M * D;
    CUtensorMap map_k = {}, map_v = {};
    if (FewSmem<D>::TMA) {
        const unsigned long long dims[2] = {(unsigned long long)D, (unsigned long long)pages * nkv * AF_PAGE}, strides[1] = {(unsigned long long)D * 2};
        const unsigned box[2] = {64, AF_PAGE};
        if (int rc = ti_tensor_map_bf16(&map_k, k, 2, dims, strides, box, true)) return rc;
        if (int rc = ti_tensor_map_bf16(&map_v, v, 2, dims, strides, box, true)) return rc;
    }
    ti_launch(attention_few_kernel<D, MT>, dim3(G), dim3(AF_THREADS), FewSmem<D>::BYTES, stream, map_k, map_v, out, q, k, v, table, table_stride, seq_slots, cu,
              kv_lens, ws_o, ws_ml, status, scale * 1.4426950408889634f, B, nq, nkv, window);
    if (int rc = ti_check_launch("attention_few")) return rc;
    const int rows = max_new * (nq / nkv);
    // More than eight parts an item: four warps a row (59.9 us in place of 62.3 at 37 parts; at two parts 90 in place of 70).
    const bool deep = 8LL * B * nkv * ((rows + M - 1) / M) < G;
    ti_launch(deep ? attention_few_join_kernel<4> : attention_few_join_kernel<1>, dim3(deep ? rows : (rows + AF_JOIN_WARPS - 1) / AF_JOIN_WARPS, nkv, B),
              dim3(32 * AF_JOIN_WARPS), 0, stream, out, cu, kv_lens, ws_o, ws_ml, B, nq, nkv, D, M, window, G);
    return ti_check_launch("attention_few_join");
}

// q [tokens, nq, D] and out [tokens, nq * D]; the tokens of sequence b are cu[b] to cu[b + 1], at most max_new; kv_lens[b] its length with them; its
// pages are row seq_slots[b] of block_table (of a pool of `pages`). `status`: the word of bounded waits. `ws`: ti_attention_few_workspace bytes, 16-byte aligned. Returns 2 for sizes outside what it takes.
extern "C" int ti_attention_few(void* out, const void* q, const void* k_cache, const void* v_cache, const int* block_table, int table_stride,
                                const int* seq_slots, const int* cu, const int* kv_lens, void* ws, long long ws_bytes, int* status, float scale, int B, int nq,
                                int nkv, int D, int page_size, int max_new, int pages, int window, cudaStream_t stream) {
    if (B == 0 || max_new == 0) return 0;
    TI_REQUIRE(B > 0 && max_new > 0 && nq > 0 && nkv > 0 && D > 0 && window >= 0, "attention_few: %d sequences, %d new tokens, %d / %d heads of %d", B,
               max_new, nq, nkv, D);
    TI_REQUIRE(scale > 0.f, "attention_few: scale must be positive");
    const int M = few_rows(max_new * (nq / nkv), D);
    const long long slabs = (max_new * (long long)(nq / nkv) + M - 1) / M;
    if (page_size != AF_PAGE || nq % nkv != 0 || nkv > 65535 || slabs * nkv * table_stride * (B < AF_MAX_SEQS ? B : AF_MAX_SEQS) >= 1LL << 31) {
        ti_fail("attention_few takes pages of %d and fewer than 2^31 tiles of %d keys; got pages of %d, %d sequences of up to %d pages, %d new tokens, %d / %d heads",
                AF_PAGE, AF_PAGE, page_size, B, table_stride, max_new, nq, nkv);
        return 2;
    }
    TI_REQUIRE(status != nullptr && aligned16(k_cache) && aligned16(v_cache), "attention_few: pages must be 16-byte aligned");
    TI_REQUIRE(((uintptr_t)q | (uintptr_t)out) % 4 == 0, "attention_few: queries and outputs must be 4-byte aligned (two elements are moved at a time)");
    if ((long long)pages * nkv * AF_PAGE > 0x7fffffffLL) {
        ti_fail("attention_few: a pool of %d pages of %d heads has more than 2^31 rows", pages, nkv);
        return 2;
    }
    TI_REQUIRE(ws != nullptr && aligned16(ws) && ws_bytes >= ti_attention_few_workspace(B, max_new, nq, nkv, D), "attention_few: work space of %lld bytes, %lld needed",
               ws_bytes, ti_attention_few_workspace(B, max_new, nq, nkv, D));
    for (int b0 = 0; b0 < B; b0 += AF_MAX_SEQS) {            // the sequences in turns of as many as a launch takes
        const int n = B - b0 < AF_MAX_SEQS ? B - b0 : AF_MAX_SEQS;
        int rc;
#define AF_LAUNCH(d, mt) \
    rc = launch_few<d, mt>((bf16*)out, (const bf16*)q, (const bf16*)k_cache, (const bf16*)v_cache, block_table, table_stride, seq_slots + b0, cu + b0, kv_lens + b0, ws, \
                             status, scale, n, nq, nkv, max_new, pages, window, stream)
#define AF_CASE(d)                                   \
    case d:                                          \
        if (M == 16) AF_LAUNCH(d, 1);                \
        else if (M == 32) AF_LAUNCH(d, 2);           \
        else AF_LAUNCH(d, 4);                        \
        break;
        switch (D) {
            AF_CASE(16) AF_CASE(32) AF_CASE(48) AF_CASE(64) AF_CASE(80) AF_CASE(96) AF_CASE(112) AF_CASE(128)
            case 256: AF_LAUNCH(256, 1); break;
            default:
                ti_fail("attention_few has no instance for head size %d", D);
                return 2;
        }
        if (rc) return rc;
    }
    return 0;
#undef AF_CASE
#undef AF_LAUNCH
}
