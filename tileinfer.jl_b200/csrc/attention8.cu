// Attention over the paged cache in 8 bits (cache8.cu), bfloat16 queries and results: one to some tens of new tokens of every sequence. The new tokens'
// keys and values are in the cache already; token i of a sequence's T stands at position L - T + i, and sees the keys up to itself (and, with a window, the
// window's last ones only).
//
//   out[i, h] = sum_j softmax_j(scale q[i, h] . sk[p(j)] ck[j]) sv[p(j)] cv[j], over the visible j; p(j) is j's page.
//
// Bound by reading the cache once, so the T x (query heads per KV head) rows that share a KV head go together (slabs of up to 24), and the work is shared out by
// length (attention_parts.cuh). A page's head is one tile, 64 x D consecutive bytes of keys and as many of values, which come as two TMA copies of
// rows of 128 swizzled bytes, whatever D is. A warp asks for them and brings the scales; four others take 16 keys of a tile each, on their own.
//
// Measured, heads of 128: one row over 65,536 positions 31.4 us (134 MB, 20.5 at the rate of a copy; 131,072 more positions take 40.7 us more, 6.6 TB/s, so that 11 us
// are launches, the first look-ups and reads, and the join); 64 sequences of 1,024 35.9 us (3.8 TB/s: the same, and 2,000 cycles a tile in each of three blocks an SM);
// 40 rows over 8 of up to 32,768 139.8 us (2.0 TB/s): a tile's chain of MMAs, exponentials and MMAs with two warps a scheduler, and codes widened twice, for two slabs.
//
// Keys and values are the MMAs' rows, the queries their columns, eight at a time: S^T = K Q^T, O^T = V^T P^T, so that a code is widened once whatever the
// number of queries, and eight or fewer cost eight. P^T's fragments are S^T's, turned by movmatrix.
//
// Codes are widened in registers to numbers of 16 bits, exactly (one instruction for two; values of four keys are first put side by side, one for two
// more). Queries are scaled by a power of two a row, so that they fit those numbers without loss. Keys' dimensions are permuted alike in both operands, so that a
// lane's share of four MMAs is 16 consecutive bytes; so are the keys, so that a warp's reads meet all banks.
//
// With z_j = (the score in base 2) + log2 sv[p(j)] and m near the maximum of z so far, P = 2^(z - m + 7) are the weights of the values' codes, rounded to 16
// bits (2^-11) as the MMA's operand, and the denominator is the 32-bit sum of P / sv. So pages of unequal scales (a page of zeros has 2^-100) cost an addition to the
// exponent. m stays until a z is more than 8 above it (P <= 2^15), so that most tiles exchange no maxima. Scores, sums and outputs stand in 32-bit.
//
// The denominator holds for value scales from 2^-100 to 2^120. With s the score without log2 sv, its terms are 2^(s - m + 7) in units of 2^10: between 2^-123 and some 2^125
// for the largest of a row. P / sv loses a term where P, below 2^-126, becomes zero: in a tile whose log2 sv is at most 90 below the largest so far, m <= max s + that
// largest, so that a lost term is below 2^-43 of the row's largest one. In other tiles, which the asking warp marks, the terms are computed from s. Sums are brought to
// another m in two steps of half the power, as the power alone may vanish where the sum times it does not. (Without these steps a page of zeros left the denominator beside
// values of 10^13; with them 40 rows over up to 32,768 positions take 140.0 us in place of 137.6, one row as long as before.)
//
// Keys and values beyond the sequence's end or before the first visible key may hold any codes: their scores are replaced and their values' codes are
// zero. A NaN code of a key that some rows see and others do not (a drafted token's own) reaches the rows that see it alone.
#include "attention_parts.cuh"
#include "e4m3.cuh"
#include "linear8.cuh"
#include "mma_util.cuh"

#include <climits>
#include <cmath>

namespace {

constexpr int A8_THREADS = 160, A8_MAX_SEQS = 256;           // four warps that compute, one that asks; sequences of one launch
constexpr float P_POWER = 7.f, SLACK = 8.f;
constexpr float SUM_UNIT = 0x1p-10f;                         // of denominators
constexpr unsigned SCALES_APART = 90;                        // beyond so many powers of two a tile's denominator has exponentials of its own

// DP: D rounded up to 64, 128 or 256. NQ: queries in eights.
template <int DP, int NQ> struct Shape8 {
    static constexpr int M = 8 * NQ, STAGES = 3, BLOCKS = DP > 128 ? 1 : NQ == 1 ? 3 : 2;
    // More than eight queries lie in shared memory (the outputs take the registers): [eight][64 dimensions][half][lane].
    static constexpr bool Q_SHARED = NQ > 1;
    static constexpr int Q = Q_SHARED ? NQ * (DP / 64) * 2 * 32 * 16 : 0;
    // Stages, queries, then the warps' shares of an item: [warp][row][DP].
    static __host__ __device__ int bytes(int D) { return STAGES * 2 * AF_PAGE * D + Q + 4 * M * DP * 4 + 1024; }
};

struct Args8 {
    bf16* out;
    const bf16* q;
    const unsigned char* v;                                  // for NaN codes that were taken out
    const float *k_scales, *v_scales;
    const int* table;
    int table_stride, slots, columns;
    FewLimits limits;
    const int *seq_slots, *cu, *kv_lens;
    float *ws_o, *ws_ml;
    int* status;
    float scale_log2e;
    int B, nq, nkv, D, window, pages;
};

// Byte i of a tile of swizzled 128-byte rows.
__device__ __forceinline__ int tile_at(int i) { return (i & ~0x70) | ((i ^ (i >> 3)) & 0x70); }
// 0xFF in the places of NaN codes.
__device__ __forceinline__ unsigned nan_codes(unsigned w) { return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu); }
// A sum times 2^x, x <= 0, also where 2^x alone is below 2^-126.
__device__ __forceinline__ float scaled(float sum, float x) {
    const float half = power2(0.5f * x);
    return sum * half * half;
}
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// An 8 x 8 matrix of 16-bit numbers, two of a row a lane, turned.
__device__ __forceinline__ unsigned turned(unsigned x) {
    unsigned r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// EXACT: D is DP, so that a lane's places in a tile are the same in every sixteen keys.
template <int DP, int NQ, bool EXACT>
__global__ void __launch_bounds__(A8_THREADS, Shape8<DP, NQ>::BLOCKS) attention8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                                        const Args8 a) {
    typedef Shape8<DP, NQ> S;
    constexpr int M = S::M, KH = DP / 64, MT = DP / 16, STAGES = S::STAGES;
    // Bytes of a key's values that a lane reads at once, and how often.
    constexpr int VB = DP == 64 ? 8 : 16, VH = DP == 256 ? 2 : 1;
    extern __shared__ __align__(128) unsigned char smem_dyn[];
    __shared__ unsigned s_units[A8_MAX_SEQS + 1], s_scan[A8_THREADS / 32];
    __shared__ int s_cu[A8_MAX_SEQS + 1], s_len[A8_MAX_SEQS], s_slot[A8_MAX_SEQS];
    __shared__ float s_ml[4][M][2], s_row[M];                                           // s_row: a row's factor of its scores
    __shared__ float4 s_scale[64];                           // of the run's tiles in turn: sk, log2 sv, SUM_UNIT / sv, below zero where sv lies apart
    __shared__ __align__(8) unsigned long long bars[2 * STAGES];
    unsigned char* ring = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    const int D = EXACT ? DP : a.D, tile_bytes = AF_PAGE * D, B = a.B, nkv = a.nkv, group = a.nq / nkv;
    const unsigned full0 = smem_u32(bars), empty0 = full0 + 8 * STAGES;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { tc::mbar_init(full0 + 8 * s, 2); tc::mbar_init(empty0 + 8 * s, 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

    // Units before every sequence.
    unsigned carry = 0;
    for (int b0 = 0; b0 < B; b0 += A8_THREADS) {
        const int b = b0 + threadIdx.x;
        unsigned v = 0;
        if (b < B) {
            const int at = a.limits.row(__ldcg(a.cu + b)), end = a.limits.row(__ldcg(a.cu + b + 1)), len = a.limits.length(__ldcg(a.kv_lens + b));
            const int slot = __ldcg(a.seq_slots + b);
            s_slot[b] = slot < a.slots ? slot : -1;          // a slot that does not exist has no pages
            s_cu[b] = at;
            if (b == B - 1) s_cu[B] = end;
            s_len[b] = len;
            const FewShape s = few_shape(a.limits.run(end - at), len, a.window, group, M);
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
        p.s = few_shape(a.limits.run(s_cu[x + 1] - s_cu[x]), s_len[x], a.window, group, M);
        const int v = (int)(u - s_units[x]), item = v / p.s.tiles;
        p.tile = v - item * p.s.tiles;
        p.kvh = item / p.s.slabs;
        p.slab = item - p.kvh * p.s.slabs;
        return p;
    };

    if (warp == 4) {
        // ---------------------------------------------------------------- copies: lane 0 asks; the lanes look up the pages of 32 tiles at once, and of the next 32
        // meanwhile, and hand the tiles' scales over, which need not be there when a tile is asked for
        struct Ahead {
            int block;                                       // the tile's page and head, -1 beyond the pool
            bool fresh, scaled;                              // with new keys; its scales are here
            float sk, sv;
        };
        bool ok = true, waited = false, placed = false;      // placed: all scales that are here have been handed over
        unsigned phase = 0;
        int stage = 0, pending = 0;                          // tiles asked for and not yet handed over
        auto look = [&](unsigned u) {
            Ahead x = {-1, false, true, 1.f, 1.f};
            if (u >= hi) return x;
            const Place p = locate(u);
            const int tile = p.s.t0 + p.tile, slot = s_slot[p.b];
            const int page = slot >= 0 && tile < a.columns ? __ldcg(a.table + (size_t)slot * a.table_stride + tile) : -1;
            // Tiles with new keys were written by the kernel before this one; the others stand since earlier steps.
            x.fresh = (tile + 1) * AF_PAGE > p.s.L - p.s.T;
            if (page >= 0 && page < a.pages) { x.block = page * nkv + p.kvh; x.scaled = false; }                     // a page that does not exist reads as zeros
            return x;
        };
        auto scales = [&](Ahead& x) {
            if (x.scaled || (x.fresh && !waited)) return;
            x.sk = __ldcg(a.k_scales + x.block);
            x.sv = __ldcg(a.v_scales + x.block);
            x.scaled = true;
        };
        unsigned top = 0;                                    // the largest exponent of sv of the tiles before these 32
        auto place = [&](const Ahead& x, unsigned u0) {
            const unsigned e = __float_as_uint(x.sv) >> 23;
            bool apart = false;
            if (max(top, __reduce_max_sync(0xffffffffu, x.scaled ? e : 0u)) > __reduce_min_sync(0xffffffffu, x.scaled ? e : 255u) + SCALES_APART) {
                unsigned largest = x.scaled ? max(e, top) : top;             // up to this tile: scales that are not here yet are those of later ones
#pragma unroll 1
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned v = __shfl_up_sync(0xffffffffu, largest, o);
                    if (lane >= o) largest = max(largest, v);
                }
                apart = e + SCALES_APART < largest;
            }
            const float inv = SUM_UNIT / x.sv;
            if (x.scaled) s_scale[(u0 - lo + lane) % 64] = make_float4(x.sk, __log2f(x.sv), apart ? -inv : inv, 0.f);
            __syncwarp();
            for (; pending > 0; --pending)
                if (lane == 0) tc::mbar_arrive(full0 + 8 * (stage < pending ? stage - pending + STAGES : stage - pending));
            placed = true;
        };
        Ahead now = look(lo + lane), then;
        for (unsigned u0 = lo; ok && u0 < hi; u0 += 32) {
            scales(now);
            if (u0 != lo) place(now, u0);
            then = look(u0 + 32 + lane);
            for (int i = 0; i < 32 && u0 + i < hi; ++i) {
                if (i == 8) scales(then);
                if (!waited && __shfl_sync(0xffffffffu, now.fresh, i)) {
                    pdl_wait();
                    waited = true;
                    placed = false;
                    scales(now);
                }
                if (pending == STAGES) place(now, u0);
                const int block = __shfl_sync(0xffffffffu, now.block, i);
                if (lane == 0) {
                    ok = tc::mbar_wait(empty0 + 8 * stage, phase ^ 1, a.status, 29);
                    if (ok) {
                        const unsigned bar = full0 + 8 * stage, to = smem_u32(ring) + stage * 2 * tile_bytes;
                        tc::mbar_expect_tx(bar, 2 * tile_bytes);
                        tc::tma_load_2d(to, &map_k, 0, block * (D / 2), bar);
                        tc::tma_load_2d(to + tile_bytes, &map_v, 0, block * (D / 2), bar);
                        if (placed) tc::mbar_arrive(bar);
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;
                if (!placed) ++pending;
                if (++stage == STAGES) { stage = 0; phase ^= 1; }
            }
            if (pending > 0) place(now, u0);
            top = max(top, __reduce_max_sync(0xffffffffu, __float_as_uint(now.sv) >> 23));
            now = then;
        }
        if (!ok) tc::drain_after_timeout();                  // a wait ran out: let what is in flight land
        __syncwarp();
        return;
    }

    pdl_enter();
    // Row r of sixteen keys is key r, with its bit 2 turned where r is odd: neighbouring rows then lie in different halves of the banks.
    const int key_g = g ^ ((g & 1) << 2), key_t0 = 2 * t, key_t1 = (2 * t + 1) ^ 4;
    const int share = warp * 16;                             // this warp's first key of a tile
    // A lane's places in sixteen keys: pieces of its two keys, values of its four.
    int k_at[2][KH], v_at[4][VH];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int kh = 0; kh < KH; ++kh) k_at[i][kh] = tile_at((share + 8 * i + key_g) * D + (t + 4 * kh) * 16);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int vh = 0; vh < VH; ++vh) {
            const int byte = (share + 8 * (e >> 1) + (e & 1 ? key_t1 : key_t0)) * D + vh * 128 + g * VB;
            v_at[e][vh] = tile_at(byte & ~15) | (byte & 15);
        }
    int stage = 0;
    unsigned phase = 0;
    bool ready = false;
    bool ok = true;                                          // once a wait has run out, all that is left is to meet the other warps
    unsigned u = lo;
    uint4* sq = reinterpret_cast<uint4*>(ring + STAGES * 2 * tile_bytes);
    float* mg = reinterpret_cast<float*>(ring + STAGES * 2 * tile_bytes + S::Q);
    while (u < hi) {
        // One segment: the tiles of one item that lie in this block's run.
        const Place at = locate(u);
        const FewShape& s = at.s;
        const unsigned seg_begin = u, seg_end = min(hi, u + (unsigned)(s.tiles - at.tile));
        const int rows = s.T * group, first_token = s_cu[at.b];
        // Queries as columns: column g of an eight; with a power of two taken out of a row, its numbers fit 16 bits without loss.
        unsigned qf[S::Q_SHARED ? 1 : KH][4][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            if (S::Q_SHARED && (n & 3) != warp) continue;    // the warps take the eights in turn
            const int r = at.slab * M + 8 * n + g, i = r / group;
            const bool real = r < rows;
            const bf16* row = a.q + ((size_t)(first_token + i) * a.nq + (size_t)at.kvh * group + (r - i * group)) * D;
            unsigned raw[KH][4][2];
            float top = 0.f;
#pragma unroll
            for (int kh = 0; kh < KH; ++kh) {
                const int d = (t + 4 * kh) * 16;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const unsigned w = real && (EXACT || d < D) ? __ldcg(reinterpret_cast<const unsigned*>(row + d + 4 * j + 2 * e)) : 0u;
                        raw[kh][j][e] = w;
                        top = fmaxf(top, fmaxf(finite_size(__uint_as_float(w << 16)), finite_size(__uint_as_float(w & 0xFFFF0000u))));
                    }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int power = max((int)(__float_as_uint(top) >> 23) - 127, -100) - 14;           // the row's largest becomes 2^14 to 2^15
            if (t == 0) s_row[8 * n + g] = power_of_two(power) * a.scale_log2e;                  // with one eight all warps write the same
            const float inverse = power_of_two(-power);
#pragma unroll
            for (int kh = 0; kh < KH; ++kh) {
                unsigned f[4][2];
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const unsigned w = raw[kh][j][e];
                        f[j][e] = pack_f16(__uint_as_float(w << 16) * inverse, __uint_as_float(w & 0xFFFF0000u) * inverse);
                        if (!S::Q_SHARED) qf[kh][j][e] = f[j][e];
                    }
                if (S::Q_SHARED) {
                    sq[((n * KH + kh) * 2) * 32 + lane] = make_uint4(f[0][0], f[0][1], f[1][0], f[1][1]);
                    sq[((n * KH + kh) * 2 + 1) * 32 + lane] = make_uint4(f[2][0], f[2][1], f[3][0], f[3][1]);
                }
            }
        }
        compute_sync();
        float rf[NQ][2];                                     // of columns 2 t and 2 t + 1
#pragma unroll
        for (int n = 0; n < NQ; ++n) { rf[n][0] = s_row[8 * n + 2 * t]; rf[n][1] = s_row[8 * n + 2 * t + 1]; }
        float o[NQ][MT][4], m[NQ][2], l[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][i][j] = 0.f;
        }
        // Columns' positions and first visible keys, wanted at edges alone.
        auto column = [&](int n, int e, int& pos, int& low) {
            const int r = at.slab * M + 8 * n + 2 * t + e;
            pos = r < rows ? s.L - s.T + r / group : -1;
            low = a.window > 0 ? max(0, pos - a.window + 1) : 0;
        };

        // Whether the next tile is there, asked while this one's values are worked on; after them where their registers leave no room (64 sequences of 1,024,
        // one row: not ahead 38.4 us, after 37.8, before 36.5; eight of up to 32,768, 40 rows: 145, 138.5, 149).
        constexpr bool EARLY = NQ == 1 && DP <= 128;
        auto ask_next = [&] {
            const bool wraps = stage + 1 == STAGES;
            ready = tc::mbar_test(full0 + 8 * (wraps ? 0 : stage + 1), wraps ? phase ^ 1 : phase, lane == 0);
        };
        bool odd = false;
        int tile = s.t0 + at.tile;
        for (; u < seg_end; ++u, ++tile) {
            if (ok) ok = tc::warp_wait_after(ready, full0 + 8 * stage, phase, lane == 0, a.status, 28);
            if (!ok) continue;
            const unsigned char* kt = ring + stage * 2 * tile_bytes;
            const unsigned char* vt = kt + tile_bytes;
            const float4 scales = s_scale[(u - lo) % 64];
            const float sk = scales.x, lv = scales.y;
            float inv = scales.z;
            const int key_base = tile * AF_PAGE + share;
            float sc[NQ][4];
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[n][j] = 0.f;
#pragma unroll
            for (int kh = 0; kh < KH; ++kh) {
                const bool there = EXACT || (t + 4 * kh) * 16 < D;
                const uint4 k0 = there ? *reinterpret_cast<const uint4*>(kt + k_at[0][kh]) : make_uint4(0, 0, 0, 0);
                const uint4 k1 = there ? *reinterpret_cast<const uint4*>(kt + k_at[1][kh]) : make_uint4(0, 0, 0, 0);
                const unsigned w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
                for (int jj = 0; jj < 2; ++jj) {
                    uint4 y[NQ];
                    if (S::Q_SHARED)
#pragma unroll
                        for (int n = 0; n < NQ; ++n) y[n] = sq[((n * KH + kh) * 2 + jj) * 32 + lane];
#pragma unroll
                    for (int j = 2 * jj; j < 2 * jj + 2; ++j) {
                        const unsigned f[4] = {e4m3_half2((unsigned short)w0[j]), e4m3_half2((unsigned short)w1[j]), e4m3_half2((unsigned short)(w0[j] >> 16)),
                                               e4m3_half2((unsigned short)(w1[j] >> 16))};
#pragma unroll
                        for (int n = 0; n < NQ; ++n) {
                            if (S::Q_SHARED) mma16816_f16(sc[n], f, j & 1 ? y[n].z : y[n].x, j & 1 ? y[n].w : y[n].y);
                            else mma16816_f16(sc[n], f, qf[kh][j][0], qf[kh][j][1]);
                        }
                    }
                }
            }
            // A tile at an edge has scores replaced: of keys that a row does not see.
            const bool edge = (tile + 1) * AF_PAGE > s.L - s.T + 1 || (a.window > 0 && tile * AF_PAGE < s.L - a.window);
            if (edge) {
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        int pos, low;
                        column(n, e, pos, low);
                        if (key_base + key_g > pos || key_base + key_g < low) sc[n][e] = -INFINITY;
                        if (key_base + 8 + key_g > pos || key_base + 8 + key_g < low) sc[n][2 + e] = -INFINITY;
                    }
            }
            bool above = inv < 0.f;                          // or a tile whose denominator is apart
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    sc[n][j] = fmaf(sc[n][j], fmaxf(rf[n][j & 1] * sk, 1.1754944e-38f), lv);           // off zero: a score of -inf stays one
                    above |= sc[n][j] > m[n][j & 1] + SLACK;
                }
            if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(m[n][e], fmaxf(sc[n][e], sc[n][2 + e]));
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                        const float down = m[n][e] - (top == -INFINITY ? 0.f : top), by = power2(down);
                        m[n][e] = top;
                        l[n][e] = scaled(l[n][e], down);
#pragma unroll
                        for (int i = 0; i < MT; ++i) { o[n][i][e] *= by; o[n][i][2 + e] *= by; }
                        if (inv < 0.f) {                     // 2^(s - m + 7) is up to 2^115: ten powers more leave room at the other end
                            const float base = (top == -INFINITY ? 0.f : top - P_POWER) + lv - 10.f;
                            l[n][e] = fmaf(power2(sc[n][e] - base) + power2(sc[n][2 + e] - base), SUM_UNIT * 0x1p-10f, l[n][e]);
                        }
                    }
                inv = fmaxf(inv, 0.f);
            }
            unsigned pf[NQ][2];
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const float b0 = m[n][0] == -INFINITY ? 0.f : m[n][0] - P_POWER, b1 = m[n][1] == -INFINITY ? 0.f : m[n][1] - P_POWER;
                const float p0 = power2(sc[n][0] - b0), p1 = power2(sc[n][1] - b1), p2 = power2(sc[n][2] - b0), p3 = power2(sc[n][3] - b1);
                l[n][0] = fmaf(p0 + p2, inv, l[n][0]);
                l[n][1] = fmaf(p1 + p3, inv, l[n][1]);
                pf[n][0] = turned(pack_f16(p0, p1));
                pf[n][1] = turned(pack_f16(p2, p3));
            }
            if (EARLY) ask_next();
#pragma unroll
            for (int vh = 0; vh < VH; ++vh) {
                // A lane's four keys: 16 (8, twice 16) bytes of each.
                unsigned w[4][VB / 4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool there = EXACT || vh * 128 + g * VB < D;
                    if (VB == 16) {
                        const uint4 v = there ? *reinterpret_cast<const uint4*>(vt + v_at[e][vh]) : make_uint4(0, 0, 0, 0);
                        w[e][0] = v.x; w[e][1] = v.y; w[e][VB / 4 - 2] = v.z; w[e][VB / 4 - 1] = v.w;
                    } else {
                        const uint2 v = there ? *reinterpret_cast<const uint2*>(vt + v_at[e][vh]) : make_uint2(0, 0);
                        w[e][0] = v.x; w[e][1] = v.y;
                    }
                }
                if (edge) {
                    // Values that nobody sees may have any code, and 0 x NaN is NaN; NaN codes that some rows see and others do not are added at the segment's end.
                    // Those that all rows see stay.
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key_base + 8 * (e >> 1) + (e & 1 ? key_t1 : key_t0);
                        const bool seen = key < s.L && key >= s.first, some = key > s.L - s.T || (a.window > 0 && key < s.L - a.window);
#pragma unroll
                        for (int j = 0; j < VB / 4; ++j) {
                            if (!seen) w[e][j] = 0;
                            else if (some) {
                                const unsigned bad = nan_codes(w[e][j]);
                                odd |= bad != 0;
                                w[e][j] &= ~bad;
                            }
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < VB / 4; ++j) {
                    // Side by side: bytes of the keys at k = 2 t and 2 t + 1, and of those eight further on. Rows g and g + 8 are a lane's neighbouring dimensions.
                    const unsigned a01 = __byte_perm(w[0][j], w[1][j], 0x5140), a23 = __byte_perm(w[0][j], w[1][j], 0x7362);
                    const unsigned b01 = __byte_perm(w[2][j], w[3][j], 0x5140), b23 = __byte_perm(w[2][j], w[3][j], 0x7362);
                    const unsigned f0[4] = {e4m3_half2((unsigned short)a01), e4m3_half2((unsigned short)(a01 >> 16)), e4m3_half2((unsigned short)b01),
                                            e4m3_half2((unsigned short)(b01 >> 16))};
                    const unsigned f1[4] = {e4m3_half2((unsigned short)a23), e4m3_half2((unsigned short)(a23 >> 16)), e4m3_half2((unsigned short)b23),
                                            e4m3_half2((unsigned short)(b23 >> 16))};
                    const int i = vh * 8 + 2 * j;
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        mma16816_f16(o[n][i], f0, pf[n][0], pf[n][1]);
                        mma16816_f16(o[n][i + 1], f1, pf[n][0], pf[n][1]);
                    }
                }
            }
            if (!EARLY) ask_next();
            tc::fence_async_smem();                          // the stage's next copies are another proxy's than these reads
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(empty0 + 8 * stage);
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        // The dimension of row g (h: g + 8) of results i: VB consecutive ones a lane.
        auto dim = [&](int i, int h) { return (i / 8) * 128 + g * VB + 2 * (i % 8) + h; };
        if (ok && __any_sync(0xffffffffu, odd)) {            // what this warp has taken out: NaN whatever its weight
            auto put_back = [&](int from, int to) {
                for (int key = max(from, (s.t0 + at.tile) * AF_PAGE); key < min(to, tile * AF_PAGE); ++key) {
                    if (key % AF_PAGE / 16 != warp) continue;
                    const int slot = s_slot[at.b], page = slot >= 0 && key / AF_PAGE < a.columns ? __ldcg(a.table + (size_t)slot * a.table_stride + key / AF_PAGE) : -1;
                    if (page < 0 || page >= a.pages) continue;
                    const unsigned char* value = a.v + (((size_t)page * nkv + at.kvh) * AF_PAGE + key % AF_PAGE) * D;
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            int pos, low;
                            column(n, e, pos, low);
                            if (key > pos || key < low) continue;
#pragma unroll
                            for (int i = 0; i < MT; ++i)
#pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    if (dim(i, h) < D && (__ldcg(value + dim(i, h)) & 0x7F) == 0x7F) o[n][i][2 * h + e] = __uint_as_float(0x7FFFFFFFu);
                        }
                }
            };
            put_back(s.L - s.T + 1, s.L);
            if (a.window > 0) put_back(s.first, min(s.L - a.window, s.L - s.T + 1));
        }

        // The warps' shares of the keys joined: row r of warp w at [w][r], its 16-byte pieces turned by the row, so that a write's lanes meet other banks.
        const int here = min(M, rows - at.slab * M);
        auto piece_at = [](int r, int piece) { return piece ^ ((r >> 1) & 3); };
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = l[n][e];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                const int r = 8 * n + 2 * t + e;
                if (r >= here) continue;
                float* to = mg + (size_t)(warp * M + r) * DP;
#pragma unroll
                for (int i = 0; i < MT; i += 2)
                    *reinterpret_cast<float4*>(to + 4 * piece_at(r, dim(i, 0) / 4)) = make_float4(o[n][i][e], o[n][i][2 + e], o[n][i + 1][e], o[n][i + 1][2 + e]);
                if (g == 0) { s_ml[warp][r][0] = m[n][e]; s_ml[warp][r][1] = sum; }
            }
        compute_sync();
        const bool whole = (int)(seg_end - seg_begin) == s.tiles;
        const size_t slot = (size_t)blockIdx.x * 2 + (seg_begin == lo ? 0 : 1);
        for (int e = threadIdx.x; e < here * (D / 4); e += 128) {
            const int r = e / (D / 4), piece = e - r * (D / 4);
            float mm = -INFINITY;
#pragma unroll
            for (int k = 0; k < 4; ++k) mm = fmaxf(mm, s_ml[k][r][0]);
            const float base = mm == -INFINITY ? 0.f : mm;
            float sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float f = power2(s_ml[k][r][0] - base);
                sum += scaled(s_ml[k][r][1], s_ml[k][r][0] - base);
                const float4 x = *reinterpret_cast<const float4*>(mg + (size_t)(k * M + r) * DP + 4 * piece_at(r, piece));
                acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
            }
            acc.x *= SUM_UNIT; acc.y *= SUM_UNIT; acc.z *= SUM_UNIT; acc.w *= SUM_UNIT;
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

// Queries in eights of a slab: rows shared out evenly among as few slabs of 24 (heads beyond 128: of 16) as hold them.
int slab_eights(long long max_rows, int D) {
    const long long most = D > 128 ? 16 : 24, slabs = (max_rows + most - 1) / most;
    return (int)(((max_rows + slabs - 1) / slabs + 7) / 8);
}
int sm_blocks(int eights, int D) { return D > 128 ? 1 : eights == 1 ? 3 : 2; }

struct Call {
    Args8 a;
    CUtensorMap k, v;
    int max_new;
    cudaStream_t stream;
};

template <int DP, int NQ, bool EXACT> int launch(const Call& c) {
    typedef Shape8<DP, NQ> S;
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(attention8_kernel<DP, NQ, EXACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::bytes(DP));
        if (e != cudaSuccess) return ti_fail("attention8: %s", cudaGetErrorString(e));
        configured = true;
    }
    const int G = S::BLOCKS * ti_sm_count();
    ti_launch(attention8_kernel<DP, NQ, EXACT>, dim3(G), dim3(A8_THREADS), S::bytes(c.a.D), c.stream, c.k, c.v, c.a);
    if (int rc = ti_check_launch("attention8")) return rc;
    join_parts(c.a.out, c.a.cu, c.a.kv_lens, c.a.ws_o, c.a.ws_ml, c.a.B, c.a.nq, c.a.nkv, c.a.D, S::M, c.max_new, c.a.window, G, c.a.limits, c.stream);
    return ti_check_launch("attention8_join");
}
template <int DP, bool EXACT> int launch_rows(const Call& c, int eights) {
    if (eights == 1) return launch<DP, 1, EXACT>(c);
    if constexpr (DP <= 128)
        if (eights == 3) return launch<DP, 3, EXACT>(c);
    return launch<DP, 2, EXACT>(c);
}

}  // namespace

int cache_widen8(void* k_out, void* v_out, int* table_out, int* slots_out, int* lens_out, int* cu_out, const void* k, const void* v, const float* k_scales, const float* v_scales,
                 const int* table, int table_stride, int slots, int columns, const int* seq_slots, const int* cu, const int* kv_lens, int B, int n, int nkv, int D, int pages, int per_seq,
                 int window, cudaStream_t stream);
extern "C" int ti_attention_prefill_tc(void* out, const void* q, const void* k_cache, const void* v_cache, int n_pages, const int* block_table, int table_stride,
                                       const int* seq_slots, const int* cu_seqlens, const int* kv_lens, int n_seqs, int n_tokens, int total_blocks, float scale, int nq,
                                       int nkv, int D, int page_size, int window, int* status, cudaStream_t stream);
extern "C" int ti_attention_prefill(void* out, const void* q, const void* k_cache, const void* v_cache, const int* block_table, int table_stride, const int* seq_slots,
                                    const int* cu_seqlens, const int* kv_lens, int n_seqs, int total_tiles, float scale, int nq, int nkv, int D, int page_size, int window,
                                    cudaStream_t stream);
// Whether a step goes through pages widened to bfloat16 and the prompts' kernels, for heads of 64 and 128 on the fifth-generation tensor cores (attention_prefill_tc.cu),
// else with mma.sync (attention_prefill.cu): the shorter by estimates in microseconds, for sequences of max_len positions. Slabs: a slab's tile (heads of 128 4.8 ns;
// of the sizes between 6.4, up to 64 3.8, of 256 9.5), 57 ns for a slab's other work. Widened: a walk along the longest sequence (19 ns a position; with mma.sync 15 and
// 0.265 for each of the head's dimensions), rounds of the SMs, the widened bytes. Microseconds in turn, 32 / 8 heads of 128: one sequence, 64 new of 8,192 62 / 170,
// 128 of 1,024 30 / 32, 256 of 4,096 122 / 94, 2,048 of 4,096 1,212 / 139; four sequences, 32 of 512 25 / 25, 128 of 128 45 / 17. Heads of 96: 68 / 321, 32 / 45,
// 135 / 166, 1,316 / 504, 24 / 29, 43 / 15; of 256: 128 / 680, 55 / 96, 278 / 349, 3,394 / 1,057, 38 / 59, 86 / 31.
extern "C" int ti_attention8_widens(int B, int max_new, int nq, int nkv, int D, int max_len) {
    if (B <= 0 || nkv <= 0 || nq % nkv != 0 || (D != 256 && (D > 128 || D % 16 != 0)) || nq / nkv > 128 || B > 65535 || max_len <= 0 || max_new * (long long)(nq / nkv) <= 24)
        return 0;
    const bool fifth = D == 64 || D == 128;
    const double rows = max_new * (double)(nq / nkv), heads = (double)B * nkv, items = heads * ceil(rows / (D > 128 ? 16 : 24)), bytes = heads * max_len * D * 6 / 5e6;
    const double tile = fifth ? 4.8 * D / 128 : D < 64 ? 3.8 : D < 128 ? 6.4 : 9.5, size = fifth ? D / 128.0 : D < 64 ? 0.5 : 1.0;
    const double slabs = 5 + 0.001 * tile * items * (max_len / 64.0) + 0.057 * items * size;
    const double waves = heads * ceil(rows / (fifth ? 256 : 128)) / ti_sm_count(), walk = (fifth ? waves : ceil(waves)) * (max_len - 0.5 * max_new);
    return 11 + (fifth ? 0.0193 : 0.015 + 0.000265 * D) * (walk > max_len ? walk : max_len) + 2 * waves + bytes < slabs;
}
// Sequences whose pages are widened at once: as many as half a gigabyte holds, one at least.
static int widened_at_once(int B, int nkv, int D, int max_len) {
    const long long one = ((long long)max_len + AF_PAGE - 1) / AF_PAGE * nkv * AF_PAGE * D * 4, fit = one > 0 ? (1LL << 29) / one : B;
    return (int)(fit < 1 ? 1 : fit < B ? fit : B);
}
// Kernels of one call.
extern "C" int ti_attention8_launches(int B, int max_new, int nq, int nkv, int D, int max_len) {
    if (B <= 0 || max_new <= 0) return 0;
    const int turn = ti_attention8_widens(B, max_new, nq, nkv, D, max_len) ? widened_at_once(B, nkv, D, max_len) : A8_MAX_SEQS;
    return 2 * ((B - 1) / turn + 1);
}
static long long up16(long long bytes) { return (bytes + 15) / 16 * 16; }

// Bytes of the work space: two slots of rows a block, or the widened pages with their table.
extern "C" long long ti_attention8_workspace(int B, int max_new, int nq, int nkv, int D, int max_len) {
    if (B <= 0 || max_new <= 0 || nq <= 0 || nkv <= 0 || D <= 0) return 0;
    if (ti_attention8_widens(B, max_new, nq, nkv, D, max_len)) {
        const long long turn = widened_at_once(B, nkv, D, max_len), pages = turn * ((max_len + AF_PAGE - 1) / AF_PAGE);
        return pages * nkv * AF_PAGE * D * 4 + up16(4 * pages) + 2 * up16(4 * turn) + up16(4 * (turn + 1));
    }
    const int eights = slab_eights(max_new * (long long)(nq / nkv), D);
    return 2LL * sm_blocks(eights, D) * ti_sm_count() * 8 * eights * (D + 2) * 4;
}

// q [n, nq, D] and out [n, nq * D]; pools [pages, nkv, 64, D] with scales [pages, nkv]; the tokens of sequence b are cu[b] to cu[b + 1], at most max_new;
// kv_lens[b] its length with them, at most max_len; its pages are row seq_slots[b] of table (`slots` rows of `columns`, table_stride apart). Ranges beyond the n rows of q and out are cut to them, a
// length beyond a row of the table to that, and a slot that does not exist has no pages. `status`: the word of bounded waits. Returns 2 for sizes outside what it takes.
extern "C" int ti_attention8_table(void* out, const void* q, const void* k, const void* v, const float* k_scales, const float* v_scales, const int* table,
                                   int table_stride, const int* seq_slots, const int* cu, const int* kv_lens, void* ws, long long ws_bytes, int* status, float scale,
                                   int B, int n, int nq, int nkv, int D, int page_size, int max_new, int max_len, int pages, int window, int slots, int columns, cudaStream_t stream) {
    if (B == 0 || n == 0 || max_new == 0) return 0;
    TI_REQUIRE(B > 0 && n > 0 && max_new > 0 && nq > 0 && nkv > 0 && D > 0 && window >= 0 && pages > 0, "attention8: %d sequences, %d new tokens, %d / %d heads of %d", B,
               max_new, nq, nkv, D);
    TI_REQUIRE(slots >= 0 && columns >= 0 && table_stride >= 0, "attention8: a table of %d x %d", slots, columns);
    TI_REQUIRE(scale > 0.f, "attention8: scale must be positive");
    const long long rows = max_new * (long long)(nq / nkv);
    const int eights = nkv > 0 && nq % nkv == 0 ? slab_eights(rows, D) : 1, M = 8 * eights;
    if (page_size != AF_PAGE || D > 256 || D % 16 != 0 || nq % nkv != 0 || nkv > 65535 ||
        (rows + M - 1) / M * nkv * columns * (B < A8_MAX_SEQS ? B : A8_MAX_SEQS) >= 1LL << 31) {
        ti_fail("attention8 takes pages of %d, heads of a multiple of 16 up to 256 and fewer than 2^31 tiles of %d keys; got pages of %d, %d sequences of up to %d pages, %d new "
                "tokens, %d / %d heads of %d", AF_PAGE, AF_PAGE, page_size, B, columns, max_new, nq, nkv, D);
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
    if (ti_attention8_widens(B, max_new, nq, nkv, D, max_len)) {
        const int per_seq = (max_len + AF_PAGE - 1) / AF_PAGE, turn = widened_at_once(B, nkv, D, max_len);
        const long long all = (long long)turn * per_seq, pool = all * nkv * AF_PAGE * D;
        TI_REQUIRE(all * nkv * AF_PAGE <= 0x7fffffffLL, "attention8: %d positions of %d heads are too many for a long run", max_len, nkv);
        TI_REQUIRE(((uintptr_t)q | (uintptr_t)out) % 16 == 0, "attention8: queries and outputs of long runs must be 16-byte aligned");
        bf16 *k16 = (bf16*)ws, *v16 = k16 + pool;
        int *table16 = (int*)(v16 + pool), *slots16 = table16 + up16(4 * all) / 4, *lens16 = slots16 + up16(4LL * turn) / 4, *cu16 = lens16 + up16(4LL * turn) / 4;
        for (int b0 = 0; b0 < B; b0 += turn) {
            const int these = B - b0 < turn ? B - b0 : turn;
            if (int rc = cache_widen8(k16, v16, table16, slots16, lens16, cu16, k, v, k_scales, v_scales, table, table_stride, slots, columns, seq_slots + b0, cu + b0, kv_lens + b0, these, n, nkv,
                                      D, pages, per_seq, window, stream)) return rc;
            // As many blocks as the runs can need: those beyond leave at once.
            const bool fifth = D == 64 || D == 128;          // generation of tensor cores
            const int tokens = (fifth ? 2 : 1) * (128 / (nq / nkv)), blocks = n / tokens + (these < n ? these : n);
            const long long most = (long long)these * (((long long)max_new + tokens - 1) / tokens);
            const int grid = blocks < most ? blocks : (int)most;
            if (int rc = fifth ? ti_attention_prefill_tc(out, q, k16, v16, (int)all, table16, per_seq, slots16, cu16, lens16, these, n, grid, scale, nq, nkv, D, page_size,
                                                         window, status, stream)
                               : ti_attention_prefill(out, q, k16, v16, table16, per_seq, slots16, cu16, lens16, these, grid, scale, nq, nkv, D, page_size, window, stream)) return rc;
        }
        return 0;
    }
    Call c;
    c.max_new = max_new;
    c.stream = stream;
    // A page's head as rows of 64 numbers of 16 bits, moved as they are.
    const unsigned long long dims[2] = {64, (unsigned long long)pages * nkv * (D / 2)}, strides[1] = {128};
    const unsigned box[2] = {64, (unsigned)D / 2};
    if (int rc = ti_tensor_map_bf16(&c.k, k, 2, dims, strides, box, true)) return rc;
    if (int rc = ti_tensor_map_bf16(&c.v, v, 2, dims, strides, box, true)) return rc;
    const long long parts = 2LL * sm_blocks(eights, D) * ti_sm_count(), positions = (long long)columns * AF_PAGE;
    const FewLimits limits = {n, max_new, positions < INT_MAX / 2 ? (int)positions : INT_MAX / 2};
    for (int b0 = 0; b0 < B; b0 += A8_MAX_SEQS) {            // the sequences in turns of as many as a launch takes
        c.a = Args8{(bf16*)out, (const bf16*)q, (const unsigned char*)v, k_scales, v_scales, table, table_stride, slots, columns, limits, seq_slots + b0, cu + b0, kv_lens + b0, (float*)ws,
                    (float*)ws + parts * M * D, status, scale * 1.4426950408889634f, B - b0 < A8_MAX_SEQS ? B - b0 : A8_MAX_SEQS, nq, nkv, D, window, pages};
        if (int rc = D == 64 ? launch_rows<64, true>(c, eights) : D == 128 ? launch_rows<128, true>(c, eights) : D == 256 ? launch_rows<256, true>(c, eights) :
                     D < 64 ? launch_rows<64, false>(c, eights) : D < 128 ? launch_rows<128, false>(c, eights) : launch_rows<256, false>(c, eights)) return rc;
    }
    return 0;
}
// The same where every slot exists and a row has as many columns as its pitch.
extern "C" int ti_attention8(void* out, const void* q, const void* k, const void* v, const float* k_scales, const float* v_scales, const int* table,
                             int table_stride, const int* seq_slots, const int* cu, const int* kv_lens, void* ws, long long ws_bytes, int* status, float scale,
                             int B, int n, int nq, int nkv, int D, int page_size, int max_new, int max_len, int pages, int window, cudaStream_t stream) {
    return ti_attention8_table(out, q, k, v, k_scales, v_scales, table, table_stride, seq_slots, cu, kv_lens, ws, ws_bytes, status, scale, B, n, nq, nkv, D, page_size, max_new,
                               max_len, pages, window, INT_MAX, table_stride, stream);
}
