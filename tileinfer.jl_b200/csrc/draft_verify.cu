// Which drafted tokens stand, and the token after them.
//
// Sequence b brings c <= K drafted tokens d_0 .. d_{c-1}, each drawn from the draft's probabilities q_i, and uniform numbers u_0 .. u_K. Token
// d_i stands while u_i q_i(d_i) < p_i(d_i), p the model's probabilities at that place; a is the number that stand before the first that does
// not. The next token is drawn by u_K from the weights max(p_a - q_a, 0) after a refusal and from p_c where all stand, so that every token is
// distributed as one drawn from p. Without q a draft is a certainty: q_i(d_i) = 1 and 0 elsewhere.
//
// The draw is in whole numbers: a weight is round(w 2^40), the token the first whose cumulative weight reaches ceil(u_K total), at least 1.
// Sums of whole numbers do not depend on their order, so neither does the token on how a row is shared out. Differences that leave no weight
// (q >= p everywhere) give way to p itself; a row of p without weight gives the token -1, which no embedding takes.
//
// Bound by reading one row of p and, after a refusal, one of q: a row is shared out among blocks that each leave the weight of a stretch, and
// the block that arrives last finds the stretch and then the token (no block waits for another). 4 drafts over 131,072 tokens: 6.4 us for one sequence (two
// dependent passes in one launch), 20.3 us for 64 (67 MB in all: 3.3 TB/s, and the last blocks' second pass).
#include "sampling_rule.cuh"

#define DV_THREADS 256
#define DV_WARPS (DV_THREADS / 32)
#define DV_MAX_CHUNKS 256

// Inclusive scan over the block of one value per thread; `scratch`: DV_WARPS + 1 words, free again after the next barrier.
__device__ __forceinline__ u64 dv_scan(u64 v, u64* scratch, u64& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < DV_WARPS; ++w) {
        const u64 s = scratch[w];
        if (w < warp) before += s;
        all += s;
    }
    total = all;
    return v + before;
}

__global__ void __launch_bounds__(DV_THREADS) verify_drafts_kernel(int* accepted, int* tokens, const float* p, long long p_seq, long long p_row,
                                                                   const float* q, long long q_seq, long long q_row, const int* drafts,
                                                                   const float* uniforms, const int* counts, int K, int vocab, int per,
                                                                   u64* sums, unsigned* tickets) {
    __shared__ u64 scratch[DV_WARPS + 1];
    __shared__ int s_found;
    __shared__ bool s_last;
    const int b = blockIdx.y, chunk = blockIdx.x, chunks = gridDim.x, lane = threadIdx.x & 31;
    const float* pb = p + (size_t)b * p_seq;
    const float* qb = q != nullptr ? q + (size_t)b * q_seq : nullptr;
    pdl_enter();

    // Every warp finds the first refusal for itself.
    const int count = counts != nullptr ? min(max(__ldcg(counts + b), 0), K) : K;
    int stand = count;
    for (int i0 = 0; i0 < count; i0 += 32) {
        const int i = i0 + lane;
        bool refused = false;
        if (i < count) {
            const int d = __ldcg(drafts + (size_t)b * K + i);
            const float u = __ldcg(uniforms + (size_t)b * (K + 1) + i);
            float mine = 0.f, theirs = 1.f;
            if (d >= 0 && d < vocab) {
                mine = __ldcg(pb + (size_t)i * p_row + d);
                if (qb != nullptr) theirs = __ldcg(qb + (size_t)i * q_row + d);
            }
            refused = !(__fmul_rn(u, theirs) < mine);
        }
        const unsigned where = __ballot_sync(0xffffffffu, refused);
        if (where) { stand = i0 + __ffs(where) - 1; break; }
    }
    const float* pr = pb + (size_t)stand * p_row;
    const bool differs = stand < count;
    const float* qr = differs && qb != nullptr ? qb + (size_t)stand * q_row : nullptr;
    const int without = differs && qb == nullptr ? __ldcg(drafts + (size_t)b * K + stand) : -1;
    auto rest = [&](int v, float pv, float qv) { return fixed_parts(v == without ? pv - 1.f : pv - qv); };
    // Four neighbours of both rows, 0 beyond the end.
    auto load4 = [&](int v, int end, float4& a, float4& c) {
        a = c = make_float4(0.f, 0.f, 0.f, 0.f);
        if (v + 3 < end) {
            a = __ldcg(reinterpret_cast<const float4*>(pr + v));
            if (qr != nullptr) c = __ldcg(reinterpret_cast<const float4*>(qr + v));
        } else if (v < end) {
            a.x = __ldcg(pr + v);
            if (v + 1 < end) a.y = __ldcg(pr + v + 1);
            if (v + 2 < end) a.z = __ldcg(pr + v + 2);
            if (qr != nullptr) {
                c.x = __ldcg(qr + v);
                if (v + 1 < end) c.y = __ldcg(qr + v + 1);
                if (v + 2 < end) c.z = __ldcg(qr + v + 2);
            }
        }
    };

    const int lo = min(vocab, chunk * per), hi = min(vocab, lo + per);
    const bool wide = ((uintptr_t)pr & 15) == 0 && ((uintptr_t)qr & 15) == 0;
    u64 part = 0;
    if (wide) {
        for (int v0 = lo + 4 * threadIdx.x; v0 < hi; v0 += 16 * DV_THREADS) {
            float4 a[4], c[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) load4(v0 + u * 4 * DV_THREADS, hi, a[u], c[u]);
            int high = 0, low = 0;                           // sixteen of them fit 32 bits
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int v = v0 + u * 4 * DV_THREADS;
                const Fixed f0 = rest(v, a[u].x, c[u].x), f1 = rest(v + 1, a[u].y, c[u].y), f2 = rest(v + 2, a[u].z, c[u].z), f3 = rest(v + 3, a[u].w, c[u].w);
                high += f0.high + f1.high + f2.high + f3.high;
                low += f0.low + f1.low + f2.low + f3.low;
            }
            part += (u64)(((long long)high << 20) + low);
        }
    } else {
        for (int v = lo + threadIdx.x; v < hi; v += DV_THREADS) {
            const Fixed f = rest(v, __ldcg(pr + v), qr != nullptr ? __ldcg(qr + v) : 0.f);
            part += (u64)(((long long)f.high << 20) + f.low);
        }
    }
    u64 part_sum;
    dv_scan(part, scratch, part_sum);
    if (threadIdx.x == 0) {
        sums[(size_t)b * chunks + chunk] = part_sum;
        __threadfence();
        s_last = atomicAdd(&tickets[b], 1u) == (unsigned)chunks - 1;
        s_found = -1;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();

    // The stretch that holds the target, a thread a stretch.
    const bool in = (int)threadIdx.x < chunks;
    u64 w_part = in ? __ldcg(sums + (size_t)b * chunks + threadIdx.x) : 0, total;
    u64 through = dv_scan(w_part, scratch, total);
    const float u = __ldcg(uniforms + (size_t)b * (K + 1) + K);
    const u32 r24 = (u32)fminf(fmaxf(u, 0.f) * 16777216.f, 16777215.f);
    const bool plain = total == 0;                            // no weight in the differences (or none to take off): the weights of p itself
    if (plain) {
        u64 whole = 0;
        for (int v = threadIdx.x; v < vocab; v += DV_THREADS) whole += fixed_weight(__ldcg(pr + v));
        __syncthreads();
        dv_scan(whole, scratch, total);
    }
    u64 target = draw_target(total, r24);
    if (target == 0) target = 1;
    __shared__ u64 s_before;
    if (threadIdx.x == 0 && plain) { s_found = total ? 0 : -1; s_before = 0; }           // searched from its beginning
    if (!plain && in && through >= target && through - w_part < target) { s_found = (int)threadIdx.x; s_before = through - w_part; }
    __syncthreads();
    int next = -1;
    if (s_found >= 0) {                                       // uniform over the block
        int v0 = s_found * per;
        const int end = plain ? vocab : min(vocab, v0 + per);
        u64 cum = s_before;
        __syncthreads();
        // Sixteen tokens a thread at a time, in runs of four: the runs' sums scanned in order, then the run that reaches the target.
        for (; v0 < end && next < 0; v0 += 16 * DV_THREADS) {
            u64 w[4][4], sum[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int v = v0 + (k * DV_THREADS + (int)threadIdx.x) * 4;
                float4 a, c;
                if (wide) load4(v, end, a, c);
                else {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        e[i] = v + i < end ? __ldcg(pr + v + i) : 0.f;
                        e[4 + i] = v + i < end && qr != nullptr ? __ldcg(qr + v + i) : 0.f;
                    }
                    a = make_float4(e[0], e[1], e[2], e[3]); c = make_float4(e[4], e[5], e[6], e[7]);
                }
                const float av[4] = {a.x, a.y, a.z, a.w}, cv[4] = {c.x, c.y, c.z, c.w};
                sum[k] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const Fixed f = plain ? fixed_parts(av[i]) : rest(v + i, av[i], cv[i]);
                    w[k][i] = (u64)(((long long)f.high << 20) + f.low);
                    sum[k] += w[k][i];
                }
            }
            if (threadIdx.x == 0) s_found = -1;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                u64 all_in, before = cum + dv_scan(sum[k], scratch, all_in) - sum[k];
                if (before < target && before + sum[k] >= target) {                      // one thread
                    int i = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (before < target) { before += w[k][e]; i = e; }
                    s_found = v0 + (k * DV_THREADS + (int)threadIdx.x) * 4 + i;
                }
                cum += all_in;
            }
            __syncthreads();
            next = s_found;
            __syncthreads();
        }
    }
    for (int i = threadIdx.x; i <= K; i += DV_THREADS)
        tokens[(size_t)b * (K + 1) + i] = i < stand ? __ldcg(drafts + (size_t)b * K + i) : i == stand ? next : -1;
    if (threadIdx.x == 0) {
        accepted[b] = stand;
        tickets[b] = 0;                                       // ready for the next launch
    }
}

// Stretches of a row: 1,024 tokens while that fills no more than two blocks to an SM, 4,096 (what a block looks through at once) beyond.
static int verify_chunks(int seqs, int vocab) {
    int chunks = (vocab + 1023) / 1024;
    if ((long long)chunks * seqs > 2LL * ti_sm_count()) chunks = (vocab + 4095) / 4096;
    if (chunks > DV_MAX_CHUNKS) chunks = DV_MAX_CHUNKS;
    return chunks;
}

extern "C" long long ti_verify_drafts_workspace(int seqs) { return seqs > 0 ? (long long)seqs * DV_MAX_CHUNKS * 8 : 0; }

// p [B, K + 1, vocab] and q [B, K, vocab] (or null) float with strides in elements, drafts [B, K], uniforms [B, K + 1], counts [B] or null; sums:
// ti_verify_drafts_workspace bytes; tickets [B] words that are zero before the first launch (the kernel leaves them zero).
extern "C" int ti_verify_drafts(int* accepted, int* tokens, const float* p, long long p_seq, long long p_row, const float* q, long long q_seq,
                                long long q_row, const int* drafts, const float* uniforms, const int* counts, int B, int K, int vocab,
                                void* sums, unsigned* tickets, cudaStream_t stream) {
    if (B == 0) return 0;
    TI_REQUIRE(B > 0 && B <= 65535 && K >= 0 && vocab > 0, "verify_drafts: %d sequences, %d drafts, vocabulary %d", B, K, vocab);
    TI_REQUIRE(vocab <= (1 << 23), "verify_drafts: vocabulary %d exceeds %d (the weights' sum has 64 bits)", vocab, 1 << 23);
    TI_REQUIRE(sums != nullptr && tickets != nullptr, "verify_drafts: work space missing");
    const int chunks = verify_chunks(B, vocab);
    int per = (vocab + chunks - 1) / chunks;
    per = (per + 3) & ~3;
    ti_launch(verify_drafts_kernel, dim3(chunks, B), dim3(DV_THREADS), 0, stream, accepted, tokens, p, p_seq, p_row, q, q_seq, q_row, drafts, uniforms,
              counts, K, vocab, per, (u64*)sums, tickets);
    return ti_check_launch("verify_drafts");
}

// ------------------------------------------------------------------------------ greedy drafts
// A drafted token stands while it is the model's own choice at its place: one warp a sequence.
__global__ void match_drafts_kernel(int* accepted, int* tokens, const int* chosen, const int* drafts, const int* counts, int B, int K) {
    const int b = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    pdl_enter();
    if (b >= B) return;
    const int count = counts != nullptr ? min(max(__ldcg(counts + b), 0), K) : K;
    int stand = count;
    for (int i0 = 0; i0 < count; i0 += 32) {
        const int i = i0 + lane;
        const bool refused = i < count && __ldcg(drafts + (size_t)b * K + i) != __ldcg(chosen + (size_t)b * (K + 1) + i);
        const unsigned where = __ballot_sync(0xffffffffu, refused);
        if (where) { stand = i0 + __ffs(where) - 1; break; }
    }
    for (int i = lane; i <= K; i += 32) tokens[(size_t)b * (K + 1) + i] = i <= stand ? __ldcg(chosen + (size_t)b * (K + 1) + i) : -1;
    if (lane == 0) accepted[b] = stand;
}

extern "C" int ti_match_drafts(int* accepted, int* tokens, const int* chosen, const int* drafts, const int* counts, int B, int K, cudaStream_t stream) {
    if (B == 0) return 0;
    TI_REQUIRE(B > 0 && K >= 0, "match_drafts: %d sequences, %d drafts", B, K);
    ti_launch(match_drafts_kernel, dim3((B + 7) / 8), dim3(256), 0, stream, accepted, tokens, chosen, drafts, counts, B, K);
    return ti_check_launch("match_drafts");
}

// out[b, i] = the sampler's uniform number of (seeds[b], counters[b] + i); the counters move on by m.
__global__ void uniforms_kernel(float* out, const u32* seeds, u32* counters, int m) {
    const int b = blockIdx.x;
    pdl_enter();
    const u32 seed = mix32(__ldcg(seeds + b)), counter = __ldcg(counters + b);
    for (int i = threadIdx.x; i < m; i += blockDim.x) out[(size_t)b * m + i] = (float)(mix32(seed ^ (counter + (u32)i)) >> 8) * 5.9604645e-8f;
    __syncthreads();                                         // every thread has read the counter
    if (threadIdx.x == 0) counters[b] = counter + (u32)m;
}

extern "C" int ti_uniforms(float* out, const unsigned* seeds, unsigned* counters, int B, int m, cudaStream_t stream) {
    if (B == 0 || m == 0) return 0;
    TI_REQUIRE(B > 0 && m > 0, "uniforms: %d x %d", B, m);
    ti_launch(uniforms_kernel, dim3(B), dim3(32), 0, stream, out, seeds, counters, m);
    return ti_check_launch("uniforms");
}
