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
// the block that arrives last finds the stretch and then the token (no block waits for another).
#include "sampling_rule.cuh"

#define DV_THREADS 256
#define DV_WARPS (DV_THREADS / 32)
#define DV_MAX_CHUNKS 256

__device__ __forceinline__ u64 fixed_weight(float w) { return __float2ull_rn(fminf(fmaxf(w, 0.f), 1.f) * 1099511627776.0f); }   // NaN: 0

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
    auto rest = [&](int v, float pv, float qv) { return fixed_weight(v == without ? pv - 1.f : pv - qv); };

    const int lo = min(vocab, chunk * per), hi = min(vocab, lo + per);
    const bool wide = ((uintptr_t)pr & 15) == 0 && ((uintptr_t)qr & 15) == 0;
    u64 part = 0, whole = 0;
    if (wide) {
        for (int v0 = lo + 4 * threadIdx.x; v0 < hi; v0 += 16 * DV_THREADS) {
            float4 a[4], c[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int v = v0 + u * 4 * DV_THREADS;
                a[u] = c[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (v + 3 < hi) {
                    a[u] = __ldcg(reinterpret_cast<const float4*>(pr + v));
                    if (qr != nullptr) c[u] = __ldcg(reinterpret_cast<const float4*>(qr + v));
                } else if (v < hi) {
                    a[u].x = __ldcg(pr + v);
                    if (v + 1 < hi) a[u].y = __ldcg(pr + v + 1);
                    if (v + 2 < hi) a[u].z = __ldcg(pr + v + 2);
                    if (qr != nullptr) {
                        c[u].x = __ldcg(qr + v);
                        if (v + 1 < hi) c[u].y = __ldcg(qr + v + 1);
                        if (v + 2 < hi) c[u].z = __ldcg(qr + v + 2);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int v = v0 + u * 4 * DV_THREADS;
                part += rest(v, a[u].x, c[u].x) + rest(v + 1, a[u].y, c[u].y) + rest(v + 2, a[u].z, c[u].z) + rest(v + 3, a[u].w, c[u].w);
                whole += fixed_weight(a[u].x) + fixed_weight(a[u].y) + fixed_weight(a[u].z) + fixed_weight(a[u].w);
            }
        }
    } else {
        for (int v = lo + threadIdx.x; v < hi; v += DV_THREADS) {
            const float a = __ldcg(pr + v);
            part += rest(v, a, qr != nullptr ? __ldcg(qr + v) : 0.f);
            whole += fixed_weight(a);
        }
    }
    u64 part_sum, whole_sum;
    dv_scan(part, scratch, part_sum);
    __syncthreads();
    dv_scan(whole, scratch, whole_sum);
    if (threadIdx.x == 0) {
        u64* mine = sums + ((size_t)b * chunks + chunk) * 2;
        mine[0] = part_sum;
        mine[1] = whole_sum;
        __threadfence();
        s_last = atomicAdd(&tickets[b], 1u) == (unsigned)chunks - 1;
        s_found = -1;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();

    // The stretch that holds the target, a thread a stretch.
    const bool in = (int)threadIdx.x < chunks;
    const u64* all = sums + ((size_t)b * chunks + threadIdx.x) * 2;
    u64 w_part = in ? __ldcg(all) : 0, w_whole = in ? __ldcg(all + 1) : 0, total, p_total;
    u64 through = dv_scan(w_part, scratch, total);
    __syncthreads();
    const u64 p_through = dv_scan(w_whole, scratch, p_total);
    const bool plain = total == 0;                            // no weight in the differences (or none to take off)
    if (plain) { total = p_total; through = p_through; w_part = w_whole; }
    const float u = __ldcg(uniforms + (size_t)b * (K + 1) + K);
    const u32 r24 = (u32)fminf(fmaxf(u, 0.f) * 16777216.f, 16777215.f);
    u64 target = draw_target(total, r24);
    if (target == 0) target = 1;
    __shared__ u64 s_before;
    if (in && through >= target && through - w_part < target) { s_found = (int)threadIdx.x; s_before = through - w_part; }
    __syncthreads();
    int next = -1;
    if (s_found >= 0) {                                       // uniform over the block
        const int first = s_found * per, end = min(vocab, first + per), mine = (per + DV_THREADS - 1) / DV_THREADS;
        const int v0 = first + (int)threadIdx.x * mine, v1 = min(end, v0 + mine);
        const u64 before = s_before;
        auto weight = [&](int v) {
            const float a = __ldcg(pr + v);
            return plain ? fixed_weight(a) : rest(v, a, qr != nullptr ? __ldcg(qr + v) : 0.f);
        };
        u64 sum = 0, all_in;
        for (int v = v0; v < v1; ++v) sum += weight(v);
        u64 cum = before + dv_scan(sum, scratch, all_in) - sum;
        __syncthreads();
        if (cum < target && cum + sum >= target) {            // one thread
            int v = v0;
            for (; v < v1; ++v) {
                cum += weight(v);
                if (cum >= target) break;
            }
            s_found = v;
        }
        __syncthreads();
        next = s_found;
    }
    for (int i = threadIdx.x; i <= K; i += DV_THREADS)
        tokens[(size_t)b * (K + 1) + i] = i < stand ? __ldcg(drafts + (size_t)b * K + i) : i == stand ? next : -1;
    if (threadIdx.x == 0) {
        accepted[b] = stand;
        tickets[b] = 0;                                       // ready for the next launch
    }
}

// Stretches of a row: of at least 1,024 tokens, about eight blocks to an SM in all.
static int verify_chunks(int seqs, int vocab) {
    int chunks = (vocab + 1023) / 1024;
    const int most = (8 * ti_sm_count() + seqs - 1) / seqs;
    if (chunks > most) chunks = most;
    if (chunks > DV_MAX_CHUNKS) chunks = DV_MAX_CHUNKS;
    return chunks < 1 ? 1 : chunks;
}

extern "C" long long ti_verify_drafts_workspace(int seqs) { return seqs > 0 ? (long long)seqs * DV_MAX_CHUNKS * 16 : 0; }

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
