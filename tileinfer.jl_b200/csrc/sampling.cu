// Sampling on the device: greedy argmax, and temperature / top-k / top-p sampling over the
// whole vocabulary by inverse-CDF in best-first order.
//
// The rule is AntoineBut/TileInfer.jl's (src/engine/sampler.jl:49-102): candidates are
// ordered best first with ties to the smaller id; temperature, then top-k, then top-p over
// the renormalised survivors (the smallest prefix whose mass reaches top_p); the token is
// the first one whose cumulative weight reaches u × total, u = sampling_uniform(seed,
// counter) (sampler.jl:34-47). The reference samples on the device only for top_k <= 64 and
// sends the logits to the host otherwise; here every setting runs on the device.
//
// Method: no sort of the vocabulary. Each token gets a 56-bit key (descending-ordered logit bits, then
// id), so best-first order is ascending key order, and every step of the rule is "the first key whose
// cumulative weight reaches X". Weights are 2^40 fixed-point integers, so sums do not depend on the
// order of the atomic additions and the result is deterministic.
//   Fast path: ONE pass over the row builds a histogram of weights and counts over 4096 bins of the
//   scaled distance from the maximum, (max - l) / T in steps of 1/128 (the bin is monotone in the
//   key, and weights vanish beyond 28.4). A selection then scans the bins for the one that holds its
//   target, gathers that bin's few tokens in a second pass, sorts them by key in shared memory and
//   scans them. top-k, top-p and the draw share the histogram: it is cut off at each bound found.
//   Exact path: a bin with more than 4096 tokens (a flat row of a large vocabulary) sends the row to a
//   radix select over the key, 8 bits a pass, with a histogram of weights per pass.
#include "sampling_rule.cuh"

// ------------------------------------------------------------------------------ greedy
// argmax with ties to the smaller id, over a vocabulary of any size, in ONE launch that uses many
// blocks: each block reduces a slice of the row and leaves its candidate in a work space; the block
// that arrives last at the row's counter (no block waits for another) reduces the candidates, writes
// the token and resets the counter for the next launch. (value, id) under "greater value, then
// smaller id" is a total order, so the result does not depend on the order of arrival.
#define AM_THREADS 256
#define AM_MAX_CHUNKS 256

__device__ __forceinline__ bool am_better(float v, int i, float bv, int bi) { return v > bv || (v == bv && i < bi); }

__device__ __forceinline__ void am_block_reduce(float& bv, int& bi, float* sv, int* si) {
    for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
        const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
        if (am_better(ov, oi, bv, bi)) { bv = ov; bi = oi; }
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) { sv[warp] = bv; si[warp] = bi; }
    __syncthreads();
    if (warp == 0) {
        bv = lane < AM_THREADS / 32 ? sv[lane] : -INFINITY;
        bi = lane < AM_THREADS / 32 ? si[lane] : 0x7fffffff;
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
            const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
            if (am_better(ov, oi, bv, bi)) { bv = ov; bi = oi; }
        }
    }
    __syncthreads();
}

__global__ void __launch_bounds__(AM_THREADS) argmax_kernel(const float* logits, long long ld, int vocab, int per_chunk,
                                                            int* __restrict__ out, int* __restrict__ out2, float* ws_val,
                                                            int* ws_idx, unsigned* counters) {
    __shared__ float sv[AM_THREADS / 32];
    __shared__ int si[AM_THREADS / 32];
    __shared__ bool last;
    const int chunk = blockIdx.x, row_id = blockIdx.y, chunks = gridDim.x;
    const float* row = logits + (size_t)row_id * ld;
    const int lo = chunk * per_chunk, hi = min(vocab, lo + per_chunk);
    pdl_enter();
    float bv = -INFINITY;
    int bi = 0x7fffffff;
    if ((((uintptr_t)row) & 15) == 0 && (lo & 3) == 0) {
        for (int i = lo + 4 * threadIdx.x; i < hi; i += 4 * AM_THREADS) {
            if (i + 3 < hi) {
                const float4 v = __ldcg(reinterpret_cast<const float4*>(row + i));
                if (am_better(v.x, i, bv, bi)) { bv = v.x; bi = i; }
                if (am_better(v.y, i + 1, bv, bi)) { bv = v.y; bi = i + 1; }
                if (am_better(v.z, i + 2, bv, bi)) { bv = v.z; bi = i + 2; }
                if (am_better(v.w, i + 3, bv, bi)) { bv = v.w; bi = i + 3; }
            } else {
                for (int j = i; j < hi; ++j) {
                    const float v = __ldcg(row + j);
                    if (am_better(v, j, bv, bi)) { bv = v; bi = j; }
                }
            }
        }
    } else {
        for (int i = lo + threadIdx.x; i < hi; i += AM_THREADS) {
            const float v = __ldcg(row + i);
            if (am_better(v, i, bv, bi)) { bv = v; bi = i; }
        }
    }
    am_block_reduce(bv, bi, sv, si);
    if (threadIdx.x == 0) {
        ws_val[(size_t)row_id * chunks + chunk] = bv;
        ws_idx[(size_t)row_id * chunks + chunk] = bi;
        __threadfence();                                   // the candidate is visible before the ticket is taken
        last = atomicAdd(&counters[row_id], 1u) == (unsigned)chunks - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    bv = -INFINITY;
    bi = 0x7fffffff;
    for (int c = threadIdx.x; c < chunks; c += AM_THREADS) {
        const float v = __ldcg(ws_val + (size_t)row_id * chunks + c);
        const int i = __ldcg(ws_idx + (size_t)row_id * chunks + c);
        if (am_better(v, i, bv, bi)) { bv = v; bi = i; }
    }
    am_block_reduce(bv, bi, sv, si);
    if (threadIdx.x == 0) {
        out[row_id] = bi == 0x7fffffff ? 0 : bi;
        if (out2 != nullptr) out2[row_id] = bi == 0x7fffffff ? 0 : bi;     // the next step's token ids, where the caller has them
        counters[row_id] = 0;                              // ready for the next launch
    }
}

// Work space: ws_val and ws_idx hold n_rows x TI_ARGMAX_CHUNKS(vocab) entries, counters n_rows words
// that are zero before the first launch (the kernel leaves them zero).
extern "C" int ti_argmax_chunks(int vocab) {
    int chunks = (vocab + 1023) / 1024;
    if (chunks < 1) chunks = 1;
    return chunks > AM_MAX_CHUNKS ? AM_MAX_CHUNKS : chunks;
}

extern "C" int ti_argmax(const float* logits, long long ld, int n_rows, int vocab, int* out, int* out2, float* ws_val, int* ws_idx,
                         unsigned* counters, cudaStream_t stream) {
    if (n_rows == 0) return 0;
    TI_REQUIRE(vocab > 0, "argmax: vocab %d", vocab);
    TI_REQUIRE(n_rows <= 65535, "argmax: %d rows in one launch", n_rows);
    TI_REQUIRE(ws_val != nullptr && ws_idx != nullptr && counters != nullptr, "argmax: work space missing");
    // Many rows: fewer, longer chunks (about 2,048 blocks in all), so that the launch is not a long queue of tiny blocks.
    int chunks = ti_argmax_chunks(vocab);
    const int fewer = 2048 / n_rows < 8 ? 8 : 2048 / n_rows;
    if (fewer < chunks) chunks = fewer;
    int per_chunk = (vocab + chunks - 1) / chunks;
    per_chunk = (per_chunk + 3) & ~3;
    ti_launch(argmax_kernel, dim3(chunks, n_rows), dim3(AM_THREADS), 0, stream, logits, ld, vocab, per_chunk, out, out2, ws_val, ws_idx,
              counters);
    return ti_check_launch("argmax");
}

// ------------------------------------------------------------------------------ sampling
// The rule by the radix select alone (any row; seven passes over the row per selection).
__device__ int sample_exact(const float* row, int vocab, float inv_t, int top_k, float top_p, u32 r24, float maxl, u64* hist,
                            u64* totals, u64* shared) {
    u64 bound = ~0ull;
    if (top_k > 0 && top_k < vocab) {
        const Selected k = select_key(row, vocab, W_COUNT, bound, (u64)top_k, maxl, inv_t, hist, totals, shared);
        bound = k.key;
    }
    // Mass of the current set (everything, or the top-k prefix).
    {
        u64 local = 0;
        for (int i = threadIdx.x; i < vocab; i += SM_THREADS) {
            const float l = row[i];
            const u64 key = ((u64)desc_key(l) << SM_ID_BITS) | (u64)i;
            if (key <= bound) local += token_weight(W_MASS, l, maxl, inv_t);
        }
        if (threadIdx.x == 0) shared[3] = 0;
        __syncthreads();
        for (int o = 16; o > 0; o >>= 1) local += __shfl_xor_sync(0xffffffffu, local, o);
        if ((threadIdx.x & 31) == 0) atomicAdd(&shared[3], local);
        __syncthreads();
    }
    u64 total = shared[3];
    __syncthreads();
    if (top_p < 1.0f) {
        // Smallest prefix whose mass reaches top_p × total.
        const u64 target = (u64)ceil((double)top_p * (double)total);
        const Selected p = select_key(row, vocab, W_MASS, bound, target, maxl, inv_t, hist, totals, shared);
        bound = p.key;
        total = p.through;
    }
    const Selected s = select_key(row, vocab, W_MASS, bound, draw_target(total, r24), maxl, inv_t, hist, totals, shared);
    return (int)(s.key & ((1ull << SM_ID_BITS) - 1));
}

__global__ void __launch_bounds__(SM_THREADS) sample_kernel(const float* logits, long long ld, int vocab,
                                                            float inv_t, int top_k, float top_p,
                                                            const u32* seeds, u32* counters,
                                                            int* __restrict__ out, int* __restrict__ out2) {
    extern __shared__ u64 dyn[];
    __shared__ float scratch[33];
    const float* row = logits + (size_t)blockIdx.x * ld;
    pdl_wait();
    pdl_launch_dependents();

    float maxl = -INFINITY;
    for_each_logit(row, vocab, [&](int, float l) { maxl = fmaxf(maxl, l); });
    maxl = block_max(maxl, scratch);
    const u32 counter = counters[blockIdx.x];
    const u32 r24 = mix32(mix32(seeds[blockIdx.x]) ^ counter) >> 8;          // u = r24 · 2^-24

    // Fast path: one histogram of the row, cut off at each bound; a crowded bin sends the row to the exact path.
    Binned h;
    h.mass = dyn;
    h.cand_key = dyn + SB_BINS;
    h.cand_w = h.cand_key + SB_CAP;
    h.scan = h.cand_w + SB_CAP;
    h.count = reinterpret_cast<u32*>(h.scan + SM_WARPS + 8);
    // Masses are summed as two 32-bit halves with the carry passed on by hand: 64-bit additions in shared
    // memory are compare-and-swap loops, and these atomics bound the pass. The halves borrow the
    // candidates' place until the pass is over.
    u32* mass_lo = reinterpret_cast<u32*>(h.cand_key);
    u32* mass_hi = mass_lo + SB_BINS;
    for (int b = threadIdx.x; b < SB_BINS; b += SM_THREADS) { mass_lo[b] = 0; mass_hi[b] = 0; h.count[b] = 0; }
    __syncthreads();
    const bool need_counts = top_k > 0 && top_k < vocab;
    for_each_logit(row, vocab, [&](int, float l) {
        const int b = token_bin(l, maxl, inv_t);
        const u64 w = token_weight(W_MASS, l, maxl, inv_t);
        if (w) {
            const u32 lo = (u32)w;
            u32 hi = (u32)(w >> 32);
            if (lo) {
                const u32 old = atomicAdd(&mass_lo[b], lo);
                hi += (old + lo < old) ? 1u : 0u;
            }
            if (hi) atomicAdd(&mass_hi[b], hi);
        }
        if (need_counts) atomicAdd(&h.count[b], 1u);      // only top-k reads the counts
    });
    __syncthreads();
    for (int b = threadIdx.x; b < SB_BINS; b += SM_THREADS) h.mass[b] = ((u64)mass_hi[b] << 32) | (u64)mass_lo[b];
    __syncthreads();
    int token = -1;
    do {
        u64 bound = ~0ull;
        if (top_k > 0 && top_k < vocab) {
            const BinSelected k = select_binned(row, vocab, W_COUNT, bound, (u64)top_k, maxl, inv_t, h);
            if (k.overflow) break;
            bound = k.sel.key;
            cut_histogram(h, k);
        }
        u64 part = 0, total;
        for (int b = threadIdx.x; b < SB_BINS; b += SM_THREADS) part += h.mass[b];
        block_scan(part, h.scan, total);
        if (top_p < 1.0f) {
            const u64 target = (u64)ceil((double)top_p * (double)total);
            const BinSelected p = select_binned(row, vocab, W_MASS, bound, target, maxl, inv_t, h);
            if (p.overflow) break;
            bound = p.sel.key;
            total = p.sel.through;
            cut_histogram(h, p);
        }
        const BinSelected d = select_binned(row, vocab, W_MASS, bound, draw_target(total, r24), maxl, inv_t, h);
        if (d.overflow) break;
        token = (int)(d.sel.key & ((1ull << SM_ID_BITS) - 1));
    } while (false);
    if (token < 0) {                                       // uniform across the block: every thread saw the same overflow
        __syncthreads();
        u64* hist = dyn;
        u64* totals = dyn + SM_WARPS * 256;
        u64* shared = totals + 256;
        token = sample_exact(row, vocab, inv_t, top_k, top_p, r24, maxl, hist, totals, shared);
    }
    if (threadIdx.x == 0) {
        out[blockIdx.x] = token;
        if (out2 != nullptr) out2[blockIdx.x] = token;
        counters[blockIdx.x] = counter + 1;
    }
}

// ------------------------------------------------------------------------------ a row shared by a cluster
// The same rule with the row shared out among the C blocks of a cluster, for steps of a few rows, where one block
// per row leaves most of the GPU idle and is bound by one SM's instruction rate (a pass over 131,072 logits takes a
// block about 15 us). Every block makes the passes over its own stretch of the row (maximum, histogram, the
// gathering of a bin's tokens) into its own shared memory; the histograms are added up, and the gathered tokens
// collected, through distributed shared memory; the scans, the sort and the choices run in block 0 alone, on the
// same integers as in the one-block kernel, so the token is the same. Block 0 tells the others what to gather
// through a few words of its shared memory; a barrier of the cluster stands before and after every such order.
template <int C>
__global__ void __launch_bounds__(SM_THREADS) sample_cluster_kernel(const float* logits, long long ld, int vocab,
                                                                    float inv_t, int top_k, float top_p,
                                                                    const u32* seeds, u32* counters,
                                                                    int* __restrict__ out, int* __restrict__ out2) {
    extern __shared__ u64 dyn[];
    __shared__ float scratch[33];
    __shared__ float my_max;
    __shared__ u64 order[4];                               // block 0's: [0] 0 gather / 1 finished, [1] bin, [2] bound, [3] mode
    const unsigned rank = cluster_rank();
    const int row_id = blockIdx.x / C;
    const float* row = logits + (size_t)row_id * ld;
    const int per = ((vocab + C - 1) / C + 3) & ~3;        // stretches begin at multiples of 4 (16-byte loads)
    const int lo = min(vocab, (int)rank * per), hi = min(vocab, lo + per);
    pdl_wait();
    pdl_launch_dependents();

    float maxl = -INFINITY;
    for_each_logit(row, lo, hi, [&](int, float l) { maxl = fmaxf(maxl, l); });
    maxl = block_max(maxl, scratch);
    if (threadIdx.x == 0) my_max = maxl;
    cluster_sync_all();
#pragma unroll
    for (int r = 0; r < C; ++r) maxl = fmaxf(maxl, ld_remote(&my_max, (unsigned)r));

    Binned h;
    h.mass = dyn;
    h.cand_key = dyn + SB_BINS;
    h.cand_w = h.cand_key + SB_CAP;
    h.scan = h.cand_w + SB_CAP;
    h.count = reinterpret_cast<u32*>(h.scan + SM_WARPS + 8);
    u32* mass_lo = reinterpret_cast<u32*>(h.cand_key);      // as in the one-block kernel: masses as two 32-bit halves
    u32* mass_hi = mass_lo + SB_BINS;
    for (int b = threadIdx.x; b < SB_BINS; b += SM_THREADS) { mass_lo[b] = 0; mass_hi[b] = 0; h.count[b] = 0; }
    __syncthreads();
    const bool need_counts = top_k > 0 && top_k < vocab;
    for_each_logit(row, lo, hi, [&](int, float l) {
        const int b = token_bin(l, maxl, inv_t);
        const u64 w = token_weight(W_MASS, l, maxl, inv_t);
        if (w) {
            const u32 wl = (u32)w;
            u32 wh = (u32)(w >> 32);
            if (wl) {
                const u32 old = atomicAdd(&mass_lo[b], wl);
                wh += (old + wl < old) ? 1u : 0u;
            }
            if (wh) atomicAdd(&mass_hi[b], wh);
        }
        if (need_counts) atomicAdd(&h.count[b], 1u);
    });
    __syncthreads();
    cluster_sync_all();                                    // every block's histogram stands
    // Each block adds up its share of the bins over all blocks and hands the sums to block 0.
    for (int b = (int)rank * (SB_BINS / C) + threadIdx.x; b < ((int)rank + 1) * (SB_BINS / C); b += SM_THREADS) {
        u64 m = 0;
        u32 c = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) {
            m += ((u64)ld_remote(&mass_hi[b], (unsigned)r) << 32) + (u64)ld_remote(&mass_lo[b], (unsigned)r);
            c += ld_remote(&h.count[b], (unsigned)r);
        }
        st_remote(&h.mass[b], 0u, m);
        st_remote(&h.count[b], 0u, c);
    }
    cluster_sync_all();                                    // block 0 holds the row's histogram

    if (rank != 0) {
        // Gather what block 0 orders, until it says that it has finished.
        while (true) {
            cluster_sync_all();                            // an order stands
            if (ld_remote(&order[0], 0u) != 0) break;
            const int bin = (int)ld_remote(&order[1], 0u), mode = (int)ld_remote(&order[3], 0u);
            const u64 bound = ld_remote(&order[2], 0u);
            if (threadIdx.x == 0) *gathered_count(h) = 0;
            __syncthreads();
            gather_bin(row, lo, hi, mode, bound, bin, maxl, inv_t, h);
            __syncthreads();
            cluster_sync_all();                            // gathered; block 0 now reads the candidates
        }
        cluster_sync_all();                                // nobody reads block 0's order any more
        return;
    }

    const u32 counter = counters[row_id];
    const u32 r24 = mix32(mix32(seeds[row_id]) ^ counter) >> 8;
    auto select = [&](int mode, u64 bound, u64 target) -> BinSelected {
        const BinChoice at = find_bin(mode, target, h);
        if (threadIdx.x == 0) {
            order[0] = 0; order[1] = (u64)at.bin; order[2] = bound; order[3] = (u64)mode;
            *gathered_count(h) = 0;
        }
        __syncthreads();
        cluster_sync_all();
        gather_bin(row, lo, hi, mode, bound, at.bin, maxl, inv_t, h);
        __syncthreads();
        cluster_sync_all();
        // The other blocks' candidates behind this block's own; the sort puts them in key order.
        long long n = (long long)*gathered_count(h);
        __syncthreads();
        for (int r = 1; r < C; ++r) {
            const u32 nr = ld_remote(gathered_count(h), (unsigned)r);
            if (n + (long long)nr <= SB_CAP)
                for (int i = threadIdx.x; i < (int)nr; i += SM_THREADS) {
                    h.cand_key[n + i] = ld_remote(&h.cand_key[i], (unsigned)r);
                    h.cand_w[n + i] = ld_remote(&h.cand_w[i], (unsigned)r);
                }
            n += (long long)nr;
        }
        __syncthreads();
        return pick_in_bin(mode, target, at, n > SB_CAP ? SB_CAP + 1 : (int)n, h);
    };
    int token = -1;
    do {
        u64 bound = ~0ull;
        if (need_counts) {
            const BinSelected k = select(W_COUNT, bound, (u64)top_k);
            if (k.overflow) break;
            bound = k.sel.key;
            cut_histogram(h, k);
        }
        u64 part = 0, total;
        for (int b = threadIdx.x; b < SB_BINS; b += SM_THREADS) part += h.mass[b];
        block_scan(part, h.scan, total);
        if (top_p < 1.0f) {
            const u64 target = (u64)ceil((double)top_p * (double)total);
            const BinSelected p = select(W_MASS, bound, target);
            if (p.overflow) break;
            bound = p.sel.key;
            total = p.sel.through;
            cut_histogram(h, p);
        }
        const BinSelected d = select(W_MASS, bound, draw_target(total, r24));
        if (d.overflow) break;
        token = (int)(d.sel.key & ((1ull << SM_ID_BITS) - 1));
    } while (false);
    __syncthreads();
    if (threadIdx.x == 0) order[0] = 1;
    __syncthreads();
    cluster_sync_all();                                    // the others see that nothing more is ordered
    cluster_sync_all();                                    // and have read it: from here on this block is alone
    if (token < 0) {                                       // a crowded bin: the exact path, by this block over the whole row
        u64* hist = dyn;
        u64* totals = dyn + SM_WARPS * 256;
        u64* shared = totals + 256;
        token = sample_exact(row, vocab, inv_t, top_k, top_p, r24, maxl, hist, totals, shared);
    }
    if (threadIdx.x == 0) {
        out[row_id] = token;
        if (out2 != nullptr) out2[row_id] = token;
        counters[row_id] = counter + 1;
    }
}

template <int C>
static int launch_sample_cluster(const float* logits, long long ld, int n_rows, int vocab, float inv_t, int top_k, float top_p,
                                 const unsigned* seeds, unsigned* counters, int* out, int* out2, size_t smem, cudaStream_t stream) {
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(sample_cluster_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return ti_fail("sample: %s", cudaGetErrorString(e));
        configured = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_rows * C);
    cfg.blockDim = dim3(SM_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ti_pdl_enabled ? 2 : 1;
    cudaLaunchKernelEx(&cfg, sample_cluster_kernel<C>, logits, ld, vocab, inv_t, top_k, top_p, seeds, counters, out, out2);
    return ti_check_launch("sample");
}

// `cluster_blocks`: blocks that share a row (1, 2, 4 or 8; 0: chosen here from the number of rows and the vocabulary).
extern "C" int ti_sample_shared(const float* logits, long long ld, int n_rows, int vocab, float temperature, int top_k,
                                float top_p, const unsigned* seeds, unsigned* counters, int* out, int* out2, int cluster_blocks,
                                cudaStream_t stream) {
    if (n_rows == 0) return 0;
    TI_REQUIRE(cluster_blocks == 0 || cluster_blocks == 1 || cluster_blocks == 2 || cluster_blocks == 4 || cluster_blocks == 8,
               "sample: %d blocks per row (0, 1, 2, 4 or 8)", cluster_blocks);
    TI_REQUIRE(vocab > 0 && vocab <= (1 << SM_ID_BITS), "sample: vocabulary %d exceeds %d", vocab, 1 << SM_ID_BITS);
    TI_REQUIRE(temperature > 0.f, "sample: temperature must be > 0 (use argmax for greedy)");
    TI_REQUIRE(top_k >= 0, "sample: top_k must be >= 0");
    TI_REQUIRE(top_p > 0.f && top_p <= 1.f, "sample: top_p must be in (0, 1]");
    // The binned path's layout (histogram, candidates, scan scratch, counts); the exact path's is smaller and shares it.
    const size_t smem = (size_t)(SB_BINS + 2 * SB_CAP + SM_WARPS + 8) * sizeof(u64) + (size_t)SB_BINS * sizeof(u32);
    static_assert((SB_BINS + 2 * SB_CAP + SM_WARPS + 8) >= (SM_WARPS * 256 + 256 + 4), "the exact path must fit the same shared memory");
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return ti_fail("sample: %s", cudaGetErrorString(e));
        configured = true;
    }
    // A few rows of a large vocabulary: a cluster of blocks per row, as many as keep the launch within one round of the SMs.
    static int sm_count = 0;                                   // asked once: the answer does not change
    if (sm_count == 0) {
        int dev = 0;
        cudaGetDevice(&dev);
        if (cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sm_count <= 0) sm_count = 1;
    }
    // Measured at a vocabulary of 131,072 on 148 SMs (us, temperature only, for 1 / 2 / 4 / 8 blocks per row): 12 rows 47 / 35 /
    // 28 / 26, 16 rows 47 / 35 / 28 / 44, 32 rows 48 / 36 / 30 / 65, 37 rows 49 / 37 / 50, 74 rows 53 / 43 / 80, 96 rows 54 / 74:
    // clusters that do not all find room at once wait for one another, the larger the earlier.
    int share = cluster_blocks;
    if (share == 0) {
        if (vocab < 32768) share = 1;                          // a pass of one block is short already
        else if (n_rows * 8 * 3 <= sm_count * 2) share = 8;
        else if (n_rows * 4 * 8 <= sm_count * 7) share = 4;
        else if (n_rows * 2 <= sm_count) share = 2;
        else share = 1;
    }
    if (share == 8) return launch_sample_cluster<8>(logits, ld, n_rows, vocab, 1.0f / temperature, top_k, top_p, seeds, counters, out, out2, smem, stream);
    if (share == 4) return launch_sample_cluster<4>(logits, ld, n_rows, vocab, 1.0f / temperature, top_k, top_p, seeds, counters, out, out2, smem, stream);
    if (share == 2) return launch_sample_cluster<2>(logits, ld, n_rows, vocab, 1.0f / temperature, top_k, top_p, seeds, counters, out, out2, smem, stream);
    ti_launch(sample_kernel, dim3(n_rows), dim3(SM_THREADS), smem, stream, logits, ld, vocab, 1.0f / temperature, top_k, top_p, seeds,
                                                        counters, out, out2);
    return ti_check_launch("sample");
}

extern "C" int ti_sample(const float* logits, long long ld, int n_rows, int vocab, float temperature, int top_k,
                         float top_p, const unsigned* seeds, unsigned* counters, int* out, int* out2, cudaStream_t stream) {
    return ti_sample_shared(logits, ld, n_rows, vocab, temperature, top_k, top_p, seeds, counters, out, out2, 0, stream);
}

// The uniform number of (seed, counter), for tests of the generator itself.
extern "C" float ti_sampling_uniform(unsigned seed, unsigned counter) {
    return (float)(mix32(mix32(seed) ^ counter) >> 8) * 5.9604645e-8f;
}
