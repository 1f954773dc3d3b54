// What the sampler draws from, as a tensor: out[row, v] = the probability of token v under a temperature, the top_k best and the smallest
// best-first prefix whose mass reaches top_p (sampling_rule.cuh), 0 for a token that the filters leave out:
//   e_v = exp((l_v - max l) / T),  p_v = e_v / sum of e over the kept tokens.
// A masked token (a logit of -inf, or NaN) has probability 0; a row without any other has zeros everywhere.
//
// Bound by reading the logits and writing as many numbers. A row is shared out among the blocks of a cluster, which hold it in shared memory from
// its one reading on: maximum, filters, sum and the writing go over that copy. Maxima and sums are exchanged through distributed shared memory,
// the sums in the order of the ranks. A filter is a radix select over the 56-bit key (descending logit, then id): a pass counts (or adds the 2^40
// fixed-point masses of) the digits of the keys that are still in question, every block adds up its share of the bins over the cluster, and the one
// whose share holds the target names the digit; a pass whose bin is kept whole ends it.
#include "sampling_rule.cuh"

#define PB_THREADS 512
#define PB_WARPS (PB_THREADS / 32)
#define PB_BINS 2048
#define PB_HELD 16384                // logits of a block's share that are held

// exp((l - max) / T) with 1 / T as the sum of two 32-bit numbers: the rounding of the quotient alone, not of 1 / T as well.
struct Temper {
    float inv, rest;
};
__device__ __forceinline__ float tempered(float l, float maxl, const Temper& t) {
    const float d = l == maxl ? 0.f : fmaxf(l - maxl, -3e38f);           // (+inf) - (+inf) too; -inf times the rest would be +inf or NaN
    return expf(fmaf(d, t.inv, d * t.rest));
}

// Inclusive scan over the block; `scratch`: PB_WARPS words.
__device__ __forceinline__ u64 pb_scan(u64 v, u64* scratch, u64& total) {
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
    for (int w = 0; w < PB_WARPS; ++w) {
        const u64 s = scratch[w];
        if (w < warp) before += s;
        all += s;
    }
    total = all;
    return v + before;
}

template <int C>
__global__ void __launch_bounds__(PB_THREADS) probabilities_kernel(float* out, long long ldo, const float* logits, long long ld, int vocab, int per,
                                                                   Temper temper, int top_k, float top_p, bool held, bool masses) {
    extern __shared__ __align__(16) unsigned char pb_smem[];
    __shared__ float scratch[33];
    __shared__ u64 scan[PB_WARPS];
    __shared__ float x_max, x_sum;                           // this block's, for the cluster
    __shared__ u64 x_total, x_found[3];
    float* copy = reinterpret_cast<float*>(pb_smem);
    u32* hist = reinterpret_cast<u32*>(pb_smem + (held ? (size_t)per * 4 : 0));          // counts, or the low halves of masses; then the high ones
    const unsigned rank = C > 1 ? cluster_rank() : 0u;
    const int row_id = blockIdx.x / C;
    const float* row = logits + (size_t)row_id * ld;
    float* p = out + (size_t)row_id * ldo;
    const int lo = min(vocab, (int)rank * per), n = min(vocab, lo + per) - lo;           // this block's share: ids [lo, lo + n), lo a multiple of 4
    auto sync_cluster = [&] {
        if (C > 1) cluster_sync_all(); else __syncthreads();
    };
    const bool row_wide = ((uintptr_t)row & 15) == 0, out_wide = ((uintptr_t)p & 15) == 0;
    pdl_enter();

    if (held) {
        if (row_wide) {
            for (int i = threadIdx.x; i < n >> 2; i += PB_THREADS)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(copy + 4 * i)), "l"(row + lo + 4 * i));
            for (int i = (n & ~3) + threadIdx.x; i < n; i += PB_THREADS) copy[i] = __ldcg(row + lo + i);
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
        } else {
            for (int i = threadIdx.x; i < n; i += PB_THREADS) copy[i] = __ldcg(row + lo + i);
        }
        __syncthreads();
    }
    // f(place in the share, logit) over the share; NaN counts as masked.
    const float* src = held ? copy : row + lo;
    const bool wide = held || row_wide;
    auto clean = [](float l) { return l == l ? l : -INFINITY; };
    auto each = [&](auto f) {
        const int n4 = wide ? n >> 2 : 0;
        for (int i = threadIdx.x; i < n4; i += PB_THREADS) {
            const float4 v = reinterpret_cast<const float4*>(src)[i];
            f(4 * i, clean(v.x)); f(4 * i + 1, clean(v.y)); f(4 * i + 2, clean(v.z)); f(4 * i + 3, clean(v.w));
        }
        for (int i = 4 * n4 + threadIdx.x; i < n; i += PB_THREADS) f(i, clean(src[i]));
    };

    float maxl = -INFINITY;
    each([&](int, float l) { maxl = fmaxf(maxl, l); });
    maxl = block_max(maxl, scratch);
    if (C > 1) {
        if (threadIdx.x == 0) x_max = maxl;
        sync_cluster();
#pragma unroll
        for (int r = 0; r < C; ++r) maxl = fmaxf(maxl, ld_remote(&x_max, (unsigned)r));
    }

    u64 bound = ~0ull;
    auto key_of = [&](int i, float l) { return ((u64)desc_key(l) << SM_ID_BITS) | (u64)(u32)(lo + i); };
    auto mass = [&](float l) { return l == maxl ? 1ull << 40 : token_weight(W_MASS, l, maxl, temper.inv); };
    auto select = [&](bool by_mass, u64 target) {
        auto width = [](int pass) { return pass < 2 ? 11 : pass == 2 ? 10 : 8; };        // the logit's 32 bits, then the id's 24
        u64 prefix = 0, base = 0;
        int shift = 56;
        for (int pass = 0; pass < 6; ++pass) {
            const int above = shift;
            shift -= width(pass);
            const u32 mask = (1u << width(pass)) - 1;
            for (int i = threadIdx.x; i < (by_mass ? 2 : 1) * PB_BINS; i += PB_THREADS) hist[i] = 0;
            __syncthreads();
            each([&](int i, float l) {
                const u64 key = key_of(i, l);
                if (key > bound || (pass > 0 && key >> above != prefix)) return;
                const u32 digit = (u32)(key >> shift) & mask;
                if (!by_mass) { atomicAdd(&hist[digit], 1u); return; }
                const u64 w = mass(l);
                const u32 w_lo = (u32)w;
                u32 w_hi = (u32)(w >> 32);
                if (w_lo) {                                  // 64-bit additions in shared memory are compare-and-swap loops: two halves and a carry
                    const u32 old = atomicAdd(&hist[digit], w_lo);
                    w_hi += (old + w_lo < old) ? 1u : 0u;
                }
                if (w_hi) atomicAdd(&hist[PB_BINS + digit], w_hi);
            });
            sync_cluster();
            constexpr int SHARE = PB_BINS / C, PER = SHARE > PB_THREADS ? SHARE / PB_THREADS : 1;
            u64 mine[PER], sum = 0;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                mine[e] = 0;
                const int bin = (int)rank * SHARE + (int)threadIdx.x * PER + e;
                if ((int)threadIdx.x * PER + e < SHARE) {
#pragma unroll
                    for (int r = 0; r < C; ++r) {
                        mine[e] += C > 1 ? ld_remote(&hist[bin], (unsigned)r) : hist[bin];
                        if (by_mass) mine[e] += (u64)(C > 1 ? ld_remote(&hist[PB_BINS + bin], (unsigned)r) : hist[PB_BINS + bin]) << 32;
                    }
                }
                sum += mine[e];
            }
            u64 total;
            u64 cum = pb_scan(sum, scan, total) - sum;
            if (threadIdx.x == 0) x_total = total;
            sync_cluster();                                  // nobody reads the bins any more
            u64 first = base;
            if (C > 1)
                for (int r = 0; r < (int)rank; ++r) first += ld_remote(&x_total, (unsigned)r);
            cum += first;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                if (mine[e] && cum < target && cum + mine[e] >= target) {
                    const u64 digit = (u64)((int)rank * SHARE + (int)threadIdx.x * PER + e);
                    for (int r = 0; r < C; ++r) {
                        if (C > 1) {
                            st_remote(&x_found[0], (unsigned)r, digit); st_remote(&x_found[1], (unsigned)r, cum); st_remote(&x_found[2], (unsigned)r, cum + mine[e]);
                        } else { x_found[0] = digit; x_found[1] = cum; x_found[2] = cum + mine[e]; }
                    }
                }
                cum += mine[e];
            }
            sync_cluster();
            prefix = (prefix << width(pass)) | x_found[0];
            base = x_found[1];
            if (x_found[2] == target) break;                 // the bin is kept whole
        }
        bound = ((prefix + 1) << shift) - 1;
    };
    if (top_k > 0 && top_k < vocab && maxl > -INFINITY) select(false, (u64)top_k);
    if (top_p < 1.f && maxl > -INFINITY) {
        u64 local = 0, total;
        each([&](int i, float l) {
            if (key_of(i, l) <= bound) local += mass(l);
        });
        pb_scan(local, scan, total);
        if (C > 1) {
            if (threadIdx.x == 0) x_total = total;           // the selection before has been read: its last barrier stands behind
            sync_cluster();
            total = 0;
#pragma unroll
            for (int r = 0; r < C; ++r) total += ld_remote(&x_total, (unsigned)r);
        }
        const u64 target = (u64)ceil((double)top_p * (double)total);
        select(true, target ? target : 1);
    }

    float sum = 0.f;
    const bool cut = bound != ~0ull;
    each([&](int i, float l) {
        if (!cut || key_of(i, l) <= bound) sum += tempered(l, maxl, temper);
    });
    sum = block_sum(sum, scratch);
    if (C > 1) {
        if (threadIdx.x == 0) x_sum = sum;
        sync_cluster();
        sum = 0.f;
#pragma unroll
        for (int r = 0; r < C; ++r) sum += ld_remote(&x_sum, (unsigned)r);
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");            // this block reads no other's memory any more
    }
    const float scale = maxl == -INFINITY ? 0.f : __fdiv_rn(1.f, sum);
    auto value = [&](int i, float l) { return scale > 0.f && (!cut || key_of(i, l) <= bound) ? tempered(l, maxl, temper) * scale : 0.f; };
    const int n4 = wide && out_wide ? n >> 2 : 0;
    for (int i = threadIdx.x; i < n4; i += PB_THREADS) {
        const float4 v = reinterpret_cast<const float4*>(src)[i];
        *reinterpret_cast<float4*>(p + lo + 4 * i) = make_float4(value(4 * i, clean(v.x)), value(4 * i + 1, clean(v.y)), value(4 * i + 2, clean(v.z)),
                                                                 value(4 * i + 3, clean(v.w)));
    }
    for (int i = 4 * n4 + threadIdx.x; i < n; i += PB_THREADS) p[lo + i] = value(i, clean(src[i]));
    if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");       // nor any other this one's
}

template <int C>
static int launch_probabilities(float* out, long long ldo, const float* logits, long long ld, int n_rows, int vocab, Temper temper, int top_k, float top_p,
                                cudaStream_t stream) {
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(probabilities_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, PB_HELD * 4 + PB_BINS * 8);
        if (e != cudaSuccess) return ti_fail("probabilities: %s", cudaGetErrorString(e));
        configured = true;
    }
    const int per = ((vocab + C - 1) / C + 3) & ~3;
    const bool held = per <= PB_HELD, masses = top_p < 1.f, filters = masses || (top_k > 0 && top_k < vocab);
    const size_t smem = (held ? (size_t)per * 4 : 0) + (filters ? (size_t)(masses ? 2 : 1) * PB_BINS * 4 : 0);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n_rows * C);
    cfg.blockDim = dim3(PB_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ti_pdl_enabled ? 2 : 1;
    cudaLaunchKernelEx(&cfg, probabilities_kernel<C>, out, ldo, logits, ld, vocab, per, temper, top_k, top_p, held, masses);
    return ti_check_launch("probabilities");
}

extern "C" int ti_probabilities(float* out, long long ldo, const float* logits, long long ld, int n_rows, int vocab, float temperature, int top_k,
                                float top_p, cudaStream_t stream) {
    if (n_rows == 0) return 0;
    TI_REQUIRE(n_rows > 0 && n_rows <= (1 << 27) && vocab > 0 && vocab <= (1 << SM_ID_BITS), "probabilities: %d rows of %d (at most %d)", n_rows, vocab,
               1 << SM_ID_BITS);
    TI_REQUIRE(temperature > 0.f, "probabilities: temperature must be > 0");
    TI_REQUIRE(top_k >= 0, "probabilities: top_k must be >= 0");
    TI_REQUIRE(top_p > 0.f && top_p <= 1.f, "probabilities: top_p must be in (0, 1]");
    const double inv = 1.0 / (double)temperature;
    const Temper temper{(float)inv, (float)(inv - (double)(float)inv)};
    // As few blocks a row as can hold it; more while the rows leave SMs idle and a share stays above 2,048.
    int share = 1;
    while (share < 8 && ((vocab + share - 1) / share > PB_HELD || (n_rows * share * 2 <= ti_sm_count() && vocab / share > 4096))) share *= 2;
    if (share == 8) return launch_probabilities<8>(out, ldo, logits, ld, n_rows, vocab, temper, top_k, top_p, stream);
    if (share == 4) return launch_probabilities<4>(out, ldo, logits, ld, n_rows, vocab, temper, top_k, top_p, stream);
    if (share == 2) return launch_probabilities<2>(out, ldo, logits, ld, n_rows, vocab, temper, top_k, top_p, stream);
    return launch_probabilities<1>(out, ldo, logits, ld, n_rows, vocab, temper, top_k, top_p, stream);
}
