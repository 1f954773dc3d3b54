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
// The best few (up to half as many as there are groups of eight threads, what sampling mostly asks for) need none of that: the top_k-th largest of the
// groups' maxima bounds the row's top_k-th largest from below, the few tokens that reach it are exchanged, and each finds its rank by comparisons.
// Rows of 131,072: 5 rows 6.8 us; 320 rows (335 MB in and out) 86 us without filters, 105 us for the best 50, 260 us for the best 257 (radix), where the
// barriers of blocks and clusters between a row's passes are what its warps wait for.
#include "sampling_rule.cuh"

#define PB_THREADS 512
#define PB_WARPS (PB_THREADS / 32)
#define PB_BINS 2048
#define PB_HELD 16384                // logits of a block's share that are held
#define PB_TOPS (PB_THREADS / 8)     // groups of eight threads of a block
#define PB_BEST 512                  // tokens that reach the bound, of a block and of the row (both lists lie where the bins do)

// exp((l - max) / T) = 2^((l - max) log2(e) / T), the factor as the sum of two 32-bit numbers: the rounding of the product alone, not of the factor as
// well. What lies below 2^-126 becomes 0; a difference beyond that, and a masked logit's, -inf or NaN, is held to one whose number is 0 and whose
// products with both parts of the factor are finite at every temperature. (expf with its range reduction took 18 instructions of a token where this
// takes five, and instructions bounded the kernel.)
struct Temper {
    float inv;                                               // 1 / T, for the sampler's weights
    float factor, rest;                                      // log2(e) / T
    float least;                                             // factor x least = -130
};
__device__ __forceinline__ float tempered(float l, float maxl, const Temper& t) {
    const float d = fmaxf(l - maxl, t.least);
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(d, t.factor, d * t.rest)));
    return e;
}
__device__ __forceinline__ float logit_of(u64 key) {         // desc_key's inverse
    const u32 asc = ~(u32)(key >> SM_ID_BITS);
    return __uint_as_float((asc & 0x80000000u) ? asc ^ 0x80000000u : ~asc);
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
__global__ void __launch_bounds__(PB_THREADS, 3) probabilities_kernel(float* out, long long ldo, const float* logits, long long ld, int vocab, int per,
                                                                   Temper temper, int top_k, float top_p, bool held) {
    extern __shared__ __align__(16) unsigned char pb_smem[];
    __shared__ float scratch[33];
    __shared__ u64 scan[PB_WARPS];
    __shared__ float x_tops[PB_TOPS], x_sum;                 // this block's, for the cluster
    __shared__ u64 x_total, x_found[3];
    __shared__ u32 x_best;
    __shared__ __align__(16) float tops[PB_TOPS * C];
    __shared__ float bar;
    __shared__ u32 first_of[C + 1];
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
    // f(place in the share, logit) over the share; `each` takes NaN for a masked logit, `each_raw` leaves that to f.
    const float* src = held ? copy : row + lo;
    const bool wide = held || row_wide;
    auto clean = [](float l) { return l == l ? l : -INFINITY; };
    auto each_raw = [&](auto f) {
        const int n4 = wide ? n >> 2 : 0;
#pragma unroll 2
        for (int i = threadIdx.x; i < n4; i += PB_THREADS) {
            const float4 v = reinterpret_cast<const float4*>(src)[i];
            f(4 * i, v.x); f(4 * i + 1, v.y); f(4 * i + 2, v.z); f(4 * i + 3, v.w);
        }
        for (int i = 4 * n4 + threadIdx.x; i < n; i += PB_THREADS) f(i, src[i]);
    };
    auto each = [&](auto f) { each_raw([&](int i, float l) { f(i, clean(l)); }); };

    // The groups' maxima: of warps where few best are asked for, of eight threads else.
    const int group_log = top_k <= PB_WARPS * C / 2 || top_k >= vocab ? 5 : 3, tops_here = PB_THREADS >> group_log, tops_all = tops_here * C;
    float maxl = -INFINITY;
    each_raw([&](int, float l) { maxl = fmaxf(maxl, l); });
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
        if (o < (1 << group_log)) maxl = fmaxf(maxl, __shfl_xor_sync(0xffffffffu, maxl, o));
    if ((threadIdx.x & ((1 << group_log) - 1)) == 0) x_tops[threadIdx.x >> group_log] = maxl;
    if (threadIdx.x == 0) x_best = 0;
    sync_cluster();
    maxl = -INFINITY;
    if ((int)threadIdx.x < tops_all) {                       // every group's maximum of the whole row
        const int i = threadIdx.x, from = i >> (9 - group_log);
        tops[i] = maxl = C > 1 ? ld_remote(&x_tops[i & (tops_here - 1)], (unsigned)from) : x_tops[i];
    }
    maxl = block_max(maxl, scratch);
    // Equal infinities are a difference of 0 (and a choice among them alone): the row as its logits' signs.
    const bool endless = maxl == INFINITY;
    u64 bound = ~0ull;
    auto key_of = [&](int i, float l) { return ((u64)desc_key(l) << SM_ID_BITS) | (u64)(u32)(lo + i); };
    // The sampler's weight of a token (token_weight), by parts of 32 bits.
    auto parts_of = [&](float l) { return fixed_parts(l == maxl ? 1.f : expf((l - maxl) * temper.inv)); };
    auto mass = [&](float l) { const Fixed f = parts_of(l); return (u64)(((long long)f.high << 20) + f.low); };
    auto mass_of_kept = [&] {                                // the whole cluster's, of the keys up to `bound`
        u64 local = 0, total;
        each([&](int i, float l) {
            if (bound == ~0ull || key_of(i, l) <= bound) local += mass(l);
        });
        pb_scan(local, scan, total);
        if (C > 1) {
            if (threadIdx.x == 0) x_total = total;           // the selection before has been read: its last barrier stands behind
            sync_cluster();
            total = 0;
#pragma unroll
            for (int r = 0; r < C; ++r) total += ld_remote(&x_total, (unsigned)r);
        }
        return total;
    };
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
    auto number = [&](float l) { return endless ? (l == maxl ? 1.f : 0.f) : tempered(l, maxl, temper); };
    float sum = 0.f;
    bool summed = false;
    const bool by_count = top_k > 0 && top_k < vocab, by_mass = top_p < 1.f;
    auto mass_target = [&](u64 total) {
        const u64 x = (u64)ceil((double)top_p * (double)total);
        return x ? x : 1ull;
    };
    if ((by_count || by_mass) && maxl > -INFINITY) {
        const int want = by_count ? top_k : tops_all / 2;    // for a prefix by mass alone: as many as the groups' maxima give
        bool few = want <= tops_all / 2 && want > 0;
        if (few) {
            const u64 row_mass = by_count ? 0 : mass_of_kept();
            u64* mine = reinterpret_cast<u64*>(hist);
            u64* all = mine + PB_BEST;
            if ((int)threadIdx.x < tops_all) {
                const float v = tops[threadIdx.x];
                int rank = 0;
                for (int i = 0; i < tops_all; i += 4) {
                    const float4 o = *reinterpret_cast<const float4*>(tops + i);
                    const int me = (int)threadIdx.x - i;
                    rank += (o.x > v || (o.x == v && 0 < me)) + (o.y > v || (o.y == v && 1 < me)) + (o.z > v || (o.z == v && 2 < me)) +
                            (o.w > v || (o.w == v && 3 < me));
                }
                if (rank == want - 1) bar = v;
            }
            __syncthreads();
            const float least = bar;
            each_raw([&](int i, float l) {
                if (l >= least) {
                    const u32 at = atomicAdd(&x_best, 1u);
                    if (at < PB_BEST) mine[at] = key_of(i, l);
                }
            });
            sync_cluster();
            if (threadIdx.x < 32) {                          // where every block's tokens begin in the row's list
                const u32 here = (int)threadIdx.x < C ? (C > 1 ? ld_remote(&x_best, threadIdx.x) : x_best) : 0u;
                u32 through = here;
#pragma unroll
                for (int o = 1; o < C; o <<= 1) {
                    const u32 before = __shfl_up_sync(0xffffffffu, through, o);
                    if ((int)threadIdx.x >= o) through += before;
                }
                if ((int)threadIdx.x < C) first_of[threadIdx.x + 1] = through;
                if (threadIdx.x == 0) first_of[0] = 0;
            }
            __syncthreads();
            const int total = (int)first_of[C];
            few = total <= PB_BEST && total >= want;         // the same for the whole cluster (NaN may leave too few)
            if (few) {
                for (int i = threadIdx.x; i < total; i += PB_THREADS) {
                    int r = 0;
#pragma unroll
                    for (int k = 1; k < C; ++k) r += (u32)i >= first_of[k];
                    all[i] = C > 1 ? ld_remote(&mine[(u32)i - first_of[r]], (unsigned)r) : mine[i];
                }
                __syncthreads();
                // Keys differ, so ranks do: what is added is added in the order of the ranks, not of the tokens' arrival. Four threads a key.
                u64 keys[PB_BEST * 4 / PB_THREADS];
                int ranks[PB_BEST * 4 / PB_THREADS];
#pragma unroll
                for (int k = 0; k < PB_BEST * 4 / PB_THREADS; ++k) {
                    const int c = k * (PB_THREADS / 4) + ((int)threadIdx.x >> 2);
                    keys[k] = ~0ull;
                    ranks[k] = 0;
                    if (k * (PB_THREADS / 4) < total) {
                        if (c < total) {
                            keys[k] = all[c];
                            for (int i = threadIdx.x & 3; i < total; i += 4) ranks[k] += all[i] < keys[k];
                        }
                        ranks[k] += __shfl_xor_sync(0xffffffffu, ranks[k], 1);
                        ranks[k] += __shfl_xor_sync(0xffffffffu, ranks[k], 2);
                    }
                }
                __syncthreads();
#pragma unroll
                for (int k = 0; k < PB_BEST * 4 / PB_THREADS; ++k)
                    if (k * (PB_THREADS / 4) + ((int)threadIdx.x >> 2) < total && (threadIdx.x & 3) == 0) all[ranks[k]] = keys[k];
                __syncthreads();
                int kept = by_count ? top_k : total;
                const u64 key = (int)threadIdx.x < kept ? all[threadIdx.x] : 0;
                if (by_mass) {
                    const u64 m = (int)threadIdx.x < kept ? mass(logit_of(key)) : 0;
                    u64 listed;
                    const u64 through = pb_scan(m, scan, listed), target = mass_target(by_count ? listed : row_mass);
                    if (threadIdx.x == 0) x_found[0] = 0;
                    __syncthreads();
                    if (through >= target && through - m < target) x_found[0] = threadIdx.x + 1;
                    __syncthreads();
                    kept = (int)x_found[0];
                    few = kept > 0;                          // else the prefix reaches beyond the list
                }
                if (few) {
                    bound = all[kept - 1];
                    sum = block_sum((int)threadIdx.x < kept ? number(logit_of(key)) : 0.f, scratch);
                    summed = true;
                }
            }
            sync_cluster();                                  // nobody reads another's list any more
        }
        if (!few) {
            if (by_count) select(false, (u64)top_k);
            if (by_mass) select(true, mass_target(mass_of_kept()));
        }
    }
    const bool cut = bound != ~0ull;
    const float least_kept = cut ? logit_of(bound) : -INFINITY;          // (a bin kept whole ends with its last key: NaN there compares as nothing)
    if (!summed) {
        // Without filters the numbers themselves take their logits' places.
        if (!cut && held) {
            const int n4 = (n + 3) >> 2;                     // the copy's end is padded to whole vectors: beyond the share it is not used
#pragma unroll 2
            for (int i = threadIdx.x; i < n4; i += PB_THREADS) {
                float4 v = reinterpret_cast<const float4*>(copy)[i];
                v.x = number(v.x); v.y = number(v.y); v.z = number(v.z); v.w = number(v.w);
                reinterpret_cast<float4*>(copy)[i] = v;
                if (4 * i + 3 < n) sum += (v.x + v.y) + (v.z + v.w);
                else sum += v.x + (4 * i + 1 < n ? v.y : 0.f) + (4 * i + 2 < n ? v.z : 0.f);
            }
        } else {
            each([&](int i, float l) {
                if (!cut || key_of(i, l) <= bound) sum += number(l);
            });
        }
        sum = block_sum(sum, scratch);
        if (C > 1) {
            if (threadIdx.x == 0) x_sum = sum;
            sync_cluster();
            sum = 0.f;
#pragma unroll
            for (int r = 0; r < C; ++r) sum += ld_remote(&x_sum, (unsigned)r);
        }
    }
    if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");     // this block reads no other's memory any more
    const float scale = __fdiv_rn(1.f, sum);
    const int n4 = wide && out_wide ? n >> 2 : 0;
    auto write = [&](auto value) {
#pragma unroll 2
        for (int i = threadIdx.x; i < n4; i += PB_THREADS) {
            const float4 v = reinterpret_cast<const float4*>(src)[i];
            *reinterpret_cast<float4*>(p + lo + 4 * i) = make_float4(value(4 * i, v.x), value(4 * i + 1, v.y), value(4 * i + 2, v.z), value(4 * i + 3, v.w));
        }
        for (int i = 4 * n4 + threadIdx.x; i < n; i += PB_THREADS) p[lo + i] = value(i, src[i]);
    };
    if (maxl == -INFINITY) write([&](int, float) { return 0.f; });
    else if (!cut && held) write([&](int, float e) { return e * scale; });
    else if (!cut) write([&](int, float l) { return number(l) * scale; });
    else write([&](int i, float l) {
        l = clean(l);
        if (l < least_kept) return 0.f;                      // all but a few end here
        return key_of(i, l) <= bound ? number(l) * scale : 0.f;
    });
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
    cudaLaunchKernelEx(&cfg, probabilities_kernel<C>, out, ldo, logits, ld, vocab, per, temper, top_k, top_p, held);
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
    // The factor from 2^-118 on (a temperature of 5e35: beyond it, differences up to 1e28 are none to 32 bits), so that `least` is a number, and up to the
    // largest of 32 bits (a temperature of 4e-39: beyond it, no two logits that differ by 1e-36 are near each other).
    double factor = 1.4426950408889634 / (double)temperature;
    factor = factor < 0x1p-118 ? 0x1p-118 : factor > 0x1.fffffep127 ? 0x1.fffffep127 : factor;
    const Temper temper{1.0f / temperature, (float)factor, (float)(factor - (double)(float)factor), (float)(-130.0 / factor)};
    // As few blocks a row as can hold it; more while the rows leave SMs idle and a share stays above 2,048.
    int share = 1;
    while (share < 8 && ((vocab + share - 1) / share > PB_HELD || (n_rows * share * 2 <= ti_sm_count() && vocab / share > 4096))) share *= 2;
    if (share == 8) return launch_probabilities<8>(out, ldo, logits, ld, n_rows, vocab, temper, top_k, top_p, stream);
    if (share == 4) return launch_probabilities<4>(out, ldo, logits, ld, n_rows, vocab, temper, top_k, top_p, stream);
    if (share == 2) return launch_probabilities<2>(out, ldo, logits, ld, n_rows, vocab, temper, top_k, top_p, stream);
    return launch_probabilities<1>(out, ldo, logits, ld, n_rows, vocab, temper, top_k, top_p, stream);
}
