// The sampler's rule in parts that its kernels share (sampling.cu draws by it, probabilities.cu writes down what it draws from): weights as
// 2^40 fixed-point integers, keys in best-first order, and the choice of the first key whose cumulative weight reaches a target.
#pragma once
#include "common.cuh"

typedef unsigned long long u64;
typedef unsigned int u32;

#define SM_THREADS 1024
#define SM_WARPS 32
#define SM_ID_BITS 24
#define SM_PASSES 7

__host__ __device__ __forceinline__ u32 mix32(u32 x) {
    x = (x ^ (x >> 16)) * 0x7feb352du;
    x = (x ^ (x >> 15)) * 0x846ca68bu;
    return x ^ (x >> 16);
}

__device__ __forceinline__ u32 desc_key(float l) {
    const u32 b = __float_as_uint(l);
    const u32 asc = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ~asc;
}

// ceil(u x total) with u = r24 / 2^24, without leaving integers: total < 2^58 and r24 < 2^24 need 128 bits.
__device__ __forceinline__ u64 draw_target(u64 total, u32 r24) {
    const u64 hi = __umul64hi(total, (u64)r24), lo = total * (u64)r24;
    u64 target = (hi << 40) | (lo >> 24);
    if (lo & 0xFFFFFFull) target += 1;
    return target;
}

// round(w 2^40) for w held to [0, 1] (NaN: 0) as high 2^20 + low, by additions that push a number's fraction out of its 24 bits: w 2^20 and what is left
// of it after rounding are exact. (A conversion to 64 bits goes through the pipe of special functions, 16 lanes a cycle at best: 64 rows 38 us.)
struct Fixed {
    int high, low;
};
__device__ __forceinline__ Fixed fixed_parts(float w) {
    const float v = fminf(fmaxf(w, 0.f), 1.f) * 1048576.f, up = v + 8388608.f;
    const float rest = fmaf(v - (up - 8388608.f), 1048576.f, 12582912.f);
    return Fixed{__float_as_int(up) - 0x4B000000, __float_as_int(rest) - 0x4B400000};
}
__device__ __forceinline__ u64 fixed_weight(float w) {
    const Fixed f = fixed_parts(w);
    return (u64)(((long long)f.high << 20) + f.low);
}

struct Selected {
    u64 key;          // the selected token's 56-bit key
    u64 before;       // weight of the keys before it (within the set)
    u64 through;      // ... including it
};

#define W_COUNT 0
#define W_MASS 1

__device__ __forceinline__ u64 token_weight(int mode, float l, float maxl, float inv_t) {
    if (mode == W_COUNT) return 1ull;
    const float e = expf((l - maxl) * inv_t);
    return __float2ull_rn(e * 1099511627776.0f);          // × 2^40
}

// First key (ascending) among keys <= bound whose cumulative weight reaches target (at
// least 1); if the set's total is smaller, the last key with weight. All threads get it.
static __device__ Selected select_key(const float* row, int vocab, int mode, u64 bound, u64 target,
                               float maxl, float inv_t, u64* hist /*[SM_WARPS][256]*/, u64* totals /*[256]*/,
                               u64* shared /*[4]*/) {
    const int warp = threadIdx.x >> 5;
    u64 prefix = 0, base = 0;
    if (target == 0) target = 1;
    for (int pass = 0; pass < SM_PASSES; ++pass) {
        const int shift = 8 * (SM_PASSES - 1 - pass);
        for (int i = threadIdx.x; i < SM_WARPS * 256; i += SM_THREADS) hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < vocab; i += SM_THREADS) {
            const float l = row[i];
            const u64 key = ((u64)desc_key(l) << SM_ID_BITS) | (u64)i;
            if (key > bound) continue;
            if (pass > 0 && (key >> (shift + 8)) != prefix) continue;
            const u64 w = token_weight(mode, l, maxl, inv_t);
            if (w) atomicAdd(&hist[warp * 256 + (int)((key >> shift) & 255)], w);
        }
        __syncthreads();
        if (threadIdx.x < 256) {
            u64 s = 0;
            for (int w = 0; w < SM_WARPS; ++w) s += hist[w * 256 + threadIdx.x];
            totals[threadIdx.x] = s;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            u64 cum = base;
            int digit = -1, last = 0;
            for (int b = 0; b < 256; ++b) {
                const u64 w = totals[b];
                if (w == 0) continue;
                if (cum + w >= target) { digit = b; break; }
                cum += w;
                last = b;
            }
            if (digit < 0) {                 // target beyond the set: settle on the last key with weight
                digit = last;
                cum -= totals[last];
            }
            shared[0] = (prefix << 8) | (u64)digit;
            shared[1] = cum;
            shared[2] = totals[digit];
        }
        __syncthreads();
        prefix = shared[0];
        base = shared[1];
    }
    Selected r;
    r.key = prefix;
    r.before = base;
    r.through = base + shared[2];
    __syncthreads();
    return r;
}

// ------------------------------------------------------------------------------ the binned fast path
// f(index, logit) for every token of the row, the block's threads sharing them out; sixteen values per
// thread are in flight at a time (one L2 round trip per value would otherwise bound a pass).
template <typename F> __device__ __forceinline__ void for_each_logit(const float* row, int lo, int hi, F f) {
    int done = lo;
    if ((reinterpret_cast<uintptr_t>(row) & 15) == 0 && (lo & 3) == 0) {
        const int first4 = lo >> 2, n4 = hi > lo ? (hi - lo) >> 2 : 0;
        const float4* row4 = reinterpret_cast<const float4*>(row) + first4;
        for (int i = threadIdx.x; i < n4; i += 4 * SM_THREADS) {
            float4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u * SM_THREADS < n4) v[u] = __ldcg(row4 + i + u * SM_THREADS);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = i + u * SM_THREADS;
                if (j < n4) { const int t = lo + 4 * j; f(t, v[u].x); f(t + 1, v[u].y); f(t + 2, v[u].z); f(t + 3, v[u].w); }
            }
        }
        done = lo + n4 * 4;
    }
    for (int i = done + threadIdx.x; i < hi; i += 4 * SM_THREADS) {
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i + u * SM_THREADS < hi) v[u] = __ldcg(row + i + u * SM_THREADS);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i + u * SM_THREADS < hi) f(i + u * SM_THREADS, v[u]);
    }
}
template <typename F> __device__ __forceinline__ void for_each_logit(const float* row, int vocab, F f) { for_each_logit(row, 0, vocab, f); }

#define SB_BINS 4096
#define SB_PER_NAT 128.0f
#define SB_CAP 4096

struct Binned {
    u64* mass;        // [SB_BINS] weights per bin
    u32* count;       // [SB_BINS] tokens per bin
    u64* cand_key;    // [SB_CAP]
    u64* cand_w;      // [SB_CAP]
    u64* scan;        // [SM_WARPS + 8] scratch of the block scans and results
};

__device__ __forceinline__ int token_bin(float l, float maxl, float inv_t) {
    const float d = (maxl - l) * inv_t * SB_PER_NAT;
    return d >= (float)(SB_BINS - 1) ? SB_BINS - 1 : (int)d;             // NaN goes to the last bin as well
}

// Inclusive block scan of one value per thread; every thread also gets the total. `scratch`: SM_WARPS + 1 words.
__device__ __forceinline__ u64 block_scan(u64 v, u64* scratch, u64& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    if (warp == 0) {
        u64 t = lane < SM_WARPS ? scratch[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 u = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += u;
        }
        scratch[lane] = t;
        if (lane == 31) scratch[SM_WARPS] = t;
    }
    __syncthreads();
    total = scratch[SM_WARPS];
    return v + (warp > 0 ? scratch[warp - 1] : 0);
}

struct BinSelected {
    Selected sel;     // key, weight before and through it (over the whole set, in the mode's weights)
    int bin;          // the bin it lies in
    u64 mass_in_bin;  // mass and count of the bin's tokens up to and including it
    u32 count_in_bin;
    bool overflow;    // the bin held more than SB_CAP tokens: nothing was selected
};

// The first key (ascending) among keys <= bound whose cumulative weight (mode: counts or masses) reaches
// target, from the histogram of the set and one gathering pass over the row, in three steps that the kernels
// below put together: the bin that holds the target (find_bin), that bin's tokens out of a stretch of the row
// (gather_bin; several blocks may each gather a stretch), and the choice among them in key order (pick_in_bin).
struct BinChoice {
    int bin;
    u64 base;         // weight of the bins before it
};

static __device__ BinChoice find_bin(int mode, u64 target, const Binned& h) {
    if (target == 0) target = 1;
    // Four bins per thread, block scan.
    u64 local[4], sum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int b = threadIdx.x * 4 + e;
        local[e] = mode == W_COUNT ? (u64)h.count[b] : h.mass[b];
        sum += local[e];
    }
    u64 total;
    const u64 incl = block_scan(sum, h.scan, total);
    u64* res = h.scan + SM_WARPS + 1;                  // res[0] bin, res[1] weight before the bin, res[2] last bin with weight
    if (threadIdx.x == 0) { res[0] = ~0ull; res[2] = 0; }
    __syncthreads();
    {
        u64 cum = incl - sum;
        int last = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (local[e] && cum < target && cum + local[e] >= target) { res[0] = (u64)(threadIdx.x * 4 + e); res[1] = cum; }
            if (local[e]) last = threadIdx.x * 4 + e;
            cum += local[e];
        }
        if (last >= 0) atomicMax(&res[2], (u64)last);
    }
    __syncthreads();
    if (res[0] == ~0ull) {                             // the target lies beyond the set: its last bin with weight
        const int last = (int)res[2];
        __syncthreads();
        if (threadIdx.x == last / 4) { res[0] = (u64)last; res[1] = incl - sum; for (int e = 0; e < last % 4; ++e) res[1] += local[e]; }
        __syncthreads();
    }
    BinChoice c;
    c.bin = (int)res[0];
    c.base = res[1];
    __syncthreads();
    return c;
}

// The counter of gathered tokens (a 32-bit word in the scan scratch).
__device__ __forceinline__ u32* gathered_count(const Binned& h) { return reinterpret_cast<u32*>(h.scan + SM_WARPS + 6); }

// Appends the tokens of row[lo, hi) that fall into `bin` (keys <= bound) to the candidates; the counter keeps
// counting beyond SB_CAP, which the caller reads as an overflow.
static __device__ void gather_bin(const float* row, int lo, int hi, int mode, u64 bound, int bin, float maxl, float inv_t, const Binned& h) {
    u32* n_cand = gathered_count(h);
    for_each_logit(row, lo, hi, [&](int i, float l) {
        if (token_bin(l, maxl, inv_t) != bin) return;
        const u64 key = ((u64)desc_key(l) << SM_ID_BITS) | (u64)i;
        if (key > bound) return;
        const u64 w = token_weight(W_MASS, l, maxl, inv_t);
        if (mode == W_MASS && w == 0) return;
        const u32 at = atomicAdd(n_cand, 1u);
        if (at < SB_CAP) { h.cand_key[at] = key; h.cand_w[at] = w; }
    });
}

// Among the n gathered tokens of `bin`, in key order, the first whose cumulative weight reaches what is left of the target.
static __device__ BinSelected pick_in_bin(int mode, u64 target, const BinChoice& at, int n, const Binned& h) {
    BinSelected r;
    if (target == 0) target = 1;
    const int bin = at.bin;
    const u64 base = at.base;
    r.bin = bin;
    r.overflow = n > SB_CAP || n == 0;
    if (r.overflow) { __syncthreads(); return r; }
    // Bitonic sort of the next power of two, then scans of counts and masses.
    int n2 = 1;
    while (n2 < n) n2 <<= 1;
    for (int i = n + threadIdx.x; i < n2; i += SM_THREADS) { h.cand_key[i] = ~0ull; h.cand_w[i] = 0; }
    __syncthreads();
    for (int size = 2; size <= n2; size <<= 1)
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            for (int t = threadIdx.x; t < (n2 >> 1); t += SM_THREADS) {
                const int lo = 2 * t - (t & (stride - 1)), hi = lo + stride;
                const bool up = (lo & size) == 0;
                const u64 a = h.cand_key[lo], b = h.cand_key[hi];
                if ((a > b) == up) {
                    h.cand_key[lo] = b; h.cand_key[hi] = a;
                    const u64 wa = h.cand_w[lo]; h.cand_w[lo] = h.cand_w[hi]; h.cand_w[hi] = wa;
                }
            }
            __syncthreads();
        }
    // Each thread owns four consecutive places; the first place whose cumulative weight reaches the rest of the target.
    const u64 rest = target - base;
    u64 wsel[4], wmass[4], ssum = 0, msum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int i = threadIdx.x * 4 + e;
        wmass[e] = i < n ? h.cand_w[i] : 0;
        wsel[e] = i < n ? (mode == W_COUNT ? 1ull : wmass[e]) : 0;
        ssum += wsel[e]; msum += wmass[e];
    }
    u64 stotal, mtotal;
    const u64 sincl = block_scan(ssum, h.scan, stotal);
    const u64 mincl = block_scan(msum, h.scan, mtotal);
    u64* pick = h.scan + SM_WARPS + 1;                 // pick[0] place, [1] weight before, [2] through, [3] mass through
    if (threadIdx.x == 0) pick[0] = ~0ull;
    __syncthreads();
    {
        u64 cum = sincl - ssum, mcum = mincl - msum;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = threadIdx.x * 4 + e;
            mcum += wmass[e];
            if (i < n && cum < rest && cum + wsel[e] >= rest) { pick[0] = (u64)i; pick[1] = cum; pick[2] = cum + wsel[e]; pick[3] = mcum; }
            cum += wsel[e];
        }
    }
    __syncthreads();
    if (pick[0] == ~0ull) {                            // beyond the bin's weight: its last token
        __syncthreads();
        if (threadIdx.x == (n - 1) / 4) { pick[0] = (u64)(n - 1); pick[1] = stotal - wsel[(n - 1) % 4]; pick[2] = stotal; pick[3] = mtotal; }
        __syncthreads();
    }
    const int place = (int)pick[0];
    r.sel.key = h.cand_key[place];
    r.sel.before = base + pick[1];
    r.sel.through = base + pick[2];
    r.mass_in_bin = pick[3];
    r.count_in_bin = (u32)(place + 1);
    __syncthreads();
    return r;
}


static __device__ BinSelected select_binned(const float* row, int vocab, int mode, u64 bound, u64 target, float maxl, float inv_t,
                                     const Binned& h) {
    const BinChoice at = find_bin(mode, target, h);
    if (threadIdx.x == 0) *gathered_count(h) = 0;
    __syncthreads();
    gather_bin(row, 0, vocab, mode, bound, at.bin, maxl, inv_t, h);
    __syncthreads();
    return pick_in_bin(mode, target, at, (int)*gathered_count(h), h);
}

// The set shrinks to the keys up to a selected one: its bin keeps what lies before and at it, later bins empty.
__device__ __forceinline__ void cut_histogram(const Binned& h, const BinSelected& at) {
    for (int b = threadIdx.x; b < SB_BINS; b += SM_THREADS) {
        if (b == at.bin) { h.mass[b] = at.mass_in_bin; h.count[b] = at.count_in_bin; }
        else if (b > at.bin) { h.mass[b] = 0; h.count[b] = 0; }
    }
    __syncthreads();
}

// ------------------------------------------------------------------------------ a row shared by a cluster of blocks
__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned remote_addr(const void* p, unsigned rank) {
    unsigned a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ u32 ld_remote(const u32* p, unsigned rank) {
    u32 v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ u64 ld_remote(const u64* p, unsigned rank) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(remote_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float ld_remote(const float* p, unsigned rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ void st_remote(u32* p, unsigned rank, u32 v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote_addr(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void st_remote(u64* p, unsigned rank, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote_addr(p, rank)), "l"(v) : "memory");
}
