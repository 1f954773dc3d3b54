// Shared by the products of e4m3 codes: the MMA, the tensor maps of codes, the choice of a kernel.
#pragma once
#include "e4m3.cuh"
#include "linear4.cuh"
#include "tcgen05.cuh"
#include "tensor_map.h"

namespace tc {

// kind::f8f6f4: 32-bit sums of e4m3 A and B, both K-major, 128 x n, 32 of k.
__device__ __forceinline__ constexpr unsigned instr_desc_e4m3(int n) { return (1u << 4) | ((unsigned)(n >> 3) << 17) | ((128u >> 4) << 24); }
__device__ __forceinline__ void umma_e4m3(unsigned tmem_d, unsigned long long desc_a, unsigned long long desc_b, unsigned idesc, unsigned accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld16(unsigned taddr, unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}

// One thread of a warp, the same one every time: what only this guards stays uniform for the compiler.
__device__ __forceinline__ bool elected() {
    unsigned one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// Whether a barrier's phase is over, asked by the lanes with `asks`. Beside MMAs that read shared memory the answer takes some 300 cycles, a ready one too, so loops
// ask for their next step before they issue this one's work.
__device__ __forceinline__ bool mbar_test(unsigned bar, unsigned parity, bool asks) {
    unsigned done;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %3, 0;\n\t"
        "mov.u32 %0, 1;\n\t"
        "@q mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "@q selp.u32 %0, 1, 0, p;\n\t}"
        : "=&r"(done) : "r"(bar), "r"(parity), "r"((unsigned)asks) : "memory");
    return done != 0;
}
// The wait that such an answer belongs to, for the whole warp.
__device__ __forceinline__ bool warp_wait_after(bool ready, unsigned bar, unsigned parity, bool asks, int* status, int code) {
    if (__all_sync(0xffffffffu, ready)) return true;
    bool ok = true;
    if (asks) ok = mbar_wait(bar, parity, status, code);
    return __all_sync(0xffffffffu, ok);
}
// A whole warp's wait: one lane tests the barrier, the others follow it.
__device__ __forceinline__ bool warp_wait(unsigned bar, unsigned parity, int* status, int code) {
    bool ok = true;
    if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity, status, code);
    return __all_sync(0xffffffffu, ok);
}

}  // namespace tc

struct Linear8 {
    void* y;
    long long ldy;
    const void* x;                       // bfloat16, or codes with x_scales [groups, n]
    long long ldx;
    const float* x_scales;
    const unsigned char* codes;          // [out, K]
    const float* scales;                 // [groups, ceil(out / 128)]
    int n, out, K, epilogue;
    XieluParams act;
    int* status;
};

// Codes [rows, K] in rows of `ld` bytes as 16-bit numbers, moved as they are: boxes of 128 bytes x box_rows, swizzled; zeros beyond the edges.
inline int linear8_map(CUtensorMap* map, const void* codes, int rows, int K, long long ld, int box_rows) {
    const unsigned long long dims[2] = {(unsigned long long)K / 2, (unsigned long long)rows}, strides[1] = {(unsigned long long)ld};
    const unsigned box[2] = {64, (unsigned)box_rows};
    return ti_tensor_map_bf16(map, codes, 2, dims, strides, box, true);
}

// Whether four neighbouring results may be written at once.
__device__ __forceinline__ bool linear8_quads(const Linear8& p) { return p.ldy % 4 == 0 && ((uintptr_t)p.y & (p.epilogue == L4_EPI_F32_OUT ? 15 : 7)) == 0; }
// Rows o to o + 3 of token t.
__device__ __forceinline__ void linear8_store(const Linear8& p, int t, int o, float4 s, bool quads, bool y32) {
    if (quads && o + 4 <= p.out && p.epilogue == L4_EPI_NONE) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(s.x, s.y), hi = __floats2bfloat162_rn(s.z, s.w);
        *reinterpret_cast<uint2*>((bf16*)p.y + (size_t)t * p.ldy + o) = make_uint2(*reinterpret_cast<const unsigned*>(&lo), *reinterpret_cast<const unsigned*>(&hi));
    } else if (quads && o + 4 <= p.out && y32) {
        *reinterpret_cast<float4*>((float*)p.y + (size_t)t * p.ldy + o) = s;
    } else {
#pragma unroll 1
        for (int i = 0; i < 4 && o + i < p.out; ++i) store_result(p.y, p.ldy, t, o + i, i == 0 ? s.x : i == 1 ? s.y : i == 2 ? s.z : s.w, p.epilogue, p.act, y32);
    }
}

// Four sums at this place of the cluster's block `rank`, and a barrier of the cluster's blocks around such reads.
__device__ __forceinline__ float4 rank_sums(const float* at, unsigned rank) {
    unsigned a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((unsigned)__cvta_generic_to_shared(at)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_meets() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// A launch in clusters of `cluster` blocks, as a programmatic dependent of the kernel before.
template <typename... KArgs, typename... Args>
inline void linear8_launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ti_pdl_enabled ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

bool linear8_takes_few(int n, int out, int K);
int linear8_few(const Linear8& a, cudaStream_t stream);
int linear8_mid(const Linear8& a, cudaStream_t stream);
int linear8_many(const Linear8& a, cudaStream_t stream);
