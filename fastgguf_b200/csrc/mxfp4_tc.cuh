// What the tensor-memory contractions on MXFP4 weights share: barriers with bounded waits, copies, tensor memory, descriptors.
//
// Every wait on an mbarrier is bounded; when it runs out the kernel raises an error flag (fg_gemm_mxfp4_error), waits (bounded) for its
// own copies in flight, frees its tensor memory and returns.
#pragma once
#include <cuda.h>
#include "mxfp4.cuh"

#define FG_ERR_PIPELINE 10003
#define FG_ERR_TENSORMAP 10004
#define MX_WAIT_LIMIT_CYCLES 2000000000ll
#define MX_WAIT_SHORT_CYCLES 1000000ll

__device__ int g_mx_error = 0;                                    // 0, or (code << 8 | role) of the first wait that ran out
__device__ long long g_mx_wait_limit = MX_WAIT_LIMIT_CYCLES;      // a variable, so that a test can make a wait run out within a millisecond

__device__ __forceinline__ void mx_raise(int role) { atomicCAS(&g_mx_error, 0, (FG_ERR_PIPELINE << 8) | role); }
__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// (a try sleeps for up to 20 us: tries that come back sooner take issue slots from the warps that work)
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity), "r"(20000) : "memory");
    return ok != 0;
}
// false when the limit ran out; once a wait has run out somewhere, every later one gives up after a short time
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
    if (mbar_try(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
        if (mbar_try(bar, parity)) return true;
        const long long waited = clock64() - t0;
        if (waited > MX_WAIT_SHORT_CYCLES) {
            if (*(volatile int *)&g_mx_error != 0) return false;
            if (waited > *(volatile long long *)&g_mx_wait_limit) return false;
        }
    }
}
// the same for a whole warp, which stays converged
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
// `bytes` (a multiple of 16) from a 16-byte aligned address
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_alloc(uint32_t where, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_alloc_pair(uint32_t where, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_free_pair(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}
__device__ __forceinline__ uint32_t mapa_u32(uint32_t local_addr, int rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_addr), "r"(rank));
    return remote;
}
// An arrival on a barrier of the pair's other CTA.  Relaxed: what it announces lies in tensor memory and is ordered by the tcgen05 fences
// around it (a release at cluster scope waits for the warp's earlier stores: 1,000 cycles an arrival).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// a copy whose completion is counted on a barrier given by its cluster address (the pair leader's)
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t cluster_bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(cluster_bar) : "memory");
}
// arrives on the barrier at this address in both CTAs of the pair once the MMAs issued so far are complete
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
    const uint16_t both = 3;
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(both) : "memory");
}
__device__ __forceinline__ void tc_free(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}
// Operands in shared memory: K-major tiles, rows of 128 bytes swizzled by 128, 8-row groups 1024 bytes apart.  Of the descriptor only the lower word (mx_desc_lo)
// changes between MMAs, by the address in units of 16 bytes; the upper one is a constant.
#define MX_DESC_HI 0x40004040
__device__ __forceinline__ uint32_t mx_desc_lo(uint32_t saddr) { return (saddr & 0x3FFFF) >> 4 | 1u << 16; }
// D (tensor memory) (+)= A B^T in bfloat16, A in tensor memory (a lane a row, two neighbouring k a column), B in shared memory
__device__ __forceinline__ void tc_mma_bf16_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(acc), "n"(MX_DESC_HI) : "memory");
}
// the same with A and D spread over the tensor memory of a pair of CTAs, B over their shared memory
__device__ __forceinline__ void tc_mma_bf16_ts_pair(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], b, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(acc), "n"(MX_DESC_HI) : "memory");
}
// D (tensor memory) (+)= A B^T of 4-bit numbers whose blocks of 32 share a power of two, 64 numbers of K; both operands in shared memory, the
// exponents in tensor memory
__device__ __forceinline__ void tc_mma_mxf4(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t ea, uint32_t eb, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %6, 0;\n\tmov.b64 a, {%1, %7};\n\tmov.b64 b, {%2, %7};\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(ea), "r"(eb), "r"(acc), "n"(MX_DESC_HI) : "memory");
}
// 512 bytes of exponents (32 rows of 16: 8 rows every 128 bytes, not swizzled) from shared memory to four columns of tensor memory, the same for each
// group of 32 lanes; the address in units of 16 bytes
__device__ __forceinline__ void tc_cp_exponents(uint32_t taddr, uint32_t saddr16) {
    asm volatile("{\n\t.reg .b64 s;\n\tmov.b64 s, {%1, %2};\n\t"
                 "tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], s;\n\t}" ::"r"(taddr), "r"(saddr16), "n"(0x4008) : "memory");
}
// sixteen columns of this lane's row, without the wait
__device__ __forceinline__ void tc_ld16_async(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&w)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "r"(w[8]), "r"(w[9]), "r"(w[10]),
                   "r"(w[11]), "r"(w[12]), "r"(w[13]), "r"(w[14]), "r"(w[15]) : "memory");
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync_all() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_dsmem_f32(uint32_t local_addr, int rank) {
    uint32_t remote;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
    return v;
}

__device__ __forceinline__ float4 ld_dsmem_f32x4(uint32_t local_addr, int rank) {
    uint32_t remote;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
    return v;
}

// ---------------------------------------------------------------------------- host side
typedef CUresult (*MxEncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                               const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static inline MxEncodeFn mx_encode_fn() {
    static std::atomic<MxEncodeFn> known;
    MxEncodeFn fn = known.load(std::memory_order_relaxed);
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            known.store(fn = (MxEncodeFn)p, std::memory_order_relaxed);
    }
    return fn;
}
// a matrix of `rows` rows of `row_bytes` bytes, `pitch` bytes apart, in boxes of box_rows x box_bytes; zeros outside
static inline int mx_make_map(CUtensorMap *map, const void *base, bool bf16_numbers, long long rows, long long row_bytes, long long pitch, int box_rows,
                              int box_bytes, CUtensorMapSwizzle swizzle) {
    MxEncodeFn fn = mx_encode_fn();
    if (!fn) return FG_ERR_TENSORMAP;
    const int size = bf16_numbers ? 2 : 1;
    cuuint64_t dims[2] = {(cuuint64_t)(row_bytes / size), (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)pitch};
    cuuint32_t box[2] = {(cuuint32_t)(box_bytes / size), (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, bf16_numbers ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)base, dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : FG_ERR_TENSORMAP;
}
static inline int mx_device() {
    int dev = 0;
    return cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 ? -1 : dev;      // (-1: nothing is kept for it)
}
static inline int mx_sm_count() {
    static std::atomic<int> known[64];
    const int dev = mx_device();
    int n = dev < 0 ? 0 : known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        int at = 0;
        if (cudaGetDevice(&at) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, at) != cudaSuccess || n <= 0) return 148;
        if (dev >= 0) known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}
// How many clusters of S CTAs (along z; S 1: CTAs) of a kernel that takes an SM to itself run at once: clusters stay inside a group of SMs, and the groups' sizes
// are no multiples of S (of 7 or 8, fewer than 16 fit).  Asked once per device and S, once the kernel is set up there.  0, or the error of the question.
struct MxClusters { std::atomic<short> n[64][9]; };
template <typename K>
static inline int mx_clusters(MxClusters &known, K kernel, int threads, int smem, int S, int &fit) {
    if (S == 1) { fit = mx_sm_count(); return 0; }
    const int dev = mx_device();
    fit = dev < 0 ? 0 : known.n[dev][S].load(std::memory_order_relaxed);
    if (fit > 0) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1, 1, S); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = S;
    cfg.attrs = attr; cfg.numAttrs = 1;
    const int rc = (int)cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg);
    if (rc) { cudaGetLastError(); return rc; }
    if (dev >= 0 && fit > 0) known.n[dev][S].store((short)fit, std::memory_order_relaxed);
    return 0;
}
