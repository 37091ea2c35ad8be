// Contractions with weights in microscaled 4-bit floating point (format: mxfp4.cuh): out[m, n] (+)= sum_k x[m, k] w[n, k] with x in
// bfloat16, for one matrix and for rows grouped by expert on a stack of matrices.  A weight is exact in bfloat16 and a product of two
// bfloat16 numbers in float32; sums are float32.
#include "mxfp4.cuh"

struct MxGemm {
    const bf16 *x;             // [M, K], rows ldx numbers apart
    const uint8_t *w, *sc;     // weights and exponents
    void *out;                 // [M, N] of out_dtype, rows ldo numbers apart
    long long ldx, ldo;
    int M, N, K, out_dtype, accumulate, x_vec;
    const int *offsets;        // grouped: rows offsets[e] .. offsets[e + 1] of x go with matrix e; null: one matrix
    int experts;
    int chunks_per_split;      // chunks of 128 numbers of K a CTA of the cluster takes
};

// Rows [begin, end) of x that matrix e takes.  Offsets that fall or leave the rows of x name no row outside it.
__device__ __forceinline__ void mx_run(const MxGemm &a, int e, int &begin, int &end) {
    begin = min(max(a.offsets[e], 0), a.M);
    end = min(max(a.offsets[e + 1], begin), a.M);
}

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
__device__ __forceinline__ void mma_bf16_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mx_store(const MxGemm &a, int m, int n, float v) {
    const size_t at = (size_t)m * a.ldo + n;
    if (a.out_dtype == FG_F32) { float *o = (float *)a.out + at; *o = a.accumulate ? *o + v : v; }
    else ((bf16 *)a.out)[at] = __float2bfloat16_rn(v);
}

// ---------------------------------------------------------------------------- few rows: weights straight from memory to the MMA
// A CTA takes 64 weight rows and a share of K, its eight warps two sets of 32 rows x four interleaved shares of the chunks of 128 numbers.
// Weight rows are the M side of mma.sync.m16n8k16, tokens its N side.  The order of k inside a chunk is free as long as both operands
// follow it: lane (g, t) of a warp reads 16 bytes - block t of the chunk, 32 numbers that share one exponent - of row g of each of
// four groups of eight rows, and feeds them to the eight MMAs of the chunk as they come, so that weights go from global memory to the
// tensor core through registers alone.  x lies in shared memory in that order.  The four shares of K are added in shared memory, the CTAs
// of a cluster (a split of K where there are few weight rows) through distributed shared memory, both in a fixed order.
#define STREAM_ROWS 64
#define STREAM_KG 4
#define STREAM_CHUNKS(NT) (32 / (NT))       // chunks of x that are staged at once: 64 KB

template <int NT>
__global__ void __launch_bounds__(256, 2)
mxfp4_stream_kernel(MxGemm a) {
    extern __shared__ __align__(16) uint8_t smem[];
    uint4 *xs = (uint4 *)smem;                                        // [chunk][NT][4][32 lanes] of 8 bfloat16
    float *red = (float *)smem;                                       // [KG][8 NT tokens][64 rows], once x is no longer needed
    const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rg = warp & 1, kg = warp >> 1;
    const int tile = blockIdx.x, S = gridDim.z;
    const int tiles_k = mx_tiles(a.K), blocks = a.K / MX_BLOCK;
    const int c_begin = blockIdx.z * a.chunks_per_split, c_end = min(tiles_k, c_begin + a.chunks_per_split);
    const uint8_t *w = a.w, *sc = a.sc;
    int m_begin, m_end;
    if (a.offsets) {
        const int e = blockIdx.y;
        mx_run(a, e, m_begin, m_end);
        w += (size_t)e * a.N * (a.K / 2);
        sc += (size_t)e * mx_scale_bytes(a.N, a.K);
    } else { m_begin = blockIdx.y * 8 * NT; m_end = min(a.M, m_begin + 8 * NT); }
    // this warp's rows: eight neighbouring rows (i8 ..) of each quarter of a tile of 128, whose exponents are 128 neighbouring bytes
    const int base = (tile >> 1) * 128, i8 = ((tile & 1) * 2 + rg) * 8;
    const uint8_t *wrow[4];
    bool row_ok[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int r = base + 32 * j + i8 + g;
        row_ok[j] = r < a.N;
        wrow[j] = w + (size_t)(row_ok[j] ? r : 0) * (a.K / 2) + t * 16;
    }
    const uint8_t *srow = sc + (size_t)(tile >> 1) * tiles_k * MX_TILE_BYTES + (i8 + g) * 16;

    for (int m0 = m_begin; m0 < m_end; m0 += 8 * NT) {
        float acc[2][NT][4];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][n][j] = 0.f;
        for (int s0 = c_begin; s0 < c_end; s0 += STREAM_CHUNKS(NT)) {
            const int s1 = min(c_end, s0 + STREAM_CHUNKS(NT));
            uint4 d[4], e4;
            auto fetch = [&](int c) {
                const bool live = c < s1 && c * 4 + t < blocks;
#pragma unroll
                for (int j = 0; j < 4; j++) d[j] = live && row_ok[j] ? __ldcs((const uint4 *)(wrow[j] + (size_t)c * 64)) : make_uint4(0, 0, 0, 0);
                e4 = c < s1 ? *(const uint4 *)(srow + (size_t)c * MX_TILE_BYTES) : make_uint4(0, 0, 0, 0);
            };
            fetch(s0 + kg);
            __syncthreads();                                          // the last use of the shared memory is over
            for (int u = threadIdx.x; u < (s1 - s0) * NT * 8 * 16; u += 256) {
                const int p = u & 15, tok = (u >> 4) % (8 * NT), c = (u >> 4) / (8 * NT), k = (s0 + c) * 128 + p * 8;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (m0 + tok < m_end && k < a.K) {
                    const bf16 *src = a.x + (size_t)(m0 + tok) * a.ldx + k;
                    if (a.x_vec) v = *(const uint4 *)src;
                    else {
                        const unsigned short *h = (const unsigned short *)src;
                        v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
                    }
                }
                // pairs (i, i + 4), as mx_unpack8 gives the weights
                const uint4 q = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                                           __byte_perm(v.y, v.w, 0x7632));
                xs[((c * NT + (tok >> 3)) * 4 + (p & 3)) * 32 + (tok & 7) * 4 + (p >> 2)] = q;
            }
            __syncthreads();
            for (int c = s0 + kg; c < s1; c += STREAM_KG) {
                const uint4 cur[4] = {d[0], d[1], d[2], d[3]};
                const uint32_t se[4] = {(e4.x >> (8 * t)) & 255, (e4.y >> (8 * t)) & 255, (e4.z >> (8 * t)) & 255, (e4.w >> (8 * t)) & 255};
                fetch(c + STREAM_KG);
                const bool small = __all_sync(0xffffffffu, mx_small(se[0]) && mx_small(se[1]) && mx_small(se[2]) && mx_small(se[3]));
                const uint4 *xc = xs + (size_t)(c - s0) * NT * 128 + lane;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    uint32_t r[4][4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        mx_unpack8(u == 0 ? cur[j].x : u == 1 ? cur[j].y : u == 2 ? cur[j].z : cur[j].w, r[j]);
                        if (small) {
                            const uint32_t f = mx_factor(se[j]);
#pragma unroll
                            for (int q = 0; q < 4; q++) r[j][q] = mul_bf16x2(r[j][q], f);
                        } else {
#pragma unroll
                            for (int q = 0; q < 4; q++) r[j][q] = mx_scale_large(r[j][q], se[j]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const uint4 b = xc[(n * 4 + u) * 32];
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            mma_bf16_16x8x16(acc[i][n], r[2 * i][0], r[2 * i + 1][0], r[2 * i][1], r[2 * i + 1][1], b.x, b.y);
                            mma_bf16_16x8x16(acc[i][n], r[2 * i][2], r[2 * i + 1][2], r[2 * i][3], r[2 * i + 1][3], b.z, b.w);
                        }
                    }
                }
            }
        }
        // sums of the four shares of K, then of the cluster's CTAs
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    red[(kg * 8 * NT + n * 8 + 2 * t + (j & 1)) * STREAM_ROWS + rg * 32 + (2 * i + (j >> 1)) * 8 + g] = acc[i][n][j];
        __syncthreads();
        const int tokens = min(8 * NT, m_end - m0), total = tokens * STREAM_ROWS;
        for (int u = threadIdx.x; u < total; u += 256) {
            float v = red[u];
#pragma unroll
            for (int q = 1; q < STREAM_KG; q++) v += red[q * 8 * NT * STREAM_ROWS + u];
            if (S == 1) {
                const int rl = u & 63, n = base + ((rl >> 3) & 3) * 32 + ((tile & 1) * 2 + (rl >> 5)) * 8 + (rl & 7);
                if (n < a.N) mx_store(a, m0 + u / STREAM_ROWS, n, v);
            } else red[u] = v;
        }
        if (S > 1) {
            cluster_sync_all();
            const uint32_t red0 = (uint32_t)__cvta_generic_to_shared(red);
            for (int u = blockIdx.z * 256 + threadIdx.x; u < total; u += 256 * S) {
                float v = 0.f;
                for (int z = 0; z < S; z++) v += ld_dsmem_f32(red0 + u * 4, z);
                const int rl = u & 63, n = base + ((rl >> 3) & 3) * 32 + ((tile & 1) * 2 + (rl >> 5)) * 8 + (rl & 7);
                if (n < a.N) mx_store(a, m0 + u / STREAM_ROWS, n, v);
            }
            cluster_sync_all();                                       // nobody overwrites or leaves what others still read
        }
    }
}

template <int NT>
static int launch_stream(MxGemm a, int y, cudaStream_t stream) {
    const int tiles_k = mx_tiles(a.K), tiles_n = 2 * mx_tiles(a.N);      // a tile: eight rows twice in each quarter of 128
    int S = 1;
    while (S < 8 && (long long)tiles_n * y * S < 296 && tiles_k > S * STREAM_KG) S *= 2;
    a.chunks_per_split = (tiles_k + S - 1) / S;
    const int staged = a.chunks_per_split < STREAM_CHUNKS(NT) ? a.chunks_per_split : STREAM_CHUNKS(NT);
    const int red = STREAM_KG * 8 * NT * STREAM_ROWS * 4, xb = staged * NT * 2048;
    const int smem = xb > red ? xb : red;
    static FgPerDevice configured;
    if (fg_needs_setup(configured)) {
        cudaError_t e = cudaFuncSetAttribute(mxfp4_stream_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, STREAM_CHUNKS(NT) * NT * 2048);
        if (e != cudaSuccess) return (int)e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles_n, y, S); cfg.blockDim = dim3(256); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = S;
    cfg.attrs = attr; cfg.numAttrs = S > 1 ? 1 : 0;
    return (int)cudaLaunchKernelEx(&cfg, mxfp4_stream_kernel<NT>, a);
}

static int mx_check(const MxGemm &a) {
    if (a.out_dtype != FG_F32 && a.out_dtype != FG_BF16) return FG_ERR_BAD_DTYPE;
    if (a.accumulate && a.out_dtype != FG_F32) return FG_ERR_BAD_DTYPE;
    if (a.M < 0 || a.N <= 0 || a.K <= 0 || a.K % MX_BLOCK || a.ldx < 0 || a.ldo < 0 || ((uintptr_t)a.w & 15) || ((uintptr_t)a.sc & 15)) return FG_ERR_BAD_SIZE;
    return 0;
}

extern "C" int fg_gemm_mxfp4(const void *x, long long ldx, const void *w, const void *scales, void *out, int out_dtype, long long ldo, int accumulate,
                             int M, int N, int K, cudaStream_t stream) {
    MxGemm a = {(const bf16 *)x, (const uint8_t *)w, (const uint8_t *)scales, out, ldx, ldo, M, N, K, out_dtype, accumulate, 0, nullptr, 0, 0};
    const int bad = mx_check(a);
    if (bad) return bad;
    if (M == 0) return 0;
    a.x_vec = ((uintptr_t)x & 15) == 0 && ldx % 8 == 0;
    if (M <= 8) return launch_stream<1>(a, 1, stream);
    if (M > 65535 * 16) return FG_ERR_BAD_SIZE;
    return launch_stream<2>(a, (M + 15) / 16, stream);
}

// offsets: [experts + 1] on the device; w, scales: the experts' matrices one after another
extern "C" int fg_gemm_mxfp4_grouped(const void *x, long long ldx, const void *w, const void *scales, const int *offsets, int experts, void *out,
                                     int out_dtype, long long ldo, int accumulate, int M, int N, int K, cudaStream_t stream) {
    MxGemm a = {(const bf16 *)x, (const uint8_t *)w, (const uint8_t *)scales, out, ldx, ldo, M, N, K, out_dtype, accumulate, 0, offsets, experts, 0};
    const int bad = mx_check(a);
    if (bad) return bad;
    if (experts <= 0 || experts > 65535 || !offsets) return FG_ERR_BAD_SIZE;
    if (M == 0) return 0;
    a.x_vec = ((uintptr_t)x & 15) == 0 && ldx % 8 == 0;
    return (long long)M <= 4ll * experts ? launch_stream<1>(a, experts, stream) : launch_stream<2>(a, experts, stream);
}
