// (included by gemm_mxfp4.cu)
// Contraction of two matrices in microscaled 4-bit floating point (format: mxfp4.cuh): out[m, n] (+)= sum_k x[m, k] w[n, k].  The tensor core
// takes the codes and the exponents as they are (tcgen05.mma kind::mxf4 with a block's power of two for 32 numbers); products
// are exact, sums float32.
//
// A tile is 128 weight rows (the M side) x BN tokens (the N side); K goes in stages of 256 (128 bytes a row of either operand).
//
//   warp 0      TMA producer: both operands, swizzled by 128 bytes, and the tiles of 512 bytes that hold the exponents of 128 rows x 128 numbers -
//               the layout in which tensor memory wants them, so they are copied as they lie
//   warp 1      MMA issuer: the stage's exponents to tensor memory (tcgen05.cp, 32 lanes x 16 bytes, for all four lane groups), then four
//               128 x BN x 64; its commit frees the stage, exponents included
//   warps 2-9   epilogue, two to a lane group: the accumulator goes to registers at once and is free for the next tile while they store
//
// One CTA an SM walks the tiles; with few tiles a cluster of CTAs splits K and sums through distributed shared memory, in rank order.
// What bounds it: the feed of the tensor pipe, busy in 65 % of active cycles at 2,048 x 28,672 x 4,096.  Measured: 200 x 8,192 x 2,048 6.8 to 8.7 us;
// 1 to 16 x 8,192 x 4,096 8.0; 2,048 x 14,336 x 4,096 54 to 63 us (4.4 to 3.8 PFLOP/s).
#pragma once

#define BOTH_ROWS 128
#define BOTH_K 256
#define BOTH_THREADS 320
#define BOTH_A_BYTES (BOTH_ROWS * BOTH_K / 2)
#define BOTH_MAX_STAGES 6
#define BOTH_SMEM (221 * 1024)

struct MxBoth {
    MxGemm g;                                       // (x, ldx, x_vec unused)
    const uint8_t *xsc;                             // exponents of x
    int bn, stages, tiles_m, n_tiles, kb_per_split, test_skip_copy;
};

__global__ void __launch_bounds__(BOTH_THREADS, 1)
mxfp4_both_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const MxBoth a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t bars[2 * BOTH_MAX_STAGES + 2];
    __shared__ uint32_t tmem_base_s;

    const int warp = warp_index(), lane = threadIdx.x & 31;
    const int bn = a.bn, stages = a.stages, S = gridDim.z, tiles_k = mx_tiles(a.g.K), all_kb = (a.g.K + BOTH_K - 1) / BOTH_K;
    const int sides = bn > 128 ? 2 : 1;             // tiles of 128 tokens whose exponents a stage holds
    // a stage: weights | tokens | exponents of the weights (two tiles of 128 numbers) | of the tokens (two each)
    const int x_at = BOTH_A_BYTES, e_at = x_at + bn * (BOTH_K / 2), stage_bytes = (e_at + 2 * (1 + sides) * MX_TILE_BYTES + 1023) & ~1023;
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = full0 + 8 * BOTH_MAX_STAGES, tfull = empty0 + 8 * BOTH_MAX_STAGES, tempty = tfull + 8;
    const uint32_t smem0 = smem_u32(smem);
    const int kb0 = blockIdx.z * a.kb_per_split, nkb = min(a.kb_per_split, all_kb - kb0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; s++) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        mbar_init(tfull, 1);
        mbar_init(tempty, 8);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 64) { tma_prefetch_map(&tmX); tma_prefetch_map(&tmW); }
    pdl_wait();                                     // (before tensor memory is allocated: no kernel in front holds any then)
    if (warp == 1) tc_alloc(smem_u32(&tmem_base_s), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;

    if (warp == 0) {
        int s = 0, ph = 0, issued = 0;
        bool ok = true;
        const int last_m = mx_tiles(a.g.M) - 1;
        for (int T = blockIdx.x; T < a.n_tiles && ok; T += gridDim.x) {
            const int mt = T % a.tiles_m, nt = T / a.tiles_m, m0 = mt * bn;
            for (int kb = kb0; kb < kb0 + nkb; kb++, issued++) {
                ok = mbar_wait_warp(empty0 + 8 * s, ph ^ 1);
                if (!ok) { mx_raise(1); break; }
                if (elect_one()) {
                    const uint32_t dst = smem0 + s * stage_bytes, bar = full0 + 8 * s;
                    const int halves = min(2, tiles_k - 2 * kb);     // tiles of 128 numbers K still has
                    mbar_expect_tx(bar, e_at + halves * (1 + sides) * MX_TILE_BYTES);
                    tma_load_2d(dst, &tmW, kb * (BOTH_K / 2), nt * BOTH_ROWS, bar);
                    if (!(a.test_skip_copy && issued == 0)) tma_load_2d(dst + x_at, &tmX, kb * (BOTH_K / 2), m0, bar);
                    // (neighbouring tiles along K are neighbours in memory)
                    bulk_load(dst + e_at, a.g.sc + ((size_t)nt * tiles_k + 2 * kb) * MX_TILE_BYTES, halves * MX_TILE_BYTES, bar);
                    for (int q = 0; q < sides; q++)                  // (past the last token: any exponents, those sums are not stored)
                        bulk_load(dst + e_at + (2 + 2 * q) * MX_TILE_BYTES, a.xsc + ((size_t)min(m0 / 128 + q, last_m) * tiles_k + 2 * kb) * MX_TILE_BYTES,
                                  halves * MX_TILE_BYTES, bar);
                }
                __syncwarp();
                if (++s == stages) { s = 0; ph ^= 1; }
            }
        }
        for (int j = max(0, issued - stages); j < issued; j++)      // copies in flight land before the CTA exits
            mbar_wait(full0 + 8 * (j % stages), (j / stages) & 1);
        for (int j = max(0, issued - stages); j < issued; j++)      // so do the last commits' arrivals
            mbar_wait(empty0 + 8 * (j % stages), (j / stages) & 1);
        __syncwarp();
    } else if (warp == 1) {
        // instruction descriptor: both operands e2m1, exponents as bytes; bits 4 and 29 name the half word of exponents a step reads
        const uint32_t idesc = (1u << 7) | (1u << 10) | ((uint32_t)(bn >> 3) << 17) | (1u << 23) | ((uint32_t)(BOTH_ROWS >> 4) << 24);
        int s = 0, ph = 0, i = 0;
        bool ok = true;
        for (int T = blockIdx.x; T < a.n_tiles && ok; T += gridDim.x, i++) {
            ok = mbar_wait_warp(tempty, (i & 1) ^ 1);
            if (!ok) { mx_raise(4); break; }
            for (int kb = 0; kb < nkb; kb++) {
                ok = mbar_wait_warp(full0 + 8 * s, ph);
                if (!ok) { mx_raise(2); break; }
                tc_fence_after();
                const uint32_t base16 = (smem0 + s * stage_bytes) >> 4, e16 = base16 + (e_at >> 4), ad = mx_desc_lo(smem0 + s * stage_bytes), bd = ad + (x_at >> 4);
                // exponents of this stage: columns 256 + 24 s: weights [half][4], tokens [half][side][4]
                const uint32_t ea = tmem + 256 + s * 24, eb = ea + 8;
                const int left = a.g.K - (kb0 + kb) * BOTH_K;
                if (elect_one()) {
                    // (a whole stage as straight code: a step's operands cost more cycles than the step where they are computed one by one)
                    if (left >= BOTH_K) {
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            tc_cp_exponents(ea + 4 * h, e16 + h * (MX_TILE_BYTES >> 4));
                            tc_cp_exponents(eb + 8 * h, e16 + (2 + h) * (MX_TILE_BYTES >> 4));
                            if (sides == 2) tc_cp_exponents(eb + 8 * h + 4, e16 + (4 + h) * (MX_TILE_BYTES >> 4));
                        }
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            tc_mma_mxf4(tmem, ad + 2 * k, bd + 2 * k, idesc | (k & 1) * (2u << 4 | 2u << 29), ea + 4 * (k >> 1), eb + 8 * (k >> 1), (kb | k) != 0);
                    } else {
                        const int steps = (left + 63) / 64, halves = (left + 127) / 128;
                        for (int h = 0; h < halves; h++) {
                            tc_cp_exponents(ea + 4 * h, e16 + h * (MX_TILE_BYTES >> 4));
                            for (int q = 0; q < sides; q++) tc_cp_exponents(eb + 8 * h + 4 * q, e16 + (2 + 2 * q + h) * (MX_TILE_BYTES >> 4));
                        }
                        for (int k = 0; k < steps; k++)
                            tc_mma_mxf4(tmem, ad + 2 * k, bd + 2 * k, idesc | (k & 1) * (2u << 4 | 2u << 29), ea + 4 * (k >> 1), eb + 8 * (k >> 1), (kb | k) != 0);
                    }
                    tc_commit(empty0 + 8 * s);
                }
                __syncwarp();
                if (++s == stages) { s = 0; ph ^= 1; }
            }
            if (elect_one()) tc_commit(tfull);                       // also after an error: the epilogue is not left waiting
            __syncwarp();
        }
    } else {
        const int lg = warp & 3, half = (warp - 2) >> 2, r = lg * 32 + lane;
        const uint32_t trow = tmem + ((uint32_t)(lg * 32) << 16);
        int i = 0;
        for (int T = blockIdx.x; T < a.n_tiles; T += gridDim.x, i++) {
            const int m0 = T % a.tiles_m * bn, n = T / a.tiles_m * BOTH_ROWS + r;
            const bool have = mbar_wait_warp(tfull, i & 1);
            if (!have) mx_raise(5);
            __syncwarp();
            tc_fence_after();
            uint32_t v[8][16];                      // columns 16 (2 q + half) ..
#pragma unroll
            for (int q = 0; q < 8; q++)
                if ((2 * q + half) * 16 < bn) tc_ld16_async(trow + (2 * q + half) * 16, v[q]);
            tc_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty);
            __syncwarp();                           // (tcgen05.ld wants a converged warp)
            if (S > 1) {
                float *part = (float *)smem;        // [bn][128]: the ring is idle
#pragma unroll
                for (int q = 0; q < 8; q++)
                    if ((2 * q + half) * 16 < bn)
#pragma unroll
                        for (int j = 0; j < 16; j++) part[((2 * q + half) * 16 + j) * BOTH_ROWS + r] = have ? __uint_as_float(v[q][j]) : 0.f;
            } else if (have && n < a.g.N) {
#pragma unroll
                for (int q = 0; q < 8; q++)
                    if ((2 * q + half) * 16 < bn) tile_store(a.g, m0 + (2 * q + half) * 16, a.g.M, n, v[q]);
            }
            if (!have) break;
        }
        tc_fence_before();
    }
    if (S > 1) {
        // the columns rank, rank + S, .. of the tile: partial sums of all CTAs of the cluster, in rank order
        cluster_sync_all();
        if (warp >= 2) {
            const int m0 = (int)blockIdx.x % a.tiles_m * bn;
            cluster_columns(a.g, smem0, m0, min(bn, a.g.M - m0), (int)blockIdx.x / a.tiles_m * BOTH_ROWS, S, threadIdx.x - 64, 256);
        }
        cluster_sync_all();                         // nobody leaves while others read its shared memory
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) { tc_fence_after(); tc_free(tmem, 512); }
}

static int both_setup() {
    static FgPerDevice configured;
    return fg_allow_shared(configured, mxfp4_both_kernel, BOTH_SMEM);
}

static int launch_both(MxBoth a, const void *x, int bn, int S, cudaStream_t stream) {
    const MxGemm &g = a.g;
    const int all_kb = (g.K + BOTH_K - 1) / BOTH_K, sides = bn > 128 ? 2 : 1;
    const int stage_bytes = (BOTH_A_BYTES + bn * (BOTH_K / 2) + 2 * (1 + sides) * MX_TILE_BYTES + 1023) & ~1023;
    a.bn = bn;
    a.test_skip_copy = g_mx_test_skip_copy;
    a.stages = (BOTH_SMEM - 1024) / stage_bytes;
    if (a.stages > BOTH_MAX_STAGES) a.stages = BOTH_MAX_STAGES;
    a.kb_per_split = (all_kb + S - 1) / S;
    S = (all_kb + a.kb_per_split - 1) / a.kb_per_split;              // no CTA without a share
    a.tiles_m = (g.M + bn - 1) / bn;
    const long long tiles = (long long)a.tiles_m * mx_tiles(g.N);
    if (tiles > 0x3fffffff) return FG_ERR_BAD_SIZE;
    a.n_tiles = (int)tiles;
    CUtensorMap tmX, tmW;
    int rc = mx_make_map(&tmX, x, false, g.M, g.K / 2, g.K / 2, bn, BOTH_K / 2, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    rc = mx_make_map(&tmW, g.w, false, g.N, g.K / 2, g.K / 2, BOTH_ROWS, BOTH_K / 2, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    rc = both_setup();
    if (rc) return rc;
    const int n_sm = mx_sm_count();
    // (all of an SM's shared memory, needed or not: see launch_tiles)
    return mx_launch(mxfp4_both_kernel, dim3(S > 1 || tiles < n_sm ? (unsigned)tiles : (unsigned)n_sm, 1, S), BOTH_THREADS, BOTH_SMEM, dim3(1, 1, S), stream, tmX, tmW, a);
}

// The tile's width and the split of K that finish first: rounds of tiles over the SMs times what a tile takes, in SM cycles.  Tiles of
// more than one start at multiples of 128 tokens, where tiles of exponents do.
static int both_plan(int M, int N, int K, int &bn, int &S) {
    static MxClusters known;
    int fit[9];
    int rc = both_setup();
    for (int s = 1; s <= 8 && !rc; s++) rc = mx_clusters(known, mxfp4_both_kernel, BOTH_THREADS, BOTH_SMEM, s, fit[s]);
    if (rc) return rc;
    const int n_sm = mx_sm_count(), all_kb = (K + BOTH_K - 1) / BOTH_K, tiles_n = mx_tiles(N), whole = (M + 15) / 16 * 16;
    const int widths[2] = {whole < 256 ? whole : 256, whole < 128 ? whole : 128};
    double best = 1e30;
    for (int i = 0; i < 2; i++) {
        const int b = widths[i];
        const long long tiles = (long long)((M + b - 1) / b) * tiles_n;
        for (int s = 1; s <= 8; s++) {
            if (s > 1 && tiles > fit[s]) continue;
            const int kb = (all_kb + s - 1) / s;
            const double tile = kb * (300 + 1.9 * b) + 2500 + 5.0 * b + (s > 1 ? 1500 + 12.0 * b : 0);
            const double cost = (double)((tiles * s + n_sm - 1) / n_sm) * tile;
            if (cost < best) { best = cost; bn = b; S = s; }
        }
    }
    return 0;
}

// x, w and their exponents in the format; bn 0: both by the rule, else (tests, measurements) tokens a tile - 128, 256, or a multiple of 16 up to 256 that takes
// all rows - and CTAs that share K, 1 to 8
extern "C" int fg_gemm_mxfp4_both_ext(const void *x, const void *x_scales, const void *w, const void *w_scales, void *out, int out_dtype, long long ldo,
                                      int accumulate, int M, int N, int K, int bn, int splits, cudaStream_t stream) {
    MxBoth a = {};
    a.g = {nullptr, (const uint8_t *)w, (const uint8_t *)w_scales, out, 0, ldo, M, N, K, out_dtype, accumulate, 0, nullptr, 0, 0};
    a.xsc = (const uint8_t *)x_scales;
    const int bad = mx_check(a.g);
    if (bad) return bad;
    if (((uintptr_t)x & 15) || ((uintptr_t)x_scales & 15)) return FG_ERR_BAD_SIZE;
    if (M == 0) return 0;
    if (bn == 0) {
        const int rc = both_plan(M, N, K, bn, splits);
        if (rc) return rc;
    } else if (bn < 16 || bn > 256 || bn % 16 || (bn % 128 && bn < M) || splits < 1 || splits > 8) return FG_ERR_BAD_SIZE;
    return launch_both(a, x, bn, splits, stream);
}
extern "C" int fg_gemm_mxfp4_both(const void *x, const void *x_scales, const void *w, const void *w_scales, void *out, int out_dtype, long long ldo,
                                  int accumulate, int M, int N, int K, cudaStream_t stream) {
    return fg_gemm_mxfp4_both_ext(x, x_scales, w, w_scales, out, out_dtype, ldo, accumulate, M, N, K, 0, 0, stream);
}
