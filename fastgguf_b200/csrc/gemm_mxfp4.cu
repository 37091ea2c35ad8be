// Contractions with weights in microscaled 4-bit floating point (format: mxfp4.cuh): out[m, n] (+)= sum_k x[m, k] w[n, k] with x in
// bfloat16, for one matrix and for rows grouped by expert on a stack of matrices.  A weight is exact in bfloat16 and a product of two
// bfloat16 numbers in float32; sums are float32.
#include "mxfp4_tc.cuh"

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

// ---------------------------------------------------------------------------- few rows: weights through a warp's own ring to the MMA
// Weight rows are the M side of mma.sync.m16n8k16, tokens its N side.  A warp takes 32 weight rows x chunks of 128 numbers of K; lane (g, t)
// of it handles 16 bytes - block t of the chunk, 32 numbers that share one exponent - of row g of each of four groups of eight rows and
// feeds them to the eight MMAs of the chunk as they come: the order of k inside a chunk is free as long as both operands follow it.  x lies
// in shared memory in the lanes' order.  Every lane copies what it will use itself, asynchronously and three chunks ahead (104 KB in flight
// on an SM, with no registers held for them), so the ring needs no barrier.
//
// What bounds it: neither memory nor issue alone.  At the memory's rate an SM gets a chunk's 2,176 bytes of 32 rows every 92 cycles, in which its four
// schedulers issue 368; unpacking them takes 192, the MMAs, loads and addresses some 70.  Measured: 8 x 28,672 x 4,096 22.6 us (2.8 TB/s): 896 units on 592
// groups of warps are two rounds for 1.51, the schedulers issue in 55 % of active cycles, DRAM is at 30 %, and a warp that does not issue waits for its copies, for
// a busy pipe and for its last result in about equal parts (1.1, 1.1 and 1.0 cycles an instruction).  One row of 128,256 x 2,048 35.1 us (4.0 TB/s):
// 6.8 rounds of seven, issue in 65 %, DRAM at 45 %.
// Blocks with exponents above 125 (a largest number of 2 and more: a table of unit variance has them in 78 % of its blocks) take mx_times_rest, a warp's chunk
// as a whole: 8 x 28,672 x 4,096 41.4 us, one row of 128,256 x 2,048 68.5, 8 x 8,192 x 2,048 8.3 from 6.0.
//
// A CTA is two groups of eight warps or four of four; a group takes a unit of 32 rows at a time, its warps a chunk each in turn.  x is staged once for all the
// units of a CTA (in parts, for each unit again, where K is longer than the room).  The warps' sums are added in shared memory, those of a cluster's
// CTAs (a split of K where there are few units, or K is long) through distributed shared memory, all in a fixed order.
#define STREAM_ROWS 32
#define STREAM_ALL 16                       // warps of a CTA, in groups of W
#define STREAM_THREADS (32 * STREAM_ALL)
#define STREAM_RING(NT) ((NT) == 1 ? 4 : 3)  // chunks in a warp's ring (at 16 tokens the partial sums take the room of one)
#define STREAM_SLOT 2176                    // 32 rows x 64 bytes, and 128 bytes of exponents
#define STREAM_CHUNKS(NT) (32 / (NT))       // chunks of x staged at once: 64 KB

// sixteen bytes, of which the first `have` are read, the others zeros
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t have = 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

template <int NT, int W>
__global__ void __launch_bounds__(STREAM_THREADS, 1)
mxfp4_stream_kernel(const MxGemm a, int units) {
    extern __shared__ __align__(16) uint8_t smem[];
    // [warp][RING] slots of weights | [group][warp][8 NT tokens][32 rows] partial sums | x: [chunk][NT][4][32 lanes] of 8 numbers
    constexpr int GROUPS = STREAM_ALL / W, RING = STREAM_RING(NT), RED = W * 8 * NT * STREAM_ROWS;
    float *red_all = (float *)(smem + STREAM_ALL * RING * STREAM_SLOT);
    uint4 *xs = (uint4 *)(red_all + GROUPS * RED);
    const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = warp / W, wl = warp % W, tid = threadIdx.x & (32 * W - 1);
    float *red = red_all + group * RED;
    const uint32_t ring = smem_u32(smem) + warp * RING * STREAM_SLOT;
    const int S = gridDim.z, tiles_k = mx_tiles(a.K), blocks = a.K / MX_BLOCK;
    const int c_begin = blockIdx.z * a.chunks_per_split, c_end = min(tiles_k, c_begin + a.chunks_per_split);
    const bool in_parts = c_end - c_begin > STREAM_CHUNKS(NT);
    const uint8_t *w = a.w, *sc = a.sc;
    pdl_wait();
    int m_begin, m_end;
    if (a.offsets) {
        const int e = blockIdx.y;
        mx_run(a, e, m_begin, m_end);
        w += (size_t)e * a.N * (a.K / 2);
        sc += (size_t)e * mx_scale_bytes(a.N, a.K);
    } else { m_begin = blockIdx.y * 8 * NT; m_end = min(a.M, m_begin + 8 * NT); }
    const size_t pitch = a.K / 2;
    const int first = blockIdx.x * GROUPS + group, stride = gridDim.x * GROUPS;
    auto group_sync = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * W) : "memory"); };

    for (int m0 = m_begin; m0 < m_end; m0 += 8 * NT) {
        // What is copied next: chunk fc of unit fu.  Unit u is eight neighbouring rows (from 8 (u % 4)) of each quarter of a tile of 128, whose
        // exponents are 128 neighbouring bytes.  Rows past the last read that one (their sums are not stored).  Blocks past the end of K get codes of zero:
        // their exponents are padding, any byte but 255, and a number under 253 or 254 may be infinite, which the zeros of x do not cancel.
        int fu = first - stride, fc = c_end, fs = 0;
        const uint8_t *row[4], *exps = nullptr;
        auto copy = [&] {
            if (fc >= c_end) {
                fu += stride;
                fc = c_begin + wl;
                if (fu < units) {
#pragma unroll
                    for (int j = 0; j < 4; j++) row[j] = w + min((fu >> 2) * 128 + 32 * j + (fu & 3) * 8 + g, a.N - 1) * pitch + t * 16;
                    exps = sc + (size_t)(fu >> 2) * tiles_k * MX_TILE_BYTES + ((fu & 3) * 8 + g) * 16;
                }
            }
            if (fu < units && fc < c_end) {
                const bool there = fc * 4 + t < blocks;
                const int at = there ? fc * 64 : -t * 16;
                const uint32_t dst = ring + fs * STREAM_SLOT + lane * 16;
#pragma unroll
                for (int j = 0; j < 4; j++) cp_async16(dst + j * 512, row[j] + at, there ? 16 : 0);
                if (t == 0) cp_async16(ring + fs * STREAM_SLOT + 2048 + g * 16, exps + (size_t)fc * MX_TILE_BYTES);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            fc += W;
            fs = fs + 1 == RING ? 0 : fs + 1;
        };
        for (int i = 0; i < RING - 1; i++) copy();
        int s = 0;                                                    // the slot that is used next
        bool staged = false;
        // (all groups walk as many rounds: the barriers of the whole CTA are met by all)
        for (int u0 = blockIdx.x * GROUPS; u0 < units; u0 += stride) {
            const int u = u0 + group;
            const bool live = u < units;
            float sum[2][NT][4];
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) sum[i][n][j] = 0.f;
            for (int s0 = c_begin; s0 < c_end; s0 += STREAM_CHUNKS(NT)) {
                const int s1 = min(c_end, s0 + STREAM_CHUNKS(NT));
                if (!staged || in_parts) {
                    __syncthreads();                                  // the last use of x is over
                    const int pieces = (s1 - s0) * NT * 128;          // of eight numbers: [chunk][token][16]
#pragma unroll 4
                    for (int q = threadIdx.x; q < pieces; q += STREAM_THREADS) {
                        const int p = q & 15, tok = (q >> 4) & (8 * NT - 1), c = (q >> 7) / NT, k = (s0 + c) * 128 + p * 8;
                        uint4 v = make_uint4(0, 0, 0, 0);
                        if (m0 + tok < m_end && k < a.K) {
                            const bf16 *src = a.x + (size_t)(m0 + tok) * a.ldx + k;
                            if (a.x_vec) v = *(const uint4 *)src;
                            else {
                                const unsigned short *h = (const unsigned short *)src;
                                v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
                            }
                        }
                        xs[((c * NT + (tok >> 3)) * 4 + (p & 3)) * 32 + (tok & 7) * 4 + (p >> 2)] = v;
                    }
                    __syncthreads();
                    staged = true;
                }
                if (!live) continue;
                for (int c = s0 + wl; c < s1; c += W) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(RING - 2) : "memory");
                    __syncwarp();                                     // the exponents were copied by other lanes
                    const uint32_t slot = ring + s * STREAM_SLOT;
                    uint32_t e[4];
                    uint4 d[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        e[j] = lds8(slot + 2048 + g * 16 + t + 4 * j);
                        d[j] = lds128(slot + j * 512 + lane * 16);
                    }
                    __syncwarp();
                    copy();                                           // into the slot that was used last
                    const uint4 *xc = xs + (c - s0) * NT * 128 + lane;
                    auto word = [&](int q, bool small) {
                        uint32_t v[4][4];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            mx_unpack8(q == 0 ? d[j].x : q == 1 ? d[j].y : q == 2 ? d[j].z : d[j].w, v[j]);
                            const uint32_t f = small ? e[j] * 0x00800080u + 129u * 0x00800080u : mx_factor(e[j]);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                v[j][i] = mul_bf16x2(v[j][i], f);
                                if (!small) v[j][i] = mx_times_rest(v[j][i], e[j]);
                            }
                        }
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            const uint4 b = xc[(n * 4 + q) * 32];
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                mma_bf16_16x8x16(sum[i][n], v[2 * i][0], v[2 * i + 1][0], v[2 * i][1], v[2 * i + 1][1], b.x, b.y);
                                mma_bf16_16x8x16(sum[i][n], v[2 * i][2], v[2 * i + 1][2], v[2 * i][3], v[2 * i + 1][3], b.z, b.w);
                            }
                        }
                    };
                    if (__all_sync(0xffffffffu, mx_small(max(max(e[0], e[1]), max(e[2], e[3]))))) {
#pragma unroll
                        for (int q = 0; q < 4; q++) word(q, true);
                    } else {
#pragma unroll 1
                        for (int q = 0; q < 4; q++) word(q, false);
                    }
                    s = s + 1 == RING ? 0 : s + 1;
                }
            }
            // ---- sums of the group's warps, then of the cluster's CTAs
            const int total = live ? min(8 * NT, m_end - m0) * STREAM_ROWS : 0;
            auto store = [&](int q, float v) {
                const int rl = q % STREAM_ROWS, n = (u >> 2) * 128 + (rl >> 3) * 32 + (u & 3) * 8 + (rl & 7);
                if (n < a.N) mx_store(a, m0 + q / STREAM_ROWS, n, v);
            };
            if (live) {
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            red[(wl * 8 * NT + n * 8 + 2 * t + (j & 1)) * STREAM_ROWS + (2 * i + (j >> 1)) * 8 + g] = sum[i][n][j];
                group_sync();
                for (int q = tid; q < total; q += 32 * W) {
                    float v = red[q];
#pragma unroll
                    for (int z = 1; z < W; z++) v += red[z * 8 * NT * STREAM_ROWS + q];
                    if (S == 1) store(q, v); else red[q] = v;
                }
                group_sync();                                         // before the next unit's sums
            }
            if (S > 1) {
                cluster_sync_all();
                const uint32_t red0 = smem_u32(red);
                for (int q = blockIdx.z * 32 * W + tid; q < total; q += 32 * W * S) {
                    float part[8];
#pragma unroll
                    for (int z = 0; z < 8; z++) part[z] = z < S ? ld_dsmem_f32(red0 + q * 4, z) : 0.f;
                    float v = part[0];
#pragma unroll
                    for (int z = 1; z < 8; z++)
                        if (z < S) v += part[z];
                    store(q, v);
                }
                cluster_sync_all();                                   // nobody overwrites or leaves what others still read
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
}

template <int NT, int W>
struct MxStreamForm {
    static constexpr int groups = STREAM_ALL / W, fixed = STREAM_ALL * (STREAM_RING(NT) * STREAM_SLOT + 8 * NT * STREAM_ROWS * 4), room_bytes = fixed + 65536;
    static int setup() {
        static FgPerDevice configured;
        return fg_allow_shared(configured, mxfp4_stream_kernel<NT, W>, room_bytes);
    }
    static int width(int S, int busy, int units, int &gx) {          // CTAs (a cluster of S each) along the units, as many as fit at once
        static MxClusters known;
        int fit = 0;
        const int rc = mx_clusters(known, mxfp4_stream_kernel<NT, W>, STREAM_THREADS, room_bytes, S, fit), most = (units + groups - 1) / groups;
        gx = fit / busy < 1 ? 1 : fit / busy > most ? most : fit / busy;
        return rc;
    }
    // The split of K that finishes first, in us: rounds of units times a warp's chunks and the sums behind them.  Fitted to us | us with groups of eight | four
    // warps, eight rows: 28,672 x 4,096: 23.5 | 22.6; 16,384 x 2,048: 9.6 | 8.9; 4,096 x 14,336: 16.6 | 13.9; 8,192 x 2,048: 6.0 | 6.6 (it splits K);
    // 2,048 x 8,192: 7.4 | 9.3; one row of 128,256 x 2,048: 42.5 | 35.1 (sums of half as many warps, half as often).
    static int plan(int units, int tiles_k, int busy, int &S, double &best) {
        best = 1e30;
        const int rc = setup();
        if (rc) return rc;
        for (int s = 1; s <= 8; s *= 2) {
            if (s < 8 && tiles_k > s * STREAM_CHUNKS(NT)) continue;  // until x fits at once
            if (best < 1e30 && tiles_k <= s / 2 * W) break;          // each warp keeps a chunk
            const int chunks = ((tiles_k + s - 1) / s + W - 1) / W;
            int gx = 1;
            const int bad = width(s, busy, units, gx);
            if (bad) return bad;
            const long long lanes = (long long)gx * groups, rounds = (units + lanes - 1) / lanes;
            const double cost = rounds * (1.1 * chunks + (W == 8 ? 0.55 : 0.2) + (s > 1 ? (W == 8 ? 0.35 : 0.45) * s : 0.0));
            if (cost < best) { best = cost; S = s; }
        }
        return 0;
    }
    static int launch(MxGemm a, int y, int busy, int units, int S, cudaStream_t stream) {      // (behind plan)
        const int tiles_k = mx_tiles(a.K);
        int gx = 1;
        const int rc = width(S, busy, units, gx);
        if (rc) return rc;
        a.chunks_per_split = (tiles_k + S - 1) / S;
        const int staged = a.chunks_per_split < STREAM_CHUNKS(NT) ? a.chunks_per_split : STREAM_CHUNKS(NT);
        return mx_launch(mxfp4_stream_kernel<NT, W>, dim3(gx, y, S), STREAM_THREADS, fixed + staged * NT * 2048, dim3(1, 1, S), stream, a, units);
    }
};
template <int NT>
static int launch_stream(const MxGemm &a, int y, int busy /* of the y, that have rows */, cudaStream_t stream) {
    const int units = 4 * mx_tiles(a.N), tiles_k = mx_tiles(a.K);
    int s8 = 1, s4 = 1;
    double eight, four;
    int rc = MxStreamForm<NT, 8>::plan(units, tiles_k, busy, s8, eight);
    if (!rc) rc = MxStreamForm<NT, 4>::plan(units, tiles_k, busy, s4, four);
    if (rc) return rc;
    return four < eight ? MxStreamForm<NT, 4>::launch(a, y, busy, units, s4, stream) : MxStreamForm<NT, 8>::launch(a, y, busy, units, s8, stream);
}

// ---------------------------------------------------------------------------- more rows: weights through tensor memory
// A tile is 128 weight rows x BN tokens.  Weight rows are the M side of tcgen05.mma and lie in TENSOR MEMORY, where a lane is a row: a
// thread takes 64 packed numbers of its row from shared memory, turns them into bfloat16 with their exponents in registers and stores them
// as 32 columns (two neighbouring k a column); tokens are the N side, bfloat16 rows in shared memory as TMA brings them.  So a weight
// crosses shared memory in its 4 bits, and the tensor core reads only the tokens there.  K goes in stages of 128.
//
//   warp 0      tokens: two boxes of 64 numbers a stage, a ring of up to four
//   warp 1      MMA issuer: eight 128 x BN x 16 a stage; its commit frees the stage's tokens and its slot of tensor memory (four of 64 columns)
//   warp 2      weights: 64 bytes a row and 512 bytes of exponents a stage, a ring of eight
//   warps 3-18  four sets of four, a set to a slot: unpack every fourth stage, and at a tile's end a quarter of its epilogue.  The first
//               stages of the next tile are unpacked BEFORE a tile's epilogue: the tensor core goes on meanwhile.
// Unpacking is bound by the integer pipe when enough warps hide the waits around it: with two warps a scheduler, half a stage each, a
// stage's took 1,500 cycles beside the 1,024 of its MMAs at 256 tokens (2,048 x 8,192 x 4,096: 133 us; with four: 94).  At few tokens a stage
// takes some 650 cycles: unpacking and the chain from a free slot to the next full one, beside MMAs of 46 cycles each.
// Measured: 77 x 8,191 x 2,080 10.1 us; 256 x 8,192 x 4,096 18.1 us (950 TFLOP/s); 2,048 x 14,336 x 4,096 162 us (1,482 TFLOP/s) in a short run, 184 to 190 at
// the power limit; at 2,048 x 28,672 x 4,096 the tensor pipe is busy in 86 % of active cycles.  Where every block has an exponent above 125: 11.1, 22.4 and
// 167 to 190 us.
//
// One CTA an SM walks the tiles.  PAIR: two CTAs of a cluster take 256 weight rows x BN tokens (tcgen05.mma.cta_group::2); each unpacks its
// own 128 rows and brings half of the tokens, which halves the bytes an SM receives per MMA.  With few tiles a cluster of single CTAs splits
// K instead; each sums a share of the columns of all partial tiles out of the others' shared memory, in rank order.
#define TILE_ROWS 128
#define TILE_K 128
#define TILE_THREADS 608
#define TILE_W_BYTES (TILE_ROWS * TILE_K / 2)
#define TILE_W_STAGE (TILE_W_BYTES + 1024)
// A set waits on a place of this ring by parity, and knows only of its own stages that they have come: a place has to be one set's, or a copy that
// is overtaken by a later one leaves the place a phase behind and the wait passes early.
#define TILE_W_STAGES 8
#define TILE_SLOTS 4            // stages in tensor memory, 64 columns each, behind the accumulator's 256
#define TILE_AHEAD 3            // stages of the next tile that are unpacked before a tile's epilogue
#define TILE_MAX_EXPERTS 1024
#define TILE_SMEM (221 * 1024)
#define TILE_UNPACK 650         // SM cycles a stage takes at few tokens: its unpacking

static_assert(TILE_W_STAGES % TILE_SLOTS == 0, "a place of the weights' ring belongs to one set of unpacking warps");
struct MxTiles {
    MxGemm g;
    int bn, xs, tiles_m, tiles_n, n_tiles;          // tokens a tile, depth of their ring (grouped: tiles_m and n_tiles follow from the offsets)
    int kb_per_split;
    int test_skip_copy;                             // tests only: the tokens of the first stage are not copied
};
static int g_mx_test_skip_copy = 0;                 // host side of fg_gemm_mxfp4_test_hook

// a tile: rows [m0, m_end) of x, weight rows from n0 (row w_row of the stack, exponents from tile sc_tile)
struct MxTile { int m0, m_end, n0, w_row, sc_tile; };

template <bool PAIR>
__device__ __forceinline__ MxTile mx_tile(const MxTiles &a, const int *cum, int T, int rank) {
    MxTile t;
    int nt, e = 0;
    if (!a.g.offsets) {
        t.m0 = T % a.tiles_m * a.bn; t.m_end = a.g.M; nt = T / a.tiles_m;
    } else {
        int hi = a.g.experts;                       // cum[e]: tiles of x in front of expert e
        while (hi - e > 1) {
            const int mid = (e + hi) >> 1;
            if (cum[mid] * a.tiles_n <= T) e = mid; else hi = mid;
        }
        int begin, end;
        mx_run(a.g, e, begin, end);
        const int local = T - cum[e] * a.tiles_n, tm = cum[e + 1] - cum[e];
        t.m0 = begin + local % tm * a.bn; t.m_end = end; nt = local / tm;
    }
    const int n128 = PAIR ? 2 * nt + rank : nt, all128 = mx_tiles(a.g.N);
    t.n0 = n128 * TILE_ROWS;
    t.w_row = e * a.g.N + t.n0;
    t.sc_tile = e * all128 + min(n128, all128 - 1);     // (a pair's second half may lie past the matrix: its rows are not stored)
    return t;
}

// What a CTA of a cluster that splits K stores of a tile: the columns rank, rank + S, .. below `count`, summed over the CTAs' partial tiles
// [column][128 rows] at `part` in their shared memory, in rank order.  A thread takes four rows of a column; the CTAs' parts are asked for together.
__device__ __forceinline__ void cluster_columns(const MxGemm &a, uint32_t part, int m0, int count, int n0, int S, int thread, int threads) {
    const int r = (thread & 31) * 4;
    for (int c = blockIdx.z + S * (thread >> 5); c < count; c += S * (threads >> 5)) {
        float4 v[8];
#pragma unroll
        for (int z = 0; z < 8; z++)
            if (z < S) v[z] = ld_dsmem_f32x4(part + (c * 128 + r) * 4, z);
        float4 t = v[0];
#pragma unroll
        for (int z = 1; z < 8; z++)
            if (z < S) { t.x += v[z].x; t.y += v[z].y; t.z += v[z].z; t.w += v[z].w; }
        const float o[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (n0 + r + j < a.N) mx_store(a, m0 + c, n0 + r + j, o[j]);
    }
}

// Sixteen columns (tokens m0 ..) of this thread's weight row n
__device__ __forceinline__ void tile_store(const MxGemm &a, int m0, int m_end, int n, const uint32_t (&v)[16]) {
    const int count = min(16, m_end - m0);
    const size_t at = (size_t)m0 * a.ldo + n;
    if (a.out_dtype == FG_BF16) {
        bf16 *o = (bf16 *)a.out + at;
#pragma unroll
        for (int j = 0; j < 16; j++, o += a.ldo)
            if (j < count) *o = __float2bfloat16_rn(__uint_as_float(v[j]));
    } else if (a.accumulate) {
        float *o = (float *)a.out + at;
#pragma unroll
        for (int j = 0; j < 16; j++, o += a.ldo)
            if (j < count) *o += __uint_as_float(v[j]);
    } else {
        float *o = (float *)a.out + at;
#pragma unroll
        for (int j = 0; j < 16; j++, o += a.ldo)
            if (j < count) *o = __uint_as_float(v[j]);
    }
}

template <bool PAIR>
__global__ void __launch_bounds__(TILE_THREADS, 1)
mxfp4_tile_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const MxTiles a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t bars[2 * TILE_W_STAGES + 2 * TILE_SLOTS + 2];
    __shared__ uint32_t tmem_base_s;
    __shared__ int cum[TILE_MAX_EXPERTS + 1];

    const int warp = warp_index(), lane = threadIdx.x & 31;
    const int bn = a.bn, xs = a.xs, S = gridDim.z, tiles_k = mx_tiles(a.g.K);
    const int rank = PAIR ? (int)(blockIdx.x & 1) : 0, first = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x, stride = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
    const int x_half = (PAIR ? bn / 2 : bn) * 128, x_bytes = 2 * x_half;
    // full[slot]: a stage's weights are in tensor memory (four warps a CTA) and its tokens in shared memory; done[slot]: its MMAs are complete
    const uint32_t wfull0 = smem_u32(&bars[0]), wempty0 = wfull0 + 8 * TILE_W_STAGES, full0 = wempty0 + 8 * TILE_W_STAGES, done0 = full0 + 8 * TILE_SLOTS,
                   tfull = done0 + 8 * TILE_SLOTS, tempty = tfull + 8;
    const uint32_t smem0 = smem_u32(smem);
    uint8_t *wring = smem + xs * x_bytes;
    const int kb0 = blockIdx.z * a.kb_per_split, nkb = min(a.kb_per_split, tiles_k - kb0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < TILE_W_STAGES; s++) { mbar_init(wfull0 + 8 * s, 1); mbar_init(wempty0 + 8 * s, 4); }
        for (int s = 0; s < TILE_SLOTS; s++) { mbar_init(full0 + 8 * s, PAIR ? 9 : 5); mbar_init(done0 + 8 * s, 1); }
        mbar_init(tfull, 1);
        mbar_init(tempty, PAIR ? 32 : 16);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 64) { tma_prefetch_map(&tmX); tma_prefetch_map(&tmW); }
    pdl_wait();                                     // (before tensor memory is allocated: no kernel in front holds any then)
    // the partner runs, and its barriers exist, before a pair allocates tensor memory together or anything arrives on them; its own tensor memory is
    // there when its first arrival on full says so
    if (PAIR) { __syncthreads(); cluster_sync_all(); }
    if (warp == 1) { if (PAIR) tc_alloc_pair(smem_u32(&tmem_base_s), 512); else tc_alloc(smem_u32(&tmem_base_s), 512); }
    if (a.g.offsets && warp == 0) {                 // tiles of x in front of each expert's run
        int sum = 0;
        for (int e0 = 0; e0 < a.g.experts; e0 += 32) {
            int begin = 0, end = 0;
            if (e0 + lane < a.g.experts) mx_run(a.g, e0 + lane, begin, end);
            int upto = (end - begin + bn - 1) / bn;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
            // (no more than rising offsets can make, which is what the host's check of the count covers)
            if (e0 + lane < a.g.experts) cum[e0 + lane + 1] = min(sum + upto, a.tiles_m + a.g.experts);
            sum = min(sum + __shfl_sync(0xffffffffu, upto, 31), a.tiles_m + a.g.experts);
        }
        if (lane == 0) cum[0] = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    const int n_tiles = a.g.offsets ? cum[a.g.experts] * a.tiles_n : a.n_tiles;

    if (warp == 0) {
        // ------------------------------------------------------------ tokens (both CTAs of a pair; they complete on the leader's barriers)
        const uint32_t full = PAIR ? mapa_u32(full0, 0) : full0;
        int g = 0, s = 0;
        bool ok = true;
        for (int T = first; T < n_tiles && ok; T += stride) {
            const int m0 = mx_tile<PAIR>(a, cum, T, rank).m0 + (PAIR ? rank * (bn / 2) : 0);
            for (int kb = kb0; kb < kb0 + nkb; kb++, g++) {
                const int was = g - xs, slot = g % TILE_SLOTS;      // `was`: the stage that used this place before
                if (was >= 0) ok = mbar_wait_warp(done0 + 8 * (was % TILE_SLOTS), (was / TILE_SLOTS) & 1);
                if (!ok) { mx_raise(1); break; }
                if (elect_one()) {
                    const uint32_t dst = smem0 + s * x_bytes, bar = full + 8 * slot;
                    if (rank == 0) mbar_expect_tx(full0 + 8 * slot, (PAIR ? 2 : 1) * x_bytes);
                    // (a test may ask for the first stage to stay incomplete: its barrier then never fires and every wait runs out)
                    if (a.test_skip_copy && g == 0) {}
                    else if (PAIR) { tma_load_2d_pair(dst, &tmX, kb * TILE_K, m0, bar); tma_load_2d_pair(dst + x_half, &tmX, kb * TILE_K + 64, m0, bar); }
                    else { tma_load_2d(dst, &tmX, kb * TILE_K, m0, bar); tma_load_2d(dst + x_half, &tmX, kb * TILE_K + 64, m0, bar); }
                }
                __syncwarp();
                if (++s == xs) s = 0;
            }
        }
        if (rank == 0)                              // copies in flight land before the CTA exits
            for (int j = max(0, g - xs); j < g; j++) mbar_wait(full0 + 8 * (j % TILE_SLOTS), (j / TILE_SLOTS) & 1);
        // so do the last commits' arrivals, which come from the tensor core, a pair's from the leader's SM
        for (int j = max(0, g - TILE_SLOTS); j < g; j++) mbar_wait(done0 + 8 * (j % TILE_SLOTS), (j / TILE_SLOTS) & 1);
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (a pair's leader alone)
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(bn >> 3) << 17) | ((uint32_t)((PAIR ? 2 : 1) * TILE_ROWS >> 4) << 24);
        const uint32_t desc0 = mx_desc_lo(smem0);
        int g = 0, s = 0, i = 0;
        bool ok = rank == 0;
        for (int T = first; T < n_tiles && ok; T += stride, i++) {
            ok = mbar_wait_warp(tempty, (i & 1) ^ 1);
            if (!ok) { mx_raise(4); break; }
            for (int kb = 0; kb < nkb; kb++, g++) {
                const int slot = g % TILE_SLOTS;
                ok = mbar_wait_warp(full0 + 8 * slot, (g / TILE_SLOTS) & 1);
                if (!ok) { mx_raise(2); break; }
                tc_fence_after();
                const uint32_t desc[2] = {desc0 + s * (x_bytes >> 4), desc0 + s * (x_bytes >> 4) + (x_half >> 4)};
                const uint32_t at = tmem + 256 + slot * 64;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        if (PAIR) tc_mma_bf16_ts_pair(tmem, at + k * 8, desc[k >> 2] + (k & 3) * 2, idesc, (kb | k) != 0);
                        else tc_mma_bf16_ts(tmem, at + k * 8, desc[k >> 2] + (k & 3) * 2, idesc, (kb | k) != 0);
                    }
                    if (PAIR) tc_commit_pair(done0 + 8 * slot); else tc_commit(done0 + 8 * slot);
                }
                __syncwarp();
                if (++s == xs) s = 0;
            }
            if (elect_one()) { if (PAIR) tc_commit_pair(tfull); else tc_commit(tfull); }      // also after an error: the epilogue is not left waiting
            __syncwarp();
        }
        if (rank == 0 && i > 0) mbar_wait_warp(tempty, (i - 1) & 1);                         // the last tile's arrivals, the partner's among them
    } else if (warp == 2) {
        // ------------------------------------------------------------ weights and exponents
        int s = 0, ph = 0, issued = 0;
        bool ok = true;
        const uint32_t ring = smem_u32(wring);
        for (int T = first; T < n_tiles && ok; T += stride) {
            const MxTile t = mx_tile<PAIR>(a, cum, T, rank);
            for (int kb = kb0; kb < kb0 + nkb; kb++, issued++) {
                ok = mbar_wait_warp(wempty0 + 8 * s, ph ^ 1);
                if (!ok) { mx_raise(6); break; }
                if (elect_one()) {
                    const uint32_t dst = ring + s * TILE_W_STAGE, bar = wfull0 + 8 * s;
                    mbar_expect_tx(bar, TILE_W_BYTES + MX_TILE_BYTES);
                    tma_load_2d(dst, &tmW, kb * (TILE_K / 2), t.w_row, bar);
                    bulk_load(dst + TILE_W_BYTES, a.g.sc + ((size_t)t.sc_tile * tiles_k + kb) * MX_TILE_BYTES, MX_TILE_BYTES, bar);
                }
                __syncwarp();
                if (++s == TILE_W_STAGES) { s = 0; ph ^= 1; }
            }
        }
        for (int j = max(0, issued - TILE_W_STAGES); j < issued; j++) mbar_wait(wfull0 + 8 * (j % TILE_W_STAGES), (j / TILE_W_STAGES) & 1);
    } else {
        // ------------------------------------------------------------ unpack, epilogue
        const int lg = warp & 3, set = (warp - 3) >> 2, r = lg * 32 + lane;
        const uint32_t trow = tmem + ((uint32_t)(lg * 32) << 16);
        const uint32_t full = PAIR ? mapa_u32(full0, 0) : full0, empty = PAIR ? mapa_u32(tempty, 0) : tempty;
        int i = 0;                                  // tiles finished
        bool ok = true;
        auto unpack = [&](int stage) {              // (stage % TILE_SLOTS == set)
            const int s = stage % TILE_W_STAGES;
            ok = mbar_wait_warp(wfull0 + 8 * s, (stage / TILE_W_STAGES) & 1);
            if (!ok) { mx_raise(3); return; }
            const uint8_t *ws = wring + s * TILE_W_STAGE, *wr = ws + r * 64;
            const uint32_t se = *(const uint32_t *)(ws + TILE_W_BYTES + lane * 16 + lg * 4);
            uint4 d[4];                             // (64 bytes a row, sixteen-byte pieces swizzled by the row)
#pragma unroll
            for (int q = 0; q < 4; q++) d[q] = *(const uint4 *)(wr + ((q ^ ((r >> 1) & 3)) << 4));
            if (stage >= TILE_SLOTS) {
                ok = mbar_wait_warp(done0 + 8 * set, (stage / TILE_SLOTS - 1) & 1);
                if (!ok) { mx_raise(7); return; }
            }
            __syncwarp();
            tc_fence_after();
#pragma unroll
            for (int q = 0; q < 4; q++) {           // a block of 32 numbers
                uint32_t out[16];
                mx_unpack32(d[q], (se >> (8 * q)) & 255, out);
                tc_st16(trow + 256 + set * 64 + q * 16, out);
            }
            tc_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) mbar_arrive_cluster(full + 8 * set); else mbar_arrive(full + 8 * set);
                mbar_arrive(wempty0 + 8 * s);
            }
            __syncwarp();                           // (tcgen05.st and ld want a converged warp)
        };
        auto epilogue = [&](int T) {
            const MxTile t = mx_tile<PAIR>(a, cum, T, rank);
            const bool have = mbar_wait_warp(tfull, i & 1);
            if (!have) { mx_raise(5); ok = false; }
            __syncwarp();
            tc_fence_after();
            uint32_t v[4][16];                      // columns 16 (4 q + set) ..
#pragma unroll
            for (int q = 0; q < 4; q++)
                if ((4 * q + set) * 16 < bn) tc_ld16_async(trow + (4 * q + set) * 16, v[q]);
            tc_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) { if (PAIR) mbar_arrive_cluster(empty); else mbar_arrive(empty); }
            __syncwarp();
            if (!PAIR && S > 1) {
                float *part = (float *)smem;        // [bn][128]: the rings are idle
#pragma unroll
                for (int q = 0; q < 4; q++)
                    if ((4 * q + set) * 16 < bn)
#pragma unroll
                        for (int j = 0; j < 16; j++) part[((4 * q + set) * 16 + j) * TILE_ROWS + r] = have ? __uint_as_float(v[q][j]) : 0.f;
                return;
            }
            const int n = t.n0 + r;
            if (!have || n >= a.g.N) return;
#pragma unroll
            for (int q = 0; q < 4; q++)
                if ((4 * q + set) * 16 < bn) tile_store(a.g, t.m0 + (4 * q + set) * 16, t.m_end, n, v[q]);
        };
        // A tight loop over this set's stages up to `limit`, what happens between tiles outside of it: the epilogue of the tile `before` comes
        // behind the first stages of the next one.
        int T = first, before = -1, st = set;
        bool more = T < n_tiles;
        int g_end = more ? nkb : 0, limit = g_end;
        while (more || before >= 0) {
            for (; st < limit && ok; st += TILE_SLOTS) unpack(st);
            if (before >= 0) { epilogue(before); i++; before = -1; }
            if (!more) break;
            if (limit < g_end && ok) { limit = g_end; continue; }
            before = T; T += stride;
            more = T < n_tiles && ok;
            if (more) { limit = g_end + min(nkb, TILE_AHEAD); g_end += nkb; }
        }
        tc_fence_before();
    }
    if (!PAIR && S > 1) {
        // the columns rank, rank + S, .. of the tile: partial sums of all CTAs of the cluster, in rank order
        cluster_sync_all();
        if (warp >= 3) {
            const MxTile t = mx_tile<PAIR>(a, cum, first, rank);
            cluster_columns(a.g, smem0, t.m0, min(bn, t.m_end - t.m0), t.n0, S, threadIdx.x - 96, 512);
        }
        cluster_sync_all();                         // nobody leaves while others read its shared memory
    }
    tc_fence_before();
    __syncthreads();
    // neither CTA of a pair leaves, or frees tensor memory, while the other's copies complete on its barriers or the MMAs read its memory
    if (PAIR) cluster_sync_all();
    if (warp == 1) { tc_fence_after(); if (PAIR) tc_free_pair(tmem, 512); else tc_free(tmem, 512); }
}

template <bool PAIR>
static int tile_setup() {
    static FgPerDevice configured;
    return fg_allow_shared(configured, mxfp4_tile_kernel<PAIR>, TILE_SMEM);
}

template <bool PAIR>
static int launch_tiles(const MxGemm &g, int bn, int S, cudaStream_t stream) {
    MxTiles a;
    a.g = g; a.bn = bn; a.test_skip_copy = g_mx_test_skip_copy;
    const int x_bytes = (PAIR ? bn / 2 : bn) * 256, room = (TILE_SMEM - 1024 - TILE_W_STAGES * TILE_W_STAGE) / x_bytes;
    a.xs = room < TILE_SLOTS ? room : TILE_SLOTS;
    const int tiles_k = mx_tiles(g.K), rows = PAIR ? 2 * TILE_ROWS : TILE_ROWS;
    a.tiles_n = (g.N + rows - 1) / rows; a.tiles_m = (g.M + bn - 1) / bn;
    a.kb_per_split = (tiles_k + S - 1) / S;
    S = (tiles_k + a.kb_per_split - 1) / a.kb_per_split;             // no CTA without a share
    const long long tiles = (long long)(g.offsets ? a.tiles_m + g.experts : a.tiles_m) * a.tiles_n;
    if (tiles > 0x3fffffff) return FG_ERR_BAD_SIZE;
    a.n_tiles = (int)tiles;
    CUtensorMap tmX, tmW;
    int rc = mx_make_map(&tmX, g.x, true, g.M, (long long)g.K * 2, g.ldx * 2, PAIR ? bn / 2 : bn, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    rc = mx_make_map(&tmW, g.w, false, (long long)(g.offsets ? g.experts : 1) * g.N, g.K / 2, g.K / 2, TILE_ROWS, TILE_K / 2, CU_TENSOR_MAP_SWIZZLE_64B);
    if (rc) return rc;
    // All of an SM's shared memory, needed or not: a CTA that allocates tensor memory shares its SM with no other that does (of a kernel on
    // another stream, say), whose cluster might wait for one of this kernel's while it waits for tensor memory.
    rc = tile_setup<PAIR>();
    if (rc) return rc;
    const int units = PAIR ? mx_sm_count() / 2 : mx_sm_count();
    const unsigned gx = S > 1 || tiles < units ? (unsigned)tiles : (unsigned)units;
    return mx_launch(mxfp4_tile_kernel<PAIR>, dim3(PAIR ? 2 * gx : gx, 1, S), TILE_THREADS, TILE_SMEM, dim3(PAIR ? 2 : 1, 1, S), stream, tmX, tmW, a);
}
// whether TMA can bring the rows of x
static bool tile_ok(const MxGemm &g) { return g.x_vec && g.ldx >= g.K; }

// The form, the tile's width and the split of K that finish first, in SM cycles.  A stage takes the longer of its unpacking and its MMAs, as
// measured at both ends (pairs: 820 cycles at 128 tokens, 1,350 at 256; single CTAs, bound by the bytes an SM receives: 950 and 1,690).  Half of a
// step counts whole rounds of tiles over the SMs, half the tiles alone: at the power limit the clock rises while SMs are idle (2,048 x 14,336 x 4,096 in
// seven rounds of 256 tokens takes 161 to 180 us, in the ten of 160 tokens, 7 % fewer by rounds, 192).
static int tile_plan(int M, int N, int K, bool &pair, int &bn, int &S) {
    static MxClusters known;
    const int tiles_k = mx_tiles(K), n_sm = mx_sm_count();
    int fit[9];
    int rc = tile_setup<false>();
    for (int s = 1; s <= 8 && !rc; s++) rc = mx_clusters(known, mxfp4_tile_kernel<false>, TILE_THREADS, TILE_SMEM, s, fit[s]);
    if (rc) return rc;
    double best = 1e30;
    for (int p = 0; p < 2; p++) {
        const int rows = p ? 2 * TILE_ROWS : TILE_ROWS, tiles_n = (N + rows - 1) / rows, units = p ? n_sm / 2 : n_sm;
        const int step = p ? 32 : 16;                                // (a CTA of a pair brings whole groups of 16 tokens)
        for (int b = step; b <= 256; b += step) {
            if (b > step && b - step >= M) break;                    // wider than the rows there are
            const long long tiles = (long long)((M + b - 1) / b) * tiles_n;
            for (int s = 1; s <= (p ? 1 : 8); s++) {
                if (s > 1 && tiles > fit[s]) continue;
                const int kb = (tiles_k + s - 1) / s;
                const double mma = p ? 300 + 4.1 * b : 210 + 5.8 * b, stage = mma > TILE_UNPACK ? mma : TILE_UNPACK;
                const double tile = kb * stage + 2500 + 4.0 * b + (s > 1 ? 2500 + 8.0 * b : 0);
                const long long rounds = (tiles * s + units - 1) / units;
                const double even = (double)(tiles * s) / units;
                const double cost = (rounds > 1 ? 0.5 * (rounds + even) : 1.0) * tile;
                if (cost < best) { best = cost; pair = p; bn = b; S = s; }
            }
        }
    }
    return 0;
}

static int mx_check(const MxGemm &a) {
    if (a.out_dtype != FG_F32 && a.out_dtype != FG_BF16) return FG_ERR_BAD_DTYPE;
    if (a.accumulate && a.out_dtype != FG_F32) return FG_ERR_BAD_DTYPE;
    if (a.M < 0 || a.N <= 0 || a.K <= 0 || a.K % MX_BLOCK || a.ldx < 0 || a.ldo < 0 || ((uintptr_t)a.w & 15) || ((uintptr_t)a.sc & 15)) return FG_ERR_BAD_SIZE;
    if (a.M > MX_MOST || a.K > MX_MOST || (long long)a.N * (a.offsets ? a.experts : 1) > MX_MOST) return FG_ERR_BAD_SIZE;
    return 0;
}

// form: 0 by the rule; 1 the kernel for few rows, 2 tiles, 3 tiles of pairs of CTAs, with `bn` tokens a tile (a multiple of 16, of pairs 32) and K split
// over `splits` CTAs (form 2): for tests and measurements
extern "C" int fg_gemm_mxfp4_ext(const void *x, long long ldx, const void *w, const void *scales, void *out, int out_dtype, long long ldo, int accumulate,
                                 int M, int N, int K, int form, int bn, int splits, cudaStream_t stream) {
    MxGemm a = {(const bf16 *)x, (const uint8_t *)w, (const uint8_t *)scales, out, ldx, ldo, M, N, K, out_dtype, accumulate, 0, nullptr, 0, 0};
    const int bad = mx_check(a);
    if (bad) return bad;
    if (M == 0) return 0;
    a.x_vec = ((uintptr_t)x & 15) == 0 && ldx % 8 == 0;
    if (form == 0) {
        bool pair = false;
        form = M > 8 && tile_ok(a) ? 2 : 1;
        if (form == 2) {
            const int rc = tile_plan(M, N, K, pair, bn, splits);
            if (rc) return rc;
        }
        if (pair) form = 3;
    } else if (form < 1 || form > 3 || (form > 1 && (!tile_ok(a) || bn < 16 || bn > 256 || bn % 16 || splits < 1 || splits > 8 || (form == 3 && (splits > 1 || bn % 32)))))
        return FG_ERR_BAD_SIZE;
    if (form == 2) return launch_tiles<false>(a, bn, splits, stream);
    if (form == 3) return launch_tiles<true>(a, bn, 1, stream);
    if (M <= 8) return launch_stream<1>(a, 1, 1, stream);
    // (as many tiles of 16 rows a launch as a grid's second dimension takes)
    for (long long m0 = 0; m0 < M; m0 += 65535 * 16) {
        MxGemm part = a;
        part.x += m0 * ldx;
        part.out = (char *)out + m0 * ldo * (out_dtype == FG_F32 ? 4 : 2);
        part.M = M - m0 < 65535 * 16 ? (int)(M - m0) : 65535 * 16;
        const int tiles = (part.M + 15) / 16, rc = launch_stream<2>(part, tiles, tiles, stream);
        if (rc) return rc;
    }
    return 0;
}
extern "C" int fg_gemm_mxfp4(const void *x, long long ldx, const void *w, const void *scales, void *out, int out_dtype, long long ldo, int accumulate,
                             int M, int N, int K, cudaStream_t stream) {
    return fg_gemm_mxfp4_ext(x, ldx, w, scales, out, out_dtype, ldo, accumulate, M, N, K, 0, 0, 0, stream);
}

// offsets: [experts + 1] on the device; w, scales: the experts' matrices one after another
extern "C" int fg_gemm_mxfp4_grouped(const void *x, long long ldx, const void *w, const void *scales, const int *offsets, int experts, void *out,
                                     int out_dtype, long long ldo, int accumulate, int M, int N, int K, cudaStream_t stream) {
    MxGemm a = {(const bf16 *)x, (const uint8_t *)w, (const uint8_t *)scales, out, ldx, ldo, M, N, K, out_dtype, accumulate, 0, offsets, experts, 0};
    if (experts <= 0 || experts > 65535 || !offsets) return FG_ERR_BAD_SIZE;
    const int bad = mx_check(a);
    if (bad) return bad;
    if (M == 0) return 0;
    a.x_vec = ((uintptr_t)x & 15) == 0 && ldx % 8 == 0;
    if (experts <= TILE_MAX_EXPERTS && tile_ok(a)) {
        // The runs' lengths are known on the device alone: a tile's width by their mean, with room for a router that prefers some experts (32 experts
        // of 2,048 x 2,048, us at 16 | 32 | 64 | 128 tokens a tile: mean 2: 15.6 | 16.4 | 17.0 | 18.4; mean 4: 27.9 | 22.6 | 23.3 | 25.2;
        // mean 16: 40.7 | 29.0 | 29.7 | 32.7; mean 32: 60.3 | 41.4 | 35.9 | 33.0; eight experts, mean 37: 22.1 | 16.5 | 10.8 | 11.9)
        const long long mean = ((long long)M + experts - 1) / experts;
        if (mean <= 2) return launch_tiles<false>(a, 16, 1, stream);
        return launch_tiles<true>(a, mean <= 8 ? 32 : mean <= 20 ? 64 : 128, 1, stream);
    }
    return (long long)M <= 4ll * experts ? launch_stream<1>(a, experts, M < experts ? M : experts, stream) : launch_stream<2>(a, experts, M < experts ? M : experts, stream);
}

#include "gemm_mxfp4_both.cuh"

// 0, or (code << 8 | role) of the first bounded wait that ran out since it was asked last
extern "C" int fg_gemm_mxfp4_error(void) {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_mx_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_mx_error, &zero, sizeof(int));
    return v;
}
// tests only: how long a wait may last, in SM cycles (0: the ordinary limit), and whether a kernel's first copy of tokens is left out
extern "C" int fg_gemm_mxfp4_test_hook(long long wait_limit_cycles, int skip_copy) {
    const long long limit = wait_limit_cycles > 0 ? wait_limit_cycles : MX_WAIT_LIMIT_CYCLES;
    g_mx_test_skip_copy = skip_copy;
    return (int)cudaMemcpyToSymbol(g_mx_wait_limit, &limit, sizeof(limit));
}
