// Microscaled 4-bit floating point (MXFP4) on the device: the format, and the step from eight packed numbers to bfloat16.
//
// A number is a sign, two exponent bits and one mantissa bit (0, 1/2, 1, 3/2, 2, 3, 4, 6); 32 neighbours along a row share
// a power of two 2^(e - 127), e a byte (255: the block is no number).  `data` [rows, K / 2] bytes, number 2 i of a row in the
// low half of byte i; `scales` [ceil(rows / 128), ceil(K / 128), 32, 4, 4] bytes: block b of row r at
// [r / 128, b / 4, r % 32, r / 32 % 4, b % 4] - tiles of 512 bytes in the order in which a block-scaled tensor instruction
// wants the exponents of 128 rows x 128 numbers, and in which a warp that takes eight rows of each quarter of a tile finds
// its exponents in 128 neighbouring bytes.  K is a multiple of 32; exponents of rows and blocks past the matrix are padding, any
// byte but 255.
#pragma once
#include "common.cuh"

#define MX_BLOCK 32
#define MX_TILE_BYTES 512      // exponents of 128 rows x 128 numbers
#define MX_MOST (0x7fffffff - 512)      // rows (of x, of all matrices of a stack) and numbers of a row are counted in 31 bits, up to the end of the last tile

__host__ __device__ __forceinline__ int mx_tiles(int n) { return (n + 127) / 128; }
__host__ __device__ __forceinline__ size_t mx_scale_bytes(int rows, int K) { return (size_t)mx_tiles(rows) * mx_tiles(K) * MX_TILE_BYTES; }
// where the exponent of block b of row r stands
__device__ __forceinline__ size_t mx_scale_at(int r, int b, int tiles_k) {
    return ((size_t)(r >> 7) * tiles_k + (b >> 2)) * MX_TILE_BYTES + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}
// 2^(e - 127) in float32
__device__ __forceinline__ float mx_power(uint32_t e) {
    return e == 255 ? __uint_as_float(0x7fffffffu) : e == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(e << 23);
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// Eight numbers (a 32-bit word) as bfloat16 times 2^-129, in order, two to a word.
// One instruction turns a byte into two half-precision numbers.  Those times 2^-20 are subnormal in half precision, exactly: 16 |q| <= 96
// units of 2^-24, a sign and an integer in the low seven bits - which are a bfloat16's mantissa, so the SAME bits are the subnormal bfloat16
// number 16 |q| 2^-133.  A word takes 15 cycles of a scheduler this way, factor included, of which bit operations on the codes take 19 to 23.
__device__ __forceinline__ void mx_unpack8(uint32_t w, uint32_t (&r)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(w));
#pragma unroll
    for (int j = 0; j < 4; j++) asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(r[j]) : "r"(0x00100010u));      // 2^-20
}
// The factor for those numbers: 2^129 2^(e - 127) as a pair of bfloat16, a finite power up to e = 125 (a scale of 1/4; weights' are far below).
// For larger e it stays there and the rest follows in two more exact steps (255: no number).
__device__ __forceinline__ bool mx_small(uint32_t e) { return e <= 125; }
__device__ __forceinline__ uint32_t mx_factor(uint32_t e) { return (min(e, 125u) + 129) * 0x00800080u; }
__device__ __forceinline__ uint32_t mx_times_rest(uint32_t r, uint32_t e) {
    const uint32_t over = max(e, 125u) - 125, half = over >> 1;
    r = mul_bf16x2(mul_bf16x2(r, (half + 127) * 0x00800080u), (over - half + 127) * 0x00800080u);
    return e == 255 ? 0x7fff7fffu : r;
}
// A block of 32 numbers with exponent e as bfloat16, in order.  Called by whole warps.
__device__ __forceinline__ void mx_unpack32(const uint4 &d, uint32_t e, uint32_t (&out)[16]) {
    const uint32_t w[4] = {d.x, d.y, d.z, d.w}, f = mx_factor(e);
#pragma unroll
    for (int u = 0; u < 4; u++) {
        uint32_t v[4];
        mx_unpack8(w[u], v);
#pragma unroll
        for (int j = 0; j < 4; j++) out[4 * u + j] = mul_bf16x2(v[j], f);
    }
    if (!__all_sync(0xffffffffu, mx_small(e))) {
#pragma unroll
        for (int j = 0; j < 16; j++) out[j] = mx_times_rest(out[j], e);
    }
}

// ---------------------------------------------------------------------------- launches
// Dependent launches: a kernel of this library waits for its predecessor before it touches any memory (weights too: the quantiser may just have
// written them).  Only the quantiser releases its successor before it ends, behind that wait, so that one never runs beside the kernel before its
// predecessor.  Readers and contractions do not: what they write may be the weights of a bfloat16 or float32 contraction (the keys of scores, a product of
// factors), which the next kernel of the stream, or the one behind that, fetches before its own wait.  Codes and exponents are read by this library alone.
template <typename... KArgs, typename... Args>
static inline int mx_launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, dim3 cluster, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (fg_pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster.x * cluster.y * cluster.z > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster.x; attr[n].val.clusterDim.y = cluster.y; attr[n++].val.clusterDim.z = cluster.z;
    }
    cfg.attrs = attr; cfg.numAttrs = n;
    return (int)cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}
