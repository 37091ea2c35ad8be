// Microscaled 4-bit floating point (MXFP4) on the device: the format, and the step from eight packed numbers to bfloat16.
//
// A number is a sign, two exponent bits and one mantissa bit (0, 1/2, 1, 3/2, 2, 3, 4, 6); 32 neighbours along a row share
// a power of two 2^(e - 127), e a byte (255: the block is no number).  `data` [rows, K / 2] bytes, number 2 i of a row in the
// low half of byte i; `scales` [ceil(rows / 128), ceil(K / 128), 32, 4, 4] bytes: block b of row r at
// [r / 128, b / 4, r % 32, r / 32 % 4, b % 4] - tiles of 512 bytes in the order in which a block-scaled tensor instruction
// wants the exponents of 128 rows x 128 numbers, and in which a warp that takes eight rows of each quarter of a tile finds
// its exponents in 128 neighbouring bytes.  K is a multiple of 32; exponents of rows and blocks past the matrix are padding.
#pragma once
#include "common.cuh"

#define MX_BLOCK 32
#define MX_TILE_BYTES 512      // exponents of 128 rows x 128 numbers

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
// bytes of a and b by four selectors of four bits; bit 3 of one asks for eight copies of its byte's top bit
template <uint32_t SEL>
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "n"(SEL));
    return d;
}
// Eight numbers (a 32-bit word) as bfloat16 times 2^-126, in order, two to a word.
// The three bits below a code's sign, put at the bottom of a bfloat16's exponent field and the top of its mantissa, are the
// number times 2^-126 (1/2 as a subnormal).  The even and the odd codes are masked to a byte each; a byte permutation puts the two of a
// word into its halves, with zeros beside them (the sign of a byte below 128, replicated); one multiplication by 2^12 + 2^6 moves sign and
// value of both into place: the copies (bits 12..15 and 6..9 of each half) do not overlap, so nothing carries.
__device__ __forceinline__ void mx_unpack8(uint32_t w, uint32_t (&r)[4]) {
    const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
    r[0] = (prmt<0xc480u>(even, odd) * 0x1040u) & 0x81c081c0u;
    r[1] = (prmt<0xd591u>(even, odd) * 0x1040u) & 0x81c081c0u;
    r[2] = (prmt<0xe6a2u>(even, odd) * 0x1040u) & 0x81c081c0u;
    r[3] = (prmt<0xf7b3u>(even, odd) * 0x1040u) & 0x81c081c0u;
}
// The factor for those numbers: 2^126 2^(e - 127) as a pair of bfloat16, which is a finite power up to e = 128 (a scale of 2; weights' are
// far below 1).  For larger e it stays at e = 128 and mx_factor_rest is the rest, a second exact step (255: no number).
__device__ __forceinline__ bool mx_small(uint32_t e) { return e <= 128; }
__device__ __forceinline__ uint32_t mx_factor(uint32_t e) { return ((min(e, 128u) + 126) << 7) * 0x00010001u; }
__device__ __forceinline__ uint32_t mx_factor_rest(uint32_t e) {
    return (e == 255 ? 0x7fffu : e <= 128 ? 0x3f80u : (e - 1) << 7) * 0x00010001u;
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
        const uint32_t rest = mx_factor_rest(e);
#pragma unroll
        for (int j = 0; j < 16; j++) out[j] = mul_bf16x2(out[j], rest);
    }
}
