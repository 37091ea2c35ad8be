// Rows to microscaled 4-bit floating point and back (format: mxfp4.cuh).  Both kernels move bytes and compute next to nothing.
#include "mxfp4.cuh"

// ---------------------------------------------------------------------------- quantise
// A block's exponent is that of its largest number minus 2 (the largest code, 6 = 1.5 * 2^2, then covers it or saturates):
// e = max(E - 2, 0) with E the exponent field of the float32 maximum.  x 2^(127 - e) is exact, and one conversion rounds it to the nearest
// code, ties to the even one, beyond 6 to 6.  An infinity or no number anywhere in a block: e = 255, codes 0.
//
// A CTA takes 128 rows x 128 numbers.  A thread reads 32 bytes of a row at a time, 8 float32 or 16 bfloat16 numbers; the four or two threads of
// a block find its maximum by shuffles.  The exponents of the tile are 512 neighbouring bytes, gathered in shared memory.
// 14,336 x 4,096: 47.1 us from float32 (5.6 TB/s), 31.0 from bfloat16 (4.8).
__device__ __forceinline__ void load_piece(const float *p, bool vec, float (&v)[8]) {
    if (vec)
        asm("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
            : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(p));
    else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = p[j];
    }
}
__device__ __forceinline__ void load_piece(const bf16 *p, bool vec, float (&v)[16]) {
    if (vec) {
        uint32_t w[8];
        asm("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
            : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
#pragma unroll
        for (int j = 0; j < 8; j++) { v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] = __bfloat162float(p[j]);
    }
}
// two numbers to a byte, the first in its low half
__device__ __forceinline__ uint32_t to_e2m1x2(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <typename T>
__global__ void __launch_bounds__(256)
mxfp4_quantize_kernel(const T *x, long long ldx, long long x_stride, uint8_t *__restrict__ data, uint8_t *__restrict__ scales, int R,
                      int K, int tiles_r, int vec) {
    constexpr int V = 32 / sizeof(T), THREADS = 128 / V, ROWS = 256 / THREADS;      // numbers a piece, threads a row, rows a pass of the CTA
    __shared__ __align__(16) uint8_t tile[MX_TILE_BYTES];
    const int tk = blockIdx.x, tr = blockIdx.y % tiles_r, mat = blockIdx.y / tiles_r, tiles_k = gridDim.x;
    const int c = threadIdx.x % THREADS, k = tk * 128 + c * V, rows = min(128, R - tr * 128);
    if (threadIdx.x < 32) ((uint4 *)tile)[threadIdx.x] = make_uint4(0, 0, 0, 0);
    pdl_wait();
    pdl_launch_dependents();
    __syncthreads();
    // (the loads are plain asm, so that passes overlap: an address that is known only here keeps them behind the wait)
    asm volatile("" : "+l"(x) : : "memory");
    const T *src = x + (size_t)mat * x_stride + k;
    uint8_t *dst = data + (size_t)mat * R * (K / 2) + k / 2;
    // (every thread walks all passes: the shuffles name all lanes)
#pragma unroll 4
    for (int r0 = 0; r0 < rows; r0 += ROWS) {
        const int rl = r0 + threadIdx.x / THREADS;
        const bool live = rl < rows && k < K;
        const size_t r = (size_t)tr * 128 + rl;
        float v[V];
        if (live) load_piece(src + r * ldx, vec, v);
        else {
#pragma unroll
            for (int j = 0; j < V; j++) v[j] = 0.f;
        }
        uint32_t top = 0;                                  // the largest magnitude's bits: order as integers, NaN above infinity
#pragma unroll
        for (int j = 0; j < V; j++) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < MX_BLOCK / V; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const uint32_t E = top >> 23;
        const uint32_t e = E == 255 ? 255 : E > 2 ? E - 2 : 0;
        const float up = __uint_as_float((254 - min(e, 253u)) << 23);      // 2^(127 - e)
        uint32_t w[V / 8];
#pragma unroll
        for (int i = 0; i < V / 8; i++) {
            w[i] = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) w[i] |= to_e2m1x2(v[8 * i + 2 * j] * up, v[8 * i + 2 * j + 1] * up) << (8 * j);
            if (E == 255) w[i] = 0;
        }
        if (live) {
            if constexpr (V == 16) *(uint2 *)(dst + r * (K / 2)) = make_uint2(w[0], w[1]);
            else *(uint32_t *)(dst + r * (K / 2)) = w[0];
            if (c % (MX_BLOCK / V) == 0) tile[(rl & 31) * 16 + (rl >> 5) * 4 + c / (MX_BLOCK / V)] = (uint8_t)e;
        }
    }
    __syncthreads();
    if (threadIdx.x < 32)
        ((uint4 *)(scales + (((size_t)mat * tiles_r + tr) * tiles_k + tk) * MX_TILE_BYTES))[threadIdx.x] = ((const uint4 *)tile)[threadIdx.x];
}

// x: `mats` matrices [R, K] (rows ldx apart, matrices x_stride apart, both in numbers) of dtype; data, scales: as the format, one matrix after another
extern "C" int fg_mxfp4_quantize(const void *x, int dtype, long long ldx, long long x_stride, void *data, void *scales, int mats, int R, int K,
                                 cudaStream_t stream) {
    if (dtype != FG_F32 && dtype != FG_BF16) return FG_ERR_BAD_DTYPE;
    if (mats < 0 || R < 0 || R > MX_MOST || K <= 0 || K > MX_MOST || K % MX_BLOCK || ldx < 0 || ((uintptr_t)data & 15) || ((uintptr_t)scales & 15)) return FG_ERR_BAD_SIZE;
    if (mats == 0 || R == 0) return 0;
    // A launch takes up to 65,535 tiles of 128 rows: whole matrices, or a share of one matrix's rows.
    const int most = 65535, rows = R < most * 128 ? R : most * 128, together = rows < R ? 1 : most / mx_tiles(R);
    const int V = dtype == FG_F32 ? 8 : 16;
    const int vec = (uintptr_t)x % 32 == 0 && ldx % V == 0 && x_stride % V == 0;
    for (long long m = 0; m < mats; m += together)
        for (long long r = 0; r < R; r += rows) {
            const int n = mats - m < together ? (int)(mats - m) : together, nr = R - r < rows ? (int)(R - r) : rows;
            const long long at = m * x_stride + r * ldx;
            uint8_t *d = (uint8_t *)data + ((size_t)m * R + r) * (K / 2), *s = (uint8_t *)scales + m * mx_scale_bytes(R, K) + mx_scale_bytes((int)r, K);
            const dim3 grid(mx_tiles(K), mx_tiles(nr) * n);
            const int rc = dtype == FG_F32
                ? mx_launch(mxfp4_quantize_kernel<float>, grid, 256, 0, dim3(1, 1, 1), stream, (const float *)x + at, ldx, x_stride, d, s, nr, K, mx_tiles(nr), vec)
                : mx_launch(mxfp4_quantize_kernel<bf16>, grid, 256, 0, dim3(1, 1, 1), stream, (const bf16 *)x + at, ldx, x_stride, d, s, nr, K, mx_tiles(nr), vec);
            if (rc) return rc;
        }
    return 0;
}

// ---------------------------------------------------------------------------- rows
// out[i] = scale * row rows[i] (null: row i).  A piece is eight numbers, which lie in one block: four bytes in, 16 or 32 out.  A thread takes four
// pieces, 256 apart, and asks for all of them before it converts the first.  The number itself is exact in either type; a scale other than 1 rounds
// once.  A row index outside the matrix gives a row of NaN.  14,336 x 4,096: 42.9 us to float32 (6.2 TB/s), 36.0 to bfloat16 (4.1: the schedulers
// issue in 82 % of cycles); 4,001 picked rows of 2,048 6.9 us to float32 (5.4), 6.3 to bfloat16.
#define ROWS_PIECES 4
__device__ __forceinline__ void store8(float *p, bool vec, const float (&v)[8]) {
    if (vec)
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
    else {
#pragma unroll
        for (int j = 0; j < 8; j++) p[j] = v[j];
    }
}
__device__ __forceinline__ void store8(bf16 *p, bool vec, const float (&v)[8]) {
    if (vec) {
        uint32_t q[4];
#pragma unroll
        for (int j = 0; j < 4; j++) { __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]); q[j] = *(uint32_t *)&t; }
        *(uint4 *)p = make_uint4(q[0], q[1], q[2], q[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) p[j] = __float2bfloat16_rn(v[j]);
    }
}
// pieces 0 .. total - 1 of the rows from r0 on; `over` is 2^64 / (pieces a row) rounded up, by which a piece's row is one multiplication
template <typename T>
__global__ void __launch_bounds__(256)
mxfp4_rows_kernel(const uint8_t *data, const uint8_t *scales, const int *rows, T *__restrict__ out,
                  long long ldo, int r0, unsigned total, unsigned long long over, int R, int K, float scale, int vec) {
    const int tiles_k = mx_tiles(K);
    const unsigned at0 = blockIdx.x * (256 * ROWS_PIECES) + threadIdx.x, per_row = K / 8;
    uint32_t w[ROWS_PIECES], e[ROWS_PIECES];
    long long to[ROWS_PIECES];
    pdl_wait();
    asm volatile("" : "+l"(data), "+l"(scales), "+l"(rows) : : "memory");       // (addresses known only here keep the loads behind the wait)
#pragma unroll
    for (int p = 0; p < ROWS_PIECES; p++) {
        const unsigned at = at0 + p * 256;
        w[p] = 0;
        e[p] = 255;
        if (at < total) {
            const unsigned i = (unsigned)__umul64hi(at, over);
            const int c = (int)(at - i * per_row) * 8, r = rows ? rows[r0 + i] : r0 + (int)i;
            to[p] = (long long)(r0 + (int)i) * ldo + c;
            if (r >= 0 && r < R) {
                w[p] = *(const uint32_t *)(data + (size_t)r * (K / 2) + c / 2);
                e[p] = scales[mx_scale_at(r, c / MX_BLOCK, tiles_k)];
            }
        }
    }
#pragma unroll
    for (int p = 0; p < ROWS_PIECES; p++) {
        if (at0 + p * 256 >= total) break;
        const float f = mx_power(e[p]);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t code = w[p] >> (4 * j);
            // the code's value bits as a float32's lowest exponent and highest mantissa bits are the number times 2^-126
            v[j] = scale * (__uint_as_float((code & 8) << 28 | (code & 7) << 22) * __uint_as_float(253u << 23) * f);
        }
        store8(out + to[p], vec, v);
    }
}

// data, scales: one matrix [R, K]; out [n, K] of out_dtype, rows ldo numbers apart
extern "C" int fg_mxfp4_rows(const void *data, const void *scales, const int *rows, void *out, int out_dtype, long long ldo, int n, int R, int K,
                             float scale, cudaStream_t stream) {
    if (out_dtype != FG_F32 && out_dtype != FG_BF16) return FG_ERR_BAD_DTYPE;
    if (n < 0 || R < 0 || K <= 0 || K > MX_MOST || K % MX_BLOCK || ldo < K || (!rows && n > R) || ((uintptr_t)data & 3)) return FG_ERR_BAD_SIZE;
    const unsigned per_row = K / 8;
    const int most = (int)(0x7fffffffu / per_row);                   // rows of a launch: pieces are counted in 31 bits
    const unsigned long long over = ~0ull / per_row + 1;
    const int vec = (uintptr_t)out % (out_dtype == FG_F32 ? 32 : 16) == 0 && ldo % 8 == 0;
    for (int r0 = 0; r0 < n; r0 += most) {
        const unsigned total = (unsigned)(n - r0 < most ? n - r0 : most) * per_row;
        const dim3 grid((total + 256 * ROWS_PIECES - 1) / (256 * ROWS_PIECES));
        const int rc = out_dtype == FG_F32
            ? mx_launch(mxfp4_rows_kernel<float>, grid, 256, 0, dim3(1, 1, 1), stream, (const uint8_t *)data, (const uint8_t *)scales, rows, (float *)out, ldo, r0, total, over, R, K, scale, vec)
            : mx_launch(mxfp4_rows_kernel<bf16>, grid, 256, 0, dim3(1, 1, 1), stream, (const uint8_t *)data, (const uint8_t *)scales, rows, (bf16 *)out, ldo, r0, total, over, R, K, scale, vec);
        if (rc) return rc;
        if (n - r0 <= most) break;                                   // (r0 + most may pass 31 bits)
    }
    return 0;
}
