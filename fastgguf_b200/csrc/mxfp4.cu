// Rows to microscaled 4-bit floating point and back (format: mxfp4.cuh).  Both kernels move bytes and compute next to nothing.
#include "mxfp4.cuh"

// ---------------------------------------------------------------------------- quantise
// A block's exponent is that of its largest number minus 2 (the largest code, 6 = 1.5 * 2^2, then covers it or saturates):
// e = max(E - 2, 0) with E the exponent field of the float32 maximum.  x 2^(127 - e) is exact, and one conversion rounds it to the nearest
// code, ties to the even one, beyond 6 to 6.  An infinity or no number anywhere in a block: e = 255, codes 0.
//
// A CTA takes 128 rows x 128 numbers: 16 threads a row with eight numbers each (loads of 16 bytes of bfloat16, two of 16 of float32), four
// threads a block, whose maximum takes two shuffles.  The exponents of the tile are 512 neighbouring bytes, gathered in shared memory.
template <typename T>
__device__ __forceinline__ void load8(const T *p, bool vec, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float *p, bool vec, float (&v)[8]) {
    if (vec) {
        const float4 a = __ldcs((const float4 *)p), b = __ldcs((const float4 *)p + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = p[j];
    }
}
template <>
__device__ __forceinline__ void load8<bf16>(const bf16 *p, bool vec, float (&v)[8]) {
    if (vec) {
        const uint4 a = __ldcs((const uint4 *)p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; j++) { v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = __bfloat162float(p[j]);
    }
}
// two numbers to a byte, the first in its low half
__device__ __forceinline__ uint32_t to_e2m1x2(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

#define QUANT_ROWS 16      // rows a pass of the CTA's 256 threads takes
template <typename T>
__global__ void __launch_bounds__(256)
mxfp4_quantize_kernel(const T *__restrict__ x, long long ldx, long long x_stride, uint8_t *__restrict__ data, uint8_t *__restrict__ scales, int R,
                      int K, int tiles_r, int vec) {
    __shared__ __align__(16) uint8_t tile[MX_TILE_BYTES];
    const int tk = blockIdx.x, tr = blockIdx.y % tiles_r, mat = blockIdx.y / tiles_r, tiles_k = gridDim.x;
    const int c = threadIdx.x & 15, k = tk * 128 + c * 8, rows = min(128, R - tr * 128);
    if (threadIdx.x < 32) ((uint4 *)tile)[threadIdx.x] = make_uint4(0, 0, 0, 0);
    pdl_wait();
    pdl_launch_dependents();
    __syncthreads();
    const T *src = x + (size_t)mat * x_stride + k;
    uint8_t *dst = data + (size_t)mat * R * (K / 2) + k / 2;
    // (whole warps leave the loop together unless the tile's rows end inside a warp's two: the shuffles name all lanes, so all walk it)
#pragma unroll 4
    for (int r0 = 0; r0 < rows; r0 += QUANT_ROWS) {
        const int rl = r0 + (threadIdx.x >> 4);
        const bool live = rl < rows && k < K;
        const size_t r = (size_t)tr * 128 + rl;
        float v[8];
        if (live) load8<T>(src + r * ldx, vec, v);
        else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = 0.f;
        }
        uint32_t top = 0;                                  // the largest magnitude's bits: order as integers, NaN above infinity
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t E = top >> 23;
        const uint32_t e = E == 255 ? 255 : E > 2 ? E - 2 : 0;
        const float up = __uint_as_float((254 - min(e, 253u)) << 23);      // 2^(127 - e)
        uint32_t w = 0;
        if (E != 255) {
#pragma unroll
            for (int j = 0; j < 4; j++) w |= to_e2m1x2(v[2 * j] * up, v[2 * j + 1] * up) << (8 * j);
        }
        if (live) {
            *(uint32_t *)(dst + r * (K / 2)) = w;
            if ((c & 3) == 0) tile[(rl & 31) * 16 + (rl >> 5) * 4 + (c >> 2)] = (uint8_t)e;
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
    if (mats < 0 || R < 0 || K <= 0 || K % MX_BLOCK || ldx < 0 || ((uintptr_t)data & 15) || ((uintptr_t)scales & 15)) return FG_ERR_BAD_SIZE;
    if (mats == 0 || R == 0) return 0;
    const int tiles_r = mx_tiles(R);
    if ((long long)tiles_r * mats > 65535) return FG_ERR_BAD_SIZE;
    const int size = dtype == FG_F32 ? 4 : 2;
    const int vec = ((uintptr_t)x & 15) == 0 && (ldx * size) % 16 == 0 && (x_stride * size) % 16 == 0;
    dim3 grid(mx_tiles(K), tiles_r * mats);
    if (dtype == FG_F32)
        return mx_launch(mxfp4_quantize_kernel<float>, grid, 256, 0, dim3(1, 1, 1), stream, (const float *)x, ldx, x_stride, (uint8_t *)data, (uint8_t *)scales, R, K, tiles_r, vec);
    return mx_launch(mxfp4_quantize_kernel<bf16>, grid, 256, 0, dim3(1, 1, 1), stream, (const bf16 *)x, ldx, x_stride, (uint8_t *)data, (uint8_t *)scales, R, K, tiles_r, vec);
}

// ---------------------------------------------------------------------------- rows
// out[i] = scale * row rows[i] (null: row i), a thread sixteen bytes of output: four float32 or eight bfloat16 numbers, which lie in one block.
// The number itself is exact in either type; a scale other than 1 rounds once.  A row index outside the matrix gives a row of NaN.
template <typename T>
__global__ void __launch_bounds__(256)
mxfp4_rows_kernel(const uint8_t *__restrict__ data, const uint8_t *__restrict__ scales, const int *__restrict__ rows, T *__restrict__ out,
                  long long ldo, long long total, int R, int K, float scale, int vec) {
    constexpr int V = 16 / sizeof(T);
    const int per_row = K / V, tiles_k = mx_tiles(K);
    pdl_wait();
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < total; at += (long long)gridDim.x * 256) {
        const long long i = at / per_row;
        const int c = (int)(at - i * per_row) * V;
        const int r = rows ? rows[i] : (int)i;
        const bool ok = r >= 0 && r < R;
        uint32_t w = 0, e = 255;
        if (ok) {
            const uint8_t *src = data + (size_t)r * (K / 2) + c / 2;
            w = V == 8 ? *(const uint32_t *)src : (uint32_t) * (const uint16_t *)src;
            e = scales[mx_scale_at(r, c / MX_BLOCK, tiles_k)];
        }
        const float p = mx_power(e);
        float v[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const uint32_t code = (w >> (4 * j)) & 15;
            // the code's value bits as a float32's lowest exponent and highest mantissa bits are the number times 2^-126
            v[j] = scale * (__uint_as_float((code >> 3 << 31) | ((code & 7) << 22)) * __uint_as_float(253u << 23) * p);
        }
        T *dst = out + (size_t)i * ldo + c;
        if (vec) {
            uint4 o;
            if constexpr (V == 4) o = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            else {
                uint32_t q[4];
#pragma unroll
                for (int j = 0; j < 4; j++) { __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]); q[j] = *(uint32_t *)&t; }
                o = make_uint4(q[0], q[1], q[2], q[3]);
            }
            *(uint4 *)dst = o;
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) dst[j] = from_f32<T>(v[j]);
        }
    }
}

// data, scales: one matrix [R, K]; out [n, K] of out_dtype, rows ldo numbers apart
extern "C" int fg_mxfp4_rows(const void *data, const void *scales, const int *rows, void *out, int out_dtype, long long ldo, int n, int R, int K,
                             float scale, cudaStream_t stream) {
    if (out_dtype != FG_F32 && out_dtype != FG_BF16) return FG_ERR_BAD_DTYPE;
    if (n < 0 || R < 0 || K <= 0 || K % MX_BLOCK || ldo < K || (!rows && n > R) || ((uintptr_t)data & 3)) return FG_ERR_BAD_SIZE;
    if (n == 0) return 0;
    const int V = out_dtype == FG_F32 ? 4 : 8;
    const int vec = ((uintptr_t)out & 15) == 0 && ldo % V == 0;
    const long long total = (long long)n * (K / V), want = (total + 255) / 256;
    dim3 grid((unsigned)(want < 148 * 64 ? want : 148 * 64));
    if (out_dtype == FG_F32)
        return mx_launch(mxfp4_rows_kernel<float>, grid, 256, 0, dim3(1, 1, 1), stream, (const uint8_t *)data, (const uint8_t *)scales, rows, (float *)out, ldo, total, R, K, scale, vec);
    return mx_launch(mxfp4_rows_kernel<bf16>, grid, 256, 0, dim3(1, 1, 1), stream, (const uint8_t *)data, (const uint8_t *)scales, rows, (bf16 *)out, ldo, total, R, K, scale, vec);
}
