// Microscaled 4-bit matrices (the OCP MXFP4 format) and their kernels.
//
// A row of K values is cut into blocks of 32 columns (the last one padded with zeros). Block b of a row
// holds one scale 2^(s - 127), s an unsigned byte, and 32 codes of the 4-bit type e2m1 (sign, two exponent
// bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives); a value is code x scale, and
// s = 255 makes its block NaN. Quantising takes s = floor(log2 max|x|) - 2 + 127 (at least 0) and rounds
// x / scale to the nearest code, ties to the even one, magnitudes above 6 to 6. Both steps are exact in
// fp32 (a power-of-two factor, one rounding), so the codes do not depend on the kernel that made them.
//
// Codes: row-major, two per byte (even column in the low half), 16 bytes per block, rows ldc bytes apart.
// Scales: tiles of 128 rows x 4 blocks (512 bytes, k tile fastest), in the order in which the tensor cores
// read them: byte (row % 32) 16 + (row % 128) / 32 4 + block % 4 of tile (row / 128, block / 4).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace vb::mx4 {

constexpr int kBlock = 32;
__host__ __device__ inline int64_t blocks(int64_t K) { return (K + kBlock - 1) / kBlock; }
__host__ __device__ inline int64_t row_bytes(int64_t K) { return 16 * blocks(K); }
__host__ __device__ inline int64_t k_tiles(int64_t K) { return (blocks(K) + 3) / 4; }
inline int64_t scale_bytes(int64_t rows, int64_t K) { return (rows + 127) / 128 * k_tiles(K) * 512; }
// offset of the scale of block `b` of `row`, ktiles tiles per 128 rows
__host__ __device__ inline int64_t scale_at(int64_t row, int64_t b, int64_t ktiles) {
    return ((row >> 7) * ktiles + (b >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (b & 3);
}

// x [rows, K] (ldx) -> codes (ldc bytes per row), scales (every byte of the tiles is written, 0 where no
// block is). codes 16-byte aligned, ldc a multiple of 16, at least row_bytes(K).
template <class T>
void quantize(const T* x, int64_t ldx, int64_t rows, int64_t K, uint8_t* codes, int64_t ldc, uint8_t* scales,
              cudaStream_t s);
// the values back: y [rows, K] (ldy), rounded to T
template <class T>
void dequantize(const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t rows, int64_t K, T* y, int64_t ldy,
                cudaStream_t s);

#ifdef __CUDACC__
// The scale byte of a block whose largest magnitude has the fp32 bits `top` (of |x|, so that the order of
// the bits is the order of the magnitudes, with Inf and NaN on top): its exponent field - 2.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
    if (top >= 0x7f800000u) return 255u;
    const int e = int(top >> 23) - 2;
    return e < 0 ? 0u : uint32_t(e);
}
// 1 / scale (s <= 252, or 255, whose codes are 0)
__device__ __forceinline__ float inv_scale(uint32_t s) { return s == 255u ? 0.0f : __uint_as_float((254u - s) << 23); }
__device__ __forceinline__ float scale_value(uint32_t s) {
    return __uint_as_float(s == 255u ? 0x7fffffffu : s == 0u ? 0x00400000u : s << 23);
}
// Eight codes (column i in bits 4i .. 4i + 3) of v[i] * inv; 0 for a NaN block.
__device__ __forceinline__ uint32_t encode8(const float* v, float inv) {
    uint32_t d;
    float2 s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = __fmul2_rn(make_float2(v[2 * i], v[2 * i + 1]), make_float2(inv, inv));
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(d)
        : "f"(s[0].x), "f"(s[0].y), "f"(s[1].x), "f"(s[1].y), "f"(s[2].x), "f"(s[2].y), "f"(s[3].x), "f"(s[3].y));
    return inv == 0.0f ? 0u : d;
}
// The eight e2m1 values of a word of codes.
__device__ __forceinline__ void decode8(uint32_t c, float* v) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(c));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
// Largest |v| of eight values, as fp32 bits.
__device__ __forceinline__ uint32_t top8(const float* v) {
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) t = max(t, __float_as_uint(v[i]) & 0x7fffffffu);
    return t;
}
#endif

}  // namespace vb::mx4
