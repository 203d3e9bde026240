// Quantising to microscaled 4-bit blocks and reading the values back (see mx4.cuh). Both are bound by
// memory: fp16 quantising reads 2 B and writes 17/32 B per element.
#include <string>

#include "common.h"
#include "dev.cuh"
#include "mx4.cuh"

namespace vb::mx4 {

using namespace vb::d;

namespace {

constexpr int kThreads = 256;
constexpr int kPass = kThreads / 16;  // rows a CTA takes at a time: 16 threads of 8 columns make 128 columns

// Eight consecutive values from column k of a row of K, zeros past its end.
template <class T, bool VEC> __device__ __forceinline__ void load8(const T* row, int64_t k, int64_t K, float* v) {
    if (VEC && k + 8 <= K) {
        Vec<T, 8>::ldg(row + k, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_f<T>(row[k + i]) : 0.0f;
    }
}

// One CTA per scale tile (128 rows x 128 columns): a thread takes 8 columns of 8 rows, 16 rows apart, the
// four threads of a block share its maximum by shuffles, and the tile's 512 scale bytes are written at
// once from shared memory (row by row they would be 4-byte pieces 16 bytes apart).
template <class T, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int64_t K,
                                                            int64_t ktiles, uint8_t* __restrict__ codes, int64_t ldc,
                                                            uint8_t* __restrict__ scales) {
    __shared__ uint32_t tile[128];
    const int64_t rt = blockIdx.x / ktiles, kt = blockIdx.x - rt * ktiles;
    const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int64_t k = kt * 128 + c * 8;
    float v[8][8];
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int64_t r = rt * 128 + p * kPass + r0;
        if (r < rows && k < K) {
            load8<T, VEC>(x + r * ldx, k, K, v[p]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] = 0.0f;
        }
    }
    const bool block = k < (K + kBlock - 1) / kBlock * kBlock;  // (the last block's padding has codes 0)
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int rr = p * kPass + r0;
        const int64_t r = rt * 128 + rr;
        uint32_t top = top8(v[p]);
        top = max(top, __shfl_xor_sync(kFull, top, 1));
        top = max(top, __shfl_xor_sync(kFull, top, 2));
        const uint32_t s = scale_byte(top);
        if (r < rows && block) *reinterpret_cast<uint32_t*>(codes + r * ldc + k / 2) = encode8(v[p], inv_scale(s));
        // the row's four scale bytes, one from each four lanes
        uint32_t w = s << (8 * ((c >> 2) & 3));
        w |= __shfl_xor_sync(kFull, w, 4);
        w |= __shfl_xor_sync(kFull, w, 8);
        if (c == 0) tile[(rr & 31) * 4 + (rr >> 5)] = w;
    }
    __syncthreads();
    if (threadIdx.x < 128) reinterpret_cast<uint32_t*>(scales)[int64_t(blockIdx.x) * 128 + threadIdx.x] = tile[threadIdx.x];
}

// A thread takes 8 columns of up to 4 rows, `stride` rows apart.
template <class T, bool VEC>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* __restrict__ codes, int64_t ldc,
                                                              const uint8_t* __restrict__ scales, int64_t rows, int64_t K,
                                                              int64_t ktiles, T* __restrict__ y, int64_t ldy, int64_t n8,
                                                              int64_t stride) {
    const int64_t t = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    const int64_t r0 = t / n8, k = (t - r0 * n8) * 8;
    if (r0 >= stride) return;
    uint32_t c[4], s[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int64_t r = r0 + p * stride;
        if (r < rows) {
            c[p] = __ldg(reinterpret_cast<const uint32_t*>(codes + r * ldc + k / 2));
            s[p] = __ldg(scales + scale_at(r, k / kBlock, ktiles));
        }
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int64_t r = r0 + p * stride;
        if (r >= rows) continue;
        float v[8];
        decode8(c[p], v);
        const float f = scale_value(s[p]);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * f;
        T* o = y + r * ldy + k;
        if (VEC && k + 8 <= K) {
            Vec<T, 8>::store(o, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < K) o[i] = from_f<T>(v[i]);
        }
    }
}

template <class T> bool aligned16(const T* p, int64_t ld) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * int64_t(sizeof(T)) % 16 == 0;
}

unsigned grid_of(int64_t n, const char* what) {
    if (n > INT32_MAX) fail(kUnsupported, std::string(what) + ": matrix too large for one launch");
    return unsigned(n);
}

}  // namespace

template <class T>
void quantize(const T* x, int64_t ldx, int64_t rows, int64_t K, uint8_t* codes, int64_t ldc, uint8_t* scales,
              cudaStream_t s) {
    if (rows <= 0) return;
    const int64_t kt = k_tiles(K);
    const unsigned grid = grid_of((rows + 127) / 128 * kt, "mx4_quantize");
    if (aligned16(x, ldx)) quantize_kernel<T, true><<<grid, kThreads, 0, s>>>(x, ldx, rows, K, kt, codes, ldc, scales);
    else quantize_kernel<T, false><<<grid, kThreads, 0, s>>>(x, ldx, rows, K, kt, codes, ldc, scales);
    VB_LAUNCH();
}

template <class T>
void dequantize(const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t rows, int64_t K, T* y, int64_t ldy,
                cudaStream_t s) {
    if (rows <= 0) return;
    const int64_t n8 = (K + 7) / 8, stride = (rows + 3) / 4, kt = k_tiles(K);
    const unsigned grid = grid_of((stride * n8 + kThreads - 1) / kThreads, "mx4_dequantize");
    if (aligned16(y, ldy))
        dequantize_kernel<T, true><<<grid, kThreads, 0, s>>>(codes, ldc, scales, rows, K, kt, y, ldy, n8, stride);
    else
        dequantize_kernel<T, false><<<grid, kThreads, 0, s>>>(codes, ldc, scales, rows, K, kt, y, ldy, n8, stride);
    VB_LAUNCH();
}

template void quantize<float>(const float*, int64_t, int64_t, int64_t, uint8_t*, int64_t, uint8_t*, cudaStream_t);
template void quantize<__half>(const __half*, int64_t, int64_t, int64_t, uint8_t*, int64_t, uint8_t*, cudaStream_t);
template void dequantize<float>(const uint8_t*, int64_t, const uint8_t*, int64_t, int64_t, float*, int64_t, cudaStream_t);
template void dequantize<__half>(const uint8_t*, int64_t, const uint8_t*, int64_t, int64_t, __half*, int64_t,
                                 cudaStream_t);

}  // namespace vb::mx4
