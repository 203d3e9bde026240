// Quantising to microscaled 4-bit blocks and reading the values back (see mx4.cuh). Both are bound by memory: at
// fp16, quantising reads 2 B and writes 17/32 B per element. A CTA takes 128 rows x 256 columns (two scale
// tiles), a warp 256 columns of one row at a time, 8 per lane, with four rows' loads in flight; matrices of at
// most 128 columns two rows of 128. [189809 x 1024] fp16: 91 and 85 us, 0.84 and 0.90 of the copy bandwidth.
#include <string>
#include <type_traits>

#include "common.h"
#include "dev.cuh"
#include "mx4.cuh"

namespace vb::mx4 {

using namespace vb::d;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kFlight = 4;  // vectors of a lane in flight, at most
// LPR lanes per row: 8 LPR columns per CTA; ROWS rows per CTA, kPass at a time. Scale tiles have 128 rows: CTAs of
// 32 rows (for matrices that give fewer than two CTAs of 128 rows to an SM) write a quarter of their tiles' words.
template <int LPR, int ROWS> struct Shape {
    static constexpr int kCols = 8 * LPR, kPass = kWarps * (32 / LPR), kRounds = ROWS / (kPass * kFlight) > 1 ? ROWS / (kPass * kFlight) : 1;
    static constexpr int kUnroll = ROWS / (kPass * kRounds);  // vectors of a lane in flight
};

// Eight consecutive values from column k of a row of K as stored, zeros past its end.
template <class T, bool VEC> struct Eight {
    T v[8];
    __device__ __forceinline__ void load(const T* row, int64_t k, int64_t K) {
        if (VEC && k + 8 <= K) {
#pragma unroll
            for (int i = 0; i < int(sizeof(T)) / 2; ++i)
                reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(row + k) + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = k + i < K ? row[k + i] : from_f<T>(0.0f);
        }
    }
};
// Largest magnitude, as the bits of its fp32 value (NaN and Inf on top). fp16: in pairs, then widened.
__device__ __forceinline__ uint32_t top_of(const float (&v)[8]) { return top8(v); }
__device__ __forceinline__ uint32_t top_of(const __half (&v)[8]) {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(v);
    // the 15 low bits order magnitudes: two 16-bit unsigned maxima per operation
    uint32_t m = __vmaxu2(__vmaxu2(u[0] & 0x7fff7fffu, u[1] & 0x7fff7fffu), __vmaxu2(u[2] & 0x7fff7fffu, u[3] & 0x7fff7fffu));
    m = max(m & 0xffffu, m >> 16);
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m))) & 0x7fffffffu;
}

template <class T, bool VEC, int LPR, int ROWS>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int64_t K,
                                                            int ktiles, int groups, uint8_t* __restrict__ codes, int64_t ldc,
                                                            uint8_t* __restrict__ scales) {
    // the scale bytes of the CTA's two tiles, written at once (row by row they would be 4-byte pieces 16 bytes apart)
    __shared__ uint32_t tile[2][ROWS];
    const int rp = int(blockIdx.x) / groups, cg = int(blockIdx.x) - rp * groups;  // part of ROWS rows, column group
    using S = Shape<LPR, ROWS>;
    constexpr int kIn = S::kUnroll;
    const int lane = threadIdx.x & (LPR - 1), sub = threadIdx.x / LPR;  // lane of the row, row of the pass
    const int64_t k = int64_t(cg) * S::kCols + lane * 8, r0 = int64_t(rp) * ROWS;
    const bool block = k < (K + kBlock - 1) / kBlock * kBlock;  // (the last block's padding has codes 0)
#pragma unroll 1
    for (int q = 0; q < S::kRounds; ++q) {
        if (r0 + q * kIn * S::kPass >= rows) {  // no rows left: their scale bytes are 0
            if ((lane & 15) == 0) {
#pragma unroll
                for (int p = 0; p < kIn; ++p) {
                    const int rr = (q * kIn + p) * S::kPass + sub;
                    tile[lane >> 4][ROWS == 128 ? (rr & 31) * 4 + (rr >> 5) : rr] = 0;
                }
            }
            continue;
        }
        Eight<T, VEC> e[kIn];
#pragma unroll
        for (int p = 0; p < kIn; ++p) {
            const int64_t r = r0 + (q * kIn + p) * S::kPass + sub;
            e[p].load(x + r * ldx, k, r < rows ? K : 0);
        }
#pragma unroll
        for (int p = 0; p < kIn; ++p) {
            const int rr = (q * kIn + p) * S::kPass + sub;
            uint32_t top = top_of(e[p].v);
            top = max(top, __shfl_xor_sync(kFull, top, 1));
            top = max(top, __shfl_xor_sync(kFull, top, 2));
            const uint32_t s = scale_byte(top);
            if (r0 + rr < rows && block) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = to_f<T>(e[p].v[i]);
                *reinterpret_cast<uint32_t*>(codes + (r0 + rr) * ldc + k / 2) = encode8(v, inv_scale(s));
            }
            if ((lane & 3) == 0)
                reinterpret_cast<uint8_t*>(tile[lane >> 4])[4 * (ROWS == 128 ? (rr & 31) * 4 + (rr >> 5) : rr) + ((lane >> 2) & 3)] = uint8_t(s);
        }
    }
    __syncthreads();
    constexpr int kTiles = S::kCols / 128;
    // word 4 (row % 32) + row / 32 of a tile
    const int t = threadIdx.x / ROWS, i = threadIdx.x % ROWS;
    if (t < kTiles && kTiles * cg + t < ktiles) {
        uint32_t* out = reinterpret_cast<uint32_t*>(scales) + ((r0 >> 7) * ktiles + kTiles * cg + t) * 128;
        if (ROWS == 128) out[i] = tile[t][i];
        else out[4 * i + ((r0 >> 5) & 3)] = tile[t][i];
    }
}

// Eight values to a 16-byte aligned address; fp32 in one 32-byte store where that is aligned.
__device__ __forceinline__ void store8(__half* p, const float* v) { Vec<__half, 8>::store(p, v); }
__device__ __forceinline__ void store8(float* p, const float* v) {
    if ((reinterpret_cast<uintptr_t>(p) & 31) == 0)
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                     "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                     : "memory");
    else Vec<float, 8>::store(p, v);
}

template <class T, bool VEC, int LPR, int ROWS>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* __restrict__ codes, int64_t ldc,
                                                              const uint8_t* __restrict__ scales, int64_t rows, int64_t K,
                                                              int ktiles, int groups, T* __restrict__ y, int64_t ldy) {
    const int rp = int(blockIdx.x) / groups, cg = int(blockIdx.x) - rp * groups;  // part of ROWS rows, column group
    using S = Shape<LPR, ROWS>;
    constexpr int kIn = S::kUnroll;
    const int lane = threadIdx.x & (LPR - 1), sub = threadIdx.x / LPR;  // lane of the row, row of the pass
    const int64_t k = int64_t(cg) * S::kCols + lane * 8, r0 = int64_t(rp) * ROWS;
    if (k >= K) return;
    const uint8_t* st = scales + ((r0 >> 7) * ktiles + (k >> 7)) * 512 + ((k >> 5) & 3);
#pragma unroll 1
    for (int q = 0; q < S::kRounds && r0 + q * kIn * S::kPass < rows; ++q) {
        uint32_t c[kIn], s[kIn];
#pragma unroll
        for (int p = 0; p < kIn; ++p) {
            const int rr = (q * kIn + p) * S::kPass + sub;
            if (r0 + rr < rows) {
                c[p] = __ldg(reinterpret_cast<const uint32_t*>(codes + (r0 + rr) * ldc + k / 2));
                s[p] = __ldg(st + (rr & 31) * 16 + ((r0 + rr) >> 5 & 3) * 4);
            }
        }
#pragma unroll
        for (int p = 0; p < kIn; ++p) {
            const int64_t r = r0 + (q * kIn + p) * S::kPass + sub;
            if (r >= rows) continue;
            float v[8];
            decode8(c[p], v);
            const float f = scale_value(s[p]);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * f;
            T* o = y + r * ldy + k;
            if (VEC && k + 8 <= K) {
                store8(o, v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (k + i < K) o[i] = from_f<T>(v[i]);
            }
        }
    }
}

template <class T> bool aligned16(const T* p, int64_t ld) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * int64_t(sizeof(T)) % 16 == 0;
}

// f(VEC, LPR, ROWS, column groups, grid): 16-byte accesses where the rows are aligned, two rows per warp for
// narrow ones, tiles in four parts of 32 rows where there are few (all parts of a tile run: each writes its scales).
template <class T, class F> void choose(const T* p, int64_t ld, int64_t rows, int64_t K, const char* what, F&& f) {
    const bool vec = aligned16(p, ld), narrow = K <= 128;
    const int64_t groups = narrow ? 1 : (K + 255) / 256, tiles = (rows + 127) / 128 * groups;
    const bool parts = tiles < 2 * device_sm_count();
    if (tiles > INT32_MAX) fail(kUnsupported, std::string(what) + ": matrix too large for one launch");
    const unsigned grid = unsigned(parts ? 4 * tiles : tiles);
    std::integral_constant<int, 16> half;
    std::integral_constant<int, 32> warp, r32;
    std::integral_constant<int, 128> r128;
    auto rest = [&](auto v, auto lanes) {
        if (parts) f(v, lanes, r32, int(groups), grid);
        else f(v, lanes, r128, int(groups), grid);
    };
    if (vec && narrow) rest(std::true_type(), half);
    else if (vec) rest(std::true_type(), warp);
    else if (narrow) rest(std::false_type(), half);
    else rest(std::false_type(), warp);
    VB_LAUNCH();
}

}  // namespace

template <class T>
void quantize(const T* x, int64_t ldx, int64_t rows, int64_t K, uint8_t* codes, int64_t ldc, uint8_t* scales,
              cudaStream_t s) {
    if (rows <= 0) return;
    choose(x, ldx, rows, K, "mx4_quantize", [&](auto vec, auto lpr, auto part, int groups, unsigned grid) {
        quantize_kernel<T, decltype(vec)::value, decltype(lpr)::value, decltype(part)::value>
            <<<grid, kThreads, 0, s>>>(x, ldx, rows, K, int(k_tiles(K)), groups, codes, ldc, scales);
    });
}

template <class T>
void dequantize(const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t rows, int64_t K, T* y, int64_t ldy,
                cudaStream_t s) {
    if (rows <= 0) return;
    choose(y, ldy, rows, K, "mx4_dequantize", [&](auto vec, auto lpr, auto part, int groups, unsigned grid) {
        dequantize_kernel<T, decltype(vec)::value, decltype(lpr)::value, decltype(part)::value>
            <<<grid, kThreads, 0, s>>>(codes, ldc, scales, rows, K, int(k_tiles(K)), groups, y, ldy);
    });
}

template void quantize<float>(const float*, int64_t, int64_t, int64_t, uint8_t*, int64_t, uint8_t*, cudaStream_t);
template void quantize<__half>(const __half*, int64_t, int64_t, int64_t, uint8_t*, int64_t, uint8_t*, cudaStream_t);
template void dequantize<float>(const uint8_t*, int64_t, const uint8_t*, int64_t, int64_t, float*, int64_t, cudaStream_t);
template void dequantize<__half>(const uint8_t*, int64_t, const uint8_t*, int64_t, int64_t, __half*, int64_t,
                                 cudaStream_t);

}  // namespace vb::mx4
