// Block norm (see block_norm.cuh). One pass over the rows: x and h are read once, x' and y written once,
// and the row stays in registers between its norms (fp32, two-pass statistics).
#include <algorithm>
#include <string>

#include "block_norm.cuh"
#include "common.h"
#include "dev.cuh"
#include "mx4.cuh"

namespace vb::k {

using namespace vb::d;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

// Eight values from column c of a row of C (zeros past its end).
template <class S, bool VEC> __device__ __forceinline__ void load8(const S* p, int c, int C, float* v) {
    if (VEC && c + 8 <= C) {
        Vec<S, 8>::load(p + c, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < C ? to_f<S>(p[c + i]) : 0.0f;
    }
}
template <class S, bool VEC> __device__ __forceinline__ void store8(S* p, int c, int C, const float* v) {
    if (VEC && c + 8 <= C) {
        Vec<S, 8>::store(p + c, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < C) p[c + i] = from_f<S>(v[i]);
    }
}

// The sum of x over the WPR warps of a row (every thread of the CTA calls it).
template <int WPR> __device__ __forceinline__ float row_sum(float x, float* red, int warp, int lane) {
    x = warp_sum(x);
    if (WPR == 1) return x;
    __syncthreads();  // the previous sum has been read
    if (lane == 0) red[warp] = x;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) s += red[warp / WPR * WPR + i];
    return s;
}

// v <- norm(v), columns c(i) .. c(i) + 7 in v[i]; columns from C on are zero before and ignored.
template <int NV, int WPR, bool VEC>
__device__ __forceinline__ void apply_norm(float (&v)[NV][8], int kind, const float* w, const float* b, int C, float eps,
                                           int c0, float* red, int warp, int lane) {
    if (kind == kNormNone) return;
    float mean = 0.0f;
    if (kind == kNormLayer) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[i][j];
        mean = row_sum<WPR>(s, red, warp, lane) / float(C);
    }
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * WPR * 256;
        if (c + 8 <= C) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] -= mean, q = __fmaf_rn(v[i][j], v[i][j], q);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < C) v[i][j] -= mean, q = __fmaf_rn(v[i][j], v[i][j], q);
        }
    }
    const float rstd = 1.0f / sqrtf(row_sum<WPR>(q, red, warp, lane) / float(C) + eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * WPR * 256;
        if (c >= C) continue;
        float p[8];
        if (w) load8<float, VEC>(w, c, C, p);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * rstd * (w ? p[j] : 1.0f);
        if (b) {
            load8<float, VEC>(b, c, C, p);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] += p[j];
        }
    }
}

// WPR warps per row, NV vectors of 8 columns per thread.
template <class T, int NV, int WPR, bool VEC>
__global__ void __launch_bounds__(kThreads) block_norm_kernel(BlockNormArgs<T> a, int64_t ktiles) {
    __shared__ float red[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = int64_t(blockIdx.x) * (kWarps / WPR) + warp / WPR;
    if (WPR == 1 && r >= a.rows) return;
    const bool live = r < a.rows;
    const int C = live ? a.C : 0;  // (a row past the end has no columns, but takes part in the sums)
    const int c0 = ((warp % WPR) * 32 + lane) * 8;
    const int64_t g = a.group ? r / a.group : 0;
    float x[NV][8], h[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) load8<T, VEC>(a.x + r * a.ldx, c0 + i * WPR * 256, C, x[i]);
    if (a.h) {
#pragma unroll
        for (int i = 0; i < NV; ++i) load8<T, VEC>(a.h + r * a.ldh, c0 + i * WPR * 256, C, h[i]);
        apply_norm<NV, WPR, VEC>(h, a.post, a.post_w, a.post_b, C, a.eps, c0, red, warp, lane);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * WPR * 256;
        if (c >= C) continue;
        if (a.h && a.gate) {
            float p[8];
            load8<T, VEC>(a.gate + g * a.ldgate, c, C, p);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] *= p[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[i][j] *= a.res_scale;
            if (a.h) x[i][j] += h[i][j];
            x[i][j] = rnd<T>(x[i][j]);  // the stream is held in T, and pre norms what is held
        }
        if (a.out) store8<T, VEC>(a.out + r * a.ldo, c, C, x[i]);
    }
    if (!a.y && !a.yc) return;
    apply_norm<NV, WPR, VEC>(x, a.pre, a.pre_w, a.pre_b, C, a.eps, c0, red, warp, lane);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * WPR * 256;
        if (a.scale && c < C) {
            float p[8];
            load8<T, VEC>(a.scale + g * a.ldmod, c, C, p);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] *= 1.0f + p[j];
        }
        if (a.shift && c < C) {
            float p[8];
            load8<T, VEC>(a.shift + g * a.ldmod, c, C, p);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] += p[j];
        }
        if (a.y && c < C) store8<T, VEC>(a.y + r * a.ldy, c, C, x[i]);
        if (a.yc) {
            // the four threads of a block share its maximum, the sixteen of 128 columns a word of scales
            uint32_t top = mx4::top8(x[i]);
            top = max(top, __shfl_xor_sync(kFull, top, 1));
            top = max(top, __shfl_xor_sync(kFull, top, 2));
            const uint32_t s = mx4::scale_byte(top);
            uint32_t w = s << (8 * ((lane >> 2) & 3));
            w |= __shfl_xor_sync(kFull, w, 4);
            w |= __shfl_xor_sync(kFull, w, 8);
            if (live && (c & ~31) < C)
                *reinterpret_cast<uint32_t*>(a.yc + r * a.ldyc + c / 2) = mx4::encode8(x[i], mx4::inv_scale(s));
            if (live && (lane & 15) == 0 && c < C)
                *reinterpret_cast<uint32_t*>(a.ys + mx4::scale_at(r, c / mx4::kBlock, ktiles)) = w;
        }
    }
}

template <class T, int NV, int WPR> void launch(const BlockNormArgs<T>& a, bool vec, cudaStream_t s) {
    const int64_t grid = (a.rows + kWarps / WPR - 1) / (kWarps / WPR);
    if (grid > INT32_MAX) fail(kUnsupported, "block_norm: too many rows for one launch");
    const int64_t kt = mx4::k_tiles(a.C);
    if (vec) block_norm_kernel<T, NV, WPR, true><<<unsigned(grid), kThreads, 0, s>>>(a, kt);
    else block_norm_kernel<T, NV, WPR, false><<<unsigned(grid), kThreads, 0, s>>>(a, kt);
    VB_LAUNCH();
}

bool aligned(const void* p, int64_t row_bytes = 0) {
    return ((reinterpret_cast<uintptr_t>(p) | uint64_t(row_bytes)) & 15) == 0;
}

}  // namespace

template <class T> void block_norm(const BlockNormArgs<T>& a, cudaStream_t s) {
    if (a.rows <= 0) return;
    if (a.C < 1 || a.C > kBlockNormMaxC) fail(kUnsupported, "block_norm: " + std::to_string(a.C) + " columns (1 to 16384)");
    const int64_t z = sizeof(T);
    const bool vec = aligned(a.x, a.ldx * z) && aligned(a.h, a.ldh * z) && aligned(a.gate, a.ldgate * z) &&
                     aligned(a.out, a.ldo * z) && aligned(a.scale, a.ldmod * z) && aligned(a.shift) && aligned(a.y, a.ldy * z) &&
                     aligned(a.post_w) && aligned(a.post_b) && aligned(a.pre_w) && aligned(a.pre_b);
    const int nv = (a.C + 255) / 256;  // vectors of 8 per lane of one warp
    // a warp per row once the rows fill the SMs' warps; with fewer rows, as many warps per row as it has
    // 256-column pieces, for latency
    if (nv == 1) return launch<T, 1, 1>(a, vec, s);
    if (a.rows >= 8 * int64_t(device_sm_count()) && nv <= 8) {
        if (nv <= 2) launch<T, 2, 1>(a, vec, s);
        else if (nv <= 4) launch<T, 4, 1>(a, vec, s);
        else launch<T, 8, 1>(a, vec, s);
        return;
    }
    if (nv <= 2) launch<T, 1, 2>(a, vec, s);
    else if (nv <= 4) launch<T, 1, 4>(a, vec, s);
    else if (nv <= 8) launch<T, 1, 8>(a, vec, s);
    else if (nv <= 16) launch<T, 2, 8>(a, vec, s);
    else if (nv <= 32) launch<T, 4, 8>(a, vec, s);
    else launch<T, 8, 8>(a, vec, s);
}

template void block_norm<float>(const BlockNormArgs<float>&, cudaStream_t);
template void block_norm<__half>(const BlockNormArgs<__half>&, cudaStream_t);

}  // namespace vb::k
