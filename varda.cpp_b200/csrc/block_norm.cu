// Block norm (see block_norm.cuh): bound by memory (x and h read once, x' and y written once). The row stays in
// registers between its norms; statistics in fp32, two passes over the registers.
//
// Two kernels. rows_kernel, for many rows, has the norms' vectors in shared memory: reading seven vectors per row
// through the L1 cache costs more than the row itself (22 KB against 8 KB at fp16 and C = 1024). Where many
// rows share a modulation it is folded into them, x' = rs x + n(h) A1 + B1 and y = n(x') A2 + B2. few_kernel reads
// the vectors with the row, and takes up to eight warps for a row.
#include <algorithm>
#include <string>
#include <type_traits>

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

// Eight columns from c of row r (zeros past C) as part of a 4-bit block: the four lanes of a block share its
// maximum, the sixteen of 128 columns a word of scale bytes. Every lane of the warp calls it.
template <class T, int LPR>
__device__ __forceinline__ void store_blocks(const BlockNormArgs<T>& a, int64_t r, int c, int C, bool live, int64_t ktiles,
                                             const float* v) {
    uint32_t top = mx4::top8(v);
    top = max(top, __shfl_xor_sync(kFull, top, 1));
    top = max(top, __shfl_xor_sync(kFull, top, 2));
    const uint32_t s = mx4::scale_byte(top);
    uint32_t w = s << (8 * ((c >> 5) & 3));
    w |= __shfl_xor_sync(kFull, w, 4);
    if (LPR > 8) w |= __shfl_xor_sync(kFull, w, 8);  // (8 lanes have a row's 64 columns: two blocks)
    if (live && (c & ~31) < C) *reinterpret_cast<uint32_t*>(a.yc + r * a.ldyc + c / 2) = mx4::encode8(v, mx4::inv_scale(s));
    if (live && (c & 127) == 0 && c < C) *reinterpret_cast<uint32_t*>(a.ys + mx4::scale_at(r, c / mx4::kBlock, ktiles)) = w;
}

// WPR warps per row, NV vectors of 8 columns per thread. EARLY: the pre-norm's modulation is loaded with the row, for
// latency; otherwise it is only fetched into L2, which leaves registers for two more CTAs per SM ([2562 x 1000] fp32, a
// modulation per row: 18.8 us early, 17.3 late, [20000 x 1000] 108 and 99; [1 x 1024] fp16 4.3 and 4.7).
template <class T, int NV, int WPR, bool VEC, bool EARLY>
__global__ void __launch_bounds__(kThreads, NV == 8 ? 1 : NV == 4 ? 2 : NV == 2 || EARLY ? 4 : 6) few_kernel(BlockNormArgs<T> a, int64_t ktiles) {
    __shared__ float red[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = int64_t(blockIdx.x) * (kWarps / WPR) + warp / WPR;
    if (WPR == 1 && r >= a.rows) return;
    const bool live = r < a.rows;
    const int C = live ? a.C : 0;  // (a row past the end has no columns, but takes part in the sums)
    const int c0 = ((warp % WPR) * 32 + lane) * 8;
    const int64_t g = a.group ? r / a.group : 0;
    float x[NV][8], h[NV][8], gt[8], sc[8], sh[8];
#pragma unroll
    for (int i = 0; i < NV; ++i) load8<T, VEC>(a.x + r * a.ldx, c0 + i * WPR * 256, C, x[i]);
    if (a.h) {
#pragma unroll
        for (int i = 0; i < NV; ++i) load8<T, VEC>(a.h + r * a.ldh, c0 + i * WPR * 256, C, h[i]);
    }
    if (NV == 1 && a.h && a.gate) load8<T, VEC>(a.gate + g * a.ldgate, c0, C, gt);
    if constexpr (EARLY) {
        if (a.scale) load8<T, VEC>(a.scale + g * a.ldmod, c0, C, sc);
        if (a.shift) load8<T, VEC>(a.shift + g * a.ldmod, c0, C, sh);
    } else if (NV == 1 && c0 < C) {
        if (a.scale) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.scale + g * a.ldmod + c0));
        if (a.shift) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.shift + g * a.ldmod + c0));
    }
    if (a.h) apply_norm<NV, WPR, VEC>(h, a.post, a.post_w, a.post_b, C, a.eps, c0, red, warp, lane);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * WPR * 256;
        if (c >= C) continue;
        if (a.h && a.gate) {
            if (NV > 1) load8<T, VEC>(a.gate + g * a.ldgate, c, C, gt);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] *= gt[j];
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
            if (!EARLY) load8<T, VEC>(a.scale + g * a.ldmod, c, C, sc);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] *= 1.0f + sc[j];
        }
        if (a.shift && c < C) {
            if (!EARLY) load8<T, VEC>(a.shift + g * a.ldmod, c, C, sh);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] += sh[j];
        }
        if (a.y && c < C) store8<T, VEC>(a.y + r * a.ldy, c, C, x[i]);
        if (a.yc) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j >= C) x[i][j] = 0.0f;  // (-0 by a negative res_scale, NaN by an infinite rstd)
            store_blocks<T, 32>(a, r, c, C, live, ktiles, x[i]);
        }
    }
}

// Eight values as four pairs, for the packed fp32 operations.
struct F8 {
    float2 p[4];
};
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Eight values as stored, loaded now and widened when they are used.
template <class T> struct Raw8;
template <> struct Raw8<__half> {
    uint4 u;
    __device__ __forceinline__ void load(const __half* p) { u = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ F8 get() const {
        const __half2* h = reinterpret_cast<const __half2*>(&u);
        return {{__half22float2(h[0]), __half22float2(h[1]), __half22float2(h[2]), __half22float2(h[3])}};
    }
    __device__ __forceinline__ void set(const F8& f) {
        __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f.p[i].x, f.p[i].y);
    }
    __device__ __forceinline__ void store(__half* p) const { *reinterpret_cast<uint4*>(p) = u; }
    __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
    // n < 8 values
    __device__ __forceinline__ void load_part(const __half* p, int n) {
        auto get = [&](int i) -> uint32_t { return i < n ? uint32_t(__half_as_ushort(p[i])) : 0u; };
        u = make_uint4(get(0) | get(1) << 16, get(2) | get(3) << 16, get(4) | get(5) << 16, get(6));
    }
    __device__ __forceinline__ void store_part(__half* p, int n) const {
        if (n & 4) *reinterpret_cast<uint2*>(p) = make_uint2(u.x, u.y);
        const uint32_t a = n & 4 ? u.z : u.x, b = n & 4 ? u.w : u.y;
        if (n & 2) *reinterpret_cast<uint32_t*>(p + (n & 4)) = a;
        if (n & 1) p[n & 6] = __ushort_as_half((unsigned short)((n & 2 ? b : a) & 0xffffu));
    }
};
template <> struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    }
    __device__ __forceinline__ F8 get() const {
        return {{make_float2(a.x, a.y), make_float2(a.z, a.w), make_float2(b.x, b.y), make_float2(b.z, b.w)}};
    }
    __device__ __forceinline__ void set(const F8& f) {
        a = make_float4(f.p[0].x, f.p[0].y, f.p[1].x, f.p[1].y), b = make_float4(f.p[2].x, f.p[2].y, f.p[3].x, f.p[3].y);
    }
    __device__ __forceinline__ void store(float* p) const {
        *reinterpret_cast<float4*>(p) = a, *reinterpret_cast<float4*>(p + 4) = b;
    }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void load_part(const float* p, int n) {
        auto get = [&](int i) -> float { return i < n ? p[i] : 0.0f; };
        a = make_float4(get(0), get(1), get(2), get(3)), b = make_float4(get(4), get(5), get(6), 0.0f);
    }
    __device__ __forceinline__ void store_part(float* p, int n) const {
        if (n & 4) *reinterpret_cast<float4*>(p) = a;
        const float4 q = n & 4 ? b : a;
        if (n & 2) *reinterpret_cast<float2*>(p + (n & 4)) = make_float2(q.x, q.y);
        if (n & 1) p[n & 6] = n & 2 ? q.z : q.x;
    }
};
// Whether the last vector of a row before the last may be read whole: rows start 16-byte aligned, so eight values from a
// multiple of 8 below C end within the row's stride (fp16) or at most 4 values into the next row (fp32), which has them
// if C is at least 4.
template <class T> __device__ __forceinline__ bool reads_on(int C) { return sizeof(T) == 2 || C >= 4; }
// Eight values from column c of a row of C; `more`: another row follows in memory, so that the row's last vector
// can be read whole (what it holds past C is cut off later). Without one that vector is left zero here, for last8
// to fill: no else branch between a row's loads.
template <class T> __device__ __forceinline__ Raw8<T> raw8(const T* row, int c, int C, bool more) {
    Raw8<T> r;
    r.zero();
    if (c < C && (c + 8 <= C || more)) r.load(row + c);
    return r;
}
template <class T> __device__ __forceinline__ void last8(Raw8<T>& r, const T* row, int c, int C, bool more) {
    if (!more && c < C && c + 8 > C) r.load_part(row + c, C - c);
}
// ... written, the last vector in pieces of 4, 2 and 1.
template <class T> __device__ __forceinline__ void put8(T* row, int c, int C, Raw8<T>& r) {
    if (c + 8 <= C) {
        r.store(row + c);
        return;
    }
    r.store_part(row + c, C - c);
}
// zeros in the columns from C on
__device__ __forceinline__ void cut(F8& f, int c, int C) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (c + 2 * i >= C) f.p[i].x = 0.0f;
        if (c + 2 * i + 1 >= C) f.p[i].y = 0.0f;
    }
}

// CTAs per SM that the registers are cut for. More rows in flight are worth some spilling at fp16 ([189809 x 1024] 299 us
// with 2, 273 with 3; 512 columns 154 with 3, 142 with 4), not at fp32 (1024 columns 553 with 2, 680 with 3).
template <class T> constexpr int rows_ctas(int nv, bool perrow) {
    if (nv >= 3) return sizeof(T) == 2 && !perrow ? 3 : 2;
    return (perrow ? 4 : sizeof(T) == 2 ? 6 : 5) - nv;
}

// Many rows: CTA b takes rows [b per, (b + 1) per), LPR lanes of a warp or WPR warps per row, NV vectors of 8
// columns per lane. Shared memory: four vectors, A1, B1, A2, B2 of the modulation's rows (the range is cut where
// that changes), or with PERROW (a modulation per row or few rows, loaded with the row) the norms' weights and
// biases; each as the first and the second four of the lanes' eights, so that a warp reads 512 consecutive bytes.
// Threads of a CTA. Eight warps per row: its vectors (96 KB with three per lane, 128 KB with four) are shared by two rows,
// or three where the registers hold them ([20000 x 8192] fp16: 555 us with one row, 336 with two, 375 with three; 6000
// columns 296 with two, 264 with three).
template <class T> constexpr int rows_threads(int nv, int wpr, bool perrow) {
    return wpr < 8 ? kThreads : nv == 3 && sizeof(T) == 2 && !perrow ? 768 : 512;
}
template <class T, int NV, int LPR, int WPR, bool PERROW>
__global__ void __launch_bounds__(rows_threads<T>(NV, WPR, PERROW), WPR == 8 ? 1 : rows_ctas<T>(NV, PERROW))
    rows_kernel(BlockNormArgs<T> a, int64_t ktiles, int64_t per) {
    constexpr int kThreads = rows_threads<T>(NV, WPR, PERROW), kWarps = kThreads / 32;
    constexpr int kLanes = LPR * WPR, kRows = kThreads / kLanes;  // lanes per row, rows at a time
    constexpr int kVecs = NV * kLanes;                             // vectors of 8 columns per row
    extern __shared__ float4 fold[];                               // [4][2][kVecs]
    __shared__ float red[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col0 = int(threadIdx.x % kLanes) * 8;  // vector i: columns col0 + i kLanes 8 .. + 7
    const bool two = a.y || a.yc;
    const int64_t end = min(a.rows, (int64_t(blockIdx.x) + 1) * per);
    int64_t lo = int64_t(blockIdx.x) * per;
    auto total = [&](float x) -> float {
        if constexpr (WPR > 1) {
            return row_sum<WPR>(x, red, warp, lane);
        } else {
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
            return x;
        }
    };
    while (lo < end) {
        const int C = a.C;
        const int64_t g = a.group ? lo / a.group : 0;
        const int64_t hi = a.group && !PERROW ? min(end, (g + 1) * a.group) : end;
        __syncthreads();  // the rows before have read the vectors
        for (int v = threadIdx.x; v < kVecs; v += kThreads) {
            const int c = v * 8;
            float w[8] = {}, b[8] = {}, m[8];
            auto put = [&](int k) {
                fold[(2 * k) * kVecs + v] = make_float4(w[0], w[1], w[2], w[3]);
                fold[(2 * k + 1) * kVecs + v] = make_float4(w[4], w[5], w[6], w[7]);
                fold[(2 * k + 2) * kVecs + v] = make_float4(b[0], b[1], b[2], b[3]);
                fold[(2 * k + 3) * kVecs + v] = make_float4(b[4], b[5], b[6], b[7]);
            };
            auto weights = [&](int kind, const float* pw, const float* pb) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = kind && pw && c + j < C ? __ldg(pw + c + j) : 1.0f;
                    b[j] = kind && pb && c + j < C ? __ldg(pb + c + j) : 0.0f;
                }
            };
            if (a.h) {
                weights(a.post, a.post_w, a.post_b);
                if (!PERROW && a.gate) {
                    load8<T, true>(a.gate + g * a.ldgate, c, C, m);
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] *= m[j], b[j] = a.post_b ? b[j] * m[j] : 0.0f;  // (0 Inf is no bias)
                }
                put(0);
            }
            weights(a.pre, a.pre_w, a.pre_b);
            if (!PERROW && a.scale) {
                load8<T, true>(a.scale + g * a.ldmod, c, C, m);
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] *= 1.0f + m[j], b[j] = a.pre_b ? b[j] * (1.0f + m[j]) : 0.0f;
            }
            if (!PERROW && a.shift) {
                load8<T, true>(a.shift + g * a.ldmod, c, C, m);
#pragma unroll
                for (int j = 0; j < 8; ++j) b[j] += m[j];
            }
            put(2);
        }
        __syncthreads();
        auto folded = [&](int k, int i) -> F8 {
            const int v = i * kLanes + int(threadIdx.x % kLanes);
            const float4 p = fold[(2 * k) * kVecs + v], q = fold[(2 * k + 1) * kVecs + v];
            return {{make_float2(p.x, p.y), make_float2(p.z, p.w), make_float2(q.x, q.y), make_float2(q.z, q.w)}};
        };
        for (int64_t r0 = lo; r0 < hi; r0 += kRows) {
            const int64_t r = r0 + threadIdx.x / kLanes;
            const bool live = r < hi;
            const int C = live ? a.C : 0;  // (a row past the end has no columns, but takes part in the sums)
            // v <- (v - mean) rstd, or v where the norm is none
            auto centre = [&](F8(&v)[NV], int kind) {
                if (kind == kNormNone) return;
                float mean = 0.0f;
                if (kind == kNormLayer) {
                    float2 s = both(0.0f);
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) s = __fadd2_rn(s, v[i].p[j]);
                    mean = total(s.x + s.y) / float(C);
                }
                float2 q = both(0.0f);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = col0 + i * kLanes * 8;
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i].p[j] = __fadd2_rn(v[i].p[j], both(-mean));
                    if (c + 8 > C) cut(v[i], c, C);
#pragma unroll
                    for (int j = 0; j < 4; ++j) q = __ffma2_rn(v[i].p[j], v[i].p[j], q);
                }
                const float rstd = 1.0f / sqrtf(total(q.x + q.y) / float(C) + a.eps);
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i].p[j] = __fmul2_rn(v[i].p[j], both(rstd));
            };
            const bool more = r + 1 < a.rows && reads_on<T>(a.C);
            Raw8<T> xr[NV], hr[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) xr[i] = raw8(a.x + r * a.ldx, col0 + i * kLanes * 8, C, more);
            if (a.h) {
#pragma unroll
                for (int i = 0; i < NV; ++i) hr[i] = raw8(a.h + r * a.ldh, col0 + i * kLanes * 8, C, more);
            }
            F8 v[NV];
            // PERROW: a lane's vectors of the modulation fly with the row
            Raw8<T> gr[NV], scr[NV], shr[NV];
            const int64_t gm = PERROW && a.group ? r / a.group : 0;
            const bool more_g = PERROW && a.group && gm < (a.rows - 1) / a.group && reads_on<T>(a.C);
            if constexpr (PERROW) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = col0 + i * kLanes * 8;
                    if (a.h && a.gate) gr[i] = raw8(a.gate + gm * a.ldgate, c, C, more_g);
                    if (two && a.scale) scr[i] = raw8(a.scale + gm * a.ldmod, c, C, more_g);
                    if (two && a.shift) shr[i] = raw8(a.shift + gm * a.ldmod, c, C, more_g);
                }
            }
            if (!more) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = col0 + i * kLanes * 8;
                    last8(xr[i], a.x + r * a.ldx, c, C, more);
                    if (a.h) last8(hr[i], a.h + r * a.ldh, c, C, more);
                }
            }
            if (a.h) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = col0 + i * kLanes * 8;
                    v[i] = hr[i].get();
                    if (c + 8 > C) cut(v[i], c, C);
                }
                centre(v, a.post);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = col0 + i * kLanes * 8;
                F8 x = xr[i].get();
                if (a.h) {
                    const F8 w = folded(0, i), b = folded(1, i);
                    F8 gt;
                    if (PERROW && a.gate) {
                        if (!more_g) last8(gr[i], a.gate + gm * a.ldgate, c, C, more_g);
                        gt = gr[i].get();
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float2 t = __ffma2_rn(v[i].p[j], w.p[j], b.p[j]);
                        if (PERROW && a.gate) t = __fmul2_rn(t, gt.p[j]);
                        x.p[j] = __ffma2_rn(x.p[j], both(a.res_scale), t);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) x.p[j] = __fmul2_rn(x.p[j], both(a.res_scale));
                }
                Raw8<T> o;  // the stream is held in T, and pre norms what is held
                o.set(x);
                if (a.out && c < C) put8(a.out + r * a.ldo, c, C, o);
                v[i] = o.get();
                if (c + 8 > C) cut(v[i], c, C);
            }
            if (!two) continue;
            centre(v, a.pre);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = col0 + i * kLanes * 8;
                const F8 w = folded(2, i), b = folded(3, i);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i].p[j] = __ffma2_rn(v[i].p[j], w.p[j], b.p[j]);
                if (PERROW && a.scale) {
                    if (!more_g) last8(scr[i], a.scale + gm * a.ldmod, c, C, more_g);
                    const F8 sc = scr[i].get();
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i].p[j] = __fmul2_rn(v[i].p[j], __fadd2_rn(sc.p[j], both(1.0f)));
                }
                if (PERROW && a.shift) {
                    if (!more_g) last8(shr[i], a.shift + gm * a.ldmod, c, C, more_g);
                    const F8 sh = shr[i].get();
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i].p[j] = __fadd2_rn(v[i].p[j], sh.p[j]);
                }
                if (a.y && c < C) {
                    Raw8<T> o;
                    o.set(v[i]);
                    put8(a.y + r * a.ldy, c, C, o);
                }
                if (a.yc) {
                    if (c + 8 > C) cut(v[i], c, C);
                    store_blocks<T, LPR>(a, r, c, C, live, ktiles, reinterpret_cast<const float*>(&v[i]));
                }
            }
        }
        lo = hi;
    }
}

template <class T, int NV, int WPR> void launch(const BlockNormArgs<T>& a, bool vec, cudaStream_t s) {
    const int64_t grid = (a.rows + kWarps / WPR - 1) / (kWarps / WPR);
    if (grid > INT32_MAX) fail(kUnsupported, "block_norm: too many rows for one launch");
    const int64_t kt = mx4::k_tiles(a.C);
    auto go = [&](auto v, auto early) {
        few_kernel<T, NV, WPR, decltype(v)::value, decltype(early)::value><<<unsigned(grid), kThreads, 0, s>>>(a, kt);
    };
    const bool early = NV == 1 && grid <= 4 * device_sm_count();  // one wave of CTAs
    if constexpr (NV == 1) {
        if (early && vec) go(std::true_type(), std::true_type());
        else if (early) go(std::false_type(), std::true_type());
    }
    if (!early && vec) go(std::true_type(), std::false_type());
    else if (!early) go(std::false_type(), std::false_type());
    VB_LAUNCH();
}

template <class T, int NV, int LPR, int WPR, bool PERROW> void launch_rows(const BlockNormArgs<T>& a, cudaStream_t s) {
    constexpr int kThreads = rows_threads<T>(NV, WPR, PERROW), kRows = kThreads / (LPR * WPR);
    constexpr int kSmem = 4 * 2 * NV * LPR * WPR * int(sizeof(float4));
    static_assert(kSmem <= 131072, "vectors of one row");
    static std::atomic<int> per_sm[64];  // resident CTAs per SM, by device
    auto* kernel = &rows_kernel<T, NV, LPR, WPR, PERROW>;
    int dev = 0, n = 0;
    VB_CUDA(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64) n = per_sm[dev].load(std::memory_order_acquire);
    if (!n) {
        VB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        VB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, kSmem));
        if (dev >= 0 && dev < 64) per_sm[dev].store(n, std::memory_order_release);
    }
    const int64_t ctas = int64_t(std::max(1, n)) * device_sm_count();
    const int64_t per = ((a.rows + ctas - 1) / ctas + kRows - 1) / kRows * kRows;  // whole rounds of a CTA
    kernel<<<unsigned((a.rows + per - 1) / per), kThreads, kSmem, s>>>(a, mx4::k_tiles(a.C), per);
    VB_LAUNCH();
}

bool aligned(const void* p, int64_t row_bytes = 0) {
    return ((reinterpret_cast<uintptr_t>(p) | uint64_t(row_bytes)) & 15) == 0;
}

}  // namespace

template <class T> void block_norm(const BlockNormArgs<T>& args, cudaStream_t s) {
    // What is not read chooses nothing: a gate and a norm without h, a modulation and a norm without y, a norm's vectors
    // without the norm, strides without their array, groups without a modulation
    BlockNormArgs<T> a = args;
    if (!a.h) a.gate = nullptr, a.post = kNormNone, a.ldh = 0;
    if (!a.y && !a.yc) a.scale = a.shift = nullptr, a.pre = kNormNone;
    if (a.post == kNormNone) a.post_w = a.post_b = nullptr;
    if (a.pre == kNormNone) a.pre_w = a.pre_b = nullptr;
    if (!a.gate) a.ldgate = 0;
    if (!a.scale && !a.shift) a.ldmod = 0;
    if (!a.gate && !a.scale && !a.shift) a.group = 0;
    if (!a.out) a.ldo = 0;
    if (!a.y) a.ldy = 0;
    if (a.rows <= 0) return;
    if (a.C < 1 || a.C > kBlockNormMaxC) fail(kUnsupported, "block_norm: " + std::to_string(a.C) + " columns (1 to 16384)");
    const int64_t z = sizeof(T);
    const bool vec = aligned(a.x, a.ldx * z) && aligned(a.h, a.ldh * z) && aligned(a.gate, a.ldgate * z) &&
                     aligned(a.out, a.ldo * z) && aligned(a.scale, a.ldmod * z) && aligned(a.shift) && aligned(a.y, a.ldy * z) &&
                     aligned(a.post_w) && aligned(a.post_b) && aligned(a.pre_w) && aligned(a.pre_b);
    const int nv = (a.C + 255) / 256;  // vectors of 8 per lane of one warp
    // a warp per row once the rows fill the SMs' warps; with fewer rows, as many warps per row as it has
    // 256-column pieces, for latency
    // rows_kernel from the rows on where it is the faster one ([2000 x 1024] fp16, vectors folded: 9.7 -> 8.0 us, and
    // [9000 x 1024] 39 -> 22; a modulation per row: [5000 x 1024] fp16 32 -> 27, but [2562 x 1000] fp32 17 -> 29, for want of
    // registers). Folding one modulation takes a CTA the time of some 50 rows
    const bool fold = !a.group || a.group >= 1024;
    constexpr bool kPerRow = sizeof(T) == 2;
    if (vec && nv <= 32 && (fold || kPerRow) && a.rows >= int64_t(fold ? 4 : 8) * device_sm_count()) {
        auto go = [&](auto n, auto lanes, auto warps) {
            constexpr int kN = decltype(n)::value, kL = decltype(lanes)::value, kW = decltype(warps)::value;
            if constexpr (kPerRow) {
                if (!fold) return launch_rows<T, kN, kL, kW, true>(a, s);
            }
            launch_rows<T, kN, kL, kW, false>(a, s);
        };
        std::integral_constant<int, 1> one;
        std::integral_constant<int, 2> n2;
        std::integral_constant<int, 3> n3;
        std::integral_constant<int, 4> n4;
        std::integral_constant<int, 8> n8;
        std::integral_constant<int, 32> warp;
        // three vectors per lane rather than four that are not full ([40000 x 768] fp16: 53 against 66 us, [20000 x 2800] 115
        // against 159, fp32 175 against 194; but [40000 x 768] fp32 92 against 83)
        if (a.C <= 64) go(one, std::integral_constant<int, 8>(), one);
        else if (a.C <= 128) go(one, std::integral_constant<int, 16>(), one);
        else if (nv <= 1) go(one, warp, one);
        else if (nv <= 2) go(n2, warp, one);
        else if (nv <= 3 && sizeof(T) == 2) go(n3, warp, one);
        else if (nv <= 4) go(n4, warp, one);
        else if (nv <= 6) go(n3, warp, n2);
        else if (nv <= 8) go(n4, warp, n2);
        else if (nv <= 12) go(n3, warp, n4);
        else if (nv <= 16) go(n4, warp, n4);
        else if (nv <= 24) go(n3, warp, n8);
        else go(n4, warp, n8);
        return;
    }
    if (nv == 1) return launch<T, 1, 1>(a, vec, s);
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
