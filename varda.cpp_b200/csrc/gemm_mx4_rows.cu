// The 4-bit product for few rows of A (gemm_mx4.cuh), on the CUDA cores: bound by reading the weights (17/32 B per
// weight) and, at these sizes, by latency: [1 x 1024] x [1024 x 4096] 3.0 us, of which the weights are 0.35.
//
// Twice an e2m1 value is a whole number (0, 1, 2, 3, 4, 6, 8, 12 and the negatives), so a block's 32
// products are 8 dp4a on int8 values looked up from the codes, exact in 32 bits; one fp32
// multiply-add per block and output applies the scales. A lane takes one block (16 bytes of codes) of the
// row at a time, a warp 32 consecutive blocks of 4 rows of W, 32 rows apart (their scale bytes are then
// neighbours), so each W row is read in coalesced 512-byte pieces. The warps of a CTA split K where it has
// more than one such piece, and join their sums in shared memory in a fixed order.
#include <string>

#include "common.h"
#include "dev.cuh"
#include "gelu.cuh"
#include "gemm_mx4.cuh"

namespace vb::mx4 {

using namespace vb::d;

namespace {

constexpr int kWarps = 8;
constexpr int kRowsW = 4;  // rows of W per warp

// Four codes (the low 16 bits of c) -> four int8, twice their values: bytes picked from the table of the
// positive and of the negative values by the code's low three bits, then chosen by its sign.
__device__ __forceinline__ int lookup4(uint32_t c) {
    const uint32_t sel = c & 0x7777u;
    const uint32_t pos = __byte_perm(0x03020100u, 0x0c080604u, sel), neg = __byte_perm(0xfdfeff00u, 0xf4f8fafcu, sel);
    const uint32_t m = __byte_perm(0x0000ff00u, 0u, (c >> 3) & 0x1111u);
    return int((pos & ~m) | (neg & m));
}
__device__ __forceinline__ void lookup32(uint4 u, int (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = lookup4(w[i]), v[2 * i + 1] = lookup4(w[i] >> 16);
}

// Scale bytes from kNear to 254 - kNear (2^-95 to 2^95) need no care: a block's sum is below 2^13.
constexpr uint32_t kNear = 32, kOne = 127;
// d scale(sa) scale(sw) / 4 (both factors are twice their values) for any scales: the power of two in two halves.
__device__ __noinline__ float far_product(int d, uint32_t sa, uint32_t sw) {
    if (sa == 255u || sw == 255u) return scale_value(255u);
    const int e = int(sa + sw) - 256, h = e >> 1;
    return float(d) * __uint_as_float(uint32_t(max(h + 127, 1)) << 23) * __uint_as_float(uint32_t(max(e - h + 127, 1)) << 23);
}

template <class T, int MR, int WK>
__global__ void __launch_bounds__(32 * kWarps) rows_kernel(GemmArgs<T> a) {
    constexpr int NG = kWarps / WK;  // groups of 4 W rows per CTA
    __shared__ float part[kWarps][kRowsW * MR];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int wk = warp % WK, gi = warp / WK;
    const int64_t nt = blockIdx.x / (32 / NG);
    const int64_t n0 = nt * 128 + (blockIdx.x % (32 / NG)) * NG + gi;  // rows n0 + 32 j
    const int64_t nb = blocks(a.K), kt = k_tiles(a.K);
    float acc[kRowsW][MR];
#pragma unroll
    for (int j = 0; j < kRowsW; ++j)
#pragma unroll
        for (int m = 0; m < MR; ++m) acc[j][m] = 0.0f;
    for (int64_t b = wk * 32 + lane; b < nb; b += WK * 32) {
        uint4 w[kRowsW];
        uint32_t sw[kRowsW], sa[MR];
        bool far = false;  // a scale whose product with a block's sum may leave fp32 before the other scale brings it back
#pragma unroll
        for (int j = 0; j < kRowsW; ++j) {
            const int64_t n = n0 + 32 * j;
            const bool in = n < a.N;
            w[j] = in ? __ldg(reinterpret_cast<const uint4*>(a.W + n * a.ldw) + b) : make_uint4(0, 0, 0, 0);
            sw[j] = in ? __ldg(a.sW + scale_at(n, b, kt)) : kOne;
            far |= sw[j] - kNear > 254u - 2 * kNear;
        }
        int av[MR][8];
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            const bool in = m < a.M;
            const uint4 u = in ? __ldg(reinterpret_cast<const uint4*>(a.A + m * a.lda) + b) : make_uint4(0, 0, 0, 0);
            sa[m] = in ? __ldg(a.sA + scale_at(m, b, kt)) : kOne;
            far |= sa[m] - kNear > 254u - 2 * kNear;
            lookup32(u, av[m]);
        }
#pragma unroll
        for (int j = 0; j < kRowsW; ++j) {
            int wv[8];
            lookup32(w[j], wv);
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                int d = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) d = __dp4a(av[m][i], wv[i], d);
                if (!far) acc[j][m] = __fmaf_rn(float(d) * scale_value(sa[m]), 0.25f * scale_value(sw[j]), acc[j][m]);
                else acc[j][m] += far_product(d, sa[m], sw[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kRowsW; ++j)
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            const float t = warp_sum(acc[j][m]);
            if (lane == 0) part[warp][m * kRowsW + j] = t;
        }
    __syncthreads();
    if (wk != 0 || lane >= kRowsW * MR) return;
    const int64_t n = n0 + 32 * (lane % kRowsW), m = lane / kRowsW;
    if (n >= a.N || m >= a.M) return;
    float y = 0.0f;
#pragma unroll
    for (int i = 0; i < WK; ++i) y += part[gi * WK + i][lane];
    if (a.bias) y += to_f<T>(a.bias[n]);
    if (a.epi == k::kEpiGelu) y = a.gelu_tanh ? gelu(y, true) : gelu2<kFineGelu<T>>(make_float2(y, y)).x;
    if (a.epi == k::kEpiResidual) y += to_f<T>(a.R[m * a.ldr + n]);
    a.Y[m * a.ldy + n] = from_f<T>(y);
}

template <class T, int MR, int WK> void launch(const GemmArgs<T>& a, cudaStream_t s) {
    const int64_t grid = (a.N + 127) / 128 * (32 / (kWarps / WK));
    if (grid > INT32_MAX) fail(kUnsupported, "gemm_mx4: too many columns for one launch");
    rows_kernel<T, MR, WK><<<unsigned(grid), 32 * kWarps, 0, s>>>(a);
    VB_LAUNCH();
}

// as many warps along K as it has pieces of 32 blocks (a power of two)
template <class T, int MR> void dispatch_k(const GemmArgs<T>& a, cudaStream_t s) {
    const int64_t nb = blocks(a.K);
    if (nb > 128) launch<T, MR, 8>(a, s);
    else if (nb > 64) launch<T, MR, 4>(a, s);
    else if (nb > 32) launch<T, MR, 2>(a, s);
    else launch<T, MR, 1>(a, s);
}

}  // namespace

template <class T> void gemm_rows(const GemmArgs<T>& a, cudaStream_t s) {
    if (a.M <= 0 || a.N <= 0) return;
    if (a.M > kFewRows) fail(kInvalidArgument, "gemm_mx4: too many rows for the few-row kernel");
    if (a.M == 1) dispatch_k<T, 1>(a, s);
    else if (a.M == 2) dispatch_k<T, 2>(a, s);
    else dispatch_k<T, kFewRows>(a, s);
}

template void gemm_rows<float>(const GemmArgs<float>&, cudaStream_t);
template void gemm_rows<__half>(const GemmArgs<__half>&, cudaStream_t);

}  // namespace vb::mx4
