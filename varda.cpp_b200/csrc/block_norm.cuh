// The norms after and before a block, fused with the block's gate and the residual scale.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace vb::k {

constexpr int kNormNone = 0, kNormLayer = 1, kNormRms = 2;

// x' = T(res_scale x + gate post(h)), y = T(pre(x') (1 + scale) + shift), or y as 4-bit blocks (mx4.cuh).
// post, pre: LayerNorm or RMSNorm over the C columns (weight w, bias b; either may be null), or the
// identity. gate, scale, shift: one row of C values per `group` consecutive rows (one for all if 0).
template <class T> struct BlockNormArgs {
    int64_t rows = 0;
    int C = 0;
    const T* x = nullptr;
    int64_t ldx = 0;
    const T* h = nullptr;  // null: no block output
    int64_t ldh = 0;
    int post = kNormNone;
    const float *post_w = nullptr, *post_b = nullptr;
    const T* gate = nullptr;
    int64_t ldgate = 0;
    float res_scale = 1.0f;
    T* out = nullptr;  // x' (may be null, may be x)
    int64_t ldo = 0;
    int pre = kNormNone;
    const float *pre_w = nullptr, *pre_b = nullptr;
    const T *scale = nullptr, *shift = nullptr;
    int64_t ldmod = 0;
    int64_t group = 0;
    T* y = nullptr;
    int64_t ldy = 0;
    uint8_t* yc = nullptr;  // 4-bit output: codes, ldyc bytes per row, and scale tiles
    int64_t ldyc = 0;
    uint8_t* ys = nullptr;
    float eps = 0.0f;
};

constexpr int kBlockNormMaxC = 16384;

// Enqueues on s: no allocation, no synchronisation. C at most kBlockNormMaxC.
template <class T> void block_norm(const BlockNormArgs<T>& a, cudaStream_t s);

}  // namespace vb::k
