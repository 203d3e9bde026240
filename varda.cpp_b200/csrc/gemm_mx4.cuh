// Products of microscaled 4-bit matrices (mx4.cuh): Y[M, N] = epilogue(A[M, K] W[N, K]^T + bias), fp32 sums,
// one rounding to T at the end (the epilogue works on the fp32 sum).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.cuh"
#include "mx4.cuh"

namespace vb::mx4 {

constexpr int kFewRows = 4;

template <class T> struct GemmArgs {
    const uint8_t* A = nullptr;  // codes [M, K], lda bytes per row
    int64_t lda = 0;
    const uint8_t* sA = nullptr;  // A's scale tiles
    const uint8_t* W = nullptr;   // codes [N, K], ldw bytes per row
    int64_t ldw = 0;
    const uint8_t* sW = nullptr;
    const T* bias = nullptr;  // [N] or null
    T* Y = nullptr;           // [M, N] ldy elements; null: the output goes to Yc, Ys as 4-bit blocks
    int64_t ldy = 0;
    uint8_t* Yc = nullptr;
    int64_t ldyc = 0;
    uint8_t* Ys = nullptr;
    const T* R = nullptr;  // residual [M, N] ldr (kEpiResidual)
    int64_t ldr = 0;
    int64_t M = 0, N = 0, K = 0;
    int epi = k::kEpiBias;
    bool gelu_tanh = false;
};

// At most kFewRows rows of A, on the CUDA cores (Y only). Enqueues on s: no allocation, no synchronisation.
template <class T> void gemm_rows(const GemmArgs<T>& a, cudaStream_t s);
// Any number of rows, Y or 4-bit output: on the tensor cores, or gemm_rows. Y and R 16-byte aligned, their rows
// a multiple of 16 bytes apart. Enqueues on s: no allocation, no synchronisation.
template <class T> void gemm(const GemmArgs<T>& a, cudaStream_t s);
// Reads and clears the device-side error flag of the bounded waits (synchronises); 0: none timed out.
int take_error();

}  // namespace vb::mx4
