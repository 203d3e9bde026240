// The 4-bit product on the tensor cores (see gemm_mx4.cuh): tcgen05.mma kind::mxf4 with block scales, which
// multiplies 64 e2m1 values of a row and column at a time, each block of 32 with its two scales, into fp32.
//
// Persistent and warp-specialised as the fp16 GEMM (gemm_tc.cu): one 320-thread CTA per SM, or clusters of
// two with cta_group::2 computing 256-row tiles together.
//   warp 0 (one lane)   TMA producer, per 256 columns of K: codes of A [128 x 128 bytes] and of W, 128-byte
//                       swizzle, and their scale tiles (512 bytes per 128 rows and 128 columns, stored in
//                       the order tcgen05.cp takes), into a ring of STAGES.
//   warp 1 (one lane)   MMA issuer: tcgen05.cp of the stage's scales into one of two tensor-memory buffers
//                       (every lane quarter gets a copy), then 4 MMAs of K = 64; in a last stage that K
//                       cuts, only those it needs. A buffer is overwritten once the MMAs of two stages ago
//                       have completed.
//   warps 2-9           epilogue: 32 columns at a time from tensor memory, bias / GELU / residual in fp32, one
//                       rounding, and a TMA store from swizzled shared memory; or 4-bit output: a lane holds
//                       one row's block of 32 columns, so its scale is the maximum of the lane's registers.
// Tensor memory at BN = 256: two accumulators would fill all 512 columns, but the scales need 48. So the
// second starts at column 192, over the last 64 columns of the first, and both epilogues read those shared
// columns first: the next tile's MMAs start when they have been read, a quarter into the epilogue.
//
// Every wait is bounded as in gemm_tc.cu: on timeout a CTA sets the device error flag, stops issuing, waits for
// its own copies and MMAs in flight, frees its tensor memory and returns.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "common.h"
#include "dev.cuh"
#include "gemm_mx4.cuh"
#include "gemm_tc.cuh"
#include "ptx.cuh"

namespace vb::mx4 {

namespace {

using namespace vb::d;
using namespace vb::ptx;

constexpr int BM = 128, BKB = 128;  // rows of a CTA's tile; bytes of codes per row and stage (256 columns)
constexpr int kEpiWarps = 8, kThreads = 32 * (2 + kEpiWarps);
constexpr unsigned long long kTimeoutNs = 4000000000ull;  // 4 s

__device__ int g_error = 0;

struct Params {
    const void* bias;
    const void* R;
    int64_t ldr;
    void* Y;
    int64_t ldy;
    uint8_t* Yc;
    int64_t ldyc;
    uint8_t* Ys;
    int64_t ktiles_out;
    int M, N, K64;  // K64: MMAs along K, ceil(K / 64)
    int gelu_tanh;
};

__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, volatile int* abort_flag) {
    if (mbar_test(b, parity)) return true;
    const uint64_t t0 = now_ns();
    for (;;) {
        if (mbar_test(b, parity)) return true;
        if (*abort_flag) return false;
        if (now_ns() - t0 > kTimeoutNs) {
            *abort_flag = 1;
            atomicExch(&g_error, 1);
            return false;
        }
    }
}
// Ignores the abort flag (to drain work in flight), still bounded.
__device__ __forceinline__ void mbar_drain(uint64_t* b, uint32_t parity) {
    const uint64_t t0 = now_ns();
    while (!mbar_test(b, parity))
        if (now_ns() - t0 > kTimeoutNs) {
            atomicExch(&g_error, 2);
            return;
        }
}

template <bool PAIR>
__device__ __forceinline__ void load_2d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
    if (PAIR) tma_load_2d_pair(dst, map, bar, x, y);
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                smem_u32(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
            : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void load_3d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    if (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
            "%4}], [%5];" ::"r"(smem_u32(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
            "[%5];" ::"r"(smem_u32(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
}

// Shared-memory descriptors. Codes: K-major, 128-byte swizzle, 8-row groups 1024 bytes apart. Scales: 32
// rows of 16 bytes without swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t codes_desc(uint32_t saddr) {
    return uint64_t((saddr & 0x3FFFF) >> 4) | uint64_t(1) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
__device__ __forceinline__ uint64_t scales_desc(uint32_t saddr) {
    return uint64_t((saddr & 0x3FFFF) >> 4) | uint64_t(128 >> 4) << 32 | uint64_t(1) << 46;
}
// Instruction descriptor of kind::mxf4: A = B = e2m1 (1), scales ue8m0, K-major, K = 64; sf: which two of a
// 32-bit column's four scale bytes (0 or 2).
__host__ __device__ constexpr uint32_t instr_desc(int m, int n, int sf) {
    return uint32_t(sf) << 4 | 1u << 7 | 1u << 10 | uint32_t(n >> 3) << 17 | 1u << 23 | uint32_t(m >> 7) << 27 | uint32_t(sf) << 29;
}
template <bool PAIR> __device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
    if (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                    uint32_t acc) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc));
}

// T: type of bias, residual and output. OUT4: 4-bit output (T is the bias's type).
template <class T, int BN, bool PAIR, bool OUT4> struct Layout {
    static constexpr int kNTiles = BN > 128 ? BN / 128 : 1;  // scale tiles of W per 128 columns of K
    static constexpr int kA = BM * BKB, kB = (PAIR ? BN / 2 : BN) * BKB;
    static constexpr int kSA = 2 * 512, kSB = 2 * 512 * kNTiles;
    static constexpr int kStage = kA + kB + kSA + kSB;
    static constexpr int kSub = OUT4 ? 0 : 32 * 32 * int(sizeof(T));  // one 32 x 32 output sub-tile
    static constexpr int kOut = kEpiWarps * 2 * kSub;
    static constexpr int kMax = 232448 - 1024 - 256;  // the 227 KB per CTA, less alignment slack and barriers
    static constexpr int kFit = (kMax - kOut) / kStage;
    static constexpr int kStages = kFit < 8 ? kFit : 8;
    static constexpr int kBars = (2 * kStages + 5) * 8;
    static constexpr int kSmem = 1024 + kStages * kStage + kOut + kBars + 16;
    static_assert(kSmem <= 232448 && kStages >= 3, "shared memory over the 227 KB per-CTA limit");
    // tensor memory columns: accumulators at 0 and kAcc1, two scale buffers (A's, then W's) at kSf
    static constexpr bool kOverlap = BN == 256;
    static constexpr int kAcc1 = kOverlap ? 192 : BN, kSf = kAcc1 + BN, kSfBuf = 2 * 4 + 2 * 4 * kNTiles;
    static constexpr int kCols = kSf + 2 * kSfBuf <= 256 ? 256 : 512;
    static_assert(kSf + 2 * kSfBuf <= kCols, "tensor memory over 512 columns");
};

template <class T, int BN, bool PAIR, int EPI, bool OUT4>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_mx4_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSW,
                    const __grid_constant__ CUtensorMap tmY, Params p) {
    using L = Layout<T, BN, PAIR, OUT4>;
    constexpr int STAGES = L::kStages;
    constexpr int UM = PAIR ? 2 * BM : BM;  // rows of one output tile (one CTA, or the pair)
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = sA + STAGES * L::kA;
    uint8_t* sOut = sB + STAGES * L::kB;
    uint8_t* sSA = sOut + L::kOut;
    uint8_t* sSB = sSA + STAGES * L::kSA;
    uint64_t* full = reinterpret_cast<uint64_t*>(sSB + STAGES * L::kSB);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0u;  // 0: the pair leader (issues the MMAs)
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        for (int b = 0; b < 2; ++b) mbar_init(&tfull[b], 1), mbar_init(&tempty[b], PAIR ? 2 * kEpiWarps : kEpiWarps);
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "r"(L::kCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "r"(L::kCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();  // both CTAs' barriers are initialised before either signals the other's
    fence_after();
    const uint32_t tmem = *tmem_slot;

    const int n_m = (p.M + UM - 1) / UM, n_n = (p.N + BN - 1) / BN;
    const int tiles = n_m * n_n, kblocks = (p.K64 + 3) / 4;
    const int unit0 = PAIR ? int(blockIdx.x >> 1) : int(blockIdx.x);
    const int units = PAIR ? int(gridDim.x >> 1) : int(gridDim.x);

    if (warp == 0 && lane == 0) {
        // ---------------- TMA producer
        int stage = 0;
        uint32_t phase = 0;
        uint32_t issued = 0, last_parity = 0;  // per-stage bit masks for the drain
        for (int tile = unit0; tile < tiles && !*abort_flag; tile += units) {
            const int mb = tile / n_n, nb = tile - mb * n_n;
            for (int kb = 0; kb < kblocks; ++kb) {
                if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag)) break;
                // a pair's copies complete on the leader's barrier, which expects both CTAs' bytes
                if (rank == 0) mbar_expect_tx(&full[stage], uint32_t((PAIR ? 2 : 1) * L::kStage));
                const uint32_t fb = PAIR ? mapa(smem_u32(&full[stage]), 0) : smem_u32(&full[stage]);
                load_2d<PAIR>(sA + stage * L::kA, &tmA, fb, kb * BKB, mb * UM + int(rank) * BM);
                load_2d<PAIR>(sB + stage * L::kB, &tmW, fb, kb * BKB, nb * BN + int(rank) * (BN / 2));
                load_3d<PAIR>(sSA + stage * L::kSA, &tmSA, fb, 0, kb * 2, (mb * UM) / 128 + int(rank));
                load_3d<PAIR>(sSB + stage * L::kSB, &tmSW, fb, 0, kb * 2, nb * BN / 128);  // all of W's, in both CTAs
                issued |= 1u << stage;
                last_parity = (last_parity & ~(1u << stage)) | (phase << stage);
                if (++stage == STAGES) stage = 0, phase ^= 1;
            }
        }
        if (*abort_flag) {  // let every load already issued land before the CTA exits
            if (rank == 0) {
                for (int s = 0; s < STAGES; ++s)
                    if (issued & (1u << s)) mbar_drain(&full[s], (last_parity >> s) & 1);
            } else {  // the peer's loads complete on the leader's barriers: give them time to land
                const uint64_t t0 = now_ns();
                while (now_ns() - t0 < 2000000ull) {
                }
            }
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {
        // ---------------- MMA issuer (the pair's leader issues for both CTAs)
        constexpr uint32_t idesc0 = instr_desc(UM, BN, 0), idesc2 = instr_desc(UM, BN, 2);
        int stage = 0, it = 0;
        uint32_t phase = 0;
        int c = 0;  // stages so far
        bool any = false;
        for (int tile = unit0; tile < tiles; tile += units, ++it) {
            if (*abort_flag) break;
            const int ab = it & 1;
            // the accumulator is free: its own last reader is done, or (overlapping accumulators) the
            // previous tile's epilogue has read the shared columns, after it had read all of the tile before
            if (L::kOverlap) {
                if (it > 0 && !mbar_wait(&tempty[ab ^ 1], uint32_t((it - 1) >> 1) & 1u, abort_flag)) break;
            } else {
                if (!mbar_wait(&tempty[ab], (uint32_t(it >> 1) & 1u) ^ 1u, abort_flag)) break;
            }
            fence_after();
            const uint32_t d = tmem + uint32_t(ab * L::kAcc1);
            // a 64-column tile of W uses half of a tile of 128 rows' scales
            const uint32_t half = BN == 64 ? uint32_t((tile % n_n) & 1) * 2u : 0u;
            bool ok = true;
            for (int kb = 0; kb < kblocks; ++kb, ++c) {
                // the scale buffer's last readers, two stages ago, are done (their commit freed that stage)
                if (c >= 2) {
                    const int u = c - 2;
                    if (!mbar_wait(&empty[u % STAGES], uint32_t(u / STAGES) & 1u, abort_flag)) ok = false;
                }
                if (!ok || !mbar_wait(&full[stage], phase, abort_flag)) {
                    ok = false;
                    break;
                }
                fence_after();
                const int n_mma = min(4, p.K64 - 4 * kb);
                const uint32_t sf = tmem + uint32_t(L::kSf + (c & 1) * L::kSfBuf), sfw = sf + 8;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (2 * j >= n_mma) break;
                    copy_scales<PAIR>(sf + 4 * j, scales_desc(smem_u32(sSA + stage * L::kSA + j * 512)));
#pragma unroll
                    for (int t = 0; t < L::kNTiles; ++t)
                        copy_scales<PAIR>(sfw + 4 * (j * L::kNTiles + t),
                                          scales_desc(smem_u32(sSB + stage * L::kSB + (2 * t + j) * 512)));
                }
                const uint64_t a0 = codes_desc(smem_u32(sA + stage * L::kA));
                const uint64_t b0 = codes_desc(smem_u32(sB + stage * L::kB));
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < n_mma)
                        mma<PAIR>(d, a0 + uint64_t(2 * j), b0 + uint64_t(2 * j), (j & 1) ? idesc2 : idesc0, sf + 4 * (j >> 1),
                                  sfw + 4 * L::kNTiles * (j >> 1) + half, (kb | j) != 0 ? 1u : 0u);
                if (PAIR) mma_commit_pair(&empty[stage]);
                else mma_commit(&empty[stage]);
                any = true;
                if (++stage == STAGES) stage = 0, phase ^= 1;
            }
            if (!ok) break;
            if (PAIR) mma_commit_pair(&tfull[ab]);
            else mma_commit(&tfull[ab]);
        }
        if (any) {  // every MMA and copy issued by this thread completes before the tensor memory is freed
            if (PAIR) mma_commit_pair_local(drain);
            else mma_commit(drain);
            mbar_drain(drain, 0);
        }
    } else if (warp >= 2) {
        // ---------------- epilogue
        const int ew = warp - 2;
        const int lg = warp & 3;   // the lane quarter this warp may access: rows 32 lg .. + 31
        const int half = ew >> 2;  // which half of the chunks
        constexpr int kChunks = BN / 64;  // 32-column chunks per warp
        uint8_t* obuf = sOut + ew * 2 * L::kSub;
        uint32_t n_out = 0;
        const T* bias = static_cast<const T*>(p.bias);
        const T* R = static_cast<const T*>(p.R);
        const uint32_t te0 = PAIR ? mapa(smem_u32(&tempty[0]), 0) : 0u, te1 = PAIR ? mapa(smem_u32(&tempty[1]), 0) : 0u;
        auto release = [&](int ab) {
            fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) mbar_arrive_cluster(ab ? te1 : te0);
                else mbar_arrive(&tempty[ab]);
            }
        };
        // the chunk of the tile that this warp takes as its c-th: with overlapping accumulators the shared
        // columns first (chunks 6 and 7 of the first, 0 and 1 of the second)
        auto chunk_of = [&](int ab, int c) -> int {
            if (!L::kOverlap) return half * kChunks + c;
            if (c == 0) return (ab ? 0 : 6) + half;
            return (ab ? 2 : 0) + half * 3 + c - 1;
        };
        int it = 0;
        for (int tile = unit0; tile < tiles; tile += units, ++it) {
            const int ab = it & 1;
            const int mb = tile / n_n, nb = tile - mb * n_n;
            const int row0 = mb * UM + int(rank) * BM + lg * 32, row = row0 + lane;
            if (!mbar_wait(&tfull[ab], uint32_t(it >> 1) & 1u, abort_flag)) break;
            fence_after();
            const uint32_t taddr = tmem + (uint32_t(lg * 32) << 16) + uint32_t(ab * L::kAcc1);
            uint32_t ra[32], rb[32];
            tmem_ld32_async(taddr + uint32_t(32 * chunk_of(ab, 0)), ra);
            tmem_wait32(ra);
            if (L::kOverlap || kChunks == 1) release(ab);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                uint32_t(&cur)[32] = (c & 1) ? rb : ra;
                uint32_t(&nxt)[32] = (c & 1) ? ra : rb;
                const int col0 = nb * BN + 32 * chunk_of(ab, c);
                if (c + 1 < kChunks) tmem_ld32_async(taddr + uint32_t(32 * chunk_of(ab, c + 1)), nxt);
                float v[32];
                const bool whole = col0 + 32 <= p.N;
                if (bias && whole) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(cur[i]) + to_f<T>(__ldg(bias + col0 + i));
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        v[i] = __uint_as_float(cur[i]) + (bias && col0 + i < p.N ? to_f<T>(bias[col0 + i]) : 0.0f);
                }
                if (EPI == k::kEpiGelu) {
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 g = p.gelu_tanh ? make_float2(gelu(v[i], true), gelu(v[i + 1], true))
                                                     : gelu_as2(make_float2(v[i], v[i + 1]));
                        v[i] = g.x, v[i + 1] = g.y;
                    }
                }
                if (EPI == k::kEpiResidual && row < p.M) {
                    const T* r = R + int64_t(row) * p.ldr + col0;
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            float b[8];
                            Vec<T, 8>::load(r + i, b);
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[i + j] += b[j];
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (col0 + i < p.N) v[i] += to_f<T>(r[i]);
                    }
                }
                if (c + 1 < kChunks) {
                    tmem_wait32(nxt);
                    if (!L::kOverlap && c + 2 == kChunks) release(ab);  // every column is in registers
                }
                if (OUT4) {
                    if (row < p.M && col0 < p.N) {
                        uint32_t top = 0;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            if (!whole && col0 + i >= p.N) v[i] = 0.0f;
                            top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
                        }
                        const uint32_t s = scale_byte(top);
                        const float inv = inv_scale(s);
                        *reinterpret_cast<uint4*>(p.Yc + int64_t(row) * p.ldyc + col0 / 2) =
                            make_uint4(encode8(v, inv), encode8(v + 8, inv), encode8(v + 16, inv), encode8(v + 24, inv));
                        p.Ys[scale_at(row, col0 / 32, p.ktiles_out)] = uint8_t(s);
                    } else if (row < p.M && col0 / 32 < int(4 * p.ktiles_out)) {
                        p.Ys[scale_at(row, col0 / 32, p.ktiles_out)] = 0;  // the last scale tile's blocks past N
                    }
                    // (a 64-column tile that is the first half of the last scale tile: its second half)
                    if (BN == 64 && row < p.M && nb == n_n - 1 && !(nb & 1))
                        p.Ys[scale_at(row, col0 / 32 + 2, p.ktiles_out)] = 0;
                } else if (!whole && (p.N * int(sizeof(T))) % 16 != 0) {
                    // a TMA store writes whole 16-byte pieces: the columns past N belong to the caller
                    if (row < p.M) {
                        T* y = static_cast<T*>(p.Y) + int64_t(row) * p.ldy + col0;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (col0 + i < p.N) y[i] = from_f<T>(v[i]);
                    }
                } else {
                    const uint32_t obi = n_out & 1;
                    if (n_out >= 2 && lane == 0) bulk_wait_read1();  // the store that used this buffer read it
                    __syncwarp();
                    uint8_t* ob = obuf + obi * L::kSub;
                    if constexpr (sizeof(T) == 2) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t o[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[i] = pack_h2(make_float2(v[8 * j + 2 * i], v[8 * j + 2 * i + 1]));
                            *reinterpret_cast<uint4*>(ob + sw64(lane, j)) = make_uint4(o[0], o[1], o[2], o[3]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<float4*>(ob + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                                make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (col0 < p.N && row0 < p.M) tma_store_2d(&tmY, ob, col0, row0);  // (rows past M are clipped)
                        bulk_commit();
                    }
                    ++n_out;
                }
            }
        }
        if (!OUT4 && lane == 0) bulk_wait_all();  // every TMA store has finished before the CTA exits
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();  // no CTA leaves while its peer may still read its shared memory or signal it
    if (warp == 1) {
        fence_after();
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kCols));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kCols));
    }
}

// Codes [rows, bytes] as bytes, box [box_rows, 128 bytes], 128-byte swizzle, zeros out of bounds.
CUtensorMap codes_map(const uint8_t* base, int64_t rows, int64_t bytes, int64_t ld, int box_rows) {
    const cuuint64_t dims[2] = {cuuint64_t(bytes), cuuint64_t(rows)}, strides[1] = {cuuint64_t(ld)};
    const cuuint32_t box[2] = {BKB, cuuint32_t(box_rows)};
    return tc::tensor_map(base, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
// Scale tiles [row tiles, k tiles, 512 bytes] as 32-bit words, box of two k tiles and box_rows row tiles.
CUtensorMap scales_map(const uint8_t* base, int64_t rows, int64_t ktiles, int box_rows) {
    const cuuint64_t dims[3] = {128, cuuint64_t(ktiles), cuuint64_t((rows + 127) / 128)};
    const cuuint64_t strides[2] = {512, cuuint64_t(ktiles) * 512};
    const cuuint32_t box[3] = {128, 2, cuuint32_t(box_rows)};
    return tc::tensor_map(base, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <class T, int BN, bool PAIR, int EPI, bool OUT4> void launch(const GemmArgs<T>& a, cudaStream_t s) {
    using L = Layout<T, BN, PAIR, OUT4>;
    static std::atomic<uint64_t> configured{0};  // per instantiation and device
    once_per_device(configured, [] {
        VB_CUDA(cudaFuncSetAttribute(gemm_mx4_kernel<T, BN, PAIR, EPI, OUT4>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     L::kSmem));
    });
    const int64_t kt = k_tiles(a.K);
    const CUtensorMap ta = codes_map(a.A, a.M, row_bytes(a.K), a.lda, BM);
    const CUtensorMap tw = codes_map(a.W, a.N, row_bytes(a.K), a.ldw, PAIR ? BN / 2 : BN);
    const CUtensorMap tsa = scales_map(a.sA, a.M, kt, 1), tsw = scales_map(a.sW, a.N, kt, L::kNTiles);
    CUtensorMap ty = ta;
    if (!OUT4) {
        const cuuint64_t dims[2] = {cuuint64_t(a.N), cuuint64_t(a.M)}, strides[1] = {cuuint64_t(a.ldy) * sizeof(T)};
        const cuuint32_t box[2] = {32, 32};
        ty = tc::tensor_map(a.Y, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, dims,
                            strides, box, sizeof(T) == 2 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
    }
    const Params p{a.bias, a.R, a.ldr, a.Y, a.ldy, a.Yc, a.ldyc, a.Ys, k_tiles(a.N), int(a.M), int(a.N), int((a.K + 63) / 64),
                   a.gelu_tanh ? 1 : 0};
    constexpr int UM = PAIR ? 2 * BM : BM;
    const int64_t tiles = ((a.M + UM - 1) / UM) * ((a.N + BN - 1) / BN);
    if (tiles > INT32_MAX / 2) fail(kUnsupported, "gemm_mx4: too many output tiles");
    if (!PAIR) {
        const int grid = int(std::min<int64_t>(tiles, device_sm_count()));
        gemm_mx4_kernel<T, BN, PAIR, EPI, OUT4><<<grid, kThreads, L::kSmem, s>>>(ta, tw, tsa, tsw, ty, p);
        VB_LAUNCH();
        return;
    }
    const int pairs = int(std::min<int64_t>(tiles, device_sm_count() / 2));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(2 * pairs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = size_t(L::kSmem);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    VB_CUDA(cudaLaunchKernelEx(&cfg, gemm_mx4_kernel<T, BN, PAIR, EPI, OUT4>, ta, tw, tsa, tsw, ty, p));
    ++launch_counter();
}

template <class T, int EPI, bool OUT4> void dispatch_tile(const GemmArgs<T>& a, cudaStream_t s) {
    auto tiles = [&](int64_t m, int64_t n) { return ((a.M + m - 1) / m) * ((a.N + n - 1) / n); };
    const int64_t sms = device_sm_count();
    // the largest tile that still gives every SM (pair) one
    if (tiles(256, 256) >= sms / 2) launch<T, 256, true, EPI, OUT4>(a, s);
    else if (tiles(128, 128) >= sms) launch<T, 128, false, EPI, OUT4>(a, s);
    else launch<T, 64, false, EPI, OUT4>(a, s);
}

}  // namespace

template <class T> void gemm(const GemmArgs<T>& a, cudaStream_t s) {
    if (a.M <= 0 || a.N <= 0) return;
    if (!a.Yc && a.M <= 8) return gemm_rows(a, s);
    switch (a.epi) {
        case k::kEpiBias:
            if (a.Yc) dispatch_tile<T, k::kEpiBias, true>(a, s);
            else dispatch_tile<T, k::kEpiBias, false>(a, s);
            break;
        case k::kEpiGelu:
            if (a.Yc) dispatch_tile<T, k::kEpiGelu, true>(a, s);
            else dispatch_tile<T, k::kEpiGelu, false>(a, s);
            break;
        case k::kEpiResidual:
            if (a.Yc) fail(kInvalidArgument, "gemm_mx4: no residual with 4-bit output");
            dispatch_tile<T, k::kEpiResidual, false>(a, s);
            break;
        default: fail(kInvalidArgument, "gemm_mx4: unknown epilogue");
    }
}

template void gemm<float>(const GemmArgs<float>&, cudaStream_t);
template void gemm<__half>(const GemmArgs<__half>&, cudaStream_t);

int take_error() {
    VB_CUDA(cudaDeviceSynchronize());
    int e = 0, zero = 0;
    VB_CUDA(cudaMemcpyFromSymbol(&e, g_error, sizeof(int)));
    if (e) VB_CUDA(cudaMemcpyToSymbol(g_error, &zero, sizeof(int)));
    return e;
}

}  // namespace vb::mx4
