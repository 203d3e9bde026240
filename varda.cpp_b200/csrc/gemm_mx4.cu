// The 4-bit product on the tensor cores (see gemm_mx4.cuh): tcgen05.mma kind::mxf4 with block scales, which
// multiplies 64 e2m1 values of a row and column at a time, each block of 32 with its two scales, into fp32.
//
// Persistent and warp-specialised: one 768-thread CTA per SM, or clusters of two with cta_group::2 computing
// 256 x 256 tiles together (each CTA loads its 128 rows of A and half of the W tile).
//   warp 0              TMA producer: codes of A [128 x 128 bytes = 256 columns of K] and of W, 128-byte
//                       swizzle, into a ring of kStages.
//   warp 2              TMA producer of their scale tiles (512 bytes per 128 rows and 128 columns, stored in
//                       the order in which tensor memory holds them) into a ring of kSlots.
//   warps 4-7           scales from shared into tensor memory, each warp its lane quarter's copy, into the buffer
//                       of the stage (as many as stages). (tcgen05.cp does the same from the MMA thread, but
//                       the tensor pipe runs it between the MMAs, some 57 cycles for 512 bytes: [189809 x 4096] x
//                       [4096 x 1024] took 470 us with it, 365 with these warps.)
//   warp 1              MMA issuer: four MMAs of K = 64 per stage; in a last stage that K cuts, only those it needs.
//                       (These three warps run their loops whole and issue through one elected lane: the operands
//                       are then uniform values. 3-5% on the long sums against one lane in a branch.)
//   warps 8-23          epilogue: a warp takes 32 rows and a quarter of the tile's columns into registers at
//                       once and hands the accumulator back, then bias / GELU / residual in fp32, one rounding
//                       and a TMA store from swizzled shared memory (the residual came by TMA into the same
//                       buffer meanwhile); or 4-bit output: a lane holds whole blocks of its row, so a
//                       block's scale is the maximum of the lane's registers.
// Tensor memory at BN = 256: two accumulators would fill all 512 columns, but the scales need some. So the
// second accumulator starts at column 128, over half of the first; since the epilogue reads all columns
// at once, the next tile's MMAs start some 1300 cycles after the last one's end.
//
// What bounds it, on [189809 x K] x [K x 4096] to fp16: at K = 64 the epilogue alone, 264 us with a bias (5.9 TB/s of
// output), 410 with GELU (its arithmetic), and 446 with GELU and 4-bit output. At K = 1024, where the MMAs take some 240 by
// themselves, 437, 539 and 540 to 575: the two do not overlap whole, as a tile's MMAs wait for the accumulator that they
// share with the tile before, and the epilogue's warps, all in step, for the MMAs (issue slots 40 to 62% used, the tensor
// pipe 33 to 43%; neither bounds it). Long sums: [189809 x 4096] x [4096 x 1024] + residual 369 us = 4320 TFLOP/s (tensor
// pipe 55%; the loads alone take 320 us, some 10 TB/s from L2). Run for seconds all of them are held by the 1 kW power limit
// (1.4 GHz: 445 us). Tried and dropped: 192-column tiles with two whole accumulators and two sets of epilogue warps (514 us
// with a bias), the same with A's rows kept in shared memory (533), plain stores instead of TMA stores (517).
//
// Every wait is bounded: when one runs out a CTA sets the device error flag, stops issuing, waits for its own copies and
// MMAs in flight, frees its tensor memory and returns. Each lane of a warp waits for itself, and the barrier may complete
// or the time run out between two lanes' looks; so no lane leaves a loop by its own answer. Lanes that gave up take part in
// the warp's instructions (tensor memory read or written in vain), and the warp votes where it has to meet anyway, before
// anything is handed on ([189809 x 256] x [256 x 4096] 276 us, as with lanes that left by themselves; with a vote at each
// wait 284; the votes left cost [189809 x 4096] x [4096 x 1024] + residual 2%).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstdlib>
#include <mutex>
#include <string>

#include "common.h"
#include "dev.cuh"
#include "gelu.cuh"
#include "gemm_mx4.cuh"
#include "gemm_tc.cuh"
#include "ptx.cuh"

namespace vb::mx4 {

namespace {

using namespace vb::d;
using namespace vb::ptx;

constexpr int BM = 128, BKB = 128;  // rows of a CTA's tile; bytes of codes per row and stage (256 columns)
constexpr int kEpiWarps = 16, kEpiWarp0 = 8, kThreads = 32 * (kEpiWarp0 + kEpiWarps);
// registers: the first two warpgroups give back to the epilogue's four (2 x 48 + 4 x 96 <= 6 x the 80 of the launch)
constexpr int kLaunchRegs = 80, kFewRegs = 48, kEpiRegs = 96;
static_assert(2 * kFewRegs + 4 * kEpiRegs <= 6 * kLaunchRegs, "register split over what the CTA is launched with");
constexpr unsigned long long kTimeoutNs = 4000000000ull;  // 4 s

__device__ int g_error = 0;

struct Params {
    const void* bias;
    void* Y;
    int64_t ldy;
    uint8_t* Yc;
    int64_t ldyc;
    uint8_t* Ys;
    int64_t ktiles_out;
    int M, N, K64;  // K64: MMAs along K, ceil(K / 64)
    int gelu_tanh;
    unsigned long long wait_ns;  // limit of each wait
    int withhold;                // test hook: block 0 never loads its first stage
};

// Bounded wait; false if this lane gave up. CL: the barrier also takes arrivals of the pair's other CTA.
template <bool CL = false>
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, volatile int* abort_flag, unsigned long long limit_ns) {
    auto test = [&] { return CL ? mbar_test_cl(b, parity) : mbar_test(b, parity); };
    if (test()) return true;
    const uint64_t t0 = now_ns();
    for (;;) {
        if (test()) return true;
        if (*abort_flag) return false;
        if (now_ns() - t0 > limit_ns) {
            *abort_flag = 1;
            atomicExch(&g_error, 1);
            return false;
        }
    }
}
// The warp's vote, and a __syncwarp (which orders its memory accesses; the vote alone does not).
__device__ __forceinline__ bool whole_warp(bool ok) {
    ok = __all_sync(kFull, ok);
    __syncwarp();
    return ok;
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

// After an abort: time for the loads already issued to land before the CTA exits (their barriers may also wait
// for arrivals that will not come, or belong to the pair's other CTA).
__device__ __forceinline__ void settle() {
    const uint64_t t0 = now_ns();
    while (now_ns() - t0 < 2000000ull) {
    }
}

template <bool PAIR>
__device__ __forceinline__ void load_codes(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
    if (PAIR) tma_load_2d_pair(dst, map, mapa(smem_u32(bar), 0), x, y);  // completes on the leader's barrier
    else tma_load_2d(dst, map, bar, x, y);
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// Arrival on a barrier of the pair that tells of tensor memory read or written, and of nothing else: the order that the PTX
// ISA gives in "tcgen05 memory consistency model", canonical synchronisation patterns, for an instruction and another
// thread that needs its end: tcgen05.ld or st, tcgen05.wait, tcgen05.fence::before_thread_sync,
// mbarrier.arrive.relaxed.cluster; there mbarrier.try_wait at cluster scope, tcgen05.fence::after_thread_sync,
// tcgen05.mma (the fence orders what came before it with the arrival, an execution ordering instruction). A release at
// cluster scope would also wait for the thread's other writes: 766 us instead of 445 on [189809 x 1024] x [1024 x 4096].
__device__ __forceinline__ void mbar_arrive_peer(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// Shared-memory descriptor of the codes: K-major, 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t codes_desc(uint32_t saddr) {
    return uint64_t((saddr & 0x3FFFF) >> 4) | uint64_t(1) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
// Instruction descriptor of kind::mxf4: A = B = e2m1 (1), scales ue8m0, K-major, K = 64; sf: which two of a
// 32-bit column's four scale bytes (0 or 2).
__host__ __device__ constexpr uint32_t instr_desc(int m, int n, int sf) {
    return uint32_t(sf) << 4 | 1u << 7 | 1u << 10 | uint32_t(n >> 3) << 17 | 1u << 23 | uint32_t(m >> 7) << 27 | uint32_t(sf) << 29;
}
// Scales into tensor memory: this lane's 16 bytes of a tile (rows lane + 32 i in column i) at column taddr.
__device__ __forceinline__ void st_scales(uint32_t taddr, uint4 v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(v.x), "r"(v.y), "r"(v.z),
                 "r"(v.w)
                 : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read0() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

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
    static constexpr int kSlots = 6;
    static constexpr int kCW = BN / 4 > 32 ? BN / 4 : 32;  // columns per epilogue warp
    static constexpr int kGroups = BN / kCW;                // epilogue warps per 32 rows
    // output staging: sub-tiles of 32 rows x kSW columns, one buffer per warp
    static constexpr int kSW = sizeof(T) == 4 ? 32 : kCW;
    static constexpr int kSub = 32 * kSW * int(sizeof(T));
    static constexpr int kOut = OUT4 ? 0 : kEpiWarps * kSub;
    static constexpr int kBias = kEpiWarps * kCW * 4;  // each epilogue warp's columns of the bias, fp32
    static constexpr int kFixed = 1024 + kOut + kSlots * (kSA + kSB) + kBias + 640;  // alignment slack, ..., barriers
    // tensor memory columns: accumulators at 0 and kAcc1, then per stage two halves of K = 128, each with A's
    // scales and W's
    static constexpr bool kOverlap = BN == 256;
    static constexpr int kAcc1 = kOverlap ? 128 : BN, kSf = kAcc1 + BN, kSfHalf = 4 + 4 * kNTiles, kSfBuf = 2 * kSfHalf;
    static constexpr int kFit = (232448 - kFixed) / (kA + kB), kFitT = (512 - kSf) / kSfBuf;
    static constexpr int kStages = kFit < kFitT ? (kFit < 8 ? kFit : 8) : (kFitT < 8 ? kFitT : 8);
    static constexpr int kSmem = kFixed + kStages * (kA + kB);
    static_assert(kStages >= 3, "shared memory over the 227 KB per-CTA limit");
    static constexpr int kCols = kSf + kStages * kSfBuf <= 256 ? 256 : 512;
    static_assert(kSf + kStages * kSfBuf <= kCols, "tensor memory over 512 columns");
    static constexpr int kBarriers = 2 * kStages + 2 * kSlots + 2 + 2 + 1 + kEpiWarps;
    static_assert(kBarriers * 8 + 16 <= 640, "barrier area");
};

template <class T, int BN, bool PAIR, int EPI, bool OUT4>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_mx4_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSW,
                    const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmR, Params p) {
    using L = Layout<T, BN, PAIR, OUT4>;
    constexpr int STAGES = L::kStages, SLOTS = L::kSlots;
    constexpr int UM = PAIR ? 2 * BM : BM;  // rows of one output tile (one CTA, or the pair)
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = sA + STAGES * L::kA;
    uint8_t* sOut = sB + STAGES * L::kB;
    uint8_t* sSc = sOut + L::kOut;
    float* sBias = reinterpret_cast<float*>(sSc + SLOTS * (L::kSA + L::kSB));
    // full: a stage's codes are in shared memory and its scales in tensor memory (the leader's, for both CTAs)
    uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sBias) + L::kBias);
    uint64_t* empty = full + STAGES;
    uint64_t* sfull = empty + STAGES;   // scale slots, in shared memory
    uint64_t* sempty = sfull + SLOTS;
    uint64_t* tfull = sempty + SLOTS;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint64_t* rfull = drain + 1;  // per epilogue warp: its residual sub-tile
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(rfull + kEpiWarps);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0u;  // 0: the pair leader (issues the MMAs)
    if (threadIdx.x == 0) {
        constexpr uint32_t ctas = PAIR ? 2 : 1;
        for (int s = 0; s < STAGES; ++s) mbar_init(&full[s], 1 + 4 * ctas), mbar_init(&empty[s], 1);
        for (int s = 0; s < SLOTS; ++s) mbar_init(&sfull[s], 1), mbar_init(&sempty[s], 4);
        for (int b = 0; b < 2; ++b) mbar_init(&tfull[b], 1), mbar_init(&tempty[b], 4 * L::kGroups * ctas);
        mbar_init(drain, 1);
        for (int w = 0; w < kEpiWarps; ++w) mbar_init(&rfull[w], 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 3) {
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

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
        if (warp == 0) {
            // ---------------- TMA producer of the codes
            const bool leader = elect_one();
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true, withhold = p.withhold && blockIdx.x == 0;
            for (int tile = unit0; ok && tile < tiles; tile += units) {
                const int mb = tile / n_n, nb = tile - mb * n_n;
                for (int kb = 0; kb < kblocks; ++kb) {
                    ok = mbar_wait(&empty[stage], phase ^ 1, abort_flag, p.wait_ns);
                    if (leader && ok && !withhold) {
                        if (rank == 0) mbar_expect_tx(&full[stage], uint32_t((PAIR ? 2 : 1) * (L::kA + L::kB)));
                        load_codes<PAIR>(sA + stage * L::kA, &tmA, &full[stage], kb * BKB, mb * UM + int(rank) * BM);
                        load_codes<PAIR>(sB + stage * L::kB, &tmW, &full[stage], kb * BKB, nb * BN + int(rank) * (BN / 2));
                    }
                    ok = whole_warp(ok);
                    if (!ok) break;
                    withhold = false;
                    if (++stage == STAGES) stage = 0, phase ^= 1;
                }
            }
        } else if (warp == 2) {
            // ---------------- TMA producer of the scales (all of the W tile's, in both CTAs of a pair)
            const bool leader = elect_one();
            int slot = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = unit0; ok && tile < tiles; tile += units) {
                const int mb = tile / n_n, nb = tile - mb * n_n;
                for (int kb = 0; kb < kblocks; ++kb) {
                    ok = mbar_wait(&sempty[slot], phase ^ 1, abort_flag, p.wait_ns);
                    if (leader && ok) {
                        mbar_expect_tx(&sfull[slot], uint32_t(L::kSA + L::kSB));
                        uint8_t* d = sSc + slot * (L::kSA + L::kSB);
                        tma_load_3d(d, &tmSA, &sfull[slot], 0, kb * 2, (mb * UM) / 128 + int(rank));
                        tma_load_3d(d + L::kSA, &tmSW, &sfull[slot], 0, kb * 2, nb * BN / 128);
                    }
                    ok = whole_warp(ok);
                    if (!ok) break;
                    if (++slot == SLOTS) slot = 0, phase ^= 1;
                }
            }
        } else if (warp == 1 && rank == 0) {
            // ---------------- MMA issuer (the pair's leader issues for both CTAs). The whole warp runs the loop and one
            // lane issues, so that descriptors and addresses are uniform values
            const bool leader = elect_one();
            constexpr uint32_t idesc0 = instr_desc(UM, BN, 0), idesc2 = instr_desc(UM, BN, 2);
            int stage = 0, it = 0;
            uint32_t phase = 0;
            bool any = false, ok = true;
            for (int tile = unit0; ok && tile < tiles; tile += units, ++it) {
                const int ab = it & 1;
                // the accumulator has been read: its own last tile's, or (overlapping accumulators) the
                // previous tile's, whose readers were done with the tile before
                if (!L::kOverlap) ok = mbar_wait<PAIR>(&tempty[ab], (uint32_t(it >> 1) & 1u) ^ 1u, abort_flag, p.wait_ns);
                else if (it > 0) ok = mbar_wait<PAIR>(&tempty[ab ^ 1], uint32_t((it - 1) >> 1) & 1u, abort_flag, p.wait_ns);
                fence_after();
                const uint32_t d = tmem + uint32_t(ab * L::kAcc1);
                // a 64-column tile of W uses half of a tile of 128 rows' scales
                const uint32_t half = BN == 64 ? uint32_t((tile % n_n) & 1) * 2u : 0u;
                for (int kb = 0; kb < kblocks; ++kb) {
                    ok = ok && mbar_wait<PAIR>(&full[stage], phase, abort_flag, p.wait_ns);
                    fence_after();
                    const int n_mma = min(4, p.K64 - 4 * kb);
                    const uint64_t a0 = codes_desc(smem_u32(sA + stage * L::kA));
                    const uint64_t b0 = codes_desc(smem_u32(sB + stage * L::kB));
                    const uint32_t sf = tmem + uint32_t(L::kSf + stage * L::kSfBuf);
                    if (leader && ok) {
                        any = true;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t sa = sf + uint32_t((j >> 1) * L::kSfHalf);
                            if (j < n_mma)
                                mma<PAIR>(d, a0 + uint64_t(2 * j), b0 + uint64_t(2 * j), (j & 1) ? idesc2 : idesc0, sa, sa + 4 + half,
                                          (kb | j) != 0 ? 1u : 0u);
                        }
                        if (PAIR) mma_commit_pair(&empty[stage]);
                        else mma_commit(&empty[stage]);
                    }
                    ok = whole_warp(ok);
                    if (!ok) break;
                    if (++stage == STAGES) stage = 0, phase ^= 1;
                }
                if (leader && ok) {
                    if (PAIR) mma_commit_pair(&tfull[ab]);
                    else mma_commit(&tfull[ab]);
                }
                __syncwarp();
            }
            if (any) {  // every MMA issued by this thread (the leader) completes before the tensor memory is freed
                if (PAIR) mma_commit_pair_local(drain);
                else mma_commit(drain);
                mbar_drain(drain, 0);
            }
        }
    } else if (warp < kEpiWarp0) {
        // ---------------- scales: shared memory -> this warp's lane quarter of tensor memory
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
        const uint32_t tq = tmem + (uint32_t((warp & 3) * 32) << 16) + uint32_t(L::kSf);
        int slot = 0, stage = 0;
        uint32_t sphase = 0, phase = 0;
        bool ok = true;
        for (int tile = unit0; ok && tile < tiles; tile += units) {
            for (int kb = 0; kb < kblocks; ++kb) {
                ok = mbar_wait(&sfull[slot], sphase, abort_flag, p.wait_ns);
                // both halves (a cut last stage's second half may hold no columns of K: it is then not used)
                const uint8_t* src = sSc + slot * (L::kSA + L::kSB) + lane * 16;
                uint4 v[2][1 + L::kNTiles];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    v[j][0] = *reinterpret_cast<const uint4*>(src + j * 512);
#pragma unroll
                    for (int t = 0; t < L::kNTiles; ++t) v[j][1 + t] = *reinterpret_cast<const uint4*>(src + L::kSA + (2 * t + j) * 512);
                }
                // the MMAs that read this buffer are done
                ok = ok && mbar_wait(&empty[stage], phase ^ 1, abort_flag, p.wait_ns);
                fence_after();
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int t = 0; t <= L::kNTiles; ++t)
                        st_scales(tq + uint32_t(stage * L::kSfBuf + j * L::kSfHalf + 4 * t), v[j][t]);
                wait_st();
                fence_before();
                ok = whole_warp(ok);
                if (!ok) break;
                if (lane == 0) {
                    if (PAIR) mbar_arrive_peer(mapa(smem_u32(&full[stage]), 0));
                    else mbar_arrive(&full[stage]);
                    mbar_arrive(&sempty[slot]);
                }
                if (++slot == SLOTS) slot = 0, sphase ^= 1;
                if (++stage == STAGES) stage = 0, phase ^= 1;
            }
        }
    } else {
        // ---------------- epilogue
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
        const int ew = warp - kEpiWarp0;
        const int lg = warp & 3;  // the lane quarter this warp may access: rows 32 lg .. + 31
        const int grp = ew >> 2;  // its columns: grp kCW .. + kCW - 1
        uint8_t* ob = sOut + ew * L::kSub;
        float* wb = sBias + ew * L::kCW;
        uint64_t* rbar = &rfull[ew];
        uint32_t rphase = 0;
        const T* bias = static_cast<const T*>(p.bias);
        const uint32_t te0 = PAIR ? mapa(smem_u32(&tempty[0]), 0) : 0u, te1 = PAIR ? mapa(smem_u32(&tempty[1]), 0) : 0u;
        // 16-byte chunk j of row r of a staged sub-tile, swizzled as the tensor map has it
        auto chunk_at = [&](int r, int j) -> uint8_t* {
            return ob + (L::kSW * sizeof(T) == 128 ? r * 128 + ((j ^ (r & 7)) << 4) : sw64(r, j));
        };
        // one lane: the residual sub-tile into the staging buffer, once the store before has read that
        auto load_residual = [&](int col0, int row0) {
            bulk_wait_read0();
            mbar_expect_tx(rbar, uint32_t(L::kSub));
            tma_load_2d(ob, &tmR, rbar, col0, row0);
        };
        int it = 0;
        for (int tile = unit0; grp < L::kGroups && tile < tiles; tile += units, ++it) {
            const int ab = it & 1;
            const int mb = tile / n_n, nb = tile - mb * n_n;
            const int row0 = mb * UM + int(rank) * BM + lg * 32, row = row0 + lane;
            const int colw = nb * BN + grp * L::kCW;
            __syncwarp();  // every lane is done with the tile before's buffers
            if (EPI == k::kEpiResidual && lane == 0) load_residual(colw, row0);
#pragma unroll
            for (int i = lane; i < L::kCW; i += 32) wb[i] = bias && colw + i < p.N ? to_f<T>(__ldg(bias + colw + i)) : 0.0f;
            __syncwarp();
            const bool ok = mbar_wait(&tfull[ab], uint32_t(it >> 1) & 1u, abort_flag, p.wait_ns);
            fence_after();
            const uint32_t taddr = tmem + (uint32_t(lg * 32) << 16) + uint32_t(ab * L::kAcc1 + grp * L::kCW);
            uint32_t acc[L::kCW / 32][32];
#pragma unroll
            for (int c = 0; c < L::kCW / 32; ++c) tmem_ld32_async(taddr + uint32_t(32 * c), acc[c]);
#pragma unroll
            for (int c = 0; c < L::kCW / 32; ++c) tmem_wait32(acc[c]);
            fence_before();
            if (!whole_warp(ok)) {
                if (EPI == k::kEpiResidual && lane == 0) mbar_drain(rbar, rphase);
                break;
            }
            if (lane == 0) {
                if (PAIR) mbar_arrive_peer(ab ? te1 : te0);
                else mbar_arrive(&tempty[ab]);
            }
            uint32_t scales = 0;  // OUT4: the scale bytes of the warp's columns
#pragma unroll
            for (int c = 0; c < L::kCW / 32; ++c) {
                const int col0 = colw + 32 * c;
                const bool whole = col0 + 32 <= p.N;
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float4 b = *reinterpret_cast<const float4*>(wb + 32 * c + i);
                    const float2 s0 = __fadd2_rn(make_float2(__uint_as_float(acc[c][i]), __uint_as_float(acc[c][i + 1])), make_float2(b.x, b.y));
                    const float2 s1 = __fadd2_rn(make_float2(__uint_as_float(acc[c][i + 2]), __uint_as_float(acc[c][i + 3])), make_float2(b.z, b.w));
                    v[i] = s0.x, v[i + 1] = s0.y, v[i + 2] = s1.x, v[i + 3] = s1.y;
                }
                if (EPI == k::kEpiGelu) {
                    if (p.gelu_tanh) {
#pragma unroll 1
                        for (int i = 0; i < 32; ++i) {
                            // (a rotation, so that the registers are not indexed and the code stays small)
                            const float g = gelu(v[0], true);
#pragma unroll
                            for (int j = 0; j < 31; ++j) v[j] = v[j + 1];
                            v[31] = g;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 g = gelu2<kFineGelu<T> && !OUT4>(make_float2(v[i], v[i + 1]));
                            v[i] = g.x, v[i + 1] = g.y;
                        }
                    }
                }
                if constexpr (OUT4) {
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (col0 + i >= p.N) v[i] = 0.0f;
                    }
                    float top = 0.0f;  // NaN if one is
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(fabsf(v[i])), "f"(fabsf(v[i + 1])));
                    const uint32_t s = scale_byte(__float_as_uint(top) & 0x7fffffffu);
                    const float inv = inv_scale(s);
                    scales |= s << (8 * c);
                    if (row < p.M && col0 < p.N)
                        *reinterpret_cast<uint4*>(p.Yc + int64_t(row) * p.ldyc + col0 / 2) =
                            make_uint4(encode8(v, inv), encode8(v + 8, inv), encode8(v + 16, inv), encode8(v + 24, inv));
                } else {
                    constexpr int kChunks = 32 * int(sizeof(T)) / 16;  // 16-byte chunks of the 32 columns
                    constexpr int kVals = 16 / int(sizeof(T));
                    const int j0 = L::kSW == 64 ? 4 * c : 0;
                    if (EPI == k::kEpiResidual) {
                        if (L::kSW == 32 && c > 0) {  // a second sub-tile through the same buffer
                            __syncwarp();
                            if (lane == 0) load_residual(col0, row0);
                        }
                        if (L::kSW == 32 || c == 0) {
                            if (!mbar_wait(rbar, rphase, abort_flag, p.wait_ns)) mbar_drain(rbar, rphase);  // (it is on its way)
                            rphase ^= 1;
                        }
#pragma unroll
                        for (int j = 0; j < kChunks; ++j) {
                            float r[kVals];
                            Vec<T, kVals>::load(reinterpret_cast<const T*>(chunk_at(lane, j0 + j)), r);
#pragma unroll
                            for (int i = 0; i < kVals; ++i) v[kVals * j + i] += r[i];
                        }
                    } else if (L::kSW == 32 || c == 0) {
                        if (lane == 0) bulk_wait_read0();  // the store before has read the buffer
                        __syncwarp();
                    }
                    // a TMA store writes whole 16-byte pieces: a row's columns past N belong to the caller
                    const bool ragged = colw + L::kCW > p.N && (p.N * int(sizeof(T))) % 16 != 0;
                    if (ragged) {
                        if (row < p.M) {
                            T* y = static_cast<T*>(p.Y) + int64_t(row) * p.ldy + col0;
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (col0 + i < p.N) y[i] = from_f<T>(v[i]);
                        }
                        continue;
                    }
#pragma unroll
                    for (int j = 0; j < kChunks; ++j) {
                        uint4 o;
                        if constexpr (sizeof(T) == 2)
                            o = make_uint4(pack_h2(make_float2(v[8 * j], v[8 * j + 1])), pack_h2(make_float2(v[8 * j + 2], v[8 * j + 3])),
                                           pack_h2(make_float2(v[8 * j + 4], v[8 * j + 5])), pack_h2(make_float2(v[8 * j + 6], v[8 * j + 7])));
                        else
                            o = make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]),
                                           __float_as_uint(v[4 * j + 3]));
                        *reinterpret_cast<uint4*>(chunk_at(lane, j0 + j)) = o;
                    }
                    if (L::kSW == 32 || c + 1 == L::kCW / 32) {
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            const int cs = L::kSW == 32 ? col0 : colw;
                            if (cs < p.N && row0 < p.M) tma_store_2d(&tmY, ob, cs, row0);  // (past M and N: clipped)
                            bulk_commit();
                        }
                    }
                }
            }
            if constexpr (OUT4) {
                // the blocks' scale bytes; 0 for the last scale tile's blocks past N
                const int b0 = colw / 32;
                if (row < p.M && b0 < int(4 * p.ktiles_out)) {
                    uint8_t* d = p.Ys + scale_at(row, b0, p.ktiles_out);
                    if (L::kCW == 64) *reinterpret_cast<uint16_t*>(d) = uint16_t(scales);
                    else *d = uint8_t(scales);
                    // (a 64-column tile that is the first half of the last scale tile: its second half)
                    if (BN == 64 && nb == n_n - 1 && !(nb & 1)) d[2] = 0;
                }
            }
        }
        if (!OUT4 && lane == 0) bulk_wait_all();  // every TMA store has finished before the CTA exits
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    if (*abort_flag) settle();  // (every thread, once no warp issues any more)
    if (PAIR) cluster_sync();  // no CTA leaves while its peer may still read its shared memory or signal it
    if (warp == 3) {
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

// Rows of the output or residual, box [32, width], 128 or 64 bytes wide and swizzled so.
template <class T> CUtensorMap rows_map(const T* base, int64_t rows, int64_t cols, int64_t ld, int width) {
    const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)}, strides[1] = {cuuint64_t(ld) * sizeof(T)};
    const cuuint32_t box[2] = {cuuint32_t(width), 32};
    return tc::tensor_map(base, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, dims,
                          strides, box, width * sizeof(T) == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

template <class T, int BN, bool PAIR, int EPI, bool OUT4> void launch(const GemmArgs<T>& a, cudaStream_t s) {
    using L = Layout<T, BN, PAIR, OUT4>;
    static std::atomic<uint64_t> configured{0};  // per instantiation and device
    once_per_device(configured, [] {
        auto* kernel = &gemm_mx4_kernel<T, BN, PAIR, EPI, OUT4>;
        VB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem));
        // the epilogue's registers come out of what the CTA is launched with
        cudaFuncAttributes f{};
        VB_CUDA(cudaFuncGetAttributes(&f, kernel));
        if (f.numRegs < kLaunchRegs) fail(kInternal, "gemm_mx4: built with fewer registers per thread than it splits");
    });
    const int64_t kt = k_tiles(a.K);
    const CUtensorMap ta = codes_map(a.A, a.M, row_bytes(a.K), a.lda, BM);
    const CUtensorMap tw = codes_map(a.W, a.N, row_bytes(a.K), a.ldw, PAIR ? BN / 2 : BN);
    const CUtensorMap tsa = scales_map(a.sA, a.M, kt, 1), tsw = scales_map(a.sW, a.N, kt, L::kNTiles);
    CUtensorMap ty = ta, tr = ta;
    if (!OUT4) {
        ty = rows_map(a.Y, a.M, a.N, a.ldy, L::kSW);
        if (EPI == k::kEpiResidual) tr = rows_map(a.R, a.M, a.N, a.ldr, L::kSW);
    }
    // failure-path test hooks (host side, no fault): VB_DEBUG_WAIT_NS shortens every wait's limit and
    // VB_DEBUG_MX4_WITHHOLD=1 makes block 0 skip its first stage's codes, so that the waits on them run out
    const char* wn = std::getenv("VB_DEBUG_WAIT_NS");
    const char* wh = std::getenv("VB_DEBUG_MX4_WITHHOLD");
    const Params p{a.bias, a.Y, a.ldy, a.Yc, a.ldyc, a.Ys, k_tiles(a.N), int(a.M), int(a.N), int((a.K + 63) / 64),
                   a.gelu_tanh ? 1 : 0, wn && *wn ? std::strtoull(wn, nullptr, 10) : kTimeoutNs, wh && *wh && std::atoi(wh) != 0};
    constexpr int UM = PAIR ? 2 * BM : BM;
    const int64_t tiles = ((a.M + UM - 1) / UM) * ((a.N + BN - 1) / BN);
    if (tiles > INT32_MAX / 2) fail(kUnsupported, "gemm_mx4: too many output tiles");
    if (!PAIR) {
        const int grid = int(std::min<int64_t>(tiles, device_sm_count()));
        gemm_mx4_kernel<T, BN, PAIR, EPI, OUT4><<<grid, kThreads, L::kSmem, s>>>(ta, tw, tsa, tsw, ty, tr, p);
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
    VB_CUDA(cudaLaunchKernelEx(&cfg, gemm_mx4_kernel<T, BN, PAIR, EPI, OUT4>, ta, tw, tsa, tsw, ty, tr, p));
    ++launch_counter();
}

template <class T, int EPI, bool OUT4> void dispatch_tile(const GemmArgs<T>& a, cudaStream_t s) {
    auto tiles = [&](int64_t m, int64_t n) { return ((a.M + m - 1) / m) * ((a.N + n - 1) / n); };
    const int64_t sms = device_sm_count();
    // 64 columns where that gives an SM no second tile ([5000 x 512] x [512 x 256]: 5.3 us, with 128 columns 4.9 where it
    // does, at 700 rows 4.4 against 4.9). The pairs' 256 columns once they have several each, sooner for long sums, whose
    // loads they halve ([20000 x 512] x [512 x 1024], 4 each: 14.5 against 12.6; [100000 x 512] x [512 x 2048], 42: 87
    // against 92; [60000 x 2048] x [2048 x 512] with GELU, 6: 40 against 44), but not for fp32 output after short ones, which the
    // stores bound ([100000 x 512] x [512 x 2048]: 174 against 139)
    const bool stores = sizeof(T) == 4 && !OUT4 && a.K <= 512;
    if (tiles(128, 64) <= sms) launch<T, 64, false, EPI, OUT4>(a, s);
    else if (a.N > 128 && !stores && tiles(256, 256) >= (a.K > 1024 ? 4 : 8) * (sms / 2)) launch<T, 256, true, EPI, OUT4>(a, s);
    else launch<T, 128, false, EPI, OUT4>(a, s);
}

}  // namespace

template <class T> void gemm(const GemmArgs<T>& a, cudaStream_t s) {
    if (a.M <= 0 || a.N <= 0) return;
    // one or two rows, or up to four with a long sum that the tensor cores would form in one CTA per 64 columns ([4 x 4096] x
    // [4096 x 1024]: 4.7 against 7.3 us, [2 x 1024] x [1024 x 4096]: 3.4 against 4.7; [4 x 1024]: 4.5 against 4.7)
    if (!a.Yc && (a.M <= 2 || (a.M <= kFewRows && a.K > 2048 && a.M * a.N <= 4096))) return gemm_rows(a, s);
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
