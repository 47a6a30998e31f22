/*
 * Grouped matrix products on the tensor cores (tcgen05), fed by TMA.
 *
 * A tile of the result is 128 lanes per CTA x up to kColumns columns of fp32 (int32)
 * sums in tensor memory.  The DENSE matrix lies along the lanes and the ragged rows
 * along the columns: N of tcgen05.mma is any multiple of 16, so a group of 5 rows
 * costs an MMA of 16 columns and not one of 128 rows, and the same kernel serves a
 * decoding batch, where all time goes into reading weights, and a training batch.
 * For the weight gradient both operands are read with their summed index, the rows,
 * along the outer dimension (MN-major), and the last rows of a group, which share a
 * block with the next group's, are cut off in shared memory.
 *
 * Wide tiles (256 columns) are computed by a pair of CTAs on neighbouring SMs, 256 x
 * 256 results: each holds 128 rows of the dense matrix and half of the ragged rows,
 * and one MMA reads both.  A single CTA would have to load 48 KB for 512 cycles of
 * MMA, more than the 49 to 63 bytes per cycle that an SM was measured to get with all
 * of them loading; the pair loads 32 KB each.  A block of a pair then takes 572 cycles, 560
 * with the loads left out and 523 with the MMAs left out: what bounds it are the MMAs, at
 * the clock that the power limit leaves (1.1 GHz without a pause, 1.65 without the loads).
 * One group of 18944 rows, 1024 x 8192: 217 us in a short run, 1470 TFLOP/s, and 264 us,
 * 1200 TFLOP/s, without a pause; 8192 rows of 16 groups, 2048 x 4096, without a pause: 146 us.
 *
 * CTAs are persistent: warp 0 loads blocks of 128 bytes of the summed index into a
 * ring of stages, one lane of warp 1 issues the MMAs, warps from 4 on read the
 * finished sums and write results while the next tile computes in the other half of
 * tensor memory.  Warp 3 works out the next tiles ahead of all of them, and warp 2
 * cuts the ends of groups off; done by the MMA warp itself either left the tensor
 * cores idle for 600 cycles per tile.
 *
 * Tiles that do not fill a wave are split along the summed index
 * (grouped_schedule.cuh): each CTA leaves its sums in the buffer, and for each piece
 * of the tile, 32 lanes x 16 columns, the warp that arrives last adds them in the
 * parts' order, so that the result does not depend on who that is.  Parts go through
 * the pieces from different ones on: arriving together, each is the last one for some,
 * and the adding is shared (512 x 512 from 16384 rows: 24 us; 62 us with one CTA adding
 * a whole tile).
 *
 * Operands whose rows do not start on multiples of 16 bytes (odd widths) cannot be
 * loaded by TMA: they are copied to rows that do first (grouped_kernels.cu), in the
 * buffer.  Warps that bring such rows into shared memory themselves, shifting each word
 * into place, were built and measured: 128 x 128 x 64 blocks took 3000 cycles instead of
 * 256 (2048 x 2049 matrices, 8192 rows: 620 us, with the copy 94 us).
 *
 * The set-up of a CTA overlaps the end of the kernel before (programmatic launch).  Each
 * warp waits for that one before it touches memory, and before its first bounded wait: the
 * kernel before may take as long as it likes.
 *
 * Every wait is bounded.  One that runs out makes the CTA leave, and the other of its pair:
 * loads and MMAs in flight are given time to land, tensor memory is freed, and the
 * buffer's first word and a word of the device's count it.
 */
#include <atomic>
#include <cstdint>

#include <cuda.h>
#include <cuda_runtime.h>

#include "aclsparse_b200_kernels.h"
#include "element_types.cuh"
#include "grouped_schedule.cuh"
#include "grouped_tc.h"
#include "plan_kernels.h"
#include "tcgen05.cuh"

namespace {

using namespace aclsp;

// CTAs on this device that gave up a wait since the program began.  The count in the buffer lives no longer than the buffer
// or until its counters are cleared, which products do themselves; nothing clears this one.
__device__ uint32_t gWaitFailures;

// Narrow tiles are for few rows, where reading the dense matrix is all: two CTAs to an SM, with half its shared memory
// each, so that one loads while the other starts or ends (32 groups of 4 rows, 2048 x 1024 matrices: 26.1 us, with one
// CTA and all of it 28.6).
template <uint32_t kColumns>
constexpr uint32_t kCtasPerSm = kColumns <= 64u ? 2u : 1u;
// Warps that write results: one or two for each quarter of the lanes of tensor memory.
template <uint32_t kColumns>
constexpr uint32_t kResultWarpsOf = kColumns <= 64u ? 4u : 8u;
template <uint32_t kColumns>
constexpr uint32_t kThreads = 128u + 32u * kResultWarpsOf<kColumns>;
constexpr uint32_t kSegments = 4;     // tiles that the schedule may be ahead
constexpr uint32_t kLeftBytes = kTileLanes * 128u;
constexpr uint32_t kRightBox = 32;  // rows of one load of a forward product's right operand
// Room for a gradient's results on their way out, per warp: two boxes of 32 rows x 128 bytes for TMA; or, where the rows
// of C are not aligned, 32 lanes x 16 results, each lane's one word longer than they are, so that the lanes write to
// different banks.
constexpr uint32_t kTurnBoxBytes = 32u * 128u;
constexpr uint32_t kTurnWarpBytes = 2u * kTurnBoxBytes;
constexpr uint64_t kDrainNs = 10000000ull;

template <uint32_t kColumns, uint32_t kCtas, bool kGradient>
struct Ring {
    static constexpr uint32_t kRightRows = kColumns / kCtas;  // of the right operand in one CTA
    static constexpr uint32_t kStageBytes = kLeftBytes + kRightRows * 128u;
    static constexpr uint32_t kTurnBytes = kGradient ? kResultWarpsOf<kColumns> * kTurnWarpBytes : 0u;
    static constexpr uint32_t kStages = ((kCtasPerSm<kColumns> == 2u ? 111u : 224u) * 1024u - kTurnBytes) / kStageBytes;
    static constexpr uint32_t kTurn = kStageBytes * kStages;           // behind the stages: results on their way out
    static constexpr uint32_t kBytes = kTurn + kTurnBytes + 1024u;     // stages start on multiples of 1024
};

// One result in the type of C; beta == 0 does not read C.
template <typename T>
__device__ __forceinline__ float ToFloat(T v);
template <>
__device__ __forceinline__ float ToFloat(float v) { return v; }
template <>
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T FromFloat(float v);
template <>
__device__ __forceinline__ float FromFloat(float v) { return v; }
template <>
__device__ __forceinline__ __half FromFloat(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 FromFloat(float v) { return __float2bfloat16_rn(v); }

// Sixteen neighbouring results of one lane.
struct Lane16 {
    float v[16];
};

// Forward: the lane is a column of C, the sixteen values belong to sixteen rows.  A warp writes 32 neighbouring
// columns of a row at a time.  Called by whole warps.
template <typename T>
__device__ __forceinline__ void StoreForward(const AclspGroupedParams& p, void* c, const Segment& s, uint32_t column,
                                             uint32_t j0, const Lane16& sums, float laneScale, float beta)
{
    const uint32_t count = s.columns - j0 < 16u ? s.columns - j0 : 16u;
    float r[16];
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j) {
        r[j] = sums.v[j] * laneScale;
    }
    if (p.rowScales != nullptr) {
        // one load for the sixteen rows, handed round: a load per row would wait for each store before it
        const uint32_t mine = threadIdx.x % 16u;
        const float scale = mine < count ? __ldg(p.rowScales + s.row0 + j0 + mine) : 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) {
            r[j] *= __shfl_sync(0xFFFFFFFFu, scale, static_cast<int>(j));
        }
    }
    if (column >= p.n) {
        return;
    }
    T* at = static_cast<T*>(c) + static_cast<int64_t>(s.row0 + j0) * p.ldc + column;
    if (beta != 0.0f) {
        T old[16];
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) {
            old[j] = j < count ? at[static_cast<int64_t>(j) * p.ldc] : FromFloat<T>(0.0f);
        }
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) {
            r[j] = fmaf(beta, ToFloat(old[j]), r[j]);
        }
    }
    if (count == 16u) {
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) {
            *at = FromFloat<T>(r[j]);
            at += p.ldc;
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) {
            if (j < count) {
                *at = FromFloat<T>(r[j]);
            }
            at += p.ldc;
        }
    }
}

// Gradient: the lane is a row of C_g, the sixteen values are neighbours in it.  Called by whole warps.  Where the rows
// are aligned, each lane writes its own in whole sectors; elsewhere (odd widths, a last column tile) the warp turns the
// values round in shared memory and writes rows element by element, sixteen lanes to one: a lane at a time to its own row
// would send every element to the memory by itself (2047 x 2049 from 8192 rows: 306 us, turned round 113 us).
template <typename T>
__device__ __forceinline__ void StoreGradient(const AclspGroupedParams& p, void* c, const Segment& s, uint32_t row,
                                              uint32_t j0, const Lane16& sums, float laneScale, float beta, uint32_t turn)
{
    const bool hasRow = row < p.m;
    T* at = static_cast<T*>(c) + static_cast<int64_t>(s.group) * p.cBatchStride + static_cast<int64_t>(row) * p.ldc +
            s.right + j0;
    const uint32_t count = s.columns - j0 < 16u ? s.columns - j0 : 16u;
    alignas(16) T out[16];
    if (beta != 0.0f) {
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) {
            const float old = hasRow && j < count ? ToFloat(at[j]) : 0.0f;
            out[j] = FromFloat<T>(fmaf(beta, old, sums.v[j] * laneScale));
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) {
            out[j] = FromFloat<T>(sums.v[j] * laneScale);
        }
    }
    const uint32_t* words = reinterpret_cast<const uint32_t*>(out);
    if (__all_sync(0xFFFFFFFFu, count == 16u && reinterpret_cast<uintptr_t>(at) % 16u == 0u)) {
        if (hasRow && reinterpret_cast<uintptr_t>(at) % 32u != 0u) {
#pragma unroll
            for (uint32_t i = 0; i < sizeof(out) / 16u; ++i) {
                reinterpret_cast<uint4*>(at)[i] = make_uint4(words[4 * i], words[4 * i + 1], words[4 * i + 2], words[4 * i + 3]);
            }
        } else if (hasRow) {
#pragma unroll
            for (uint32_t i = 0; i < sizeof(out) / 32u; ++i) {
                const uint32_t eight[8] = {words[8 * i],     words[8 * i + 1], words[8 * i + 2], words[8 * i + 3],
                                           words[8 * i + 4], words[8 * i + 5], words[8 * i + 6], words[8 * i + 7]};
                Store32(reinterpret_cast<unsigned char*>(at) + 32u * i, eight);
            }
        }
        return;
    }
    constexpr uint32_t kPitch = 16u * sizeof(T) + 4u;
    const uint32_t lane = threadIdx.x % 32u;
    __syncwarp();
#pragma unroll
    for (uint32_t i = 0; i < sizeof(out) / 4u; ++i) {
        asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(turn + lane * kPitch + 4u * i), "r"(words[i]) : "memory");
    }
    __syncwarp();
    const uint32_t column = lane % 16u;
    T* to = at - static_cast<int64_t>(lane) * p.ldc + static_cast<int64_t>(lane / 16u) * p.ldc + column;
    const uint32_t rowsLeft = p.m - (row - lane) > 32u || row - lane >= p.m ? (row - lane >= p.m ? 0u : 32u) : p.m - (row - lane);
#pragma unroll 4
    for (uint32_t r = lane / 16u; r < rowsLeft; r += 2u) {
        if (column < count) {
            const uint32_t address = turn + r * kPitch + column * static_cast<uint32_t>(sizeof(T));
            if constexpr (sizeof(T) == 4) {
                uint32_t v;
                asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(v) : "r"(address) : "memory");
                *reinterpret_cast<uint32_t*>(to) = v;
            } else {
                uint16_t v;
                asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(v) : "r"(address) : "memory");
                *reinterpret_cast<uint16_t*>(to) = v;
            }
        }
        to += 2 * p.ldc;
    }
}

template <bool kGradient, typename T>
__device__ __forceinline__ void StoreResults(const AclspGroupedParams& p, void* c, const Segment& s, uint32_t row,
                                             uint32_t j0, const Lane16& sums, float laneScale, float beta, uint32_t turn)
{
    if constexpr (kGradient) {
        StoreGradient<T>(p, c, s, row, j0, sums, laneScale, beta, turn);
    } else {
        StoreForward<T>(p, c, s, row, j0, sums, laneScale, beta);
    }
}

// Calls f with a value of C's type: outside the loops over a tile's columns, which are then straight code.
template <typename F>
__device__ __forceinline__ void WithOutType(uint32_t type, F f)
{
    if (type == ACLSP_TYPE_F32) {
        f(float{});
    } else if (type == ACLSP_TYPE_F16) {
        f(__half{});
    } else {
        f(__nv_bfloat16{});
    }
}

template <bool kInt8>
__device__ __forceinline__ float SumToFloat(uint32_t bits)
{
    return kInt8 ? __int2float_rn(static_cast<int32_t>(bits)) : __uint_as_float(bits);
}

template <bool kInt8>
__device__ __forceinline__ uint32_t AddSums(uint32_t a, uint32_t b)
{
    return kInt8 ? a + b : __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}

template <bool kInt8, uint32_t kColumns, bool kGradient, uint32_t kCtas>
__global__ void __launch_bounds__(kThreads<kColumns>, kCtasPerSm<kColumns>)
    GroupedTensorKernel(const __grid_constant__ CUtensorMap leftMap, const __grid_constant__ CUtensorMap rightMap,
                        const __grid_constant__ CUtensorMap outMap, void* __restrict__ c, uint32_t* __restrict__ buffer,
                        const AclspGroupedParams p, const uint32_t leftMn, const uint32_t outMapped, const uint32_t joinBlocks)
{
    using R = Ring<kColumns, kCtas, kGradient>;
    constexpr uint32_t kBlock = kInt8 ? 128u : 64u;         // elements of the summed index in a block
    constexpr uint32_t kStepElements = kInt8 ? 32u : 16u;   // and in one MMA
    constexpr uint32_t kResultWarps = kResultWarpsOf<kColumns>;
    constexpr uint32_t kColumnStep = 16u * kCtas;           // N of the MMA is a multiple of this
    extern __shared__ unsigned char dynamic[];
    __shared__ uint64_t full[R::kStages];
    __shared__ uint64_t empty[R::kStages];
    __shared__ uint64_t sumsFull[2];
    __shared__ uint64_t sumsEmpty[2];
    __shared__ uint64_t segmentFull[kSegments];
    __shared__ uint64_t segmentEmpty[kSegments];
    __shared__ Segment segments[kSegments];
    __shared__ uint64_t drained;
    __shared__ uint64_t cutFull[R::kStages];  // a block whose last rows are to be cut off has landed in this CTA
    __shared__ uint64_t cutDone[R::kStages];  // first CTA: a block's last rows are cut off, in both CTAs
    __shared__ uint32_t tmemAddress;
    __shared__ uint32_t gaveUp;

    const uint32_t warp = threadIdx.x / 32u;
    const uint32_t lane = threadIdx.x % 32u;
    const uint32_t rank = kCtas == 2 ? blockIdx.x % 2u : 0u;  // in the pair; rank 0 issues the MMAs
    const Workers workers{blockIdx.x / kCtas, gridDim.x / kCtas};
    const uint32_t ring = (SmemAddress(dynamic) + 1023u) & ~1023u;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < R::kStages; ++i) {
            BarInit(SmemAddress(full + i), 1);
            BarInit(SmemAddress(empty + i), 1);
            BarInit(SmemAddress(cutFull + i), 1);
            BarInit(SmemAddress(cutDone + i), kCtas);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            BarInit(SmemAddress(sumsFull + i), 1);
            BarInit(SmemAddress(sumsEmpty + i), kResultWarps * kCtas);
        }
        for (uint32_t i = 0; i < kSegments; ++i) {
            BarInit(SmemAddress(segmentFull + i), 1);
            BarInit(SmemAddress(segmentEmpty + i), 1u + kResultWarps + (rank == 0u ? 1u : 0u) + (kGradient ? 1u : 0u));
        }
        BarInit(SmemAddress(&drained), 1);
        gaveUp = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        FenceProxyAsync();
        TmaPrefetch(&leftMap);
        TmaPrefetch(&rightMap);
    }
    if (warp == 2) {
        TmemAlloc<kCtas>(SmemAddress(&tmemAddress), 2u * kColumns);
        TmemFenceBefore();
    }
    __syncthreads();
    if constexpr (kCtas == 2) {
        ClusterSync();  // the other CTA's barriers are ready too
    }
    TmemFenceAfter();
    const uint32_t tmem = tmemAddress;
    LetNextKernelStart();  // each warp waits for the previous one itself, before it touches global memory or waits for another warp
    volatile uint32_t* const stop = &gaveUp;
    const uint64_t limit = p.waitLimitNs;

    // The next segment of the schedule, for one of the warps that follow it; parts == 0 ends it.
    uint32_t taken = 0;
    auto nextSegment = [&](Segment* s) {
        const uint32_t i = taken % kSegments;
        if (!__all_sync(0xFFFFFFFFu, BarWait(SmemAddress(segmentFull + i), taken / kSegments & 1u, stop, limit))) {
            return false;
        }
        *s = segments[i];
        __syncwarp();
        if (lane == 0) {
            BarArrive(SmemAddress(segmentEmpty + i));
        }
        ++taken;
        return s->parts != 0u;
    };
    // Gradient: rows of block b that belong to the group.  The last block of a group may hold rows behind it; those of
    // the last MMA's share are somebody else's and are overwritten with zeros, in both operands, so that no infinity or
    // NaN of theirs gets in.
    auto validRows = [&](const Segment& s, uint32_t b) {
        return s.rows - b * kBlock < kBlock ? s.rows - b * kBlock : kBlock;
    };
    auto cutRows = [&](uint32_t valid, uint32_t left) {
        const uint32_t vectors = (kStepElements - valid % kStepElements) % kStepElements * 8u;
        for (uint32_t i = lane; i < vectors; i += 32u) {
#pragma unroll
            for (uint32_t block = 0; block < 2u + R::kRightRows / 64u; ++block) {
                const uint32_t address = left + block * 8192u + valid * 128u + i * 16u;
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(address), "r"(0) : "memory");
            }
        }
        FenceProxyAsync();
        __syncwarp();
    };

    if (warp == 0) {
        constexpr uint32_t kBox = kGradient ? 64u : kRightBox;
        WaitForPreviousKernel();
        Segment s;
        uint32_t stage = 0;
        uint32_t parity = 0;
        bool good = true;
        while (good && nextSegment(&s)) {
            const uint32_t share = (s.columns + kColumnStep - 1u) / kColumnStep * 16u;  // of the columns, in this CTA
            const uint32_t boxes = (share + kBox - 1u) / kBox;
            const uint32_t bytes = kLeftBytes + boxes * kBox * 128u;
            const uint32_t leftAt = s.left + rank * kTileLanes;
            const uint32_t rightAt = (kGradient ? s.right : s.row0) + rank * share;
            if (ElectLane()) {
                for (uint32_t b = s.block0; b < s.block1; ++b) {
                    if (!BarWait(SmemAddress(empty + stage), parity ^ 1u, stop, limit)) {
                        good = false;
                        break;
                    }
                    const uint32_t left = ring + stage * R::kStageBytes;
                    const uint32_t right = left + kLeftBytes;
                    const bool cut = kGradient && validRows(s, b) % kStepElements != 0u;
                    // A pair's blocks are announced to the first CTA, except those whose last rows are cut off: each
                    // CTA's warp 2 sees to its share first, and the MMAs wait for that.
                    uint32_t bar = SmemAddress((cut ? cutFull : full) + stage);
                    if (cut) {
                        BarExpect(bar, bytes);
                        if (rank == 0u) {
                            BarArrive(SmemAddress(full + stage));
                        }
                    } else if (rank == 0u) {
                        BarExpect(bar, kCtas * bytes);
                    } else {
                        bar = PeerAddress(bar, 0);
                    }
                    const int32_t at = static_cast<int32_t>(b * kBlock);
                    if constexpr (kGradient) {
                        const int32_t row = static_cast<int32_t>(s.row0) + at;
                        for (uint32_t i = 0; i < 2; ++i) {
                            TmaLoad2<kCtas>(left + i * 8192u, &leftMap, bar, static_cast<int32_t>(leftAt + i * 64u), row);
                        }
                        for (uint32_t i = 0; i < boxes; ++i) {
                            TmaLoad2<kCtas>(right + i * 8192u, &rightMap, bar, static_cast<int32_t>(rightAt + i * 64u), row);
                        }
                    } else {
                        if (leftMn == 0u) {
                            TmaLoad3<kCtas>(left, &leftMap, bar, at, static_cast<int32_t>(leftAt), static_cast<int32_t>(s.group));
                        } else {
                            for (uint32_t i = 0; i < (kInt8 ? 1u : 2u); ++i) {
                                TmaLoad3<kCtas>(left + i * 8192u, &leftMap, bar, static_cast<int32_t>(leftAt + i * 64u), at,
                                                static_cast<int32_t>(s.group));
                            }
                        }
                        for (uint32_t i = 0; i < boxes; ++i) {
                            TmaLoad2<kCtas>(right + i * kBox * 128u, &rightMap, bar, at,
                                            static_cast<int32_t>(rightAt + i * kBox));
                        }
                    }
                    stage = stage + 1u == R::kStages ? 0u : stage + 1u;
                    parity ^= stage == 0u ? 1u : 0u;
                }
            }
            __syncwarp();
            good = __all_sync(0xFFFFFFFFu, good) != 0;
        }
    } else if (warp == 1 && rank == 0u) {
        // One lane does it all: with the warp's votes and an election for each block, a block took 570 cycles to issue, and
        // the tensor cores need 512 for 256 columns, 384 for 192 (1024 x 1024 gradients of 2 x 4096 rows: 36.6 us then, 31.0
        // now).
        WaitForPreviousKernel();
        if (ElectLane()) {
            const bool leftT = kGradient || leftMn != 0u;
            const uint32_t shape = MmaShape(kCtas, kInt8, p.inType == ACLSP_TYPE_BF16, leftT, kGradient);
            // 32 bytes of the summed index per instruction: inside a 128-byte row, or as many rows as it has elements
            const uint32_t leftStep = (leftT ? kStepElements * 128u : 32u) >> 4;
            const uint32_t rightStep = (kGradient ? kStepElements * 128u : 32u) >> 4;
            const uint64_t leftBase = OperandDescriptor(ring, 8192u);
            const uint64_t rightBase = OperandDescriptor(ring + kLeftBytes, 8192u);
            uint32_t stage = 0;
            uint32_t parity = 0;
            uint32_t tile = 0;
            uint32_t cuts = 0;  // a bit per stage: the parity of its next cut block
            bool good = true;
            struct Work {
                uint32_t columns, length, block0, block1;
            };
            // What this lane needs of the next segment; false at the end.
            auto take = [&](Work* w) {
                const uint32_t i = taken % kSegments;
                if (!BarWait(SmemAddress(segmentFull + i), taken / kSegments & 1u, stop, limit)) {
                    good = false;
                    return false;
                }
                const Segment& s = segments[i];
                *w = Work{s.columns, kGradient ? s.rows : p.k, s.block0, s.block1};
                const bool more = s.parts != 0u;
                BarArrive(SmemAddress(segmentEmpty + i));
                ++taken;
                return more;
            };
            Work w;
            bool more = take(&w);
            while (more) {
                const uint32_t half = tile & 1u;
                good = BarWait(SmemAddress(sumsEmpty + half), (tile >> 1 & 1u) ^ 1u, stop, limit);
                if (!good) {
                    break;
                }
                ++tile;
                TmemFenceAfter();
                const uint32_t d = tmem + half * kColumns;
                const uint32_t instruction = shape | MmaColumns((w.columns + kColumnStep - 1u) / kColumnStep * kColumnStep);
                Work next;
                if (w.block0 == w.block1) {
                    more = take(&next);
                }
                for (uint32_t b = w.block0; b < w.block1; ++b) {
                    good = BarWait(SmemAddress(full + stage), parity, stop, limit);
                    if (!good) {
                        break;
                    }
                    const uint32_t valid = w.length - b * kBlock < kBlock ? w.length - b * kBlock : kBlock;
                    if constexpr (kGradient) {
                        if (valid % kStepElements != 0u) {
                            good = BarWait(SmemAddress(cutDone + stage), cuts >> stage & 1u, stop, limit);
                            cuts ^= 1u << stage;
                            if (!good) {
                                break;
                            }
                        }
                    }
                    const uint64_t left = leftBase + stage * (R::kStageBytes >> 4);
                    const uint64_t right = rightBase + stage * (R::kStageBytes >> 4);
#pragma unroll
                    for (uint32_t i = 0; i < 4u; ++i) {
                        if (i * kStepElements < valid) {
                            Mma<kInt8, kCtas>(d, left + i * leftStep, right + i * rightStep, instruction,
                                              b != w.block0 || i != 0u ? 1u : 0u);
                        }
                    }
                    MmaCommit<kCtas>(SmemAddress(empty + stage));
                    if (b == w.block0) {
                        more = take(&next);  // while this tile computes
                    }
                    stage = stage + 1u == R::kStages ? 0u : stage + 1u;
                    parity ^= stage == 0u ? 1u : 0u;
                }
                if (!good) {
                    break;
                }
                MmaCommit<kCtas>(SmemAddress(sumsFull + half));
                w = next;
            }
            if (!good) {  // not under instructions that still read tensor memory
                uint32_t never = 0;
                MmaCommit<kCtas>(SmemAddress(&drained));
                (void)BarWait(SmemAddress(&drained), 0, &never, kWaitLimitNs);
            }
        }
        __syncwarp();
    } else if (kGradient && warp == 2) {
        WaitForPreviousKernel();
        Segment s;
        uint32_t block = 0;  // of all that this CTA loads: the stage is block % kStages
        uint32_t cuts = 0;   // a bit per stage: the parity of its next cut block
        while (nextSegment(&s)) {
            const uint32_t count = s.block1 - s.block0;
            const uint32_t valid = count != 0u ? validRows(s, s.block1 - 1u) : 0u;
            if (valid % kStepElements != 0u) {
                const uint32_t stage = (block + count - 1u) % R::kStages;
                if (!__all_sync(0xFFFFFFFFu, BarWait(SmemAddress(cutFull + stage), cuts >> stage & 1u, stop, limit))) {
                    break;
                }
                cuts ^= 1u << stage;
                cutRows(valid, ring + stage * R::kStageBytes);
                if (lane == 0) {
                    const uint32_t done = SmemAddress(cutDone + stage);
                    if (rank == 0u) {
                        BarArrive(done);
                    } else {
                        BarArrivePeer(PeerAddress(done, 0));
                    }
                }
            }
            block += count;
        }
    } else if (warp == 3) {
        AclspGroupedParams own = p;
        if (p.offsets != nullptr) {  // without them the schedule needs nothing from memory
            WaitForPreviousKernel(own.offsets);
        }
        auto schedule = [&]() {
            if constexpr (kGradient) {
                return GradientSchedule(own, workers, kTileLanes * kCtas, kColumns, kBlock, joinBlocks);
            } else {
                return ForwardSchedule(own, workers, kTileLanes * kCtas, kColumns, (p.k + kBlock - 1u) / kBlock, joinBlocks);
            }
        }();
        bool more = true;
        for (uint32_t given = 0; more; ++given) {
            Segment s;
            more = schedule.Next(&s);
            s.parts = more ? s.parts : 0u;
            const uint32_t i = given % kSegments;
            if (given == kSegments) {
                WaitForPreviousKernel();  // the first wait that others have to end
            }
            if (!__all_sync(0xFFFFFFFFu, BarWait(SmemAddress(segmentEmpty + i), (given / kSegments & 1u) ^ 1u, stop, limit))) {
                break;
            }
            if (lane == 0) {
                segments[i] = s;
                BarArrive(SmemAddress(segmentFull + i));
            }
            __syncwarp();
        }
    } else if (warp >= 4) {
        AclspGroupedParams own = p;
        WaitForPreviousKernel(own.rowScales, own.colScales, own.alphaPtr, own.betaPtr);
        const float alpha = p.alphaPtr != nullptr ? *own.alphaPtr : p.alpha;
        const float beta = p.betaPtr != nullptr ? *own.betaPtr : p.beta;
        const uint32_t tmemLane = threadIdx.x % 128u;
        const uint32_t firstChunk = (warp - 4u) / 4u * 16u;  // of the columns: warps that share lanes take turns
        constexpr uint32_t kChunkStep = kResultWarps / 4u * 16u;
        const uint32_t turn = ring + R::kTurn + (warp - 4u) * kTurnWarpBytes;
        uint32_t* const counters = buffer + kGroupedHeaderWords;
        uint4* const partials = reinterpret_cast<uint4*>(counters + kGroupedCounters);
        uint32_t boxes = 0;  // that this warp has sent out
        constexpr uint32_t kSlotVectors = kTileLanes * kColumns / 4u;
        Segment s;
        uint32_t tile = 0;
        // This warp has read its share of the sums: the tensor memory may be written again.
        auto release = [&](uint32_t half) {
            TmemFenceBefore();
            __syncwarp();
            if (lane == 0) {
                const uint32_t bar = SmemAddress(sumsEmpty + half);
                if (rank == 0u) {
                    BarArrive(bar);
                } else {
                    BarArrivePeer(PeerAddress(bar, 0));
                }
            }
        };
        while (nextSegment(&s)) {
            const uint32_t half = tile & 1u;
            if (!__all_sync(0xFFFFFFFFu, BarWait(SmemAddress(sumsFull + half), tile >> 1 & 1u, stop, limit))) {
                break;
            }
            ++tile;
            TmemFenceAfter();
            const uint32_t from = tmem + half * kColumns + (warp % 4u * 32u << 16);
            const uint32_t row = s.left + rank * kTileLanes + tmemLane;  // of the first operand
            const bool nothing = s.block0 == s.block1;  // an empty group's gradient: no sums were made
            float laneScale = alpha;
            if (!kGradient && p.colScales != nullptr && row < p.n) {
                laneScale *= __ldg(own.colScales + static_cast<int64_t>(s.group) * p.n + row);
            }
            if (kGradient && s.parts == 1u && outMapped != 0u && beta == 0.0f) {
                if constexpr (kGradient) {
                    // Through shared memory and TMA, two boxes per warp under way: the stores of a tile take longer than
                    // short sums, and a warp that issues them itself waits for each (2000 rows of 64 groups, 512 x 1024 fp16:
                    // 25.5 us with its own stores, 18.4 so).
                    WithOutType(p.outType, [&](auto type) {
                        using T = decltype(type);
                        constexpr uint32_t kBoxColumns = 128u / sizeof(T);
                        constexpr uint32_t kOwn = kColumns / (kResultWarps / 4u);  // columns of this warp
                        const uint32_t begin = (warp - 4u) / 4u * kOwn;
                        const uint32_t end = s.columns < begin + kOwn ? s.columns : begin + kOwn;
                        const uint32_t row0 = row - lane;
                        for (uint32_t j0 = begin; j0 < end; j0 += kBoxColumns) {
                            const uint32_t box = turn + (boxes++ & 1u) * kTurnBoxBytes;
                            if (ElectLane()) {
                                StoresRead<1>();
                            }
                            __syncwarp();
#pragma unroll
                            for (uint32_t q = 0; q < kBoxColumns / 16u; ++q) {
                                uint32_t bits[16];
                                TmemLoad16(from + j0 + 16u * q, bits);
                                TmemLoadWait();
                                alignas(16) T out[16];
#pragma unroll
                                for (uint32_t j = 0; j < 16; ++j) {
                                    out[j] = FromFloat<T>(nothing ? 0.0f : SumToFloat<kInt8>(bits[j]) * laneScale);
                                }
                                const uint4* vectors = reinterpret_cast<const uint4*>(out);
                                constexpr uint32_t kVectors = sizeof(out) / 16u;
#pragma unroll
                                for (uint32_t v = 0; v < kVectors; ++v) {
                                    const uint32_t at = box + lane * 128u + ((q * kVectors + v) ^ (lane & 7u)) * 16u;
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "r"(vectors[v].x),
                                                 "r"(vectors[v].y), "r"(vectors[v].z), "r"(vectors[v].w)
                                                 : "memory");
                                }
                            }
                            FenceProxyAsync();
                            __syncwarp();
                            if (ElectLane()) {
                                if (row0 < p.m) {
                                    TmaStore3(&outMap, box, static_cast<int32_t>(s.right + j0), static_cast<int32_t>(row0),
                                              static_cast<int32_t>(s.group));
                                }
                                StoreGroup();
                            }
                            __syncwarp();
                        }
                    });
                }
                release(half);
                continue;
            }
            if (s.parts == 1u) {
                WithOutType(p.outType, [&](auto type) {
                    for (uint32_t j0 = firstChunk; j0 < s.columns; j0 += kChunkStep) {
                        uint32_t bits[16];
                        Lane16 sums;
                        __syncwarp();
                        TmemLoad16(from + j0, bits);
                        TmemLoadWait();
#pragma unroll
                        for (uint32_t j = 0; j < 16; ++j) {
                            sums.v[j] = nothing ? 0.0f : SumToFloat<kInt8>(bits[j]);
                        }
                        StoreResults<kGradient, decltype(type)>(own, c, s, row, j0, sums, laneScale, beta, turn);
                    }
                });
                release(half);
                continue;
            }
            // Partial sums lie four columns of a lane to a vector: [columns / 4][lanes][4].
            uint4* const mine = partials + static_cast<size_t>(s.slot * kCtas + rank) * kSlotVectors + tmemLane;
            for (uint32_t j0 = firstChunk; j0 < s.columns; j0 += kChunkStep) {
                uint32_t bits[16];
                __syncwarp();
                TmemLoad16(from + j0, bits);
                TmemLoadWait();
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    __stcg(mine + (j0 / 4u + j) * kTileLanes,
                           make_uint4(bits[4 * j], bits[4 * j + 1], bits[4 * j + 2], bits[4 * j + 3]));
                }
            }
            release(half);
            if (kGradient && ElectLane()) {
                StoresRead<0>();  // the room may be needed again
            }
            // the warp's sums first, then the fence of the lanes that count them
            __syncwarp();
            __threadfence();
            const uint32_t pieces = s.columns > firstChunk ? (s.columns - firstChunk + kChunkStep - 1u) / kChunkStep : 0u;
            uint32_t lasts = 0;
            uint32_t* const tileCounters = counters + (s.counter * kCtas + rank) * kTileCounters + warp % 4u;
            // Two pieces at a time, from one that differs from part to part on.
            for (uint32_t i = 0; i < pieces; ++i) {
                const uint32_t inTwo = i % 2u;
                const uint32_t j0 = firstChunk + (2u * s.part + i) % pieces * kChunkStep;
                if (inTwo == 0u) {
                    bool last = false;
                    if (lane < 2u && i + lane < pieces) {
                        uint32_t* const counter =
                            tileCounters + (firstChunk + (2u * s.part + i + lane) % pieces * kChunkStep) / 16u * 4u;
                        last = atomicAdd(counter, 1u) + 1u == s.parts;
                        if (last) {
                            *counter = 0;  // clear for the next product
                        }
                    }
                    lasts = __ballot_sync(0xFFFFFFFFu, last);
                    if (lasts != 0u) {
                        __threadfence();
                        __syncwarp();
                    }
                }
                if ((lasts >> inTwo & 1u) == 0u) {
                    continue;
                }
                const uint4* const at = partials + tmemLane + j0 / 4u * kTileLanes;
                uint32_t total[16];
                constexpr uint32_t kTogether = kColumns <= 64u ? 2u : 4u;  // parts under way together
                for (uint32_t k = 0; k < s.parts; k += kTogether) {
                    uint4 v[kTogether][4];
#pragma unroll
                    for (uint32_t q = 0; q < kTogether; ++q) {
                        if (k + q < s.parts) {
                            const uint32_t slot = (s.slot - s.part + k + q) * kCtas + rank;
#pragma unroll
                            for (uint32_t j = 0; j < 4; ++j) {
                                v[q][j] = __ldcg(at + static_cast<size_t>(slot) * kSlotVectors + j * kTileLanes);
                            }
                        }
                    }
#pragma unroll
                    for (uint32_t q = 0; q < kTogether; ++q) {
                        if (k + q < s.parts) {
#pragma unroll
                            for (uint32_t j = 0; j < 4; ++j) {
                                const uint32_t w[4] = {v[q][j].x, v[q][j].y, v[q][j].z, v[q][j].w};
#pragma unroll
                                for (uint32_t e = 0; e < 4; ++e) {
                                    total[4 * j + e] = k + q == 0u ? w[e] : AddSums<kInt8>(total[4 * j + e], w[e]);
                                }
                            }
                        }
                    }
                }
                Lane16 sums;
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) {
                    sums.v[j] = SumToFloat<kInt8>(total[j]);
                }
                WithOutType(p.outType, [&](auto type) {
                    StoreResults<kGradient, decltype(type)>(own, c, s, row, j0, sums, laneScale, beta, turn);
                });
            }
        }
        __syncwarp();
        if (kGradient && ElectLane()) {
            StoresDone();
        }
    }

    __syncthreads();
    if constexpr (kCtas == 2) {
        if (threadIdx.x == 0 && *stop != 0u) {
            StorePeer(PeerAddress(SmemAddress(&gaveUp), rank ^ 1u), 1u);
        }
        ClusterSync();  // neither CTA leaves while the other may still reach its shared memory
    }
    // Where a wait ran out, in any warp of this CTA or of the pair's other one, loads and MMAs may still be under way, also
    // those of warps that ended as they should: neither CTA may free its tensor memory or leave its shared memory under
    // them, so both give them time to land.
    if (*stop != 0u) {
        if (threadIdx.x == 0) {
            atomicAdd(buffer, 1u);
            atomicAdd(&gWaitFailures, 1u);
            const uint64_t began = Nanoseconds();
            while (Nanoseconds() - began < kDrainNs) {
            }
        }
        __syncthreads();
    }
    if (warp == 2) {
        TmemFenceAfter();
        TmemFree<kCtas>(tmem, 2u * kColumns);
    }
}

// ---- host side ----

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn Encoder()
{
    static const EncodeFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<EncodeFn>(f);
    }();
    return fn;
}

// A map of `rank` dimensions (innermost first) of elements of a type whose boxes are 128 bytes wide and `boxRows` rows
// high.
bool Encode(CUtensorMap* map, uint32_t type, const void* base, uint32_t rank, const uint64_t* sizes,
            const uint64_t* strideElements, uint32_t boxRows)
{
    const uint64_t bytes = type == ACLSP_TYPE_I8 ? 1u : type == ACLSP_TYPE_F32 ? 4u : 2u;
    cuuint64_t dims[3];
    cuuint64_t strides[2];
    cuuint32_t box[3] = {static_cast<cuuint32_t>(128u / bytes), boxRows, 1};
    cuuint32_t ones[3] = {1, 1, 1};
    for (uint32_t i = 0; i < rank; ++i) {
        dims[i] = sizes[i];
        if (i > 0) {
            strides[i - 1] = strideElements[i - 1] * bytes;
        }
    }
    const CUtensorMapDataType element = type == ACLSP_TYPE_I8     ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                        : type == ACLSP_TYPE_F32  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                        : type == ACLSP_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                  : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return Encoder()(map, element, rank, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool kInt8, uint32_t kColumns, bool kGradient>
void Launch(const CUtensorMap& left, const CUtensorMap& right, const CUtensorMap* out, void* c, void* buffer,
            const AclspGroupedParams& p, uint32_t leftMn, uint32_t sms, cudaStream_t s)
{
    constexpr uint32_t kCtas = kColumns == 256u ? 2u : 1u;
    constexpr uint32_t kBytes = Ring<kColumns, kCtas, kGradient>::kBytes;
    auto kernel = GroupedTensorKernel<kInt8, kColumns, kGradient, kCtas>;
    // once per device: a small product takes the GPU about as long as this call takes the host with its launch
    static std::atomic<uint64_t> allowed{0};
    int device = 0;
    (void)cudaGetDevice(&device);
    const uint64_t bit = 1ull << (device & 63);
    if ((allowed.load(std::memory_order_relaxed) & bit) == 0u) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kBytes)) == cudaSuccess) {
            allowed.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    AclspCountLaunches(1);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(sms * kCtasPerSm<kColumns> / kCtas * kCtas);
    config.blockDim = dim3(kThreads<kColumns>);
    config.dynamicSmemBytes = kBytes;
    config.stream = s;
    cudaLaunchAttribute attributes[2] = {};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = kCtas;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = kCtas > 1u ? 2u : 1u;
    cudaLaunchKernelEx(&config, kernel, left, right, out != nullptr ? *out : left, c, static_cast<uint32_t*>(buffer), p, leftMn,
                       out != nullptr ? 1u : 0u, kColumns >= 256u ? kJoinBlocksWide : kJoinBlocks);
}

}  // namespace

cudaError_t AclspGroupedTotalWaitFailures(cudaStream_t s, uint32_t* count)
{
    const cudaError_t err = cudaMemcpyFromSymbolAsync(count, gWaitFailures, sizeof(*count), 0, cudaMemcpyDeviceToHost, s);
    return err != cudaSuccess ? err : cudaStreamSynchronize(s);
}

// The width of a tile.  What a choice costs is the number of turns that the workers take for all tiles times what a turn
// takes: the blocks of the summed index at the rate that an SM gets operands from L2 (a block of a 128 x 32 tile is 20 KB,
// of a 128 x 64 one 24 KB, of 128 x 128 32 KB; in a pair's 256 x 256 tile each CTA loads 32 KB), or writing the results
// of the tile before, where that is longer; and the results of the last one.  The host knows the rows of an average group
// only; larger groups are cut into more tiles, which read the dense matrix again, from L2, smaller ones leave columns
// unused.  Measured, us: 1003 rows of 4 groups, 776 x 1001: 10.4 with 128 columns, 14.5 with 256; 5719 rows, 1056 x 1968
// int8: 23.2 with 128, 24.9 with 256; 512 x 512 from 16384 rows: 24.6 with 128, 36.3 with 256.
uint32_t AclspGroupedColumns(const AclspGroupedParams& p)
{
    struct Choice {
        uint32_t columns;
        uint32_t workers;
        uint64_t block;    // relative cost of a block
        uint64_t results;  // and of reading a tile's sums and writing its results
    };
    constexpr Choice kChoices[] = {{256, 74, 32, 320}, {128, 148, 32, 160}, {64, 148, 24, 100}, {32, 148, 20, 60}};
    const uint64_t bytes = p.inType == ACLSP_TYPE_I8 ? 1u : 2u;
    const uint64_t groups = p.groups < p.rows ? p.groups : (p.rows > 0 ? p.rows : 1u);  // that can have rows
    const uint64_t average = (p.rows + groups - 1u) / groups;
    const uint64_t length = p.weightGrad != 0 ? average : p.k;
    const uint64_t blocks = (length * bytes + 127u) / 128u;
    uint32_t best = 0;
    uint64_t least = ~0ull;
    for (const Choice& c : kChoices) {
        if (p.weightGrad != 0 && c.columns < 128u) {
            break;  // two blocks of 64 columns are the least that the gradient's loads make
        }
        const uint64_t lanes = kTileLanes * (c.columns == 256u ? 2u : 1u);
        const uint64_t down = ((p.weightGrad != 0 ? p.m : p.n) + lanes - 1u) / lanes;
        const uint64_t across = ((p.weightGrad != 0 ? p.n : average) + c.columns - 1u) / c.columns;
        const uint64_t tiles = (p.weightGrad != 0 ? p.groups : groups) * down * across;
        const uint64_t turns = (tiles + c.workers - 1u) / c.workers;
        const uint64_t results = p.inType == ACLSP_TYPE_I8 ? c.results + c.results / 2u : c.results;
        const uint64_t cost = turns * (blocks * c.block > results ? blocks * c.block : results) + results;
        if (cost < least) {
            least = cost;
            best = c.columns;
        }
    }
    return best;
}

// Both sides' times, in ns beside what is common to them: without tensor cores the matrices at 5.0 TB/s or, where that is
// longer, the products one by one; with them the matrices at 5.8 TB/s, and 3.7 us of set-up, ring and join.  The bound
// on the rows is for groups that the host does not know: all rows may be in one, whose matrix is then read once for
// every four.  Measured, us, with and without tensor cores: 8 rows, 1024 x 1024: 7.0, 5.1; 16 rows: 6.9, 8.1; 16 rows of 8
// groups, 2048 x 1024: 12.8, 11.3; 4096 x 4096: 46, 54; 4 rows, 4096 x 4096: 11.7, 11.9; 2 rows: 11.7, 8.1.
bool AclspGroupedFewRows(const AclspGroupedParams& p)
{
    const uint64_t bytes = p.inType == ACLSP_TYPE_I8 ? 1u : 2u;
    const uint64_t strides = static_cast<uint64_t>(p.aOuter) | static_cast<uint64_t>(p.bOuter) |
                             (p.groups > 1u ? static_cast<uint64_t>(p.bBatchStride) : 0u);
    if (p.weightGrad != 0 || p.bInner != 1 || strides * bytes % 16u != 0u || p.n > 1u << 24 || p.rows > 16u ||
        (p.rows > 8u && 2u * p.groups < p.rows)) {
        return false;
    }
    const uint64_t matrix = static_cast<uint64_t>(p.n) * p.k;
    const uint64_t read = matrix * bytes * (p.groups < p.rows ? p.groups : p.rows);
    const uint64_t products = matrix * p.rows / (p.inType == ACLSP_TYPE_I8 ? 25000u : 7000u);
    return (read / 5000u > products ? read / 5000u : products) <= read / 5800u + 3700u;
}

AclspGroupedOperands AclspGroupedDescribe(const AclspGroupedParams& p)
{
    AclspGroupedOperands o{};
    if (p.weightGrad != 0) {
        o.left = {p.m, p.rows, 1, static_cast<uint64_t>(p.aInner), 0, 0, 0};
        o.right = {p.n, p.rows, 1, static_cast<uint64_t>(p.bInner), 0, 0, 0};
    } else {
        const bool kContiguous = p.bInner == 1;
        o.left = {kContiguous ? p.k : p.n, kContiguous ? p.n : p.k, p.groups,
                  static_cast<uint64_t>(kContiguous ? p.bOuter : p.bInner), static_cast<uint64_t>(p.bBatchStride), 0, 0};
        o.right = {p.k, p.rows, 1, static_cast<uint64_t>(p.aOuter), 0, 0, 0};
    }
    if (AclspGroupedFewRows(p)) {
        o.bufferBytes = kGroupedCountersEnd;
        return o;
    }
    o.bufferBytes = kGroupedCountersEnd + 2ull * kGroupedMaxCtas * kTileLanes * AclspGroupedColumns(p) * 4u;
    const uint64_t bytes = p.inType == ACLSP_TYPE_I8 ? 1u : 2u;
    for (AclspGroupedOperand* x : {&o.left, &o.right}) {
        const bool strides = x->ld * bytes % 16u == 0u && (x->batches == 1u || x->batchStride * bytes % 16u == 0u);
        if (!strides && x->rowElements != 0u && x->rows != 0u) {
            x->copyOffset = (o.bufferBytes + 255u) / 256u * 256u;
            x->copyBytes = x->batches * x->rows * ((x->rowElements * bytes + 15u) / 16u * 16u);
            o.bufferBytes = x->copyOffset + x->copyBytes;
        }
    }
    return o;
}

bool AclspGroupedTensorLaunch(const void* a, const void* b, void* c, void* buffer, const AclspGroupedParams& given,
                              cudaStream_t s)
{
    AclspGroupedParams p = given;
    p.waitLimitNs = p.waitLimitNs != 0u ? p.waitLimitNs : kWaitLimitNs;
    constexpr uint32_t kLongest = 1u << 28;  // block and tile numbers stay far inside 32 bits
    constexpr uint64_t kFarthest = 1ull << 40;  // strides that a tensor map takes, in bytes
    const uint32_t columns = AclspGroupedColumns(p);
    const uint64_t bytes = p.inType == ACLSP_TYPE_I8 ? 1u : 2u;
    const uint64_t down = ((p.weightGrad != 0 ? p.m : p.n) + kTileLanes - 1u) / kTileLanes;
    const uint64_t tiles = p.weightGrad != 0 ? p.groups * down * ((p.n + columns - 1u) / columns)
                                             : (static_cast<uint64_t>(p.rows) / columns + p.groups) * down;
    if (p.rows > kLongest || p.k > kLongest || (p.weightGrad == 0 && p.k == 0) || p.rows == 0 || tiles > 1u << 30 ||
        Encoder() == nullptr) {
        return false;
    }
    AclspGroupedOperands o = AclspGroupedDescribe(p);
    const void* bases[2] = {p.weightGrad != 0 ? a : b, p.weightGrad != 0 ? b : a};
    const AclspGroupedOperand* const operands[2] = {&o.left, &o.right};
    for (uint32_t i = 0; i < 2; ++i) {
        const AclspGroupedOperand& x = *operands[i];
        const uint64_t batch = x.batches > 1u ? x.batchStride : 0u;
        if (x.copyBytes == 0u && (reinterpret_cast<uintptr_t>(bases[i]) % 16u != 0u || x.ld * bytes >= kFarthest ||
                                  batch * bytes >= kFarthest)) {
            return false;
        }
    }
    AclspGroupedCopyRows(&o, &bases[0], &bases[1], buffer, p, s);
    uint32_t sms = AclspSmCount();
    sms = sms == 0 || sms > kGroupedMaxCtas ? kGroupedMaxCtas : sms;
    CUtensorMap left;
    CUtensorMap right;
    const uint64_t leftSizes[3] = {o.left.rowElements, o.left.rows, o.left.batches};
    const uint64_t leftStrides[2] = {o.left.ld, o.left.batches > 1u ? o.left.batchStride : o.left.ld};
    const uint64_t rightSizes[2] = {o.right.rowElements, o.right.rows};
    const uint64_t rightStride[1] = {o.right.ld};
    if (p.weightGrad != 0) {
        if (!Encode(&left, p.inType, bases[0], 2, leftSizes, leftStrides, 64) ||
            !Encode(&right, p.inType, bases[1], 2, rightSizes, rightStride, 64)) {
            return false;
        }
        // Results through TMA where C allows it.  A store that ends behind the last column, between two multiples of 16
        // bytes, was seen to write on to the next one, so the rows must end on one.
        CUtensorMap out;
        const uint64_t outBytes = p.outType == ACLSP_TYPE_F32 ? 4u : 2u;
        const uint64_t outSizes[3] = {p.n, p.m, p.groups};
        const uint64_t outStrides[2] = {static_cast<uint64_t>(p.ldc),
                                        static_cast<uint64_t>(p.groups > 1u ? p.cBatchStride : p.ldc)};
        const bool outMapped = reinterpret_cast<uintptr_t>(c) % 16u == 0u && p.n * outBytes % 16u == 0u &&
                               outStrides[0] * outBytes % 16u == 0u &&
                               outStrides[1] * outBytes % 16u == 0u && outStrides[0] * outBytes < kFarthest &&
                               outStrides[1] * outBytes < kFarthest &&
                               Encode(&out, p.outType, c, 3, outSizes, outStrides, 32);
        (columns == 256u ? Launch<false, 256, true> : Launch<false, 128, true>)(left, right, outMapped ? &out : nullptr, c,
                                                                                buffer, p, 1u, sms, s);
        return true;
    }
    const uint32_t leftMn = p.bInner == 1 ? 0u : 1u;
    const uint32_t leftBox = leftMn != 0 ? static_cast<uint32_t>(128u / bytes) : kTileLanes;
    if (!Encode(&left, p.inType, bases[0], 3, leftSizes, leftStrides, leftBox) ||
        !Encode(&right, p.inType, bases[1], 2, rightSizes, rightStride, kRightBox)) {
        return false;
    }
    const bool int8 = p.inType == ACLSP_TYPE_I8;
    auto run = int8 ? (columns == 32u    ? Launch<true, 32, false>
                       : columns == 64u  ? Launch<true, 64, false>
                       : columns == 128u ? Launch<true, 128, false>
                                         : Launch<true, 256, false>)
                    : (columns == 32u    ? Launch<false, 32, false>
                       : columns == 64u  ? Launch<false, 64, false>
                       : columns == 128u ? Launch<false, 128, false>
                                         : Launch<false, 256, false>);
    run(left, right, nullptr, c, buffer, p, leftMn, sms, s);
    return true;
}
