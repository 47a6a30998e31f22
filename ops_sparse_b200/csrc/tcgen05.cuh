/*
 * The sm_100a instructions that the grouped products use, as inline PTX: barriers
 * in shared memory with bounded waits, tiled TMA loads (this GPU's memory, no
 * multicast), tensor memory, and tcgen05.mma with its two descriptors.
 */
#ifndef ACLSPARSE_B200_TCGEN05_CUH_
#define ACLSPARSE_B200_TCGEN05_CUH_

#include <cstdint>

#include <cuda.h>

namespace aclsp {

__device__ __forceinline__ uint32_t SmemAddress(const void* p)
{
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// One lane of a converged warp.  TMA and tcgen05 instructions take their operands from uniform registers: behind this
// branch the compiler knows that one lane is active, behind `lane == 0` it goes round the lanes for each of them
// (four MMAs and a commit then took 550 cycles to issue, and 240 this way).
__device__ __forceinline__ bool ElectLane()
{
    uint32_t elected;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(elected));
    return elected != 0;
}

__device__ __forceinline__ void BarInit(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void BarArrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}

// The address of the same variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t PeerAddress(uint32_t address, uint32_t rank)
{
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(there) : "r"(address), "r"(rank));
    return there;
}

__device__ __forceinline__ void BarArrivePeer(uint32_t peerBar)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(peerBar) : "memory");
}

__device__ __forceinline__ void StorePeer(uint32_t peerAddress, uint32_t value)
{
    asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(peerAddress), "r"(value) : "memory");
}

__device__ __forceinline__ void ClusterSync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

__device__ __forceinline__ void BarExpect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool BarTry(uint32_t bar, uint32_t parity)
{
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}

__device__ __forceinline__ uint64_t Nanoseconds()
{
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;\n" : "=l"(t));
    return t;
}

constexpr uint64_t kWaitLimitNs = 4000000000ull;  // where nothing else is asked for

// Waits for the phase of `parity` to end, `limit` nanoseconds at most.  `*gaveUp` is shared by the CTA: a wait that runs
// out sets it, and every other wait then gives up too, so that the CTA leaves in bounded time.
__device__ __forceinline__ bool BarWait(uint32_t bar, uint32_t parity, volatile uint32_t* gaveUp, uint64_t limit)
{
    // The clock is looked at rarely: reading it takes longer than most waits.
    uint64_t began = 0;
    for (uint32_t spin = 0;; ++spin) {
        if (BarTry(bar, parity)) {
            return true;
        }
        if (spin % 256u == 255u) {
            const uint64_t now = Nanoseconds();
            began = began == 0u ? now : began;
            if (*gaveUp != 0u || now - began > limit) {
                *gaveUp = 1u;
                return false;
            }
        }
    }
}

__device__ __forceinline__ void TmaPrefetch(const CUtensorMap* map)
{
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory");
}

// A box of a matrix or of a batch of them into this CTA's shared memory.  With kCtas == 2 the barrier may be the
// other CTA's of the pair.
template <uint32_t kCtas>
__device__ __forceinline__ void TmaLoad2(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y)
{
    if constexpr (kCtas == 2) {
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], "
            "[%2];\n" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
    } else {
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n" ::"r"(
                dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
    }
}

template <uint32_t kCtas>
__device__ __forceinline__ void TmaLoad3(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y, int32_t z)
{
    if constexpr (kCtas == 2) {
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, "
            "%5}], [%2];\n" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
    } else {
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n" ::"r"(
                dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
    }
}

// A box of shared memory into a batch of matrices; what lies outside them is not written.  The thread's stores form
// groups: at most kLeft of them may still be reading shared memory after the wait (none under way after StoresDone).
__device__ __forceinline__ void TmaStore3(const CUtensorMap* map, uint32_t src, int32_t x, int32_t y, int32_t z)
{
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];\n" ::"l"(map), "r"(src), "r"(x),
                 "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void StoreGroup() { asm volatile("cp.async.bulk.commit_group;\n" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void StoresRead()
{
    asm volatile("cp.async.bulk.wait_group.read %0;\n" ::"n"(kLeft) : "memory");
}
__device__ __forceinline__ void StoresDone() { asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory"); }

// A kernel launched with programmatic serialization starts while the one before it in the stream still runs: nothing of
// that one's may be read, nor anything written, before this wait.  The other call lets the next such kernel start.
__device__ __forceinline__ void WaitForPreviousKernel() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
// The same, for a kernel that reads through these pointers with __ldg: such loads count as loads of memory that never
// changes, which the compiler may move ahead of the wait, so the pointers are made known only behind it.
template <typename T>
__device__ __forceinline__ void KnownFromHere(T*& pointer)
{
    asm volatile("" : "+l"(pointer)::"memory");
}
template <typename... T>
__device__ __forceinline__ void WaitForPreviousKernel(T*&... pointers)
{
    WaitForPreviousKernel();
    (KnownFromHere(pointers), ...);
}
__device__ __forceinline__ void LetNextKernelStart() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }

// Writes of this thread to shared memory become visible to the asynchronous proxy (TMA, tcgen05.mma).
__device__ __forceinline__ void FenceProxyAsync()
{
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
}

// Tensor memory: of this CTA, or with kCtas == 2 of both CTAs of the pair, each of which calls.
template <uint32_t kCtas>
__device__ __forceinline__ void TmemAlloc(uint32_t smemResult, uint32_t columns)
{
    if constexpr (kCtas == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smemResult), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smemResult), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
}

template <uint32_t kCtas>
__device__ __forceinline__ void TmemFree(uint32_t address, uint32_t columns)
{
    if constexpr (kCtas == 2) {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(address), "r"(columns) : "memory");
    } else {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(address), "r"(columns) : "memory");
    }
}

__device__ __forceinline__ void TmemFenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void TmemFenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }

// `bar` gets one arrival, in both CTAs of a pair, when every tcgen05.mma that this thread has issued so far is done.
template <uint32_t kCtas>
__device__ __forceinline__ void MmaCommit(uint32_t bar)
{
    if constexpr (kCtas == 2) {
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar),
                     "h"(static_cast<uint16_t>(3))
                     : "memory");
    } else {
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
    }
}

// D (128 lanes per CTA x N columns of tensor memory at d) = A * B, or += when accumulate.  In a pair each CTA holds its
// own 128 rows of A and half of B's N columns, at the same shared-memory addresses.
#define ACLSP_MMA(group, kind)                                                                              \
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"                                                \
                 "tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n}\n" ::"r"(d),      \
                 "l"(a), "l"(b), "r"(shape), "r"(accumulate)                                                \
                 : "memory")
template <bool kInt8, uint32_t kCtas>
__device__ __forceinline__ void Mma(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, uint32_t accumulate)
{
    if constexpr (kInt8 && kCtas == 2) {
        ACLSP_MMA("2", "i8");
    } else if constexpr (kInt8) {
        ACLSP_MMA("1", "i8");
    } else if constexpr (kCtas == 2) {
        ACLSP_MMA("2", "f16");
    } else {
        ACLSP_MMA("1", "f16");
    }
}
#undef ACLSP_MMA

// 16 columns of this warp's 32 lanes: thread i gets lane i's.
__device__ __forceinline__ void TmemLoad16(uint32_t address, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(address));
}

// 32 bytes to a 32-byte aligned address: one whole sector.
__device__ __forceinline__ void Store32(void* p, const uint32_t (&r)[8])
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

__device__ __forceinline__ void TmemLoadWait() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }

// Shared-memory descriptor of an operand in rows of 128 bytes with the 128-byte swizzle, eight rows (1024 bytes) per
// swizzle pattern.  Summed index contiguous: a row holds one row of the operand, `blockBytes` is not used.  Otherwise a
// row holds 128 bytes of operand rows at one summed index, and the next 128 bytes of them lie `blockBytes` further on.
__device__ __forceinline__ uint64_t OperandDescriptor(uint32_t smem, uint32_t blockBytes)
{
    return static_cast<uint64_t>((smem >> 4) & 0x3FFFu) | static_cast<uint64_t>((blockBytes >> 4) & 0x3FFFu) << 16 |
           static_cast<uint64_t>(1024u >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// Instruction descriptor without N: dense, (128 per CTA) x N, sums fp32 (fp16 or bf16 operands) or int32 (int8 operands).
__device__ __forceinline__ uint32_t MmaShape(uint32_t ctas, bool int8, bool bf16, bool aTransposed, bool bTransposed)
{
    const uint32_t sums = int8 ? 2u : 1u;
    const uint32_t operand = int8 || bf16 ? 1u : 0u;  // int8: 1 signed; fp16: 0, bf16: 1
    return sums << 4 | operand << 7 | operand << 10 | (aTransposed ? 1u : 0u) << 15 | (bTransposed ? 1u : 0u) << 16 |
           ctas * (128u / 16u) << 24;
}
__device__ __forceinline__ uint32_t MmaColumns(uint32_t n) { return n / 8u << 17; }

}  // namespace aclsp

#endif  // ACLSPARSE_B200_TCGEN05_CUH_
