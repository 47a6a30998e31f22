/*
 * Operands that a tensor map cannot describe (rows that do not start on 16-byte
 * boundaries) on their way to the tensor cores: warps read them in 4-byte words,
 * shift the bytes into place and write the swizzled rows that tcgen05.mma reads.
 *
 * A warp reads one row's 128 bytes with one load, 32 neighbouring words, whatever
 * the row's alignment; sixteen rows are in flight before the first one is needed.
 * The word behind the 32 that a shifted row needs comes with one more load for all
 * sixteen, lane j's for row j.  Words that reach over the matrix's first or last byte
 * are put together from its bytes, so that nothing outside it is read.
 */
#ifndef ACLSPARSE_B200_PANEL_LOAD_CUH_
#define ACLSPARSE_B200_PANEL_LOAD_CUH_

#include <cstdint>

namespace aclsp {

constexpr uint32_t kPanelWarps = 8;   // as many as rows of the swizzle pattern
constexpr uint32_t kPanelBatch = 16;  // rows that a warp has in flight

// Rows of 128 bytes in shared memory and where they come from.  Shared row r holds matrix row origin + r % kBlockRows,
// the 128 bytes from byte firstByte + r / kBlockRows * 128 on; rows beyond `rows` matrix rows and bytes beyond rowBytes
// are zeros.
struct Panel {
    const unsigned char* base;
    const unsigned char* end;  // one past the matrix's last byte
    int64_t pitch;             // bytes from row to row
    uint32_t origin;
    uint32_t rows;
    int64_t firstByte;
    int64_t rowBytes;
};

// A word of the matrix that may reach over one of its ends (rare: not worth registers where it is called).
__device__ __noinline__ uint32_t WordFromBytes(const unsigned char* at, const unsigned char* begin, const unsigned char* end)
{
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (at + i >= begin && at + i < end) {
            v |= static_cast<uint32_t>(__ldg(at + i)) << (8 * i);
        }
    }
    return v;
}

// A word, or zero, without a branch: sixteen of these are to be in flight together.
__device__ __forceinline__ uint32_t WordIf(bool wanted, const unsigned char* at)
{
    uint32_t v;
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %2, 0;\nmov.b32 %0, 0;\n@p ld.global.nc.b32 %0, [%1];\n}\n"
                 : "=r"(v)
                 : "l"(at), "r"(wanted ? 1u : 0u));
    return v;
}

// What a warp's sixteen rows warp, warp + 8, .. of a panel have in common.  They are eight rows of the matrix apart, a
// multiple of 8 bytes: all of them start at the same byte of a word, and lie at the same place of the swizzle pattern.
template <uint32_t kBlockRows>
struct PanelLane {
    static constexpr uint32_t kPerBlock = kBlockRows / kPanelWarps;  // of a warp's rows
    static constexpr uint32_t kBlocks = kPanelBatch / kPerBlock;

    const unsigned char* first;  // byte 0 of row `warp`
    uint32_t shift;              // of it in its word
    uint32_t rows;               // of the warp's rows: those that the matrix has (per block)
    uint32_t stored;             // and those that the panel has

    __device__ __forceinline__ PanelLane(const Panel& p, uint32_t warp, uint32_t panelRows)
        : first(p.base + static_cast<int64_t>(p.origin + warp) * p.pitch + p.firstByte),
          shift(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(first)) & 3u),
          rows(p.rows > warp ? (p.rows - warp + kPanelWarps - 1u) / kPanelWarps : 0u),
          stored(panelRows > warp ? (panelRows - warp + kPanelWarps - 1u) / kPanelWarps : 0u)
    {
    }
    // Whether the warp's row j is to be read.
    __device__ __forceinline__ bool Has(uint32_t j) const { return j % kPerBlock < rows && j < stored; }
    // Bytes of a row in block i that are the matrix's.
    static __device__ __forceinline__ int32_t Valid(const Panel& p, uint32_t i)
    {
        const int64_t left = p.rowBytes - p.firstByte - 128 * static_cast<int64_t>(i);
        return left <= 0 ? 0 : (left < 128 ? static_cast<int32_t>(left) : 128);
    }
};

// The words of a warp's rows: this lane's of each, and the one behind row `lane`'s.
struct PanelWords {
    uint32_t word[kPanelBatch];
    uint32_t behind;
};

template <uint32_t kBlockRows>
__device__ __forceinline__ void PanelRead(const Panel& p, uint32_t warp, uint32_t lane, uint32_t panelRows, PanelWords* w)
{
    using Lane = PanelLane<kBlockRows>;
    const Lane l(p, warp, panelRows);
    const int64_t step = p.pitch * kPanelWarps;
    // Whether a word of this warp's may reach over an end of the matrix: in its first row, or in its last one.
    const bool atEnd = l.first - l.shift < p.base ||
                       l.first + static_cast<int64_t>(Lane::kPerBlock - 1u) * step + 128u * Lane::kBlocks + 4u > p.end;
    const uint32_t ownRow = lane % kPanelBatch;
    const unsigned char* own = l.first - l.shift + static_cast<int64_t>(ownRow % Lane::kPerBlock) * step +
                               (ownRow / Lane::kPerBlock * 128u + 128u);
    const int32_t ownValid = Lane::kBlocks == 1u || ownRow < Lane::kPerBlock ? Lane::Valid(p, 0) : Lane::Valid(p, 1);
    const bool ownWanted = lane < kPanelBatch && l.Has(ownRow) && ownValid + static_cast<int32_t>(l.shift) > 128;
    w->behind = WordIf(ownWanted && !atEnd, own);
#pragma unroll
    for (uint32_t i = 0; i < Lane::kBlocks; ++i) {
        const int32_t valid = Lane::Valid(p, i);
        const bool wanted = valid > 0 && static_cast<int32_t>(4u * lane) < valid + static_cast<int32_t>(l.shift) && !atEnd;
        const unsigned char* at = l.first - l.shift + (i * 128u + 4u * lane);
#pragma unroll
        for (uint32_t j = i * Lane::kPerBlock; j < (i + 1u) * Lane::kPerBlock; ++j) {
            w->word[j] = WordIf(wanted && l.Has(j), at);
            at += step;
        }
    }
    if (atEnd) {
        if (ownWanted) {
            w->behind = WordFromBytes(own, p.base, p.end);
        }
#pragma unroll
        for (uint32_t i = 0; i < Lane::kBlocks; ++i) {
            const int32_t valid = Lane::Valid(p, i);
            const bool wanted = valid > 0 && static_cast<int32_t>(4u * lane) < valid + static_cast<int32_t>(l.shift);
            const unsigned char* at = l.first - l.shift + (i * 128u + 4u * lane);
#pragma unroll
            for (uint32_t j = i * Lane::kPerBlock; j < (i + 1u) * Lane::kPerBlock; ++j) {
                const bool inside = at >= p.base && at + 4 <= p.end;
                w->word[j] = WordIf(wanted && l.Has(j) && inside, at);
                if (wanted && l.Has(j) && !inside) {
                    w->word[j] = WordFromBytes(at, p.base, p.end);
                }
                at += step;
            }
        }
    }
}

template <uint32_t kBlockRows>
__device__ __forceinline__ void PanelWrite(const Panel& p, uint32_t warp, uint32_t lane, uint32_t panelRows,
                                           const PanelWords& w, uint32_t smem)
{
    using Lane = PanelLane<kBlockRows>;
    const Lane l(p, warp, panelRows);
    // the 128-byte swizzle: 16-byte pieces of a row change places with the row's number modulo 8
    const uint32_t to = smem + warp * 128u + ((lane / 4u ^ warp) << 4) + lane % 4u * 4u;
#pragma unroll
    for (uint32_t i = 0; i < Lane::kBlocks; ++i) {
        const int32_t mine = Lane::Valid(p, i) - static_cast<int32_t>(4u * lane);
        const uint32_t mask = mine >= 4 ? 0xFFFFFFFFu : (mine <= 0 ? 0u : (1u << (8 * mine)) - 1u);
#pragma unroll
        for (uint32_t j = i * Lane::kPerBlock; j < (i + 1u) * Lane::kPerBlock; ++j) {
            const uint32_t behind = __shfl_sync(0xFFFFFFFFu, w.behind, static_cast<int>(j));
            const uint32_t next = __shfl_down_sync(0xFFFFFFFFu, w.word[j], 1);
            const uint32_t v = __funnelshift_r(w.word[j], lane == 31u ? behind : next, 8u * l.shift) & mask;
            if (j < l.stored) {
                asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(to + j * kPanelWarps * 128u), "r"(v) : "memory");
            }
        }
    }
}

}  // namespace aclsp

#endif  // ACLSPARSE_B200_PANEL_LOAD_CUH_
