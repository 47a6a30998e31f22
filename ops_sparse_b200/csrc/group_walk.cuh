/*
 * How a kernel finds its tile of a grouped product.  The sizes of the groups are
 * known on the device only, so the tiles are numbered there: group after group,
 * a group of `size` rows being cut into ceil(size / tileRows) pieces of nearly
 * equal length (a multiple of 16 rows, so that no piece pays for a much larger
 * neighbour), each piece with `across` tiles along the other dimension.
 *
 * A warp walks the groups 32 at a time: each lane loads two offsets, a running
 * maximum makes them ascending whatever the array holds (every row is in one
 * group at most, so the number of tiles stays bounded), a prefix sum numbers the
 * tiles.  Tiles are asked for in ascending order, so the walk only goes forward.
 */
#ifndef ACLSPARSE_B200_GROUP_WALK_CUH_
#define ACLSPARSE_B200_GROUP_WALK_CUH_

#include <cstdint>

namespace aclsp {

// An offset inside the matrix.
__device__ __forceinline__ uint32_t ClampOffset(int32_t v, uint32_t rows)
{
    return v < 0 ? 0u : (static_cast<uint32_t>(v) > rows ? rows : static_cast<uint32_t>(v));
}

// The largest value of the lanes up to this one.
__device__ __forceinline__ uint32_t RunningMax(uint32_t v)
{
    for (uint32_t d = 1; d < 32u; d *= 2u) {
        const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, v, d);
        v = threadIdx.x % 32u >= d && up > v ? up : v;
    }
    return v;
}

// The rows of 32 groups from `base` on, one per lane.  Ends ascend whatever the array holds: none is below the largest
// offset before it, of which *reached is the one before these groups, and then behind them.  Called by a whole warp.
__device__ __forceinline__ void RowsOfGroups(const int32_t* offsets, uint32_t groups, uint32_t rows, uint32_t base,
                                             uint32_t* reached, uint32_t* begin, uint32_t* size)
{
    const uint32_t lane = threadIdx.x % 32u;
    const uint32_t g = base + lane;
    uint32_t first = 0;
    uint32_t last = 0;
    if (offsets == nullptr) {
        last = g == 0 ? rows : 0u;
    } else if (g < groups) {
        first = ClampOffset(__ldg(offsets + g), rows);
        last = ClampOffset(__ldg(offsets + g + 1), rows);
    }
    const uint32_t top = RunningMax(first > last ? first : last);
    uint32_t before = __shfl_up_sync(0xFFFFFFFFu, top, 1);
    before = lane == 0 ? 0u : before;
    before = before > *reached ? before : *reached;
    *begin = first > before ? first : before;
    const uint32_t until = last > *begin ? last : *begin;
    *size = g < groups ? until - *begin : 0u;
    const uint32_t all = __shfl_sync(0xFFFFFFFFu, top, 31);
    *reached = all > *reached ? all : *reached;
}

// One tile: `count` rows from row `row0` on, of group `group`; `across` is its place along the other dimension.
struct GroupTile {
    uint32_t group;
    uint32_t row0;
    uint32_t count;
    uint32_t across;
};

class GroupWalk {
public:
    __device__ __forceinline__ GroupWalk(const int32_t* offsets, uint32_t groups, uint32_t rows, uint32_t tileRows,
                                         uint32_t across)
        : offsets_(offsets), groups_(groups), rows_(rows), tileRows_(tileRows), across_(across)
    {
        Load();
    }

    // Tile `t`; false when there are fewer.  Called by a whole warp, with ascending t.
    __device__ __forceinline__ bool Find(uint32_t t, GroupTile* tile)
    {
        while (t >= end_) {
            if (base_ + 32u >= groups_) {
                return false;
            }
            base_ += 32u;
            Load();
        }
        // the lane whose tiles include t: the first one whose inclusive prefix is beyond it
        const uint32_t ballot = __ballot_sync(0xFFFFFFFFu, t < inclusive_);
        const int lane = __ffs(static_cast<int>(ballot)) - 1;
        const uint32_t begin = __shfl_sync(0xFFFFFFFFu, begin_, lane);
        const uint32_t size = __shfl_sync(0xFFFFFFFFu, size_, lane);
        const uint32_t pieces = (size + tileRows_ - 1u) / tileRows_;
        tile->group = base_ + static_cast<uint32_t>(lane);
        tile->row0 = begin;
        if (pieces == 1u) {  // a decoding batch's case, where each division shows
            tile->across = t - (__shfl_sync(0xFFFFFFFFu, inclusive_, lane) - across_);
            tile->count = size;
            return true;
        }
        const uint32_t local = t - (__shfl_sync(0xFFFFFFFFu, inclusive_, lane) - pieces * across_);
        // Bands of eight pieces, all tiles across for each: the tiles that run at one time share their operands
        // (a wave of 148 tiles reads about 8 + 19 different ones), also in a group far larger than the L2 cache.
        const uint32_t band = local / (kBand * across_);
        const uint32_t inBand = local - band * kBand * across_;
        const uint32_t width = pieces - band * kBand < kBand ? pieces - band * kBand : kBand;
        const uint32_t piece = band * kBand + inBand % width;
        const uint32_t length = ((size + pieces - 1u) / pieces + 15u) / 16u * 16u;
        const uint32_t from = piece * length < size ? piece * length : size;
        tile->across = inBand / width;
        tile->row0 = begin + from;
        tile->count = size - from < length ? size - from : length;
        return true;
    }

    // Number of tiles in all groups.  Asked for before the first tile, so each lane takes eight groups at a time, whose
    // loads are under way together (256 rows over 512 groups, 1024 x 1024 matrices: 69 us, 78 with a walk of 32 groups at a
    // time).
    __device__ __forceinline__ uint32_t Count() const
    {
        constexpr uint32_t kEach = 8;
        if (groups_ <= 32u) {
            return end_;
        }
        uint32_t sum = 0;
        uint32_t reached = 0;
        for (uint32_t base = 0; base < groups_; base += 32u * kEach) {
            const uint32_t g0 = base + threadIdx.x % 32u * kEach;
            uint32_t bounds[kEach + 1];
            uint32_t top = 0;
#pragma unroll
            for (uint32_t i = 0; i <= kEach; ++i) {
                bounds[i] = g0 < groups_ && g0 + i <= groups_ ? ClampOffset(__ldg(offsets_ + g0 + i), rows_) : 0u;
            }
#pragma unroll
            for (uint32_t i = 0; i <= kEach; ++i) {
                top = bounds[i] > top ? bounds[i] : top;
            }
            top = RunningMax(top);
            uint32_t before = __shfl_up_sync(0xFFFFFFFFu, top, 1);
            before = threadIdx.x % 32u == 0u || before < reached ? reached : before;
#pragma unroll
            for (uint32_t i = 0; i < kEach; ++i) {
                const uint32_t begin = bounds[i] > before ? bounds[i] : before;
                const uint32_t size = bounds[i + 1] > begin ? bounds[i + 1] - begin : 0u;  // none behind the last group
                sum += (size + tileRows_ - 1u) / tileRows_;
                before = begin > bounds[i + 1] ? begin : bounds[i + 1];
            }
            const uint32_t last = __shfl_sync(0xFFFFFFFFu, top, 31);
            reached = last > reached ? last : reached;
        }
        return __reduce_add_sync(0xFFFFFFFFu, sum) * across_;
    }

private:
    static constexpr uint32_t kBand = 8;

    __device__ __forceinline__ void Load()
    {
        const uint32_t lane = threadIdx.x % 32u;
        RowsOfGroups(offsets_, groups_, rows_, base_, &reached_, &begin_, &size_);
        uint32_t sum = (size_ + tileRows_ - 1u) / tileRows_ * across_;
        for (int d = 1; d < 32; d *= 2) {
            const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, sum, d);
            sum += static_cast<int>(lane) >= d ? up : 0u;
        }
        inclusive_ = sum + end_;
        end_ = __shfl_sync(0xFFFFFFFFu, inclusive_, 31);
    }

    const int32_t* offsets_;
    uint32_t groups_;
    uint32_t rows_;
    uint32_t tileRows_;
    uint32_t across_;
    uint32_t base_ = 0;       // first group of the 32 that the lanes hold
    uint32_t end_ = 0;        // tiles of all groups up to the last of them
    uint32_t reached_ = 0;    // largest offset before them
    uint32_t begin_ = 0;      // this lane's group: first row, rows, tiles up to its end
    uint32_t size_ = 0;
    uint32_t inclusive_ = 0;
};

// The rows of one group after another, for a kernel whose warps all ask for the same groups in ascending order; the same
// rows as above.
class GroupRows {
public:
    __device__ __forceinline__ GroupRows(const int32_t* offsets, uint32_t rows) : offsets_(offsets), rows_(rows) {}

    __device__ __forceinline__ void Find(uint32_t g, uint32_t* first, uint32_t* last)
    {
        if (offsets_ == nullptr) {
            *first = 0;
            *last = rows_;
            return;
        }
        uint32_t top = 0;
        for (uint32_t i = seen_ + threadIdx.x % 32u; i <= g; i += 32u) {
            const uint32_t v = ClampOffset(__ldg(offsets_ + i), rows_);
            top = v > top ? v : top;
        }
        top = __reduce_max_sync(0xFFFFFFFFu, top);
        reached_ = top > reached_ ? top : reached_;
        seen_ = g + 1u;
        const uint32_t end = ClampOffset(__ldg(offsets_ + g + 1), rows_);
        *first = reached_;
        *last = end > reached_ ? end : reached_;
    }

private:
    const int32_t* offsets_;
    uint32_t rows_;
    uint32_t seen_ = 0;     // offsets that have been looked at
    uint32_t reached_ = 0;  // the largest of them
};

}  // namespace aclsp

#endif  // ACLSPARSE_B200_GROUP_WALK_CUH_
