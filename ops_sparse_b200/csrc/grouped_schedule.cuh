/*
 * Which part of which tile a worker - a CTA, or a pair of them - of the tensor-core
 * kernel works on, in order.  One warp of each CTA asks and tells the others
 * through shared memory.
 *
 * A tile is (128 per CTA) x tileColumns results; its summed index is cut into blocks
 * of 128 bytes.  Forward products run whole tiles in waves of one per worker; the
 * tiles left after the last full wave are each split along the summed index into as
 * many equal parts as there are workers for them, where that saves more time than
 * joining the parts' sums costs.  Weight gradients, whose tiles differ in length with
 * their groups, are split where there are few of them, into parts of about the same
 * length.  A tile's parts are equal and start together, so that they also end
 * together: with runs of blocks that ignore the tiles' borders every worker is busy to
 * the last, but one that begins a tile after the end of another arrives late, alone,
 * and the others' sums wait for it (512 x 512 from 16384 rows: 73 us).
 */
#ifndef ACLSPARSE_B200_GROUPED_SCHEDULE_CUH_
#define ACLSPARSE_B200_GROUPED_SCHEDULE_CUH_

#include <cstdint>

#include "aclsparse_b200_kernels.h"
#include "group_walk.cuh"

namespace aclsp {

constexpr uint32_t kTileLanes = 128;      // results along the first operand per CTA: lanes of tensor memory
constexpr uint32_t kGroupedMaxCtas = 148;
constexpr uint32_t kMinSplitBlocks = 4;   // shortest run of blocks worth a worker of its own
constexpr uint32_t kWholeTileWaves = 2;   // gradient: with this many tiles per worker nothing is split
// A counter per quarter of a tile's lanes in a CTA and sixteen of its columns.
constexpr uint32_t kTileCounters = 4u * 256u / 16u;
constexpr uint32_t kGroupedCounters = kWholeTileWaves * kGroupedMaxCtas * kTileCounters;

struct Segment {
    uint32_t group;
    uint32_t row0;      // forward: first row of the tile; gradient: first row of the group
    uint32_t rows;      // forward: rows of the tile; gradient: rows of the group
    uint32_t left;      // first result index along the lanes
    uint32_t right;     // gradient: first column
    uint32_t columns;   // results along the other dimension
    uint32_t block0;    // blocks [block0, block1) of the summed index
    uint32_t block1;
    uint32_t parts;     // parts of the tile; 1: the result is complete here
    uint32_t part;      // which one this is
    uint32_t slot;      // parts > 1: where its sums are left; those of the tile's other parts lie around it, in order
    uint32_t counter;   // and the tile's counters
};

struct Workers {
    uint32_t index;
    uint32_t count;
};

class ForwardSchedule {
public:
    __device__ __forceinline__ ForwardSchedule(const AclspGroupedParams& p, Workers workers, uint32_t tileLanes,
                                               uint32_t tileRows, uint32_t blocks, uint32_t joinBlocks)
        : walk_(p.offsets, p.groups, p.rows, tileRows, (p.n + tileLanes - 1u) / tileLanes), workers_(workers),
          tileLanes_(tileLanes), blocks_(blocks), length_(blocks)
    {
        tiles_ = walk_.Count();
        tile_ = workers.index;
        whole_ = tiles_ / workers.count * workers.count;
        const uint32_t left = tiles_ - whole_;
        // one part per SM: a second one there would only share its loads (one int8 row, 4096 x 4096: 8.9 us, 9.4 with two)
        const uint32_t most = workers.count < kGroupedMaxCtas ? workers.count : kGroupedMaxCtas;
        if (left != 0u && 2u * left <= most && blocks > kMinSplitBlocks + joinBlocks) {
            const uint32_t parts = most / left;
            const uint32_t length = (blocks + parts - 1u) / parts;
            length_ = length > kMinSplitBlocks ? length : kMinSplitBlocks;
            length_ = length_ + joinBlocks < blocks ? length_ : blocks;
        }
        parts_ = length_ < blocks ? (blocks + length_ - 1u) / length_ : 1u;
    }

    __device__ __forceinline__ bool Next(Segment* s)
    {
        uint32_t t = tile_;
        s->block0 = 0;
        s->block1 = blocks_;
        s->parts = 1;
        s->part = 0;
        if (t >= whole_ && parts_ > 1u) {
            // the parts of what is left of the tiles, one per worker
            const uint32_t local = workers_.index / parts_;
            t = whole_ + local;
            if (done_ || t >= tiles_) {
                return false;
            }
            done_ = true;
            s->parts = parts_;
            s->part = workers_.index - local * parts_;
            s->slot = workers_.index;
            s->counter = local;
            s->block0 = s->part * length_;
            s->block1 = s->block0 + length_ < blocks_ ? s->block0 + length_ : blocks_;
        } else if (t >= tiles_) {
            return false;
        }
        tile_ += workers_.count;
        GroupTile tile;
        if (!walk_.Find(t, &tile)) {
            return false;
        }
        s->group = tile.group;
        s->row0 = tile.row0;
        s->rows = tile.count;
        s->left = tile.across * tileLanes_;
        s->right = 0;
        s->columns = tile.count;
        return true;
    }

private:
    GroupWalk walk_;
    Workers workers_;
    uint32_t tileLanes_;
    uint32_t blocks_;
    uint32_t length_;  // of a part
    uint32_t parts_;
    uint32_t tiles_;
    uint32_t whole_;   // tiles in full waves
    uint32_t tile_;
    bool done_ = false;
};

class GradientSchedule {
public:
    __device__ __forceinline__ GradientSchedule(const AclspGroupedParams& p, Workers workers, uint32_t tileLanes,
                                                uint32_t tileColumns, uint32_t blockRows, uint32_t joinBlocks)
        : workers_(workers), tileLanes_(tileLanes), offsets_(p.offsets), groups_(p.groups), rows_(p.rows), n_(p.n),
          tileColumns_(tileColumns), blockRows_(blockRows), across_((p.n + tileColumns - 1u) / tileColumns),
          perGroup_(across_ * ((p.m + tileLanes - 1u) / tileLanes))
    {
        const uint32_t tiles = groups_ * perGroup_;
        next_ = workers_.index;
        // Few tiles: parts so short that there are just no more of them than the workers take in one turn (in two, where
        // there are more tiles than workers).
        if (tiles < kWholeTileWaves * workers_.count) {
            const uint32_t most = tiles <= workers_.count ? workers_.count : kWholeTileWaves * workers_.count;
            uint32_t longest;
            uint32_t all;
            Sum(&all, &longest);
            // ceil(blocks / length) summed over the tiles is at most all / length + tiles
            uint32_t length = most > tiles ? (all + most - tiles - 1u) / (most - tiles) : longest;
            length = length > kMinSplitBlocks ? length : kMinSplitBlocks;
            length_ = length + joinBlocks < longest ? length : length_;
        }
        Load();
    }

    __device__ __forceinline__ bool Next(Segment* s)
    {
        while (next_ >= end_) {
            if (base_ + 32u >= groups_) {
                return false;
            }
            base_ += 32u;
            Load();
        }
        const uint32_t ballot = __ballot_sync(0xFFFFFFFFu, next_ < inclusive_);
        const int lane = __ffs(static_cast<int>(ballot)) - 1;
        s->group = base_ + static_cast<uint32_t>(lane);
        s->row0 = __shfl_sync(0xFFFFFFFFu, begin_, lane);
        s->rows = __shfl_sync(0xFFFFFFFFu, size_, lane);
        const uint32_t blocks = (s->rows + blockRows_ - 1u) / blockRows_;
        const uint32_t parts = Parts(blocks, length_);
        const uint32_t inGroup = next_ - (__shfl_sync(0xFFFFFFFFu, inclusive_, lane) - parts * perGroup_);
        const uint32_t tile = inGroup / parts;
        s->parts = parts;
        s->part = inGroup - tile * parts;
        s->slot = next_;
        s->counter = s->group * perGroup_ + tile;
        const uint32_t length = (blocks + parts - 1u) / parts;
        s->block0 = s->part * length < blocks ? s->part * length : blocks;
        s->block1 = s->block0 + length < blocks ? s->block0 + length : blocks;
        s->left = tile / across_ * tileLanes_;
        s->right = tile % across_ * tileColumns_;
        s->columns = n_ - s->right < tileColumns_ ? n_ - s->right : tileColumns_;
        next_ += workers_.count;
        return true;
    }

private:
    // Parts of a tile: none longer than `length`, and none empty.  An empty group's tile is one part of no blocks.
    static __device__ __forceinline__ uint32_t Parts(uint32_t blocks, uint32_t length)
    {
        if (blocks <= length) {
            return 1u;
        }
        const uint32_t parts = (blocks + length - 1u) / length;
        const uint32_t even = (blocks + parts - 1u) / parts;
        return (blocks + even - 1u) / even;
    }

    // The blocks of all tiles, and the longest tile's.
    __device__ __forceinline__ void Sum(uint32_t* blocks, uint32_t* longest) const
    {
        uint32_t sum = 0;
        uint32_t top = 0;
        uint32_t reached = 0;
        for (uint32_t base = 0; base < groups_; base += 32u) {
            uint32_t begin, size;
            RowsOfGroups(offsets_, groups_, rows_, base, &reached, &begin, &size);
            const uint32_t own = (size + blockRows_ - 1u) / blockRows_;
            sum += perGroup_ * own;
            top = own > top ? own : top;
        }
        *blocks = __reduce_add_sync(0xFFFFFFFFu, sum);
        *longest = __reduce_max_sync(0xFFFFFFFFu, top);
    }

    // The parts of 32 groups, numbered.
    __device__ __forceinline__ void Load()
    {
        const uint32_t lane = threadIdx.x % 32u;
        RowsOfGroups(offsets_, groups_, rows_, base_, &reached_, &begin_, &size_);
        uint32_t sum = base_ + lane < groups_ ? perGroup_ * Parts((size_ + blockRows_ - 1u) / blockRows_, length_) : 0u;
        for (int d = 1; d < 32; d *= 2) {
            const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, sum, d);
            sum += static_cast<int>(lane) >= d ? up : 0u;
        }
        inclusive_ = sum + end_;
        end_ = __shfl_sync(0xFFFFFFFFu, inclusive_, 31);
    }

    Workers workers_;
    uint32_t tileLanes_;
    const int32_t* offsets_;
    uint32_t groups_;
    uint32_t rows_;
    uint32_t n_;
    uint32_t tileColumns_;
    uint32_t blockRows_;
    uint32_t across_;
    uint32_t perGroup_;
    uint32_t length_ = 0xFFFFFFFFu;  // longest part
    uint32_t next_;                  // number of the next part
    uint32_t base_ = 0;
    uint32_t end_ = 0;
    uint32_t reached_ = 0;  // largest offset before the groups that the lanes hold
    uint32_t begin_ = 0;
    uint32_t size_ = 0;
    uint32_t inclusive_ = 0;
};

}  // namespace aclsp

#endif  // ACLSPARSE_B200_GROUPED_SCHEDULE_CUH_
