/*
 * Which part of which tile a worker - a CTA, or a pair of them - of the tensor-core
 * kernel works on, in order.  One warp of each CTA asks and tells the others
 * through shared memory.
 *
 * A tile is (128 per CTA) x tileColumns results; its summed index is cut into blocks of
 * 128 bytes.  Forward products run whole tiles in waves of one per worker, and what
 * is left after the last full wave is split along the summed index over all of them
 * where that saves more time than joining the partial sums costs.  Weight
 * gradients, whose tiles differ in length with their groups, run whole tiles
 * round robin when there are many and are split into equal runs of blocks when
 * there are few.
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
constexpr uint32_t kWholeTileWaves = 4;   // gradient: with this many tiles per worker nothing is split
constexpr uint32_t kGroupedCounters = kWholeTileWaves * kGroupedMaxCtas;

struct Segment {
    uint32_t group;
    uint32_t row0;      // forward: first row of the tile; gradient: first row of the group
    uint32_t rows;      // forward: rows of the tile; gradient: rows of the group
    uint32_t left;      // first result index along the lanes
    uint32_t right;     // gradient: first column
    uint32_t columns;   // results along the other dimension
    uint32_t block0;    // blocks [block0, block1) of the summed index
    uint32_t block1;
    uint32_t parts;     // workers that share the tile; 1: the result is complete here
    uint32_t counter;   // parts > 1: the tile's counter,
    uint32_t firstWorker;  // its first worker, whose partial sums are in slot firstSlot; worker w's after it in slot 2 * w
    uint32_t firstSlot;
    uint32_t slot;      // this worker's slot
};

struct Workers {
    uint32_t index;
    uint32_t count;
};

// The workers that share units [start, start + length) of runs of `per` units each.
__device__ __forceinline__ void SetParts(Segment* s, const Workers& w, uint32_t start, uint32_t length, uint32_t per,
                                         uint32_t counter)
{
    s->firstWorker = start / per;
    s->parts = (start + length - 1u) / per - s->firstWorker + 1u;
    // a worker's run holds two partial tiles at most: one that it continues (slot 0) and one that it begins (slot 1)
    s->firstSlot = 2u * s->firstWorker + (s->firstWorker * per < start ? 1u : 0u);
    s->slot = w.index == s->firstWorker ? s->firstSlot : 2u * w.index;
    s->counter = counter;
}

class ForwardSchedule {
public:
    __device__ __forceinline__ ForwardSchedule(const AclspGroupedParams& p, Workers workers, uint32_t tileLanes,
                                               uint32_t tileRows, uint32_t blocks, uint32_t joinBlocks)
        : walk_(p.offsets, p.groups, p.rows, tileRows, (p.n + tileLanes - 1u) / tileLanes), workers_(workers),
          tileLanes_(tileLanes), blocks_(blocks)
    {
        const uint32_t tiles = walk_.Count();
        walk_.Restart();
        waves_ = tiles / workers_.count;
        const uint32_t units = (tiles - waves_ * workers_.count) * blocks;
        per_ = (units + workers_.count - 1u) / workers_.count;
        per_ = per_ > kMinSplitBlocks ? per_ : kMinSplitBlocks;
        per_ = per_ + joinBlocks < blocks ? per_ : blocks;
        unit_ = workers_.index * per_ < units ? workers_.index * per_ : units;
        unitEnd_ = unit_ + per_ < units ? unit_ + per_ : units;
    }

    __device__ __forceinline__ bool Next(Segment* s)
    {
        uint32_t t;
        s->block0 = 0;
        s->block1 = blocks_;
        s->parts = 1;
        if (wave_ < waves_) {
            t = wave_ * workers_.count + workers_.index;
            ++wave_;
        } else {
            if (unit_ >= unitEnd_) {
                return false;
            }
            const uint32_t local = unit_ / blocks_;
            const uint32_t start = local * blocks_;
            t = waves_ * workers_.count + local;
            s->block0 = unit_ - start;
            const uint32_t until = s->block0 + (unitEnd_ - unit_);
            s->block1 = until < blocks_ ? until : blocks_;
            unit_ += s->block1 - s->block0;
            SetParts(s, workers_, start, blocks_, per_, local);
        }
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
    uint32_t waves_;
    uint32_t wave_ = 0;
    uint32_t per_;
    uint32_t unit_;
    uint32_t unitEnd_;
};

class GradientSchedule {
public:
    __device__ __forceinline__ GradientSchedule(const AclspGroupedParams& p, Workers workers, uint32_t tileLanes,
                                                uint32_t tileColumns, uint32_t blockRows)
        : workers_(workers), tileLanes_(tileLanes), offsets_(p.offsets), groups_(p.groups), rows_(p.rows), n_(p.n), tileColumns_(tileColumns), blockRows_(blockRows),
          across_((p.n + tileColumns - 1u) / tileColumns), perGroup_(across_ * ((p.m + tileLanes - 1u) / tileLanes))
    {
        total_ = groups_ * perGroup_;
        split_ = total_ < kWholeTileWaves * workers_.count;
        tile_ = workers_.index;
        if (split_) {
            Load();
            while (base_ + 32u < groups_) {
                base_ += 32u;
                Load();
            }
            const uint32_t units = end_;
            per_ = (units + workers_.count - 1u) / workers_.count;
            per_ = per_ > kMinSplitBlocks ? per_ : kMinSplitBlocks;
            unit_ = workers_.index * per_ < units ? workers_.index * per_ : units;
            unitEnd_ = unit_ + per_ < units ? unit_ + per_ : units;
            if (base_ != 0u) {
                base_ = 0;
                end_ = 0;
                Load();
            }
        }
    }

    __device__ __forceinline__ bool Next(Segment* s)
    {
        uint32_t inGroup;
        s->parts = 1;
        if (!split_) {
            if (tile_ >= total_) {
                return false;
            }
            s->group = tile_ / perGroup_;
            inGroup = tile_ % perGroup_;
            tile_ += workers_.count;
            uint32_t last;
            GroupRows(offsets_, s->group, rows_, &s->row0, &last);
            s->rows = last - s->row0;
            s->block0 = 0;
            s->block1 = (s->rows + blockRows_ - 1u) / blockRows_;
        } else {
            if (unit_ >= unitEnd_) {
                return false;
            }
            while (unit_ >= end_ && base_ + 32u < groups_) {
                base_ += 32u;
                Load();
            }
            const uint32_t ballot = __ballot_sync(0xFFFFFFFFu, unit_ < inclusive_);
            const int lane = __ffs(static_cast<int>(ballot)) - 1;
            s->group = base_ + static_cast<uint32_t>(lane);
            s->row0 = __shfl_sync(0xFFFFFFFFu, begin_, lane);
            s->rows = __shfl_sync(0xFFFFFFFFu, size_, lane);
            const uint32_t blocks = (s->rows + blockRows_ - 1u) / blockRows_;
            const uint32_t units = blocks > 0u ? blocks : 1u;
            const uint32_t first = __shfl_sync(0xFFFFFFFFu, inclusive_, lane) - units * perGroup_;
            inGroup = (unit_ - first) / units;
            const uint32_t start = first + inGroup * units;
            s->block0 = unit_ - start;
            const uint32_t until = s->block0 + (unitEnd_ - unit_);
            s->block1 = until < units ? until : units;
            unit_ += s->block1 - s->block0;
            if (blocks == 0u) {
                s->block1 = 0;  // an empty group: beta * C
            } else {
                SetParts(s, workers_, start, units, per_, s->group * perGroup_ + inGroup);
            }
        }
        s->left = inGroup / across_ * tileLanes_;
        s->right = inGroup % across_ * tileColumns_;
        s->columns = n_ - s->right < tileColumns_ ? n_ - s->right : tileColumns_;
        return true;
    }

private:
    // Units of 32 groups: a group has perGroup_ tiles of as many units as its rows make blocks, an empty one of one.
    __device__ __forceinline__ void Load()
    {
        const uint32_t lane = threadIdx.x % 32u;
        const uint32_t g = base_ + lane;
        begin_ = 0;
        size_ = 0;
        uint32_t sum = 0;
        if (g < groups_) {
            uint32_t last;
            GroupRows(offsets_, g, rows_, &begin_, &last);
            size_ = last - begin_;
            const uint32_t blocks = (size_ + blockRows_ - 1u) / blockRows_;
            sum = perGroup_ * (blocks > 0u ? blocks : 1u);
        }
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
    uint32_t total_;
    bool split_;
    uint32_t tile_;
    uint32_t per_ = 1;
    uint32_t unit_ = 0;
    uint32_t unitEnd_ = 0;
    uint32_t base_ = 0;
    uint32_t end_ = 0;
    uint32_t begin_ = 0;
    uint32_t size_ = 0;
    uint32_t inclusive_ = 0;
};

}  // namespace aclsp

#endif  // ACLSPARSE_B200_GROUPED_SCHEDULE_CUH_
