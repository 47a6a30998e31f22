/* Internal: the tensor-core form of the grouped products (grouped_tc_kernels.cu) and the layout of their buffer:
 * a header whose first word counts waits that ran out, the split tiles' counters, then partial sums. */
#ifndef ACLSPARSE_B200_GROUPED_TC_H_
#define ACLSPARSE_B200_GROUPED_TC_H_

#include <cstdint>

#include <cuda_runtime.h>

#include "aclsparse_b200_kernels.h"

constexpr uint32_t kGroupedHeaderWords = 16;
// What writing and joining partial sums costs, in blocks of the summed index: a tile is split only where more is saved.
constexpr uint32_t kJoinBlocks = 8;
constexpr uint32_t kJoinBlocksWide = 48;  // tiles of 256 columns

// Columns of a tile: rows of a group that one tile takes (forward), columns of C_g (gradient).
uint32_t AclspGroupedColumns(const AclspGroupedParams& p);

// Launches the product; false, and nothing launched, where there is nothing to sum over or the tiles are too many to
// number.
bool AclspGroupedTensorLaunch(const void* a, const void* b, void* c, void* buffer, const AclspGroupedParams& p,
                              cudaStream_t stream);

// SMs of the current device, 0 when none can be queried (handle.cpp).
uint32_t AclspSmCount();

#endif  // ACLSPARSE_B200_GROUPED_TC_H_
