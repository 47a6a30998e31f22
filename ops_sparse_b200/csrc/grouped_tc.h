/* Internal: the tensor-core form of the grouped products (grouped_tc_kernels.cu) and the layout of their buffer:
 * a header whose first word counts waits that ran out, the split tiles' counters, then partial sums. */
#ifndef ACLSPARSE_B200_GROUPED_TC_H_
#define ACLSPARSE_B200_GROUPED_TC_H_

#include <cstdint>

#include <cuda_runtime.h>

#include "aclsparse_b200_kernels.h"
#include "grouped_schedule.cuh"

constexpr uint32_t kGroupedHeaderWords = 16;
// Where the partial sums begin; what is before them is what Preprocess clears.
constexpr uint32_t kGroupedCountersEnd = 4u * (kGroupedHeaderWords + aclsp::kGroupedCounters);
// What writing and joining partial sums costs, in blocks of the summed index: a tile is split only where more is saved
// (4 rows of 4 groups, 1024 x 1024 matrices, tensor cores: 8.45 us with 8, 8.8 with 12; 8192 rows through 2048 x 4096
// ones, 256 columns: 124 us with 48, 126 with 24, 129 with 8).
constexpr uint32_t kJoinBlocks = 8;
constexpr uint32_t kJoinBlocksWide = 48;

// Forward products of so few rows that a kernel without tensor cores (grouped_kernels.cu) is faster, where the bases too
// are on multiples of 16 bytes.  They need no partial sums.
bool AclspGroupedFewRows(const AclspGroupedParams& p);

// Columns of a tile: rows of a group that one tile takes (forward), columns of C_g (gradient).
uint32_t AclspGroupedColumns(const AclspGroupedParams& p);

// An operand as rows of contiguous elements, one batch of them per group (forward's dense matrix) or a single one.
struct AclspGroupedOperand {
    uint64_t rowElements;
    uint64_t rows;
    uint64_t batches;
    uint64_t ld;
    uint64_t batchStride;
    // Rows that do not start on multiples of 16 bytes, which a tensor map asks for, are copied to ones that do, behind
    // the partial sums; 0 where there is no need.
    uint64_t copyBytes;
    uint64_t copyOffset;
};
struct AclspGroupedOperands {
    AclspGroupedOperand left;   // along the lanes: B, or A in the gradient
    AclspGroupedOperand right;  // along the columns
    uint64_t bufferBytes;
};
AclspGroupedOperands AclspGroupedDescribe(const AclspGroupedParams& p);

// Copies the operands that need it, in one launch, and makes bases, ld and batchStride those of the copies.  Batches
// whose group has no rows are left out.
void AclspGroupedCopyRows(AclspGroupedOperands* o, const void** left, const void** right, void* buffer,
                          const AclspGroupedParams& p, cudaStream_t stream);

// Launches the product; false, and nothing launched, where a base is not 16-byte aligned, there is nothing to sum over
// or the sizes are too large to number tiles and blocks.
bool AclspGroupedTensorLaunch(const void* a, const void* b, void* c, void* buffer, const AclspGroupedParams& p,
                              cudaStream_t stream);

// CTAs on the current device that gave up a wait since the program began; waits for the stream.
cudaError_t AclspGroupedTotalWaitFailures(cudaStream_t stream, uint32_t* count);

// SMs of the current device, 0 when none can be queried (handle.cpp).
uint32_t AclspSmCount();

#endif  // ACLSPARSE_B200_GROUPED_TC_H_
