/*
 * B200 additions to the aclsparse API.  The reference library drives one
 * device through one stream and has no multi-device code, so the entry points
 * in this header have no counterpart there; they carry the pieces of the
 * multi-GPU path that have to run where the matrix lives, a product that needs
 * no buffer, and the dense products of ragged row groups (experts) that stand
 * between the sparse operators of a mixture-of-experts layer.
 */
#ifndef ACLSPARSE_B200_EXT_H_
#define ACLSPARSE_B200_EXT_H_

#include "cann_ops_sparse.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The library is built with hidden visibility: only what this header declares is exported. */
#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/* Row-block boundaries that balance the non-zeros of a CSR matrix over `parts`
 * devices.  Writes parts+1 int32 values to the DEVICE array `bounds`
 * (asynchronously, on the handle's stream):
 *     bounds[g] = min{ r : rowOffsets[r] - base >= ceil(g * nnz / parts) },  bounds[parts] = rows.
 * Device g then owns rows [bounds[g], bounds[g+1]); x (or B) is replicated and
 * y (or C) is reassembled by an all-gather.  Needs int32 row offsets with unit
 * stride.  No counterpart in the reference. */
aclsparseStatus_t aclsparseB200RowBlockBounds(aclsparseHandle_t handle, aclsparseConstSpMatDescr_t matA, int parts,
                                              void* bounds);

/* y = alpha * A * x + beta * y for a CSR matrix (int32 indices, fp32 data, unit strides, host scalars)
 * WITHOUT an external buffer and without allocating anything: the plan and the per-tile carries that
 * aclsparseSpMV keeps in the caller's buffer live in an 8 MiB device array built into the library.
 * For callers that cannot allocate device memory when they need the product - a latency-critical loop
 * whose memory was fixed at start-up, a host framework whose allocator owns the device, a plug-in that
 * is only handed its operands.  Asynchronous on `stream`.
 *   - Matrices whose plan exceeds the built-in scratch (roughly rows * 4 + (rows + nnz) * 0.012 bytes
 *     > 8 MiB) are refused with ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES and a message on stderr.
 *   - The first call on a device loads the library's device code (with it the scratch array) and looks up
 *     the scratch's device address: that call can take device memory once and must be made at start-up,
 *     outside any stream capture.  Every later call on that device allocates nothing.
 *   - All calls on a device share the scratch: calls that overlap on the GPU race; keep them in stream order.
 * This entry point has no counterpart in the reference. */
aclsparseStatus_t aclsparseB200SpMVNoAlloc(aclrtStream stream, int64_t rows, int64_t cols, int64_t nnz,
                                           const int32_t* rowOffsets, const int32_t* colInd, const float* values,
                                           aclsparseIndexBase_t idxBase, const float* x, float* y, float alpha,
                                           float beta);

/* Mirrors of an output vector / matrix: after this call every element that aclsparseSpMV (aclsparseSpMM)
 * writes to `vec` (`mat`) is also stored at the same element position of each of the `count` (at most 7)
 * buffers `mirrors[0..count)`, by the product kernels themselves.  With the result buffers of the other
 * GPUs of the node as mirrors (peer-mapped pointers, each advanced to this device's row block) the product
 * and the reassembly of a row-block-sharded y / C over NVLink become one kernel; the caller follows it with
 * a barrier across the devices.  A mirror has the layout (stride, leading dimension, order) of the vector
 * or matrix itself.  count == 0 clears the list.  The host array `mirrors` is copied.  beta scales the
 * values of `vec` / `mat` only; mirrors are never read.  No counterpart in the reference. */
aclsparseStatus_t aclsparseB200DnVecSetMirrors(aclsparseDnVecDescr_t vec, int count, void* const* mirrors);
aclsparseStatus_t aclsparseB200DnMatSetMirrors(aclsparseDnMatDescr_t mat, int count, void* const* mirrors);

/* The same with ONE mirror that is an NVLink multicast address (a cuMulticast / symmetric-memory mapping
 * bound to the result buffers of all GPUs of the node, advanced to this device's row block): the kernels
 * store to it with multimem.st, NVSwitch replicates each store to every GPU, and a device sends its block
 * once instead of once per peer.  Replaces any mirror list; SetMirrors(.., 0, NULL) clears it.  Only on
 * devices and buffers for which such a mapping exists.  No counterpart in the reference. */
aclsparseStatus_t aclsparseB200DnVecSetMulticastMirror(aclsparseDnVecDescr_t vec, void* multicast);
aclsparseStatus_t aclsparseB200DnMatSetMulticastMirror(aclsparseDnMatDescr_t mat, void* multicast);

/* Barrier across the GPUs of a node that share a row-block-sharded result: enqueues, on `stream`, one
 * small kernel that tells every peer "my row block is in your buffer" and waits until every peer has said
 * the same.  `localState` is this rank's AclspNodeBarrierState (aclsparse_b200_kernels.h; 128 bytes of
 * zero-filled memory that all ranks can address), `peerStates[r]` rank r's as this device addresses it.
 * The wait is bounded by `spinLimit` polls per peer (0 picks the default, about a second): a peer that
 * never arrives makes the kernel give up and record it, nothing hangs and nothing traps.
 * aclsparseB200NodeBarrierStatus synchronises `stream`, reads that record and clears it: it returns
 * ACL_SPARSE_STATUS_EXECUTION_FAILED when a barrier since the last call gave up (and, if `missingRank` is
 * non-null, stores the rank that was missing), ACL_SPARSE_STATUS_SUCCESS otherwise.
 * No counterpart in the reference, which is single-device. */
aclsparseStatus_t aclsparseB200NodeBarrier(aclrtStream stream, void* localState, void* const* peerStates, int world,
                                           int rank, unsigned spinLimit);
aclsparseStatus_t aclsparseB200NodeBarrierStatus(aclrtStream stream, void* localState, int* missingRank);

/* How many warps of SpMV products over the plan in `externalBuffer` gave up waiting for a bulk copy since the
 * plan was built (the SpMV row-block kernel waits for its copies at most about a quarter of a second each; a
 * warp whose wait runs out computes its remaining rows with plain loads, so the results are right either way,
 * and counts itself here).  Synchronises `stream` and reads the counter from the plan header.  A diagnostic:
 * anything but 0 means the copy engine did not deliver in time.  No counterpart in the reference. */
aclsparseStatus_t aclsparseB200SpMVWaitFailures(aclrtStream stream, const void* externalBuffer, unsigned* count);

/* The same barrier as the END of every product written into `vec` / `mat`, instead of a kernel of its own:
 * the last kernel of aclsparseSpMV / aclsparseSpMM (fp32) runs it in the CTA that finishes last, after
 * that CTA has seen all others fence their stores, so a sharded step is the product kernels alone.  The
 * arguments are those of aclsparseB200NodeBarrier; world <= 1 or localState == NULL removes it.  A product
 * that has nothing to launch (no rows) runs no barrier: such a rank calls aclsparseB200NodeBarrier.  The
 * wait is bounded as above and reported through aclsparseB200NodeBarrierStatus. */
aclsparseStatus_t aclsparseB200DnVecSetClosingBarrier(aclsparseDnVecDescr_t vec, void* localState,
                                                      void* const* peerStates, int world, int rank,
                                                      unsigned spinLimit);
aclsparseStatus_t aclsparseB200DnMatSetClosingBarrier(aclsparseDnMatDescr_t mat, void* localState,
                                                      void* const* peerStates, int world, int rank,
                                                      unsigned spinLimit);

/* Grouped matrix product: the product of a block-diagonal matrix of ragged dense row blocks with one dense
 * matrix per block, as a mixture-of-experts layer computes it once its rows are sorted by expert:
 *     C[r, :] = alpha * rowScales[r] * (A[r, :] * op(B_g)) .* colScales[g, :] + beta * C[r, :]
 * for the rows r of group g, groupOffsets[g] <= r < groupOffsets[g + 1].
 *   matA  rows x k, row-major.  matC  rows x n, row-major.  matB  one batch entry per group
 *         (aclsparseDnMatSetStridedBatch), op(B_g) is k x n, row- or column-major, op N / T (H is T).
 *   groupOffsets  DEVICE array of groups + 1 int32, ascending; NULL with a single group: all rows.  Its content is
 *         never trusted with an address: values are clamped to [0, rows], and to the largest one before them, so that
 *         every row is in one group at most.
 *   rowScales (rows floats) and colScales (groups x n floats), DEVICE arrays, may be NULL: ones.
 *   types  A, B fp16 or bf16 with C of that type or fp32: fp32 sums; A, B int8 with C fp32, fp16 or bf16: exact
 *         int32 sums, k <= 131071.  The compute type is ACL_FLOAT.  The result is formed in fp32 and rounded once
 *         to the type of C.  Others, also mirrors and closing barriers on C: NOT_SUPPORTED.
 * A and B should start on multiples of 16 bytes: rows of any width and leading dimension run on the tensor cores, a
 * matrix that is merely shifted does not and takes many times as long.
 * Rows of C outside [groupOffsets[0], groupOffsets[groups]) are left as they are; beta == 0 does not read C; an
 * empty group costs nothing; k == 0 gives beta * C; alpha == 0 multiplies the sums like any other alpha (an infinity or a
 * NaN in them gives NaN).  C must not overlap A or B.  Results do not depend on
 * scheduling.  The buffer holds partial sums of products split along k: 64-byte aligned, one call at a time.
 * Preprocess clears its counters; it is optional: a product that finds no Preprocess of its matC for this buffer
 * on this stream clears them itself, with one more launch.  A Preprocess holds until another one or another operator is
 * given the buffer, or GetBufferSize is asked for this matC again; until then nothing else may write to the buffer, so
 * memory that has had another use in between, or comes from another allocation at the same address, needs one of the two
 * first.  Asynchronous on the handle's stream.
 * No counterpart in the reference. */
aclsparseStatus_t aclsparseB200GroupedMMGetBufferSize(aclsparseHandle_t handle, aclsparseOperation_t opB,
                                                      const void* alpha, aclsparseConstDnMatDescr_t matA,
                                                      const int32_t* groupOffsets, aclsparseConstDnMatDescr_t matB,
                                                      const float* rowScales, const float* colScales, const void* beta,
                                                      aclsparseDnMatDescr_t matC, aclDataType computeType,
                                                      size_t* bufferSize);
aclsparseStatus_t aclsparseB200GroupedMMPreprocess(aclsparseHandle_t handle, aclsparseOperation_t opB,
                                                   const void* alpha, aclsparseConstDnMatDescr_t matA,
                                                   const int32_t* groupOffsets, aclsparseConstDnMatDescr_t matB,
                                                   const float* rowScales, const float* colScales, const void* beta,
                                                   aclsparseDnMatDescr_t matC, aclDataType computeType,
                                                   void* externalBuffer);
aclsparseStatus_t aclsparseB200GroupedMM(aclsparseHandle_t handle, aclsparseOperation_t opB, const void* alpha,
                                         aclsparseConstDnMatDescr_t matA, const int32_t* groupOffsets,
                                         aclsparseConstDnMatDescr_t matB, const float* rowScales,
                                         const float* colScales, const void* beta, aclsparseDnMatDescr_t matC,
                                         aclDataType computeType, void* externalBuffer);

/* The gradient of the grouped product with respect to its weights:
 *     C_g = alpha * A_g^T * B_g + beta * C_g,
 * A_g and B_g being the rows groupOffsets[g] .. groupOffsets[g + 1] of matA (rows x m, row-major) and matB
 * (rows x n, row-major), C_g batch entry g of matC (m x n, row- or column-major).  With y = x * W_g^T the gradient of
 * W_g is the product of A = dy and B = x.  fp16 or bf16 with C of that type or fp32 (beta = 1 accumulates);
 * an empty group gives beta * C_g.  groupOffsets, the buffer, Preprocess and everything else as above. */
aclsparseStatus_t aclsparseB200GroupedMMWeightGradGetBufferSize(
    aclsparseHandle_t handle, const void* alpha, aclsparseConstDnMatDescr_t matA, aclsparseConstDnMatDescr_t matB,
    const int32_t* groupOffsets, const void* beta, aclsparseDnMatDescr_t matC, aclDataType computeType,
    size_t* bufferSize);
aclsparseStatus_t aclsparseB200GroupedMMWeightGradPreprocess(
    aclsparseHandle_t handle, const void* alpha, aclsparseConstDnMatDescr_t matA, aclsparseConstDnMatDescr_t matB,
    const int32_t* groupOffsets, const void* beta, aclsparseDnMatDescr_t matC, aclDataType computeType,
    void* externalBuffer);
aclsparseStatus_t aclsparseB200GroupedMMWeightGrad(aclsparseHandle_t handle, const void* alpha,
                                                   aclsparseConstDnMatDescr_t matA, aclsparseConstDnMatDescr_t matB,
                                                   const int32_t* groupOffsets, const void* beta,
                                                   aclsparseDnMatDescr_t matC, aclDataType computeType,
                                                   void* externalBuffer);

/* How many CTAs of grouped products over `externalBuffer` gave up a wait since its counters were last cleared: by
 * Preprocess, by this call, or by a product that found no current Preprocess (every one in a capture) and cleared them
 * itself, so that without Preprocess it speaks of the last product alone.  Every wait of those kernels is bounded, at four
 * seconds from the end of the kernel before; a CTA whose wait runs out leaves its tiles unfinished and counts itself here,
 * the other one of its pair too.  Anything but 0 means that results since then are not to be used; the call then clears
 * the counters, so that the next product can use the buffer again.  The buffer has been through a Preprocess or a
 * product.  Synchronises `stream`; in a capture: NOT_SUPPORTED.  No counterpart in the reference. */
aclsparseStatus_t aclsparseB200GroupedMMWaitFailures(aclrtStream stream, void* externalBuffer, unsigned* count);

/* The same count over every grouped product of this process on the current device, whatever its buffer and whether that
 * still exists.  Nothing clears it: a reading that is larger than the one before means that a product which ended
 * between them is incomplete.  Synchronises `stream`, and counts what has ended by then; in a capture: NOT_SUPPORTED. */
aclsparseStatus_t aclsparseB200GroupedMMTotalWaitFailures(aclrtStream stream, unsigned* count);

/* Rows of a matrix in 8 bits with one scale each, the operand of the int8 product above:
 *     scales[r] = max_k |X[r, k]| * (1 / 127)   (in fp32, 1 / 127 being its nearest fp32 number),
 *     Q[r, k]   = X[r, k] / scales[r], the exact quotient rounded to the nearest integer, ties to even
 * (and held to +-127, which only matters where the scale is subnormal).
 * matX fp32, fp16 or bf16, matQ int8, both rows x cols, row-major with any leading dimension; scales: DEVICE array of
 * rows floats.  A row of zeros, and one so small that its scale rounds to zero, gives zeros with the scale 0.  A row
 * that holds an infinity or a NaN gives zeros with that scale, infinite or NaN: a product with it is then NaN
 * throughout, never silently finite.  Asynchronous on the handle's stream.  No counterpart in the reference. */
aclsparseStatus_t aclsparseB200QuantizeRows(aclsparseHandle_t handle, aclsparseConstDnMatDescr_t matX,
                                            aclsparseDnMatDescr_t matQ, float* scales);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif

#endif /* ACLSPARSE_B200_EXT_H_ */
