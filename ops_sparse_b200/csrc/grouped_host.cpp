/*
 * Host layer of the grouped matrix products and of the row quantisation
 * (include/aclsparse_b200_ext.h): validation, buffer sizing, the bookkeeping of
 * the buffer's counters and the calls into the launch shim.  The checks come in
 * the order of aclsparseSpMM's: handle and scalars, descriptors, operations,
 * types, dimensions, storage, buffer.  No counterpart in the reference.
 */
#include <cstdint>

#include <cuda_runtime.h>

#include "aclsparse_b200_ext.h"
#include "aclsparse_b200_kernels.h"
#include "grouped_tc.h"
#include "internal.h"
#include "plan_layout.h"

namespace {

// A sum of k int8 products stays inside int32: k * 128 * 128 <= 2^31 - 1.
constexpr int64_t kMaxInt8Sum = 131071;

uint32_t KernelType(aclDataType t)
{
    return t == ACL_FLOAT16 ? ACLSP_TYPE_F16 : t == ACL_BF16 ? ACLSP_TYPE_BF16 : t == ACL_INT8 ? ACLSP_TYPE_I8 : ACLSP_TYPE_F32;
}

bool IsFloatType(aclDataType t) { return t == ACL_FLOAT || t == ACL_FLOAT16 || t == ACL_BF16; }

aclsparseStatus_t CheckCall(const char* api, aclsparseHandle_t handle, const void* alpha, const void* beta)
{
    if (handle == nullptr) {
        ACLSP_LOGE(api, "handle is nullptr");
        return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    }
    if (alpha == nullptr || beta == nullptr || handle->signature != kHandleSignature) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t CheckMats(const char* api, const aclsparseDnMatDescr* a, const aclsparseDnMatDescr* b,
                            const aclsparseDnMatDescr* c)
{
    if (a == nullptr || b == nullptr || c == nullptr) {
        ACLSP_LOGE(api, "matA, matB, or matC is nullptr");
        return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    }
    if (a->signature != kDnMatSignature || b->signature != kDnMatSignature || c->signature != kDnMatSignature) {
        ACLSP_LOGE(api, "invalid descriptor signature");
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    return ACL_SPARSE_STATUS_SUCCESS;
}

bool HasStorage(const aclsparseDnMatDescr* d) { return d->rows == 0 || d->cols == 0 || d->values != nullptr; }

// Elements lie on multiples of their own size, as a typed pointer's do.
bool IsElementAligned(const aclsparseDnMatDescr* d)
{
    const uintptr_t bytes = d->valueType == ACL_INT8 ? 1u : d->valueType == ACL_FLOAT ? 4u : 2u;
    return reinterpret_cast<uintptr_t>(d->values) % bytes == 0;
}

// The checks that both products share once types and dimensions are known to be right.
aclsparseStatus_t CheckStorage(const char* api, const aclsparseDnMatDescr* a, const aclsparseDnMatDescr* b,
                               const aclsparseDnMatDescr* c, int32_t groups, const int32_t* offsets)
{
    if (c->numMirrors != 0 || c->barrier.world > 1) {
        ACLSP_LOGE(api, "mirrors and closing barriers are not supported on the result of a grouped product");
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    if (offsets == nullptr && groups != 1) {
        ACLSP_LOGE(api, "groupOffsets is nullptr with %d groups", groups);
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (!HasStorage(a) || !HasStorage(b) || !HasStorage(c) || !IsElementAligned(a) || !IsElementAligned(b) ||
        !IsElementAligned(c) || reinterpret_cast<uintptr_t>(offsets) % sizeof(int32_t) != 0) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    return ACL_SPARSE_STATUS_SUCCESS;
}

// Validates a forward product and describes it to the kernels (all but the scalars).
aclsparseStatus_t DescribeForward(const char* api, const aclsparseDnMatDescr* a, const aclsparseDnMatDescr* b,
                                  const aclsparseDnMatDescr* c, aclsparseOperation_t opB, const int32_t* offsets,
                                  const float* rowScales, const float* colScales, aclDataType computeType,
                                  AclspGroupedParams* p)
{
    aclsparseStatus_t st = CheckMats(api, a, b, c);
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    if (opB != ACL_SPARSE_OP_NON_TRANSPOSE && opB != ACL_SPARSE_OP_TRANSPOSE &&
        opB != ACL_SPARSE_OP_CONJUGATE_TRANSPOSE) {
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    if (a->order != ACL_SPARSE_ORDER_ROW || c->order != ACL_SPARSE_ORDER_ROW || a->batchCount != 1 ||
        c->batchCount != 1) {
        ACLSP_LOGE(api, "matA and matC must be single row-major matrices");
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    const aclDataType in = a->valueType;
    const aclDataType out = c->valueType;
    const bool types = in == ACL_INT8 ? IsFloatType(out)
                                      : (in == ACL_FLOAT16 || in == ACL_BF16) && (out == in || out == ACL_FLOAT);
    if (b->valueType != in || !types || computeType != ACL_FLOAT) {
        ACLSP_LOGE(api, "unsupported data type combination A=%d B=%d C=%d compute=%d", static_cast<int>(in),
                   static_cast<int>(b->valueType), static_cast<int>(out), static_cast<int>(computeType));
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    const bool plain = opB == ACL_SPARSE_OP_NON_TRANSPOSE;
    const int64_t bK = plain ? b->rows : b->cols;
    const int64_t bN = plain ? b->cols : b->rows;
    if (a->rows != c->rows || a->cols != bK || bN != c->cols) {
        ACLSP_LOGE(api, "matrix dimensions do not match");
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (in == ACL_INT8 && a->cols > kMaxInt8Sum) {
        ACLSP_LOGE(api, "int8 sums of more than %lld products do not fit int32", static_cast<long long>(kMaxInt8Sum));
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    st = CheckStorage(api, a, b, c, b->batchCount, offsets);
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    if (reinterpret_cast<uintptr_t>(rowScales) % sizeof(float) != 0 ||
        reinterpret_cast<uintptr_t>(colScales) % sizeof(float) != 0) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    *p = AclspGroupedParams{};
    p->rows = static_cast<uint32_t>(a->rows);
    p->groups = static_cast<uint32_t>(b->batchCount);
    p->n = static_cast<uint32_t>(c->cols);
    p->k = static_cast<uint32_t>(a->cols);
    p->inType = KernelType(in);
    p->outType = KernelType(out);
    p->aOuter = a->ld;
    p->aInner = 1;
    const bool kContiguous = (b->order == ACL_SPARSE_ORDER_ROW) != plain;
    p->bOuter = kContiguous ? b->ld : 1;
    p->bInner = kContiguous ? 1 : b->ld;
    p->bBatchStride = b->batchStride;
    p->ldc = c->ld;
    p->offsets = offsets;
    p->rowScales = rowScales;
    p->colScales = colScales;
    return ACL_SPARSE_STATUS_SUCCESS;
}

// Validates a weight gradient and describes it; *swap says that A and B change places (a column-major C_g is the
// row-major product B_g^T * A_g).
aclsparseStatus_t DescribeGradient(const char* api, const aclsparseDnMatDescr* a, const aclsparseDnMatDescr* b,
                                   const aclsparseDnMatDescr* c, const int32_t* offsets, aclDataType computeType,
                                   AclspGroupedParams* p, bool* swap)
{
    aclsparseStatus_t st = CheckMats(api, a, b, c);
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    if (a->order != ACL_SPARSE_ORDER_ROW || b->order != ACL_SPARSE_ORDER_ROW || a->batchCount != 1 ||
        b->batchCount != 1) {
        ACLSP_LOGE(api, "matA and matB must be single row-major matrices");
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    const aclDataType in = a->valueType;
    const aclDataType out = c->valueType;
    if ((in != ACL_FLOAT16 && in != ACL_BF16) || b->valueType != in || (out != in && out != ACL_FLOAT) ||
        computeType != ACL_FLOAT) {
        ACLSP_LOGE(api, "unsupported data type combination A=%d B=%d C=%d compute=%d", static_cast<int>(in),
                   static_cast<int>(b->valueType), static_cast<int>(out), static_cast<int>(computeType));
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    if (a->rows != b->rows || a->cols != c->rows || b->cols != c->cols) {
        ACLSP_LOGE(api, "matrix dimensions do not match");
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    st = CheckStorage(api, a, b, c, c->batchCount, offsets);
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    *swap = c->order == ACL_SPARSE_ORDER_COL;
    const aclsparseDnMatDescr* left = *swap ? b : a;
    const aclsparseDnMatDescr* right = *swap ? a : b;
    *p = AclspGroupedParams{};
    p->rows = static_cast<uint32_t>(a->rows);
    p->groups = static_cast<uint32_t>(c->batchCount);
    p->m = static_cast<uint32_t>(left->cols);
    p->n = static_cast<uint32_t>(right->cols);
    p->weightGrad = 1;
    p->inType = KernelType(in);
    p->outType = KernelType(out);
    p->aOuter = 1;
    p->aInner = left->ld;
    p->bOuter = 1;
    p->bInner = right->ld;
    p->ldc = c->ld;
    p->cBatchStride = c->batchStride;
    p->offsets = offsets;
    return ACL_SPARSE_STATUS_SUCCESS;
}

void SetScalars(const aclsparseContext* h, const void* alpha, const void* beta, AclspGroupedParams* p)
{
    if (h->pointerMode == ACL_SPARSE_POINTER_MODE_DEVICE) {
        p->alphaPtr = static_cast<const float*>(alpha);
        p->betaPtr = static_cast<const float*>(beta);
    } else {
        p->alpha = *static_cast<const float*>(alpha);
        p->beta = *static_cast<const float*>(beta);
    }
}

aclsparseStatus_t CheckBuffer(const char* api, const void* buffer)
{
    if (buffer == nullptr) {
        ACLSP_LOGE(api, "buffer is nullptr");
        return ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES;
    }
    if (reinterpret_cast<uintptr_t>(buffer) % ACLSP_WS_ALIGN != 0) {
        ACLSP_LOGE(api, "buffer=%p; expected 64-byte alignment", buffer);
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t Enqueued(const char* api)
{
    const cudaError_t err = cudaPeekAtLastError();
    if (err != cudaSuccess) {
        ACLSP_LOGE(api, "kernel enqueue failed: %s", cudaGetErrorString(err));
        return ACL_SPARSE_STATUS_EXECUTION_FAILED;
    }
    return ACL_SPARSE_STATUS_SUCCESS;
}

bool IsCapturing(aclrtStream stream)
{
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &status) != cudaSuccess) {
        (void)cudaGetLastError();  // the legacy stream while another one captures: the launch will say so
        return false;
    }
    return status != cudaStreamCaptureStatusNone;
}

// Preprocess: the buffer's counters are cleared, and the record says so.  Inside a capture nothing has run yet, so
// nothing is recorded: the products of a graph clear the counters themselves and do not depend on what the buffer
// held before a replay.
aclsparseStatus_t Preprocess(const char* api, aclsparseContext* h, aclsparseDnMatDescr* c, void* buffer)
{
    (void)cudaGetLastError();
    const bool capturing = IsCapturing(h->stream);
    aclsp_b200_grouped_preprocess_kernel_do(buffer, h->stream);
    const aclsparseStatus_t st = Enqueued(api);
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    const uint64_t serial = AclspPublishPlan(buffer);
    c->grouped = GroupedPlanRecord{};
    if (!capturing) {
        c->grouped = GroupedPlanRecord{buffer, h->stream, h->streamEpoch, serial};
    }
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t Execute(const char* api, aclsparseContext* h, const void* a, const void* b, aclsparseDnMatDescr* c,
                          void* buffer, const AclspGroupedParams& p)
{
    (void)cudaGetLastError();
    const GroupedPlanRecord& r = c->grouped;
    const bool clear = r.buffer == buffer && r.stream == h->stream && r.streamEpoch == h->streamEpoch &&
                       AclspPlanIsCurrent(buffer, r.serial) && !IsCapturing(h->stream);
    if (!clear) {
        aclsp_b200_grouped_preprocess_kernel_do(buffer, h->stream);
        AclspForgetPlan(buffer);  // whatever plan the buffer held is gone
    }
    if ((p.weightGrad == 0 && p.rows == 0) || p.n == 0 || (p.weightGrad != 0 && p.m == 0)) {
        (void)cudaGetLastError();
        return ACL_SPARSE_STATUS_SUCCESS;  // nothing to write, which needs no GPU either; the buffer counts no failures
    }
    aclsp_b200_grouped_mm_kernel_do(a, b, c->values, buffer, &p, h->stream);
    return Enqueued(api);
}

constexpr const char* kMm = "aclsparseB200GroupedMM";
constexpr const char* kGrad = "aclsparseB200GroupedMMWeightGrad";

}  // namespace

extern "C" aclsparseStatus_t aclsparseB200GroupedMMGetBufferSize(
    aclsparseHandle_t handle, aclsparseOperation_t opB, const void* alpha, aclsparseConstDnMatDescr_t matA,
    const int32_t* groupOffsets, aclsparseConstDnMatDescr_t matB, const float* rowScales, const float* colScales,
    const void* beta, aclsparseDnMatDescr_t matC, aclDataType computeType, size_t* bufferSize)
{
    aclsparseStatus_t st = CheckCall(kMm, handle, alpha, beta);
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    if (bufferSize == nullptr) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    AclspGroupedParams p;
    st = DescribeForward(kMm, matA, matB, matC, opB, groupOffsets, rowScales, colScales, computeType, &p);
    if (st == ACL_SPARSE_STATUS_SUCCESS) {
        *bufferSize = static_cast<size_t>(aclsp_b200_grouped_buffer_bytes(&p));
        // The caller is about to bring a buffer.  It may lie where the last one did, with anything in it.
        matC->grouped = GroupedPlanRecord{};
    }
    return st;
}

extern "C" aclsparseStatus_t aclsparseB200GroupedMMPreprocess(
    aclsparseHandle_t handle, aclsparseOperation_t opB, const void* alpha, aclsparseConstDnMatDescr_t matA,
    const int32_t* groupOffsets, aclsparseConstDnMatDescr_t matB, const float* rowScales, const float* colScales,
    const void* beta, aclsparseDnMatDescr_t matC, aclDataType computeType, void* externalBuffer)
{
    aclsparseStatus_t st = CheckCall(kMm, handle, alpha, beta);
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    AclspGroupedParams p;
    st = DescribeForward(kMm, matA, matB, matC, opB, groupOffsets, rowScales, colScales, computeType, &p);
    if (st == ACL_SPARSE_STATUS_SUCCESS) {
        st = CheckBuffer(kMm, externalBuffer);
    }
    return st != ACL_SPARSE_STATUS_SUCCESS ? st : Preprocess(kMm, handle, matC, externalBuffer);
}

extern "C" aclsparseStatus_t aclsparseB200GroupedMM(aclsparseHandle_t handle, aclsparseOperation_t opB,
                                                    const void* alpha, aclsparseConstDnMatDescr_t matA,
                                                    const int32_t* groupOffsets, aclsparseConstDnMatDescr_t matB,
                                                    const float* rowScales, const float* colScales, const void* beta,
                                                    aclsparseDnMatDescr_t matC, aclDataType computeType,
                                                    void* externalBuffer)
{
    aclsparseStatus_t st = CheckCall(kMm, handle, alpha, beta);
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    AclspGroupedParams p;
    st = DescribeForward(kMm, matA, matB, matC, opB, groupOffsets, rowScales, colScales, computeType, &p);
    if (st == ACL_SPARSE_STATUS_SUCCESS) {
        st = CheckBuffer(kMm, externalBuffer);
    }
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    SetScalars(handle, alpha, beta, &p);
    return Execute(kMm, handle, matA->values, matB->values, matC, externalBuffer, p);
}

extern "C" aclsparseStatus_t aclsparseB200GroupedMMWeightGradGetBufferSize(
    aclsparseHandle_t handle, const void* alpha, aclsparseConstDnMatDescr_t matA, aclsparseConstDnMatDescr_t matB,
    const int32_t* groupOffsets, const void* beta, aclsparseDnMatDescr_t matC, aclDataType computeType,
    size_t* bufferSize)
{
    aclsparseStatus_t st = CheckCall(kGrad, handle, alpha, beta);
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    if (bufferSize == nullptr) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    AclspGroupedParams p;
    bool swap = false;
    st = DescribeGradient(kGrad, matA, matB, matC, groupOffsets, computeType, &p, &swap);
    if (st == ACL_SPARSE_STATUS_SUCCESS) {
        *bufferSize = static_cast<size_t>(aclsp_b200_grouped_buffer_bytes(&p));
        // The caller is about to bring a buffer.  It may lie where the last one did, with anything in it.
        matC->grouped = GroupedPlanRecord{};
    }
    return st;
}

extern "C" aclsparseStatus_t aclsparseB200GroupedMMWeightGradPreprocess(
    aclsparseHandle_t handle, const void* alpha, aclsparseConstDnMatDescr_t matA, aclsparseConstDnMatDescr_t matB,
    const int32_t* groupOffsets, const void* beta, aclsparseDnMatDescr_t matC, aclDataType computeType,
    void* externalBuffer)
{
    aclsparseStatus_t st = CheckCall(kGrad, handle, alpha, beta);
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    AclspGroupedParams p;
    bool swap = false;
    st = DescribeGradient(kGrad, matA, matB, matC, groupOffsets, computeType, &p, &swap);
    if (st == ACL_SPARSE_STATUS_SUCCESS) {
        st = CheckBuffer(kGrad, externalBuffer);
    }
    return st != ACL_SPARSE_STATUS_SUCCESS ? st : Preprocess(kGrad, handle, matC, externalBuffer);
}

extern "C" aclsparseStatus_t aclsparseB200GroupedMMWeightGrad(aclsparseHandle_t handle, const void* alpha,
                                                              aclsparseConstDnMatDescr_t matA,
                                                              aclsparseConstDnMatDescr_t matB,
                                                              const int32_t* groupOffsets, const void* beta,
                                                              aclsparseDnMatDescr_t matC, aclDataType computeType,
                                                              void* externalBuffer)
{
    aclsparseStatus_t st = CheckCall(kGrad, handle, alpha, beta);
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    AclspGroupedParams p;
    bool swap = false;
    st = DescribeGradient(kGrad, matA, matB, matC, groupOffsets, computeType, &p, &swap);
    if (st == ACL_SPARSE_STATUS_SUCCESS) {
        st = CheckBuffer(kGrad, externalBuffer);
    }
    if (st != ACL_SPARSE_STATUS_SUCCESS) {
        return st;
    }
    SetScalars(handle, alpha, beta, &p);
    return Execute(kGrad, handle, swap ? matB->values : matA->values, swap ? matA->values : matB->values, matC,
                   externalBuffer, p);
}

extern "C" aclsparseStatus_t aclsparseB200GroupedMMWaitFailures(aclrtStream stream, void* externalBuffer,
                                                                unsigned* count)
{
    if (externalBuffer == nullptr || count == nullptr) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (IsCapturing(stream)) {
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;  // nothing has run yet, and a wait would end the capture
    }
    auto s = static_cast<cudaStream_t>(stream);
    uint32_t value = 0;  // the buffer's first word
    if (cudaMemcpyAsync(&value, externalBuffer, sizeof(value), cudaMemcpyDeviceToHost, s) != cudaSuccess ||
        cudaStreamSynchronize(s) != cudaSuccess) {
        (void)cudaGetLastError();
        return ACL_SPARSE_STATUS_EXECUTION_FAILED;
    }
    *count = value;
    if (value != 0) {
        aclsp_b200_grouped_preprocess_kernel_do(externalBuffer, stream);
        return Enqueued("aclsparseB200GroupedMMWaitFailures");
    }
    return ACL_SPARSE_STATUS_SUCCESS;
}

extern "C" aclsparseStatus_t aclsparseB200GroupedMMTotalWaitFailures(aclrtStream stream, unsigned* count)
{
    if (count == nullptr) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (IsCapturing(stream)) {
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    uint32_t value = 0;
    if (AclspGroupedTotalWaitFailures(static_cast<cudaStream_t>(stream), &value) != cudaSuccess) {
        (void)cudaGetLastError();
        return ACL_SPARSE_STATUS_EXECUTION_FAILED;
    }
    *count = value;
    return ACL_SPARSE_STATUS_SUCCESS;
}

extern "C" aclsparseStatus_t aclsparseB200QuantizeRows(aclsparseHandle_t handle, aclsparseConstDnMatDescr_t matX,
                                                       aclsparseDnMatDescr_t matQ, float* scales)
{
    constexpr const char* api = "aclsparseB200QuantizeRows";
    if (handle == nullptr) {
        ACLSP_LOGE(api, "handle is nullptr");
        return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    }
    if (handle->signature != kHandleSignature) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (matX == nullptr || matQ == nullptr) {
        ACLSP_LOGE(api, "matX or matQ is nullptr");
        return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    }
    if (matX->signature != kDnMatSignature || matQ->signature != kDnMatSignature) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (matX->order != ACL_SPARSE_ORDER_ROW || matQ->order != ACL_SPARSE_ORDER_ROW || matX->batchCount != 1 ||
        matQ->batchCount != 1 || !IsFloatType(matX->valueType) || matQ->valueType != ACL_INT8 ||
        matQ->numMirrors != 0 || matQ->barrier.world > 1) {
        ACLSP_LOGE(api, "a single row-major fp32, fp16 or bf16 matX and a single row-major int8 matQ are supported");
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    if (matX->rows != matQ->rows || matX->cols != matQ->cols) {
        ACLSP_LOGE(api, "matrix dimensions do not match");
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if ((scales == nullptr && matX->rows > 0) || reinterpret_cast<uintptr_t>(scales) % sizeof(float) != 0 ||
        !HasStorage(matX) || !HasStorage(matQ) || !IsElementAligned(matX)) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (matX->rows == 0) {
        return ACL_SPARSE_STATUS_SUCCESS;
    }
    (void)cudaGetLastError();
    aclsp_b200_quantize_rows_kernel_do(matX->values, matQ->values, scales, static_cast<uint32_t>(matX->rows),
                                       static_cast<uint32_t>(matX->cols), matX->ld, matQ->ld,
                                       KernelType(matX->valueType), handle->stream);
    return Enqueued(api);
}
