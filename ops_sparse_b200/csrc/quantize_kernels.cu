/*
 * Rows in 8 bits: scale s = max|x| / 127 of every row, q = x / s to the nearest
 * integer, ties to even.
 *
 * The quotient that is rounded is the exact one, not its fp32 value: next to a
 * tie the fp32 quotient can land on the other side.  q0 = rint(fl(x / s)) is off
 * by one at most, and the remainder r = x - q0 * s tells: one FMA gives it
 * exactly near a tie (it is a multiple of the last place of s, and at most s in
 * size), |r| > s / 2 moves q0 towards x, and |r| == s / 2 is a tie that the even
 * neighbour gets.
 */
#include <cstdint>

#include <cuda_runtime.h>

#include "aclsparse_b200_kernels.h"
#include "element_types.cuh"
#include "plan_kernels.h"

namespace {

using aclsp::kBF16;
using aclsp::kF16;
using aclsp::kF32;

constexpr int kThreads = 256;

// x / s to the nearest integer, ties to even; s > 0 finite, |x| <= 127.5 s.
__device__ __forceinline__ int RoundQuotient(float x, float s)
{
    float q = rintf(__fdiv_rn(x, s));
    const float r = fmaf(-q, s, x);
    const float twice = 2.0f * fabsf(r);
    const bool odd = (static_cast<int>(q) & 1) != 0;
    if (twice > s || (twice == s && odd)) {
        q += r > 0.0f ? 1.0f : -1.0f;
    }
    return static_cast<int>(fminf(fmaxf(q, -127.0f), 127.0f));
}

template <int kIn>
__global__ void __launch_bounds__(kThreads) QuantizeRowsKernel(const void* __restrict__ x, signed char* __restrict__ q,
                                                               float* __restrict__ scales, uint32_t rows,
                                                               uint32_t cols, int64_t ldx, int64_t ldq)
{
    __shared__ float warpMax[kThreads / 32];
    for (uint32_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int64_t from = static_cast<int64_t>(row) * ldx;
        float top = 0.0f;
        bool nan = false;
        for (uint32_t i = threadIdx.x; i < cols; i += kThreads) {
            const float v = fabsf(aclsp::LoadIn<kIn>(x, from + i));
            nan = nan || v != v;
            top = fmaxf(top, v);
        }
        for (int d = 16; d > 0; d /= 2) {
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        }
        if (threadIdx.x % 32 == 0) {
            warpMax[threadIdx.x / 32] = top;
        }
        nan = __syncthreads_or(nan) != 0;
        for (int w = 0; w < kThreads / 32; ++w) {
            top = fmaxf(top, warpMax[w]);
        }
        const float scale = nan ? __int_as_float(0x7FC00000) : __fdiv_rn(top, 127.0f);
        const bool zeros = !(scale > 0.0f && scale <= 3.402823466e38f);
        if (threadIdx.x == 0) {
            scales[row] = scale;
        }
        signed char* to = q + static_cast<int64_t>(row) * ldq;
        for (uint32_t i = threadIdx.x; i < cols; i += kThreads) {
            to[i] = zeros ? 0 : static_cast<signed char>(RoundQuotient(aclsp::LoadIn<kIn>(x, from + i), scale));
        }
        __syncthreads();
    }
}

}  // namespace

extern "C" void aclsp_b200_quantize_rows_kernel_do(const void* x, void* q, float* scales, uint32_t rows, uint32_t cols,
                                                   int64_t ldx, int64_t ldq, uint32_t xType, void* stream)
{
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    signed char* out = static_cast<signed char*>(q);
    const uint32_t grid = rows < 148u * 8u ? rows : 148u * 8u;
    AclspCountLaunches(1);
    if (xType == ACLSP_TYPE_F16) {
        QuantizeRowsKernel<kF16><<<grid, kThreads, 0, s>>>(x, out, scales, rows, cols, ldx, ldq);
    } else if (xType == ACLSP_TYPE_BF16) {
        QuantizeRowsKernel<kBF16><<<grid, kThreads, 0, s>>>(x, out, scales, rows, cols, ldx, ldq);
    } else {
        QuantizeRowsKernel<kF32><<<grid, kThreads, 0, s>>>(x, out, scales, rows, cols, ldx, ldq);
    }
}
