/*
 * Grouped matrix products: one dense matrix per ragged group of rows (forward),
 * and the gradient of those matrices, a sum over a ragged group of rows.
 *
 * PlainKernel: 64 x 64 tiles of the result, operands staged through shared
 * memory element by element with any strides, products and sums in registers
 * (fp32 FMA; int32 for int8).
 */
#include <cstdint>

#include <cuda_runtime.h>

#include "aclsparse_b200_kernels.h"
#include "element_types.cuh"
#include "group_walk.cuh"
#include "grouped_schedule.cuh"
#include "grouped_tc.h"
#include "plan_kernels.h"

namespace {

using aclsp::GroupTile;
using aclsp::GroupWalk;
using aclsp::kBF16;
using aclsp::kF16;
using aclsp::kI8;

// The part of the buffer that Preprocess clears, and where partial sums begin.
constexpr uint32_t kCountersEnd = 4u * (kGroupedHeaderWords + aclsp::kGroupedCounters);

template <int kIn>
struct Plain {
    using Sum = float;
    static __device__ __forceinline__ float Load(const void* p, int64_t i) { return aclsp::LoadIn<kIn>(p, i); }
};
template <>
struct Plain<kI8> {
    using Sum = int32_t;
    static __device__ __forceinline__ int32_t Load(const void* p, int64_t i)
    {
        return __ldg(static_cast<const signed char*>(p) + i);
    }
};

// c[at] = scaled + beta * c[at] in the type of C, rounded once; beta == 0 does not read C.
__device__ __forceinline__ void StoreResult(uint32_t type, void* c, int64_t at, float scaled, float beta)
{
    if (type == ACLSP_TYPE_F32) {
        float* out = static_cast<float*>(c) + at;
        *out = beta == 0.0f ? scaled : fmaf(beta, *out, scaled);
    } else if (type == ACLSP_TYPE_F16) {
        __half* out = static_cast<__half*>(c) + at;
        *out = __float2half_rn(beta == 0.0f ? scaled : fmaf(beta, __half2float(*out), scaled));
    } else {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(c) + at;
        *out = __float2bfloat16_rn(beta == 0.0f ? scaled : fmaf(beta, __bfloat162float(*out), scaled));
    }
}

constexpr int kPlainTile = 64;
constexpr int kPlainStep = 16;
constexpr int kPlainThreads = 256;

template <int kIn>
__global__ void __launch_bounds__(kPlainThreads) PlainKernel(const void* __restrict__ a, const void* __restrict__ b,
                                                             void* __restrict__ c, const AclspGroupedParams p)
{
    using Sum = typename Plain<kIn>::Sum;
    __shared__ Sum left[kPlainStep][kPlainTile + 1];
    __shared__ Sum right[kPlainStep][kPlainTile + 1];
    const float alpha = p.alphaPtr != nullptr ? *p.alphaPtr : p.alpha;
    const float beta = p.betaPtr != nullptr ? *p.betaPtr : p.beta;
    const uint32_t across = (p.n + kPlainTile - 1u) / kPlainTile;
    const uint32_t down = (p.m + kPlainTile - 1u) / kPlainTile;
    GroupWalk walk(p.offsets, p.weightGrad != 0 ? 0u : p.groups, p.rows, kPlainTile, across);
    const int tid = static_cast<int>(threadIdx.x);
    const int ti = tid / 16 * 4;
    const int tj = tid % 16;
    for (uint32_t t = blockIdx.x;; t += gridDim.x) {
        // this tile: rows i0.. of the left operand, columns j0.. of the right one, the sum over k0 <= k < k1
        uint32_t group, i0, iCount, j0, k0, k1;
        if (p.weightGrad != 0) {
            if (t >= p.groups * down * across) {
                break;
            }
            group = t / (down * across);
            i0 = t / across % down * kPlainTile;
            iCount = p.m - i0;
            j0 = t % across * kPlainTile;
            aclsp::GroupRows(p.offsets, group, p.rows, &k0, &k1);
        } else {
            GroupTile tile;
            if (!walk.Find(t, &tile)) {
                break;
            }
            group = tile.group;
            i0 = tile.row0;
            iCount = tile.count;
            j0 = tile.across * kPlainTile;
            k0 = 0;
            k1 = p.k;
        }
        const uint32_t jCount = p.n - j0;
        const int64_t bBase = p.weightGrad != 0 ? 0 : static_cast<int64_t>(group) * p.bBatchStride;
        Sum sum[4][4] = {};
        for (uint32_t k = k0; k < k1; k += kPlainStep) {
            for (int e = tid; e < kPlainTile * kPlainStep; e += kPlainThreads) {
                // neighbouring threads take neighbouring addresses of whichever index is contiguous
                const int li = p.aInner == 1 ? e / kPlainStep : e % kPlainTile;
                const int lk = p.aInner == 1 ? e % kPlainStep : e / kPlainTile;
                Sum v = 0;
                if (static_cast<uint32_t>(li) < iCount && k + lk < k1) {
                    v = Plain<kIn>::Load(a, static_cast<int64_t>(i0 + li) * p.aOuter +
                                                static_cast<int64_t>(k + lk) * p.aInner);
                }
                left[lk][li] = v;
                const int rj = p.bInner == 1 ? e / kPlainStep : e % kPlainTile;
                const int rk = p.bInner == 1 ? e % kPlainStep : e / kPlainTile;
                Sum w = 0;
                if (static_cast<uint32_t>(rj) < jCount && k + rk < k1) {
                    w = Plain<kIn>::Load(b, bBase + static_cast<int64_t>(j0 + rj) * p.bOuter +
                                                static_cast<int64_t>(k + rk) * p.bInner);
                }
                right[rk][rj] = w;
            }
            __syncthreads();
            for (int kk = 0; kk < kPlainStep; ++kk) {
                for (int x = 0; x < 4; ++x) {
                    for (int y = 0; y < 4; ++y) {
                        sum[x][y] += left[kk][ti + x] * right[kk][tj + 16 * y];
                    }
                }
            }
            __syncthreads();
        }
        const int64_t cBase = p.weightGrad != 0 ? static_cast<int64_t>(group) * p.cBatchStride : 0;
        for (int x = 0; x < 4; ++x) {
            if (static_cast<uint32_t>(ti + x) >= iCount) {
                continue;
            }
            const uint32_t i = i0 + ti + x;
            const float rowScale = p.rowScales != nullptr ? p.rowScales[i] * alpha : alpha;
            for (int y = 0; y < 4; ++y) {
                const uint32_t j = tj + 16 * y;
                if (j < jCount) {
                    float s = static_cast<float>(sum[x][y]) * rowScale;
                    if (p.colScales != nullptr) {
                        s *= p.colScales[static_cast<int64_t>(group) * p.n + j0 + j];
                    }
                    StoreResult(p.outType, c, cBase + static_cast<int64_t>(i) * p.ldc + j0 + j, s, beta);
                }
            }
        }
    }
}

}  // namespace

extern "C" uint64_t aclsp_b200_grouped_buffer_bytes(const AclspGroupedParams* params)
{
    // two partial tiles per CTA at most
    return kCountersEnd + 2ull * aclsp::kGroupedMaxCtas * aclsp::kTileLanes * AclspGroupedColumns(*params) * 4u;
}

extern "C" void aclsp_b200_grouped_preprocess_kernel_do(void* buffer, void* stream)
{
    AclspCountLaunches(1);
    cudaMemsetAsync(buffer, 0, kCountersEnd, static_cast<cudaStream_t>(stream));
}

extern "C" void aclsp_b200_grouped_mm_kernel_do(const void* a, const void* b, void* c, void* buffer,
                                                const AclspGroupedParams* params, void* stream)
{
    const AclspGroupedParams& p = *params;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (AclspGroupedTensorLaunch(a, b, c, buffer, p, s)) {
        return;
    }
    AclspCountLaunches(1);
    const uint32_t grid = 148u * 4u;
    if (p.inType == ACLSP_TYPE_F16) {
        PlainKernel<kF16><<<grid, kPlainThreads, 0, s>>>(a, b, c, p);
    } else if (p.inType == ACLSP_TYPE_BF16) {
        PlainKernel<kBF16><<<grid, kPlainThreads, 0, s>>>(a, b, c, p);
    } else {
        PlainKernel<kI8><<<grid, kPlainThreads, 0, s>>>(a, b, c, p);
    }
}
