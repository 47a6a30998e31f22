/*
 * Grouped matrix products: one dense matrix per ragged group of rows (forward),
 * and the gradient of those matrices, a sum over a ragged group of rows.
 *
 * The work is done on the tensor cores (grouped_tc_kernels.cu).  Here are the
 * kernels around that: FewRowsKernel for a few tokens, CopyRowsKernel, which brings
 * operands of odd widths to rows that TMA can load, and PlainKernel for what is left:
 * bases that are not 16-byte aligned, sums over nothing, and sizes beyond 2^28.  It
 * computes 64 x 64 tiles, operands staged through shared memory element by element, products and sums in
 * registers (fp32 FMA; int32 for int8).
 */
#include <cstdint>
#include <cstring>

#include <cuda_runtime.h>

#include "aclsparse_b200_kernels.h"
#include "element_types.cuh"
#include "group_walk.cuh"
#include "grouped_schedule.cuh"
#include "grouped_tc.h"
#include "plan_kernels.h"
#include "tcgen05.cuh"

namespace {

using aclsp::GroupTile;
using aclsp::GroupWalk;
using aclsp::kBF16;
using aclsp::kF16;
using aclsp::kI8;


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
    aclsp::GroupRows groupRows(p.offsets, p.rows);
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
            groupRows.Find(group, &k0, &k1);
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

// ---- products of a few rows ----

constexpr uint32_t kFewThreads = 256;
constexpr uint32_t kFewDense = 2;  // rows of the dense matrix that a warp reads side by side

// 16 bytes of a row in words, or one element alone in the first; zeros where `in` is false.
template <uint32_t kBytes>
struct Words {
    static constexpr uint32_t kCount = (kBytes + 3u) / 4u;
    uint32_t w[kCount];
    __device__ __forceinline__ void Load(const unsigned char* at, bool in)
    {
#pragma unroll
        for (uint32_t i = 0; i < kCount; ++i) {
            w[i] = 0;
        }
        if (!in) {
            return;
        }
        if constexpr (kBytes == 16u) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(at));
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (kBytes == 2u) {
            w[0] = __ldg(reinterpret_cast<const uint16_t*>(at));
        } else {
            w[0] = __ldg(at);
        }
    }
};

// The two 16-bit numbers of a word, exact.
template <int kIn>
__device__ __forceinline__ float2 Pair(uint32_t w)
{
    if constexpr (kIn == kBF16) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    } else {
        __half2 h;
        memcpy(&h, &w, sizeof(h));
        return __half22float2(h);
    }
}

// sum[d][r] += dense[d] . row[r] over the elements of the words.
template <int kIn, uint32_t kBytes, uint32_t kRows, typename Sum>
__device__ __forceinline__ void AddProducts(Sum (&sum)[kFewDense][kRows], const Words<kBytes> (&dense)[kFewDense],
                                            const Words<kBytes> (&row)[kRows])
{
#pragma unroll
    for (uint32_t i = 0; i < Words<kBytes>::kCount; ++i) {
        if constexpr (kIn == kI8) {
            // bytes behind a single element are zeros
#pragma unroll
            for (uint32_t d = 0; d < kFewDense; ++d) {
#pragma unroll
                for (uint32_t r = 0; r < kRows; ++r) {
                    sum[d][r] = __dp4a(static_cast<int>(dense[d].w[i]), static_cast<int>(row[r].w[i]), sum[d][r]);
                }
            }
        } else {
            float2 x[kRows];
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
                x[r] = Pair<kIn>(row[r].w[i]);
            }
#pragma unroll
            for (uint32_t d = 0; d < kFewDense; ++d) {
                const float2 w = Pair<kIn>(dense[d].w[i]);
#pragma unroll
                for (uint32_t r = 0; r < kRows; ++r) {
                    sum[d][r] = fmaf(w.x, x[r].x, sum[d][r]);
                    if constexpr (kBytes == 16u) {
                        sum[d][r] = fmaf(w.y, x[r].y, sum[d][r]);
                    }
                }
            }
        }
    }
}

// The lanes' values v[0 .. kCount), added over the warp: lane 32 / kCount * i gets the sum of v[i].  At each step a lane
// gives half of its values away and keeps the other half, so that kCount values take little more than one would.
template <uint32_t kCount, typename Sum>
__device__ __forceinline__ Sum AddLanes(Sum (&v)[kCount])
{
    const uint32_t lane = threadIdx.x % 32u;
    uint32_t apart = 16;
#pragma unroll
    for (uint32_t half = kCount / 2u; half > 0u; half /= 2u) {
#pragma unroll
        for (uint32_t i = 0; i < half; ++i) {
            const bool upper = (lane & apart) != 0u;
            const Sum keep = upper ? v[i + half] : v[i];
            const Sum give = upper ? v[i] : v[i + half];
            v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, static_cast<int>(apart));
        }
        apart /= 2u;
    }
#pragma unroll
    for (uint32_t d = 16u / kCount; d > 0u; d /= 2u) {
        v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], static_cast<int>(d));
    }
    return v[0];
}

struct FewOperands {
    const unsigned char* a;
    const unsigned char* b;
    void* c;
    float alpha;
    float beta;
};

// kRows rows of a group from row0 on, of which `count` are its own, times kFewDense rows of its matrix from j0 on.  Called by
// whole warps.
template <int kIn, uint32_t kRows>
__device__ __forceinline__ void FewRows(const AclspGroupedParams& p, const FewOperands& o, uint32_t group, uint32_t row0,
                                        uint32_t count, uint32_t j0)
{
    using Sum = typename Plain<kIn>::Sum;
    constexpr uint32_t kElement = kIn == kI8 ? 1u : 2u;
    constexpr uint32_t kPer = 16u / kElement;
    constexpr uint32_t kTogether = kRows == 4u ? 2u : 4u;  // loads of a row under way
    const uint32_t lane = threadIdx.x % 32u;
    const unsigned char* dense[kFewDense];
    const unsigned char* row[kRows];
#pragma unroll
    for (uint32_t d = 0; d < kFewDense; ++d) {  // the last row again where there are no more
        const uint32_t j = j0 + d < p.n ? j0 + d : p.n - 1u;
        dense[d] = o.b + (static_cast<int64_t>(group) * p.bBatchStride + static_cast<int64_t>(j) * p.bOuter) * kElement;
    }
#pragma unroll
    for (uint32_t r = 0; r < kRows; ++r) {
        row[r] = o.a + static_cast<int64_t>(row0 + (r < count ? r : count - 1u)) * p.aOuter * kElement;
    }
    Sum sum[kFewDense][kRows] = {};
    const uint32_t vectors = p.k / kPer;
    for (uint32_t v = lane; v < vectors; v += 32u * kTogether) {
        Words<16> w[kTogether][kFewDense];
        Words<16> x[kTogether][kRows];
#pragma unroll
        for (uint32_t u = 0; u < kTogether; ++u) {
            const bool in = v + 32u * u < vectors;
            const int64_t at = static_cast<int64_t>(v + 32u * u) * 16;
#pragma unroll
            for (uint32_t d = 0; d < kFewDense; ++d) {
                w[u][d].Load(dense[d] + at, in);
            }
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
                x[u][r].Load(row[r] + at, in);
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < kTogether; ++u) {
            AddProducts<kIn, 16, kRows>(sum, w[u], x[u]);
        }
    }
    if (vectors * kPer != p.k) {  // elements behind the last whole vector, fewer than a warp has lanes
        const uint32_t e = vectors * kPer + lane;
        Words<kElement> w[kFewDense];
        Words<kElement> x[kRows];
#pragma unroll
        for (uint32_t d = 0; d < kFewDense; ++d) {
            w[d].Load(dense[d] + static_cast<int64_t>(e) * kElement, e < p.k);
        }
#pragma unroll
        for (uint32_t r = 0; r < kRows; ++r) {
            x[r].Load(row[r] + static_cast<int64_t>(e) * kElement, e < p.k);
        }
        AddProducts<kIn, kElement, kRows>(sum, w, x);
    }
    constexpr uint32_t kCount = kFewDense * kRows;
    Sum all[kCount];
#pragma unroll
    for (uint32_t i = 0; i < kCount; ++i) {
        all[i] = sum[i / kRows][i % kRows];
    }
    const float total = static_cast<float>(AddLanes<kCount>(all));
    const uint32_t mine = lane / (32u / kCount);
    const uint32_t j = j0 + mine / kRows;
    if (lane % (32u / kCount) == 0u && j < p.n && mine % kRows < count) {
        const uint32_t i = row0 + mine % kRows;
        float scale = o.alpha;
        if (p.colScales != nullptr) {
            scale *= __ldg(p.colScales + static_cast<int64_t>(group) * p.n + j);
        }
        float s = total * scale;
        if (p.rowScales != nullptr) {
            s *= __ldg(p.rowScales + i);
        }
        StoreResult(p.outType, o.c, static_cast<int64_t>(i) * p.ldc + j, s, o.beta);
    }
}

// A warp takes kFewDense neighbouring rows of a group's matrix and forms their dot products with up to four of the group's
// rows at a time, fp32 (int32) sums in registers, added over the lanes at the end.  For so few rows reading the matrix is
// all, and this starts reading as soon as it knows its group: no ring to fill, no tensor memory, no partial sums to
// join.  Bound by latency, then HBM.  Two tokens, 4 matrices of 1024 x 1024 bf16: 3.4 us (tensor cores: 8.6); one int8
// token, 4096 x 4096: 3.8 us (8.9); one bf16 token, 4096 x 4096: 7.4 us (11.6).  Only for rows on multiples of 16 bytes:
// loads of single elements and of shifted vectors were measured, and the tensor cores are faster with the copy (3 rows,
// 528 x 3823: 18 and 25 us against 12.7).
template <int kIn>
__global__ void __launch_bounds__(kFewThreads, 2) FewRowsKernel(const FewOperands operands,
                                                                const AclspGroupedParams given)
{
    AclspGroupedParams p = given;
    FewOperands o = operands;
    aclsp::WaitForPreviousKernel(o.a, o.b, p.offsets, p.rowScales, p.colScales, p.alphaPtr, p.betaPtr);
    aclsp::LetNextKernelStart();
    o.alpha = p.alphaPtr != nullptr ? *p.alphaPtr : p.alpha;
    o.beta = p.betaPtr != nullptr ? *p.betaPtr : p.beta;
    constexpr uint32_t kWhole = 1u << 30;  // rows of a tile: a group is never cut
    GroupWalk walk(p.offsets, p.groups, p.rows, kWhole, (p.n + kFewDense - 1u) / kFewDense);
    const uint32_t warps = gridDim.x * (kFewThreads / 32u);
    GroupTile tile;
    for (uint32_t t = blockIdx.x * (kFewThreads / 32u) + threadIdx.x / 32u; walk.Find(t, &tile); t += warps) {
        const uint32_t j0 = tile.across * kFewDense;
        for (uint32_t r = 0; r < tile.count; r += 4u) {
            const uint32_t left = tile.count - r;
            if (left == 1u) {
                FewRows<kIn, 1>(p, o, tile.group, tile.row0 + r, 1, j0);
            } else if (left == 2u) {
                FewRows<kIn, 2>(p, o, tile.group, tile.row0 + r, 2, j0);
            } else {
                FewRows<kIn, 4>(p, o, tile.group, tile.row0 + r, left < 4u ? left : 4u, j0);
            }
        }
    }
}

template <int kIn>
void LaunchFewRows(const void* a, const void* b, void* c, const AclspGroupedParams& p, cudaStream_t s)
{
    const FewOperands o{static_cast<const unsigned char*>(a), static_cast<const unsigned char*>(b), c, 0.0f, 0.0f};
    const uint64_t live = p.groups < p.rows ? p.groups : p.rows;
    const uint64_t units = live * ((p.n + kFewDense - 1u) / kFewDense);
    const uint64_t blocks = (units + kFewThreads / 32u - 1u) / (kFewThreads / 32u);
    constexpr uint64_t kMostBlocks = 148u * 8u;
    AclspCountLaunches(1);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<uint32_t>(blocks < kMostBlocks ? blocks : kMostBlocks));
    config.blockDim = dim3(kFewThreads);
    config.stream = s;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    cudaLaunchKernelEx(&config, FewRowsKernel<kIn>, o, p);
}

// The word at `at`, zeros in place of bytes outside [begin, end).
__device__ __forceinline__ uint32_t WordOf(const unsigned char* at, const unsigned char* begin, const unsigned char* end)
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

constexpr uint32_t kCopyThreads = 256;

// Division of numbers below 2^31 by a divisor known to the host, which makes factor = floor(2^(31 + bits) / divisor) + 1
// with 2^(bits - 1) < divisor <= 2^bits: the quotient's error, number / 2^(31 + bits) at most, is less than 1 / divisor.
struct Divisor {
    uint64_t factor;
    uint32_t shift;
    uint32_t divisor;
    __device__ __forceinline__ uint64_t Quotient(uint64_t v) const
    {
        return v >> 31 == 0u ? static_cast<uint32_t>(v) * factor >> shift : v / divisor;
    }
};

Divisor DivisorOf(uint32_t d)
{
    uint32_t bits = 0;
    while ((1ull << bits) < d) {
        ++bits;
    }
    return Divisor{(1ull << (31u + bits)) / d + 1u, 31u + bits, d};
}

// Rows to copy, in bytes.
struct CopyJob {
    const unsigned char* src;
    unsigned char* dst;
    Divisor rows;
    uint32_t batches;
    int64_t rowBytes;
    int64_t pitch;
    int64_t batchPitch;
    Divisor dstVectors;  // of 16 bytes, in a row
    int64_t dstBatchPitch;
};
struct CopyJobs {
    CopyJob job[2];
};

// A thread per 16 bytes of a copied row: it reads the two aligned vectors that they come from, shifts them into place
// and writes one, the last of a row with what lies behind it.  Every byte is read from memory and written once; the second
// vector is the next thread's first and comes from L1.  One launch for both operands: blockIdx.y is the job.  Bound by
// instructions more than by HBM: 52 matrices of 880 x 1137 fp16, 104 MB, 39 us (70 with five words in place of the two
// vectors, divisions by the hardware's integer code and a grid of eight blocks per SM, which idled where matrices are
// left out).  Measured and left: two to four vectors of a thread under way together (fewer threads then: 84 to 104 us with
// the product, 70 so), going down the rows from a fixed place in them, without divisions (105 us), a warp per row
// (13 us for 51 rows of 4462 bytes), and a warp per 512 bytes of a row (short last stretches, 11 us for 5005 rows of 1554
// bytes).
__global__ void __launch_bounds__(kCopyThreads) CopyRowsKernel(const __grid_constant__ CopyJobs jobs, const int32_t* offsets)
{
    const CopyJob& c = jobs.job[blockIdx.y];
    const unsigned char* src = c.src;
    aclsp::WaitForPreviousKernel(src, offsets);
    aclsp::LetNextKernelStart();
    const uint32_t vectors = c.dstVectors.divisor;
    const uint32_t rows = c.rows.divisor;
    const uint64_t all = static_cast<uint64_t>(rows) * c.batches * vectors;
    const unsigned char* const end = src + (c.batches - 1) * c.batchPitch + (rows - 1) * c.pitch + c.rowBytes;
    const uint64_t threads = static_cast<uint64_t>(gridDim.x) * kCopyThreads;
#pragma unroll 2
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * kCopyThreads + threadIdx.x; i < all; i += threads) {
        uint64_t row = c.dstVectors.Quotient(i);
        const int64_t byte = static_cast<int64_t>(i - row * vectors) * 16;
        uint32_t batch = 0;
        if (c.batches > 1u) {
            batch = static_cast<uint32_t>(c.rows.Quotient(row));
            row -= static_cast<uint64_t>(batch) * rows;
            if (__ldg(offsets + batch) >= __ldg(offsets + batch + 1)) {
                continue;  // nobody reads this matrix
            }
        }
        const unsigned char* from = src + batch * c.batchPitch + static_cast<int64_t>(row) * c.pitch + byte;
        const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from)) & 15u;
        from -= shift;
        uint32_t w[8];
        if (from >= src && from + 32 <= end) {
            const uint4 low = __ldg(reinterpret_cast<const uint4*>(from));
            const uint4 high = __ldg(reinterpret_cast<const uint4*>(from) + 1);
            w[0] = low.x, w[1] = low.y, w[2] = low.z, w[3] = low.w;
            w[4] = high.x, w[5] = high.y, w[6] = high.z, w[7] = high.w;
        } else {  // next to an end of the matrix
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                w[k] = WordOf(from + 4 * k, src, end);
            }
        }
        // by eight bytes, by four, and by what is left of the shift
#pragma unroll
        for (uint32_t k = 0; k < 6; ++k) {
            w[k] = (shift & 8u) != 0u ? w[k + 2] : w[k];
        }
#pragma unroll
        for (uint32_t k = 0; k < 5; ++k) {
            w[k] = (shift & 4u) != 0u ? w[k + 1] : w[k];
        }
        uint32_t v[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            v[k] = __funnelshift_r(w[k], w[k + 1], 8u * (shift & 3u));
        }
        unsigned char* const to = c.dst + batch * c.dstBatchPitch + static_cast<int64_t>(row) * vectors * 16 + byte;
        *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

}  // namespace

void AclspGroupedCopyRows(AclspGroupedOperands* o, const void** left, const void** right, void* buffer,
                          const AclspGroupedParams& p, cudaStream_t stream)
{
    const int64_t bytes = p.inType == ACLSP_TYPE_I8 ? 1 : 2;
    CopyJobs jobs{};
    uint32_t count = 0;
    AclspGroupedOperand* const operands[2] = {&o->left, &o->right};
    const void** const bases[2] = {left, right};
    for (uint32_t i = 0; i < 2; ++i) {
        AclspGroupedOperand* const x = operands[i];
        if (x->copyBytes == 0u) {
            continue;
        }
        CopyJob& c = jobs.job[count++];
        c.src = static_cast<const unsigned char*>(*bases[i]);
        c.dst = static_cast<unsigned char*>(buffer) + x->copyOffset;
        c.rows = DivisorOf(static_cast<uint32_t>(x->rows));
        c.batches = static_cast<uint32_t>(x->batches);
        c.rowBytes = static_cast<int64_t>(x->rowElements) * bytes;
        c.pitch = static_cast<int64_t>(x->ld) * bytes;
        c.batchPitch = static_cast<int64_t>(x->batchStride) * bytes;
        const int64_t dstPitch = (c.rowBytes + 15) / 16 * 16;
        c.dstVectors = DivisorOf(static_cast<uint32_t>(dstPitch / 16));
        c.dstBatchPitch = dstPitch * static_cast<int64_t>(x->rows);
        *bases[i] = c.dst;
        x->ld = static_cast<uint64_t>(dstPitch / bytes);
        x->batchStride = x->rows * x->ld;
    }
    if (count == 0u) {
        return;
    }
    AclspCountLaunches(1);
    cudaLaunchConfig_t config{};
    uint64_t most = 0;
    for (uint32_t i = 0; i < count; ++i) {
        const uint64_t own = static_cast<uint64_t>(jobs.job[i].rows.divisor) * jobs.job[i].batches * jobs.job[i].dstVectors.divisor;
        most = own > most ? own : most;
    }
    // two vectors to a thread, in large copies more: 24 blocks per SM were measured like 16 and 32
    constexpr uint64_t kMostBlocks = 148u * 24u;
    const uint64_t blocks = (most + kCopyThreads * 2u - 1u) / (kCopyThreads * 2u);
    config.gridDim = dim3(static_cast<uint32_t>(blocks < kMostBlocks ? blocks : kMostBlocks), count);
    config.blockDim = dim3(kCopyThreads);
    config.stream = stream;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    cudaLaunchKernelEx(&config, CopyRowsKernel, jobs, p.offsets);
}

extern "C" uint64_t aclsp_b200_grouped_buffer_bytes(const AclspGroupedParams* params)
{
    return AclspGroupedDescribe(*params).bufferBytes;
}

extern "C" void aclsp_b200_grouped_preprocess_kernel_do(void* buffer, void* stream)
{
    AclspCountLaunches(1);
    cudaMemsetAsync(buffer, 0, kGroupedCountersEnd, static_cast<cudaStream_t>(stream));
}

extern "C" void aclsp_b200_grouped_mm_kernel_do(const void* a, const void* b, void* c, void* buffer,
                                                const AclspGroupedParams* params, void* stream)
{
    const AclspGroupedParams& p = *params;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (AclspGroupedFewRows(p) && (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) % 16u == 0u) {
        (p.inType == ACLSP_TYPE_F16    ? LaunchFewRows<kF16>
         : p.inType == ACLSP_TYPE_BF16 ? LaunchFewRows<kBF16>
                                       : LaunchFewRows<kI8>)(a, b, c, p, s);
        return;
    }
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
