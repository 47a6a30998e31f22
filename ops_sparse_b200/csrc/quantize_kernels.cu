/*
 * Rows in 8 bits: scale s = max|x| * (1/127) of every row, q = x / s to the nearest
 * integer, ties to even.
 *
 * The quotient that is rounded is the exact one, not an fp32 value of it: next to a
 * tie that can land on the other side.  t = x * (1 / s) is off by less than 1e-4
 * (|x / s| <= 127 and two roundings), so its nearest integer q0 is off by one at
 * most, and the remainder r = x - q0 * s tells: one FMA gives it exactly near a tie
 * (a multiple of the last place of s, at most s in size), |r| > s / 2 moves q0
 * towards x, |r| == s / 2 is a tie that the even neighbour gets.  That is one
 * multiplication and two additions per element (the rounding is the addition of
 * 1.5 * 2^23, whose sum holds q0 in its low byte); the correction is a rare branch.
 * A division per element would cost more than reading and writing the element.
 *
 * Bound by HBM: the row is read once, kept in registers between its maximum and its
 * quotients, and written (16384 x 8192 bf16: 74.5 us, 5.4 TB/s, 78 without a pause; 64 x 4096:
 * 2.6 us).  A row is a warp's where rows are short and many, a block's otherwise.  Rows of
 * more than 8192 16-bit or 4096 32-bit elements take a form that spills 80 bytes a thread,
 * and what passes twice that length is read twice, the second time from L2 (8192 x 14336 bf16:
 * 81 us, 4.4 TB/s; 4096 x 28672: 85).  Rows that do not start on 16-byte boundaries are read
 * element by element (16384 x 8001 fp16: 147 us).
 */
#include <cstdint>

#include <cuda_runtime.h>

#include "aclsparse_b200_kernels.h"
#include "element_types.cuh"
#include "plan_kernels.h"
#include "tcgen05.cuh"

namespace {

using aclsp::kBF16;
using aclsp::kF16;
using aclsp::kF32;

constexpr uint32_t kThreads = 256;
constexpr float kShift = 12582912.0f;      // 1.5 * 2^23
constexpr float kSmallestScale = 1e-30f;   // below it 1 / s and s / 2 may not be exact enough: plain division instead

// max|x| as bits: unsigned integers are in the order of the absolute values, and NaNs above them all; so are the
// 16-bit types' halves of a word, two at a time.
__device__ __forceinline__ uint32_t AbsBits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

__device__ __forceinline__ float BitsToMax(uint32_t bits)
{
    return __uint_as_float(bits > 0x7F800000u ? 0x7FC00000u : bits);
}

// One load of kVec neighbouring elements as they are, and elements out of it.
template <int kIn, int kVec>
struct Chunk {
    uint32_t w[kVec == 1 ? 1 : 4];

    __device__ __forceinline__ void Load(const void* base, int64_t element)
    {
        if constexpr (kVec == 1) {
            if constexpr (kIn == kF32) {
                w[0] = __ldg(static_cast<const uint32_t*>(base) + element);
            } else {
                w[0] = __ldg(static_cast<const unsigned short*>(base) + element);
            }
        } else {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(base) +
                                                                  element * (kIn == kF32 ? 4 : 2)));
            w[0] = v.x;
            w[1] = v.y;
            w[2] = v.z;
            w[3] = v.w;
        }
    }
    __device__ __forceinline__ uint32_t Top(uint32_t top) const
    {
#pragma unroll
        for (int i = 0; i < (kVec == 1 ? 1 : 4); ++i) {
            if constexpr (kIn == kF32) {
                top = max(top, AbsBits(__uint_as_float(w[i])));
            } else {
                top = __vmaxu2(top, w[i] & 0x7FFF7FFFu);
            }
        }
        return top;
    }
    // The answer of Top as the bits of an fp32 number.
    static __device__ __forceinline__ uint32_t TopBits(uint32_t top)
    {
        if constexpr (kIn == kF32) {
            return top;
        }
        const uint32_t half = max(top & 0xFFFFu, top >> 16);
        if constexpr (kIn == kBF16) {
            return half << 16;
        }
        return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(half))));
    }
    __device__ __forceinline__ float Get(int i) const
    {
        if constexpr (kIn == kF32) {
            return __uint_as_float(w[i]);
        } else {
            const uint32_t bits = i % 2 == 0 ? w[i / 2] & 0xFFFFu : w[i / 2] >> 16;
            if constexpr (kIn == kBF16) {
                return __uint_as_float(bits << 16);
            } else {
                return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
            }
        }
    }
};

// The quantisation of one row: q(x) in the low byte of the answer.
struct RowScale {
    float scale;
    float inverse;
    float half;
    bool zeros;  // the scale is zero, infinite or NaN
    bool small;

    __device__ __forceinline__ explicit RowScale(float top)
    {
        scale = top * (1.0f / 127.0f);
        zeros = !(scale > 0.0f && scale <= 3.402823466e38f);
        small = scale < kSmallestScale;
        inverse = __fdiv_rn(1.0f, scale);
        half = 0.5f * scale;
    }
    // Bytes of kVec elements, in the low bytes of q.
    template <int kVec>
    __device__ __forceinline__ void Round(const float (&x)[kVec], uint32_t (&q)[kVec]) const
    {
        bool close = small;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const float t = fmaf(x[e], inverse, kShift);
            q[e] = __float_as_uint(t);
            close = close || fabsf(fmaf(kShift - t, scale, x[e])) >= half;
        }
        if (close) {
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                q[e] = Careful(small ? rintf(__fdiv_rn(x[e], scale)) : __uint_as_float(q[e]) - kShift, x[e]);
            }
        }
    }
    __device__ __forceinline__ uint32_t Careful(float q, float x) const
    {
        const float r = fmaf(-q, scale, x);
        const float twice = 2.0f * fabsf(r);
        const bool odd = (static_cast<int>(q) & 1) != 0;
        if (twice > scale || (twice == scale && odd)) {
            q += r > 0.0f ? 1.0f : -1.0f;
        }
        return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(q, -127.0f), 127.0f)));
    }
};

template <int kVec>
__device__ __forceinline__ void StoreBytes(signed char* to, const uint32_t (&q)[kVec])
{
    if constexpr (kVec == 1) {
        *to = static_cast<signed char>(q[0]);
    } else {
        uint32_t w[kVec / 4];
#pragma unroll
        for (int i = 0; i < kVec / 4; ++i) {
            w[i] = __byte_perm(__byte_perm(q[4 * i], q[4 * i + 1], 0x0040), __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040), 0x5410);
        }
        if constexpr (kVec == 8) {
            *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
        } else {
            *reinterpret_cast<uint32_t*>(to) = w[0];
        }
    }
}

// kLanes threads per row (32 or kThreads), kHold loads of kVec elements each; with kTwice the loads that do not fit are
// read again.  Elements behind the last whole vector (fewer than kVec) are one thread's each.  The overlap of loads and
// arithmetic is that of the blocks on an SM: persistent blocks that ask for their next row before they work on the
// present one need so many registers more that they are slower (16384 x 8192 bf16: 94 us against 86).
template <int kIn, int kVec, uint32_t kLanes, int kHold, bool kTwice>
__global__ void __launch_bounds__(kThreads, kVec == 1 ? 8 : 6) QuantizeRowsKernel(const void* x, signed char* __restrict__ q,
                                                               float* __restrict__ scales, uint32_t rows,
                                                               uint32_t cols, int64_t ldx, int64_t ldq)
{
    __shared__ uint32_t warpTop[kThreads / 32];
    aclsp::WaitForPreviousKernel(x);
    aclsp::LetNextKernelStart();
    constexpr uint32_t kRows = kThreads / kLanes;
    const uint32_t lane = threadIdx.x % kLanes;
    const uint32_t row = blockIdx.x * kRows + threadIdx.x / kLanes;
    if (row >= rows) {
        return;  // whole warps, and whole blocks where a block is a row
    }
    const int64_t from = static_cast<int64_t>(row) * ldx;
    const uint32_t vectors = cols / kVec;
    const uint32_t rest = vectors * kVec + lane;  // this thread's element behind the vectors
    const bool hasRest = kVec > 1 && rest < cols;
    Chunk<kIn, kVec> hold[kHold];
    float last = 0.0f;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
        const uint32_t v = lane + static_cast<uint32_t>(i) * kLanes;
        if (v < vectors) {
            hold[i].Load(x, from + static_cast<int64_t>(v) * kVec);
        } else {
            hold[i] = {};
        }
    }
    if (hasRest) {
        last = aclsp::LoadIn<kIn>(x, from + rest);
    }
    uint32_t packed = 0;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
        packed = hold[i].Top(packed);
    }
    if constexpr (kTwice) {
        for (uint32_t v = lane + kHold * kLanes; v < vectors; v += kLanes) {
            Chunk<kIn, kVec> c;
            c.Load(x, from + static_cast<int64_t>(v) * kVec);
            packed = c.Top(packed);
        }
    }
    uint32_t top = max(Chunk<kIn, kVec>::TopBits(packed), AbsBits(last));
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if constexpr (kLanes > 32) {
        if (threadIdx.x % 32u == 0u) {
            warpTop[threadIdx.x / 32u] = top;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < kThreads / 32u; ++w) {
            top = max(top, warpTop[w]);
        }
    }
    const RowScale s(BitsToMax(top));
    if (lane == 0) {
        scales[row] = s.scale;
    }
    signed char* const to = q + static_cast<int64_t>(row) * ldq;
    auto store = [&](const Chunk<kIn, kVec>& c, uint32_t v) {
        float f[kVec];
        uint32_t b[kVec] = {};
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            f[e] = c.Get(e);
        }
        if (!s.zeros) {
            s.Round(f, b);
        }
        StoreBytes<kVec>(to + static_cast<int64_t>(v) * kVec, b);
    };
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
        const uint32_t v = lane + static_cast<uint32_t>(i) * kLanes;
        if (v < vectors) {
            store(hold[i], v);
        }
    }
    if constexpr (kTwice) {
        for (uint32_t v = lane + kHold * kLanes; v < vectors; v += kLanes) {
            Chunk<kIn, kVec> c;
            c.Load(x, from + static_cast<int64_t>(v) * kVec);
            store(c, v);
        }
    }
    if (hasRest) {
        const float f[1] = {last};
        uint32_t b[1] = {};
        if (!s.zeros) {
            s.Round(f, b);
        }
        to[rest] = static_cast<signed char>(b[0]);
    }
}

template <int kIn, int kVec, uint32_t kLanes, int kHold, bool kTwice>
void LaunchForm(const void* x, signed char* q, float* scales, uint32_t rows, uint32_t cols, int64_t ldx, int64_t ldq,
                cudaStream_t s)
{
    constexpr uint32_t kRows = kThreads / kLanes;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((rows + kRows - 1u) / kRows);
    config.blockDim = dim3(kThreads);
    config.stream = s;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    cudaLaunchKernelEx(&config, QuantizeRowsKernel<kIn, kVec, kLanes, kHold, kTwice>, x, q, scales, rows, cols, ldx, ldq);
}

template <int kIn, int kVec>
void Launch(const void* x, signed char* q, float* scales, uint32_t rows, uint32_t cols, int64_t ldx, int64_t ldq,
            cudaStream_t s)
{
    // As many loads as a row needs of each thread, so that none is masked off for nothing.
    const uint32_t vectors = (cols + kVec - 1u) / kVec;
    if (vectors <= 4u * 32u && rows >= 2048u) {
        LaunchForm<kIn, kVec, 32, 4, false>(x, q, scales, rows, cols, ldx, ldq, s);
    } else if (vectors <= 2u * kThreads) {
        LaunchForm<kIn, kVec, kThreads, 2, false>(x, q, scales, rows, cols, ldx, ldq, s);
    } else if (vectors <= 4u * kThreads) {
        LaunchForm<kIn, kVec, kThreads, 4, false>(x, q, scales, rows, cols, ldx, ldq, s);
    } else {
        LaunchForm<kIn, kVec, kThreads, kVec == 1 ? 16 : 8, true>(x, q, scales, rows, cols, ldx, ldq, s);
    }
}

}  // namespace

extern "C" void aclsp_b200_quantize_rows_kernel_do(const void* x, void* q, float* scales, uint32_t rows, uint32_t cols,
                                                   int64_t ldx, int64_t ldq, uint32_t xType, void* stream)
{
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    signed char* out = static_cast<signed char*>(q);
    AclspCountLaunches(1);
    // 16-byte loads where every row starts on one's boundary and its bytes on the matching one of Q.
    const int64_t bytes = xType == ACLSP_TYPE_F32 ? 4 : 2;
    const int64_t wide = 16 / bytes;
    const bool vector = reinterpret_cast<uintptr_t>(x) % 16u == 0u && ldx % wide == 0 &&
                        reinterpret_cast<uintptr_t>(q) % static_cast<uint64_t>(wide) == 0u && ldq % wide == 0;
    if (xType == ACLSP_TYPE_F16) {
        vector ? Launch<kF16, 8>(x, out, scales, rows, cols, ldx, ldq, s) : Launch<kF16, 1>(x, out, scales, rows, cols, ldx, ldq, s);
    } else if (xType == ACLSP_TYPE_BF16) {
        vector ? Launch<kBF16, 8>(x, out, scales, rows, cols, ldx, ldq, s) : Launch<kBF16, 1>(x, out, scales, rows, cols, ldx, ldq, s);
    } else {
        vector ? Launch<kF32, 4>(x, out, scales, rows, cols, ldx, ldq, s) : Launch<kF32, 1>(x, out, scales, rows, cols, ldx, ldq, s);
    }
}
