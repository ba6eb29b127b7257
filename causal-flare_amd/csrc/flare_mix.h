// flare_mix.h -- helpers of the short convolution, the state space scan and softmax attention.
#pragma once

#include "flare_common.h"
#include "flare_mfma.h"

namespace flare {
namespace mix {

using mfma::kLn2;
using mfma::kLog2e;

// Function `fn`<element type>(...) for the element type code `dtype`.
#define FLARE_BY_DTYPE(dtype, fn, ...)                               \
    ((dtype) == FLARE_F32    ? fn<float> __VA_ARGS__                 \
     : (dtype) == FLARE_BF16 ? fn<__hip_bfloat16> __VA_ARGS__        \
                             : fn<__half> __VA_ARGS__)

inline bool known_dtype(int dtype) { return dtype == FLARE_F32 || dtype == FLARE_BF16 || dtype == FLARE_F16; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// log(1 + e^x): the larger part exactly, and log(1 + e) of e = e^-|x| <= 1 as 2 artanh(s), s = e /
// (2 + e) <= 1/3, whose series keeps the relative accuracy of the small steps of x far below 0
// (the first term left out, s^17 / 17, is below 2^-29 of the sum).  A third of the instructions
// of log1pf, which were a fifth of the scan's backward.
__device__ __forceinline__ float softplus(float x) {
    const float e = __expf(-fabsf(x)), s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
    float p = 1.0f / 15.0f;
    p = p * q + 1.0f / 13.0f;
    p = p * q + 1.0f / 11.0f;
    p = p * q + 1.0f / 9.0f;
    p = p * q + 1.0f / 7.0f;
    p = p * q + 1.0f / 5.0f;
    p = p * q + 1.0f / 3.0f;
    return fmaxf(x, 0.0f) + 2.0f * (s + s * (q * p));
}

// a of the lower and b of the upper 32 lanes, then the other halves (permlane32_swap); the same
// for each 16 of 32 lanes (permlane16_swap).  What add(first, second) leaves is thus the sum
// of a over lanes l and l ^ 32 (or 16) in one half of the lanes and that of b in the other.
struct Halves {
    float first, second;
};
__device__ __forceinline__ Halves swap32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b),
                                                    false, false);
    const unsigned lo = r[0], hi = r[1];      // a bit cast of r[1] itself reads r[0]
    return Halves{__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
}
__device__ __forceinline__ Halves swap16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b),
                                                    false, false);
    const unsigned lo = r[0], hi = r[1];
    return Halves{__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
}

// VEC consecutive elements of one row as floats, one load where VEC is more than 1.
template <typename T, int VEC>
struct Pack {
    T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void load_row(const T* p, float (&out)[VEC]) {
    typedef Pack<T, VEC> P;
    struct alignas(VEC * sizeof(T)) A { P p; };
    const A a = *reinterpret_cast<const A*>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = to_f32(a.p.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_row(T* p, const float (&in)[VEC]) {
    typedef Pack<T, VEC> P;
    struct alignas(VEC * sizeof(T)) A { P p; } a;
#pragma unroll
    for (int i = 0; i < VEC; ++i) a.p.v[i] = from_f32<T>(in[i]);
    *reinterpret_cast<A*>(p) = a;
}

// The sums of each column of partial [R, cols], handed to put(column, sum): 64 columns a workgroup,
// 16 threads to a column, each over its share of the rows in order.
template <typename Put>
__global__ __launch_bounds__(1024) void column_sums_kernel(const float* partial, int64_t R, int64_t cols, Put put) {
    __shared__ float red[16][65];
    const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
    const int64_t col = (int64_t)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (col < cols) {
        const int64_t per = (R + 15) / 16, r0 = part * per, r1 = min(r0 + per, R);
        int64_t r = r0;
        for (; r + 8 <= r1; r += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = partial[(r + i) * cols + col];
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i];
        }
        for (; r < r1; ++r) s += partial[r * cols + col];
    }
    red[part][lane] = s;
    __syncthreads();
    if (part == 0 && col < cols) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += red[i][lane];
        put(col, t);
    }
}
template <typename Put>
int launch_column_sums(const float* partial, int64_t R, int64_t cols, Put put, hipStream_t stream) {
    column_sums_kernel<<<dim3((unsigned)ceil_div(cols, 64)), 1024, 0, stream>>>(partial, R, cols, put);
    return check_launch("column_sums");
}

}  // namespace mix
}  // namespace flare
