// Shared by the operators that run next to a neighbor list: element types,
// matrix instructions over 32 x 32 tiles, and the scores of the two
// attentions.  Target: gfx950, wave64.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/tonari_operators.h"

#include <cmath>
#include <cstdint>
#include <type_traits>

namespace tnr {
namespace op {

constexpr int kWave = 64;
constexpr float kLog2e = 1.4426950408889634f;

using bf16 = __bf16;
using f16 = _Float16;

template <typename T, int N>
using Vec = T __attribute__((ext_vector_type(N)));
using f32x16 = Vec<float, 16>;

__device__ __forceinline__ int lane_of() { return (int)__lane_id(); }
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float nan_of() { return __int_as_float(0x7fc00000); }
__device__ __forceinline__ float inf_of() { return __int_as_float(0x7f800000); }

// The pair of values that a lane and the lane 32 away hold.
struct Halves {
    float low, high;
};
__device__ __forceinline__ Halves halves_of(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}
__device__ __forceinline__ float sum_halves(float x) {
    const Halves h = halves_of(x);
    return h.low + h.high;
}
__device__ __forceinline__ float max_halves(float x) {
    const Halves h = halves_of(x);
    return fmaxf(h.low, h.high);
}

// Workgroups go to the 8 XCDs in turn; in this order each XCD takes a run of
// the work, so that what neighbours share, or write next to each other, meets
// in one L2.
__device__ __forceinline__ uint32_t xcd_order(uint32_t block, uint32_t blocks) {
    const uint32_t each = blocks / 8, left = blocks % 8, xcd = block % 8, at = block / 8;
    return xcd * each + (xcd < left ? xcd : left) + at;
}

template <int CTRL>
__device__ __forceinline__ float dpp_of(float x) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float sum_of(float a, float b) { return a + b; }
__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }

// f over the lanes whose numbers differ in the bits from `from` (a power of two)
// up, in all of them: rotations within 16 lanes, then swaps of rows.
template <float (*F)(float, float)>
__device__ __forceinline__ float join_lanes(float x, int from) {
    if (from <= 1) x = F(x, dpp_of<0xb1>(x));
    if (from <= 2) x = F(x, dpp_of<0x4e>(x));
    if (from <= 4) x = F(x, dpp_of<0x124>(x));
    if (from <= 8) x = F(x, dpp_of<0x128>(x));
    if (from <= 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x),
                                                        false, false);
        x = F(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    if (from <= 32) {
        const Halves h = halves_of(x);
        x = F(h.low, h.high);
    }
    return x;
}

// ------------------------------------------------------------------ scores

// x = scale q.k and, with a cap c, u = c tanh(x / c).  Scores are held in
// units of log 2, so that the softmax takes exp2.
struct ScoreRule {
    float scale, cap;       // cap 0: none
    float scale2, inv, cap2;  // scale log2(e), scale / cap, cap log2(e)
    static ScoreRule of(float scale, float cap) {
        return {scale, cap, scale * kLog2e, cap > 0.f ? scale / cap : 0.f, cap * kLog2e};
    }
};

// tanh within 1e-8 of its value for |y| <= 0.6 (least squares over Chebyshev
// points of tanh(y) / y in y^2), where exp would cancel; beyond, by exp.
constexpr float kTanhNear = 0.6f;
__device__ __forceinline__ float tanh_near(float y) {
    const float z = y * y;
    float f = fmaf(z, -0.006276389583945274f, 0.021116215735673904f);
    f = fmaf(z, f, -0.053875137120485306f);
    f = fmaf(z, f, 0.13332924246788025f);
    f = fmaf(z, f, -0.3333333134651184f);
    return fmaf(y * z, f, y);
}
__device__ __forceinline__ float tanh_far(float y) {
    const float e = exp2_of(y * (2.f * kLog2e));
    return fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f);
}
__device__ __forceinline__ float tanh_of(float y) {
    return fabsf(y) <= kTanhNear ? tanh_near(y) : tanh_far(y);
}

// ------------------------------------------------------------------- types

template <typename T>
__device__ __forceinline__ T rounded(float x) {
    return (T)x;
}

// N values of 16 bytes or fewer, as floats.
template <typename T, int N>
__device__ __forceinline__ void load_floats(const T* p, float (&x)[N]) {
    const Vec<T, N> v = *(const Vec<T, N>*)p;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)v[i];
}
template <typename T, int N>
__device__ __forceinline__ void store_floats(T* p, const float (&x)[N]) {
    Vec<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = rounded<T>(x[i]);
    *(Vec<T, N>*)p = v;
}

// Sum of n floats by a workgroup of 1,024, in its first thread.
__device__ __forceinline__ float block_sum(const float* x, int64_t n) {
    __shared__ float waves[16];
    float part[8] = {};
    int64_t i = threadIdx.x;
    for (; i + 7 * 1024 < n; i += 8 * 1024)
#pragma unroll
        for (int u = 0; u < 8; ++u) part[u] += x[i + u * 1024];
    for (; i < n; i += 1024) part[0] += x[i];
    float sum = join_lanes<sum_of>(((part[0] + part[1]) + (part[2] + part[3])) +
                                       ((part[4] + part[5]) + (part[6] + part[7])),
                                   1);
    if (lane_of() == 0) waves[threadIdx.x / kWave] = sum;
    __syncthreads();
    sum = 0.f;
    if (threadIdx.x == 0)
        for (int w = 0; w < 16; ++w) sum += waves[w];
    return sum;
}

// A head's slope: the sum of its rows, one workgroup each.
__global__ __launch_bounds__(1024) inline void k_slopes(const float* turn, int64_t rows,
                                                        float* grad_slopes) {
    const float sum = block_sum(turn + (int64_t)blockIdx.x * rows, rows);
    if (threadIdx.x == 0) grad_slopes[blockIdx.x] = sum;
}

}  // namespace op
}  // namespace tnr
