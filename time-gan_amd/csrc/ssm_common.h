// Shared by the kernels of the state-space operators (short_conv.hip, scan.hip): element types, the two
// nonlinearities, and the search for a row's slot among the rows of a one-token call.
#pragma once
#include "../../include/tgru.h"
#include "tgru_internal.h"

namespace tgru {
namespace ssm {

constexpr float kLog2e = 1.44269504088896f;
constexpr float kLn2 = 0.693147180559945f;

// Element types of the sequence tensors: float, __bf16, _Float16.  Conversions to and from float are the compiler's
// (to nearest even); everything between load and store is float.
template <typename X>
__device__ __forceinline__ float to_float(X v) { return (float)v; }
template <typename X>
__device__ __forceinline__ X from_float(float v) { return (X)v; }

// 1 / (1 + exp(-v)) on the hardware exp2 / rcp units: about 2 ulp; 0 and 1 at the far ends.
__device__ __forceinline__ float sigmoid(float v) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * v));
}

// log(1 + exp(v)) = max(v, 0) + log1p(exp(-|v|)) with log1p(e) = 2 atanh(e / (2 + e)): e is in [0, 1], so the atanh
// argument s is in [0, 1/3] and its Taylor series in s^2 <= 1/9 is cut after nine terms (the next one is below
// 9^-9 / 19, 2^-32 of the result).  Unlike log2(1 + e) on the hardware unit it keeps its relative precision where the
// result is small -- step sizes of 0.001 are v = -6.9.
__device__ __forceinline__ float softplus(float v) {
    const float e = __builtin_amdgcn_exp2f(-kLog2e * fabsf(v));
    const float s = e * __builtin_amdgcn_rcpf(2.f + e);
    const float q = s * s;
    float p = 1.f / 17.f;
    p = __builtin_fmaf(p, q, 1.f / 15.f);
    p = __builtin_fmaf(p, q, 1.f / 13.f);
    p = __builtin_fmaf(p, q, 1.f / 11.f);
    p = __builtin_fmaf(p, q, 1.f / 9.f);
    p = __builtin_fmaf(p, q, 1.f / 7.f);
    p = __builtin_fmaf(p, q, 1.f / 5.f);
    p = __builtin_fmaf(p, q, 1.f / 3.f);
    p = __builtin_fmaf(p, q, 1.f);
    return __builtin_fmaf(2.f * s, p, fmaxf(v, 0.f));
}

__device__ __forceinline__ int clamped_length(const int32_t *lengths, int b, int T) {
    return lengths ? min(max(lengths[b], 0), T) : T;
}

// The first row j in [from, to) with slots[j] == slot, or `to`.  All 64 lanes of the wave call it with the same
// arguments; 256 rows are looked at per trip, their loads in flight together.
__device__ __forceinline__ int find_slot(const int32_t *__restrict__ slots, int from, int to, int slot) {
    const int lane = threadIdx.x & 63;
    for (int base = from; base < to; base += 256) {
        int v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = slots[min(base + 64 * k + lane, to - 1)];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned long long hit = __ballot(base + 64 * k + lane < to && v[k] == slot);
            if (hit) return base + 64 * k + __ffsll(hit) - 1;
        }
    }
    return to;
}

inline bool known_dtype(int dtype) { return dtype == TGRU_DTYPE_F32 || dtype == TGRU_DTYPE_BF16 || dtype == TGRU_DTYPE_F16; }
inline size_t dtype_bytes(int dtype) { return dtype == TGRU_DTYPE_F32 ? 4 : 2; }

}  // namespace ssm
}  // namespace tgru
