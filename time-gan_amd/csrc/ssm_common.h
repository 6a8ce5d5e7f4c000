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

// 1 / (1 + exp(-v)) on the hardware exp2 / rcp units; 0 and 1 at the far ends.  The relative error below 0 is mostly that of
// exp2's argument, a rounded product with a rounded constant: 1.22 |v| half steps, and about 5 from exp2, the sum and the
// reciprocal; above 0 those 5 at most.  Measured, v sigmoid(v) against 64 bits: 2.8 half steps above 0, 5.7 at -5, 9.5 at -10,
// 17 at -20, 64 at -80.
__device__ __forceinline__ float sigmoid(float v) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * v));
}

// log(1 + exp(v)) = max(v, 0) + log1p(e), e = exp(-|v|) in [0, 1].  log1p(e) = log(w) + (e - (w - 1)) for the rounded
// sum w = 1 + e: what the sum lost is added back (divided by w it would be exact to first order; w is in [1, 2] and the
// term below half a step of w), so the result keeps its relative precision where it is small -- step sizes of 0.001 are
// v = -6.9.  The slope is the sigmoid of v.  Measured against 64 bits: 10 half steps at v in [-10, 0), 2.4 above, 18 at
// -15, nearly all of it the rounding of exp2's argument.
__device__ __forceinline__ void softplus_slope(float v, float &value, float &slope) {
    const float e = __builtin_amdgcn_exp2f(-kLog2e * fabsf(v)), w = 1.f + e, r = __builtin_amdgcn_rcpf(w);
    value = fmaxf(v, 0.f) + __builtin_fmaf(kLn2, __builtin_amdgcn_logf(w), e - (w - 1.f));
    slope = v < 0.f ? e * r : r;
}
__device__ __forceinline__ float softplus(float v) {
    float value, slope;
    softplus_slope(v, value, slope);
    return value;
}

__device__ __forceinline__ int clamped_length(const int32_t *lengths, int b, int T) {
    return lengths ? min(max(lengths[b], 0), T) : T;
}

// The first row j in [from, to) with slots[j] == slot, or `to`.  All 64 lanes of the wave call it with the same
// arguments; 256 rows are looked at per trip, their loads in flight together.  Every wave of every row goes through all slots,
// so a call's search grows with the square of its rows.  Measured, scan with 256 channels (16 waves a row), fp32, 16 states:
// nothing at 300 rows, 30 us become 98 at 4096, 0.4 ms become 15 at 65536, 0.8 become 59 at 131072.
__device__ __forceinline__ int find_slot(const int32_t *__restrict__ slots, int from, int to, int slot) {
    const int lane = threadIdx.x & 63;
    for (int base = from; base < to; base += 256) {
        int v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = slots[min(base + 64 * k + lane, to - 1)];
        asm volatile("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));      // (else each is loaded when its turn comes)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned long long hit = __ballot(base + 64 * k + lane < to && v[k] == slot);
            if (hit) return base + 64 * k + __ffsll(hit) - 1;
        }
    }
    return to;
}

// p[r0 * stride] + ... + p[(r1 - 1) * stride], in an order that is fixed by r0 and r1; sixteen loads in flight, because a
// thread's rows are one chain of round trips to memory (the scan's parameter gradients of 2048 sequences: 17 us, four loads 49).
__device__ __forceinline__ float sum_rows(const float *__restrict__ p, long stride, int r0, int r1) {
    constexpr int U = 16;
    float s[U];
#pragma unroll
    for (int q = 0; q < U; ++q) s[q] = 0.f;
    int r = r0;
    for (; r + U <= r1; r += U)
#pragma unroll
        for (int q = 0; q < U; ++q) s[q] += p[(long)(r + q) * stride];
    for (; r + 4 <= r1; r += 4)
#pragma unroll
        for (int q = 0; q < 4; ++q) s[q] += p[(long)(r + q) * stride];
    for (; r < r1; ++r) s[0] += p[(long)r * stride];
#pragma unroll
    for (int w = U / 2; w > 0; w >>= 1)
#pragma unroll
        for (int q = 0; q < w; ++q) s[q] += s[q + w];
    return s[0];
}

// Whether a one-token call with slots is refused because its search would take seconds (2^44 row pairs and waves: about 4 s).
inline bool search_too_long(const int32_t *slots, int B, long waves_per_row) {
    return slots && (double)B * B * waves_per_row >= 17592186044416.0;
}

inline bool known_dtype(int dtype) { return dtype == TGRU_DTYPE_F32 || dtype == TGRU_DTYPE_BF16 || dtype == TGRU_DTYPE_F16; }
inline size_t dtype_bytes(int dtype) { return dtype == TGRU_DTYPE_F32 ? 4 : 2; }

}  // namespace ssm
}  // namespace tgru
