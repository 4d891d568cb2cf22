// Device helpers of the operators that serve a packed batch.
#pragma once

#include "serve.h"

namespace fn {

// The rows of a request (its tokens times `mul`) are cut in items of `div` rows.  Item numbers: request b has those from
// cu[b] mul / div + b on, which leaves each request at least as many as it needs without a sum over the requests; the
// spare ones are empty.
__device__ __forceinline__ int first_item(const int32_t *cu, int b, int mul, int div) {
    return (int) ((long long) cu[b] * mul / div) + b;
}
// the last request whose items start at or before `item`: every lane looks at one of 64 of those left
__device__ __forceinline__ int request_of(const int32_t *cu, int B, int item, int mul, int div) {
    int lo = 0, n = B;
    const int lane = threadIdx.x & 63;
    while (n > 1) {
        const int step = (n + 63) / 64, i = lane * step;
        const bool le = i < n && first_item(cu, lo + i, mul, div) <= item;
        const int k = max(1, __popcll(__ballot(le))) - 1;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}
inline size_t item_count(int B, int T, int mul, int div) { return (size_t) ((long long) T * mul / div) + B; }

// over the lanes l, l ^ 16, l ^ 32, l ^ 48: the same bits in each
__device__ __forceinline__ float max_quarters(float x) {
    float2 r = swap16(x);
    r = swap32(fmaxf(r.x, r.y));
    return fmaxf(r.x, r.y);
}
__device__ __forceinline__ float sum_quarters(float x) {
    float2 r = swap16(x);
    r = swap32(r.x + r.y);
    return r.x + r.y;
}

// e^x = 2^t (1 + r log 2), t = x log2 e as rounded and r what the rounding left, with log2 e in two parts: off by less than
// 2^-22 of the value.  For |x| up to 1e38, whose t is finite: 0 where e^x is below fp32's normal range, and from EXP_INF on
// no finite value (a NaN where r is negative).
__device__ __forceinline__ float exp_(float x) {
    const float t = x * 1.44269504f, r = fmaf(x, 1.925963e-8f, fmaf(x, 1.44269504f, -t)), e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, r * 0.693147181f, e);
}
// the least x with t = 128 or more, where 2^t is infinite; r is 3.5e-7 there, so that e^x is too
constexpr float EXP_INF = 0x1.62e43p+6f;  // 88.72284
// 1 / (1 + e^-x) of any x, within 2^-21 of the value; 0 where it is below fp32's normal range.  The argument is held in the
// range of exp_ by a minimum and a maximum that keep a NaN (fminf and fmaxf drop it).
__device__ __forceinline__ float gate_of(float x) {
    const float y = __builtin_elementwise_minimum(__builtin_elementwise_maximum(-x, -88.0f), EXP_INF);
    return __builtin_amdgcn_rcpf(1.0f + exp_(y));
}

}  // namespace fn
