// Running log-sum-exp of a row segment, shared by the kernels that read whole
// rows of logits (draft verification, distillation).
//
// A partial sum is the pair (m, s): s the sum of exp(v - m) over the segment, m
// a reference at most kHeadroom below the largest v. A thread takes its logits in
// batches of 16: the batch's maximum first, then sixteen exponentials against one
// reference, added as a tree in binary32 and once per batch into a binary64 sum.
// At its end a thread brings the sum to its largest v itself, so that the reference
// of a row is its maximum, however the row is cut.
// Its error has three parts. An exponential is ex2.approx of a product rounded
// once, |v - m| 2^-23 + 2^-22 relative. A new reference, the thread's maximum, and
// the join of lanes, warps and parts, scales a sum by one more of them; references
// rise by more than kHeadroom, so the terms that count, within 25 of the largest,
// see at most six, and their distances add up to that 25 and twice kHeadroom (a v
// above m): 4e-6 + 11 * 2^-22 in all. The trees are four additions deep (2^-22).
// Together below 7e-6 (6e-6 where the reference stays, as in distillation).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "rsc_common.cuh"

namespace rsc {

// Logits of one 16-byte load.
template <typename T>
constexpr int kVecElems = 16 / static_cast<int>(sizeof(T));

template <typename T>
__device__ __forceinline__ float elem_to_float(T x);
template <>
__device__ __forceinline__ float elem_to_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float elem_to_float<__nv_bfloat16>(__nv_bfloat16 x) {
    return __bfloat162float(x);
}
template <>
__device__ __forceinline__ float elem_to_float<__half>(__half x) { return __half2float(x); }

// The elements of one 16-byte word as binary32.
template <typename T>
__device__ __forceinline__ void unpack(const uint4 &w, float *f);
template <>
__device__ __forceinline__ void unpack<float>(const uint4 &w, float *f) {
    f[0] = __uint_as_float(w.x);
    f[1] = __uint_as_float(w.y);
    f[2] = __uint_as_float(w.z);
    f[3] = __uint_as_float(w.w);
}
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4 &w, float *f) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
template <>
__device__ __forceinline__ void unpack<__half>(const uint4 &w, float *f) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = *reinterpret_cast<const __half2 *>(&u[i]);
        const float2 g = __half22float2(h);
        f[2 * i] = g.x;
        f[2 * i + 1] = g.y;
    }
}

// exp(d): ex2.approx of the product with log2(e).
__device__ __forceinline__ float exp_fast(float d) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fmul_rn(d, 1.4426950408889634f)));
    return r;
}

constexpr float kHeadroom = 4.0f;

// Adds kN scaled logits to (m, s) and raises `top` to their largest. A logit of -inf adds nothing; +inf makes m
// +inf and s NaN, and NaN makes s NaN (callers that read NaN as -inf fold it
// beforehand).
template <int kN>
__device__ __forceinline__ void sum_batch(float &m, float &top, double &s, const float *v) {
    float b = v[0];
#pragma unroll
    for (int i = 1; i < kN; ++i) b = fmaxf(b, v[i]);
    top = fmaxf(top, b);
    if (b > m + kHeadroom) {
        // m = -inf only while s is 0 or NaN, which the product keeps.
        s *= m == kNegInf ? 1.0 : static_cast<double>(exp_fast(__fsub_rn(m, b)));
        m = b;
    }
    // Against a maximum of -inf every logit is -inf or NaN: 0 keeps -inf - m
    // from being NaN.
    const float ref = m == kNegInf ? 0.0f : m;
    float e[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) e[i] = exp_fast(__fsub_rn(v[i], ref));
#pragma unroll
    for (int w = 1; w < kN; w *= 2) {
#pragma unroll
        for (int i = 0; i + w < kN; i += 2 * w) e[i] = __fadd_rn(e[i], e[i + w]);
    }
    s = __dadd_rn(s, static_cast<double>(e[0]));
}

// A thread's sum brought to its largest v.
__device__ __forceinline__ void sum_to_top(float &m, float top, double &s) {
    if (top > m) s *= static_cast<double>(exp_fast(__fsub_rn(m, top)));
    m = top;
}

// The sums of `width` neighbouring lanes joined, in every one of them: the
// largest reference first, then each lane's sum brought to it by one exponential.
__device__ __forceinline__ void sum_join_lanes(float &m, double &s, int width) {
    float top = m;
    for (int o = width / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // A lane at -inf holds 0 or NaN, which stays.
    if (m != kNegInf) s *= static_cast<double>(exp_fast(__fsub_rn(m, top)));
    for (int o = width / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    m = top;
}

}  // namespace rsc
