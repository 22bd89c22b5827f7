// What the model operators share: element types, packed rows, the gate of the recurrence.
#pragma once

#include "common.hpp"

#include <cfloat>
#include <type_traits>

namespace dnatok {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_float(float v) { return (T)v; }

// Calls fn with a value of the element type that a DNATOK_F32 / _BF16 / _F16 argument names (checked before).
template <typename Fn>
inline void with_type(int32_t dtype, Fn fn)
{
    if (dtype == DNATOK_F32) fn(float{});
    else if (dtype == DNATOK_BF16) fn(__bf16{});
    else fn(_Float16{});
}

// The packed axis as spans b = 0 .. count() - 1, tokens at(b) .. at(b + 1).  Without offsets these are the rows, all of one length.
// With offsets the tokens in front of the first row and those behind the last one, which are in no row (the buffer may
// be longer than its rows), are spans too, mostly empty: so a span starts at the axis' first token and one ends at its last,
// whatever the offsets are.  row(b): the span's row, or -1.
struct Rows {
    const int64_t *offsets;
    int64_t n, total, length;
    __device__ __forceinline__ int64_t count() const { return offsets ? n + 2 : n; }
    __device__ __forceinline__ int64_t row(int64_t b) const { return !offsets ? b : b > 0 && b <= n ? b - 1 : -1; }
    __device__ __forceinline__ int64_t at(int64_t b) const
    {
        if (!offsets) return b * length;
        const int64_t v = offsets[b <= 0 ? 0 : b > n ? n : b - 1];
        return b <= 0 ? 0 : b > n + 1 ? total : v;
    }
};

// The gate of the recurrence: f = 1 / (1 + E) and k = 1 - f = E f with E = exp(-g), each to a part in 2^24 / (|g| + 4) of itself however
// small it is (what is left of a rounded 1 - k or 1 - f would not be), so that a channel that forgets once in a million
// tokens keeps its rate, and one that keeps a millionth of a state keeps that much, and passes that much of a gradient on.
// (E is at most 2^126, beyond that its reciprocal would be 0 and E f with it: f is 2^-126 where it should be less.  `minimum` keeps a NaN.)
struct Gate {
    float f, k;
};
__device__ __forceinline__ Gate gate_of(float g)
{
    const float e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(-1.44269504f * g, 126.0f));
    const float f = __builtin_amdgcn_rcpf(1.0f + e);
    return Gate{f, e * f};
}
// Both in one number: k where it is the smaller, otherwise -f.  The larger is 1 - the smaller, to half a unit.
__device__ __forceinline__ float one_number(const Gate &g) { return g.k <= 0.5f ? g.k : -g.f; }
__device__ __forceinline__ Gate gate_from(float m)
{
    const float large = 1.0f - __builtin_fabsf(m);
    return m >= 0.0f ? Gate{large, m} : Gate{-m, large};
}
// v, or the largest number of its sign for an infinity: what is taken off v in proportion, so that an infinity stays one.
__device__ __forceinline__ float finite(float v) { return __builtin_amdgcn_fmed3f(v, -FLT_MAX, FLT_MAX); }
// f h + k x without the rounding of an f (or k) next to 1, which over many steps would be a wrong rate: the larger one's part with
// the smaller's share taken off it, and the smaller one's added.
__device__ __forceinline__ float next_state(const Gate &g, float h, float x)
{
    const bool keeps = g.k <= 0.5f;
    const float p = keeps ? h : x, q = keeps ? x : h, s = keeps ? g.k : g.f;
    return fmaf(s, q, fmaf(-s, finite(p), p));
}

}  // namespace dnatok
