// What the model operators share: element types, packed rows, the gate of the recurrence.
#pragma once

#include "common.hpp"

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

// The gate of the recurrence: k = 1 - f = 1 / (1 + exp(g)), to full relative precision however small (1 - f would be what
// is left of a rounded f).  The steps below use k alone, so that a channel that forgets once in a million tokens
// keeps its rate; each rounds once, by at most half a unit of the larger of what goes in.
__device__ __forceinline__ float gate_taken(float g)
{
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(1.44269504f * g));
}
__device__ __forceinline__ float next_state(float k, float h, float x) { return fmaf(k, x - h, h); }     // f h + (1 - f) x
__device__ __forceinline__ float forget(float k, float v) { return fmaf(-k, v, v); }                     // f v
__device__ __forceinline__ float slope(float k) { return fmaf(-k, k, k); }                               // f (1 - f)

}  // namespace dnatok
