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

// Row b of a packed batch is the tokens at(b) .. at(b + 1); without offsets all rows have one length.
struct Rows {
    const int64_t *offsets;
    int64_t n, total;
    __device__ __forceinline__ int64_t at(int64_t b) const { return offsets ? offsets[b] : b * (total / n); }
};

// sigmoid(g) and 1 - sigmoid(g), each to full relative precision: with e = exp(-|g|) they are 1 / (1 + e) and
// e / (1 + e), and only the one that is at most a half (`small`) enters the state's update, so that a channel
// that forgets once in a million tokens keeps its rate and a channel that forgets at once keeps x.
struct Gate {
    float small, big;
    bool mostly_kept;                                   // g >= 0: the old state has the larger share

    __device__ __forceinline__ explicit Gate(float g)
    {
        const float e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(g));
        big = __builtin_amdgcn_rcpf(1.0f + e);
        small = e * big;
        mostly_kept = g >= 0.0f;
    }
    // f h + (1 - f) x
    __device__ __forceinline__ float next(float h, float x) const
    {
        return mostly_kept ? fmaf(small, x - h, h) : fmaf(small, h - x, x);
    }
    __device__ __forceinline__ float keep() const { return mostly_kept ? small : big; }              // 1 - f
    __device__ __forceinline__ float forget(float v) const { return mostly_kept ? fmaf(-small, v, v) : small * v; }   // f v
    __device__ __forceinline__ float slope() const { return small * big; }                           // f (1 - f)
};

}  // namespace dnatok
