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
    int64_t n, total, length;
    __device__ __forceinline__ int64_t at(int64_t b) const { return offsets ? offsets[b] : b * length; }
};

// The gate of the recurrence as one signed number: of f = sigmoid(g) and 1 - f the one that is at most a half, e / (1 + e)
// with e = exp(-|g|), with g's sign.  The state's update uses only that one, so that a channel that forgets
// once in a million tokens keeps its rate (1 - f is not what is left of a rounded f), and a channel that forgets at once
// keeps x.
__device__ __forceinline__ float gate_share(float g)
{
    const float e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(g));
    return copysignf(e * __builtin_amdgcn_rcpf(1.0f + e), g);
}
__device__ __forceinline__ bool mostly_kept(float share) { return (int32_t)__float_as_uint(share) >= 0; }   // (f >= 1/2)
__device__ __forceinline__ float next_state(float share, float h, float x)        // f h + (1 - f) x
{
    return fmaf(share, x - h, mostly_kept(share) ? h : x);
}
__device__ __forceinline__ float forget(float share, float v)                     // f v
{
    return fmaf(-share, v, mostly_kept(share) ? v : 0.0f);
}
__device__ __forceinline__ float taken(float share)                               // 1 - f
{
    return mostly_kept(share) ? share : 1.0f + share;
}
__device__ __forceinline__ float slope(float share)                               // f (1 - f)
{
    return fabsf(share) * (1.0f - fabsf(share));
}

}  // namespace dnatok
