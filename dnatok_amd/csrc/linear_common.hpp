// Linear attention with a decay for each head, over packed rows: T_t = g T_(t-1) + k_t v_t^T, y_t = scale q_t T_t.
//
// Every product that the operator and its gradients need is one walk over a row,
//   T_t = D_(t-1) + b_t c_t^T,  D_t = g T_t,  out_t = scale a_t T_t:
// y = walk(q, k, v), dq = walk(dy, v, k), and from the row's other end dv = walk(k, q, dy) and dk = walk(v, dy, q), whose T is the
// gradient of the state.  What is in front of a row's first token (h0, or the gradient of the last state) enters as
// T forwards, so that it decays on its way in, and as D backwards; what is left behind its last token is the same.
//
// Steps are taken in chunks of 64: with the scores P[t][s] = a_t b_s g^(t - s) for s <= t of one chunk, and T in front of it,
//   out_t = scale (g^(t + 1) a_t T + sum_s P[t][s] c_s),   T' = g^64 T + sum_s g^(63 - s) b_s c_s^T
// (backwards each decay comes a step later): four products on the matrix cores, 16 x 16 x 32 for 16-bit operands and 16 x 16 x 4
// in 32 bits.  The chunk's operands lie in LDS; T stays in registers, where the result of one product is the operand of
// the next as it is: a lane has column l % 16 and rows 4 (l / 16) .. + 3 of a tile of T, and which of the rows of a contraction a lane
// has is free as long as the other operand's are the same.
#pragma once

#include "lm_common.hpp"

namespace dnatok {

struct Operand {
    const void *p;
    int64_t token, head;                           // elements between tokens and between heads
    int32_t shared, dim;                           // heads of the walk that share one here
};

struct WalkArgs {
    Operand a, b, c;
    const float *log_decay;
    const int64_t *offsets;
    int64_t n_rows, total, length;
    int32_t heads;
    bool reverse, decayed;
    float scale, start_scale, end_scale;
    const float *start;                            // [rows, heads, b.dim, c.dim], or transposed; NULL: zeros
    bool transposed;
    float *end;
    void *out;                                     // [total, heads, c.dim]
    bool out32;                                    // of 32 bits, whatever the operands are
    bool exact;                                    // whether states of 32 bits come of it
    float *slots;                                  // states at the cuts [cuts, heads, b.dim, c.dim], as `start` is laid out
    int64_t cut, cuts;                             // tokens from one to the next
    int64_t first_item;                            // of the launch
};

constexpr int kOutside = 64;                       // workgroups that clear what is in no row
constexpr int kChunk = 64;
// A wave to sixteen columns of the state.
constexpr int threads_of(int columns) { return columns * 4; }

// The walk itself, and what its pieces add to the state (linear_walk_*.hip); w.cuts pieces more than rows.
template <typename T> void launch_walk(const WalkArgs &w, hipStream_t s);
template <typename T> void launch_pieces(const WalkArgs &w, hipStream_t s);

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// ---- pieces of the packed axis --------------------------------------------------------------------

// The axis is cut where rows begin and at the multiples of w.cut inside rows.  Pieces are numbered cuts first: piece m - 1 begins at the
// m-th multiple, and is none if a row begins there or none is there; those that begin the rows come behind.  (Long pieces are
// the first ones, and no search is needed for a row.  In the order of the axis, where rows begin at multiples every second piece is
// none, and workgroups are dealt out so that half of the CUs got only those: 64 rows of 8,192 tokens took twice the time.)
struct Piece {
    int64_t row, lo, hi;
    bool front, back;                              // whether it begins and ends its row
    bool none;
};

__device__ __forceinline__ int64_t row_at(const WalkArgs &w, int64_t r)
{
    if (!w.offsets) return r * w.length;
    const int64_t v = w.offsets[r];
    return v < 0 ? 0 : v > w.total ? w.total : v;
}

// The last row r with before(r) <= item, or -1, where before ascends: all threads of a workgroup look at once.
template <typename Before> __device__ __forceinline__ int64_t last_row(int64_t n_rows, int64_t item, Before before)
{
    int64_t lo = -1, hi = n_rows;                  // (lo holds, hi does not)
    while (hi - lo > 1) {
        const int64_t step = (hi - lo - 1 + blockDim.x - 1) / blockDim.x;
        const int64_t r = lo + step * (threadIdx.x + 1);
        const int n = __syncthreads_count(r < hi && before(r) <= item);
        const int64_t from = lo + step * n;
        hi = from + step < hi ? from + step : hi;
        lo = from;
    }
    return lo;
}

__device__ __forceinline__ int64_t uniform(int64_t v)
{
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

__device__ __forceinline__ Piece piece_of(const WalkArgs &w, int64_t item)
{
    Piece p{};
    int64_t at;
    if (item < w.cuts) {
        at = (item + 1) * w.cut;
        p.row = last_row(w.n_rows, at, [&](int64_t r) { return row_at(w, r); });
        p.none = p.row < 0;
    } else {
        p.row = item - w.cuts;
        at = row_at(w, p.row);
    }
    if (p.none) return p;
    const int64_t begin = row_at(w, p.row), end = row_at(w, p.row + 1);
    p.lo = at;
    p.hi = end;
    p.row = uniform(p.row);
    if (w.cuts) {
        const int64_t next = (at / w.cut + 1) * w.cut;
        p.hi = next < end ? next : end;
    }
    if (p.hi < p.lo) p.hi = p.lo;
    p.front = p.lo == begin;
    p.back = p.hi == end || end < begin;
    p.none = item < w.cuts && (at <= begin || at >= end);
    p.lo = uniform(p.lo);
    p.hi = uniform(p.hi);
    const int flags = __builtin_amdgcn_readfirstlane(p.front | p.back << 1 | p.none << 2);
    p.front = flags & 1;
    p.back = flags & 2;
    p.none = flags & 4;
    return p;
}

// ---- the state -------------------------------------------------------------------------------------

// What is left of a state after n steps (one at least): by the factor, or by 1 - it.  (A factor next to 1, rounded once and multiplied
// thousands of times, would be a wrong rate.)  keeps: not if a step leaves nothing at all, whatever the state is.
constexpr float kNothingLeft = -1e30f;
struct Left {
    float factor, lost;
    bool keeps;
};
__device__ __forceinline__ Left left_after(float log_decay, float n)
{
    // factor s - lost s: one of them is 0, and the other the more exact one
    const float lost = -expm1f(n * log_decay);
    const bool keeps = !(log_decay <= kNothingLeft);
    return lost < 0.5f ? Left{1.0f, lost, keeps} : Left{expf(n * log_decay), 0.0f, keeps};
}
// (An infinity stays one as long as anything is left of a state, also where the factor has become 0, and a NaN stays one; a decay that is
// NaN makes one.)
__device__ __forceinline__ float decayed(float s, const Left &l)
{
    const float v = fmaf(-l.lost, s, l.factor * s);
    return __builtin_fabsf(s) < INFINITY ? v : l.keeps ? s + 0.0f * l.factor : 0.0f;
}

__device__ __forceinline__ float log_decay_of(const float *log_decay, int head)
{
    return __builtin_elementwise_maximum(log_decay[head], kNothingLeft);        // (so that -inf times no step at all is 0; keeps a NaN)
}

}  // namespace dnatok
