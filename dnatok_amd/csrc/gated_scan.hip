// Gated linear recurrence over packed rows, its backward pass and its single step.
//
//   f_t = sigmoid(gate_t),   h_t = f_t h_(t-1) + (1 - f_t) x_t   in every channel of a row,
//
// from a given state or from zero.  Values, gates and outputs have 16 or 32 bits, states always 32.
//
// A piece of the token axis maps the state in front of it to the state behind it by h -> A h + H, and two pieces
// that follow each other compose: A = A2 A1, H = A2 H1 + H2.  A row's first token is a piece with A = 0 (its state comes
// from h0 alone), so rows need no structure of their own: the whole packed axis is cut into tiles of one size, whether
// it holds one contig or a hundred thousand reads, and the state crosses a tile's edge only where a row does.
//
// A workgroup takes a tile by 64 or 128 channels (lanes lie along the channels, so that a token is one contiguous piece
// of memory); its waves follow each other in time, and each holds its tokens in registers.  One pass
// over them gives the wave's (A, H); these are composed in LDS; the tile's own goes to memory for the tiles behind it;
// the state in front of the tile comes from the tiles before it; a second pass over the registers gives the
// states.  So every value and gate is read from memory once.  The backward pass does the same from the other side
// with what flows towards earlier tokens, and runs the states of a wave's tokens again from the one in front of them,
// which the forward pass has left: 4 bytes for 24 tokens instead of a state for each.
//
// The state in front of a tile: a 64-bit word per tile and channel holds the tile's (A, H); the sixteenth tile of a group
// leaves the same for the group, and then the state at the group's end in its place (marked).  A word says by itself
// whether it is there (a fill kernel has put a pattern that none has), so nothing has to be ordered by a fence.  A tile
// takes the nearest group in front whose state is there, and runs that state through the groups and then the tiles
// between, one after the other.  A group's state is the one in front of it run through the group's word in the same one step, so
// the result is the same to the last bit wherever the state is found and whoever came first.  (With tiles alone, states
// one by one, a contig's tiles followed each other every 0.16 us and more: 4,000,000 tokens x 64 in 2517 us, in an early form with
// groups 855, now 523; its bytes take 323.)
//
// Tokens in no row, in front of the first or behind the last one, are spans of their own that give zeros.
//
// Rounding: f and k = 1 - f are each right to a few units of themselves (more by the gate's size), so what is small stays right: what a closed gate
// leaves, what an open one takes.  A wave's tokens and a tile's waves are joined by rounded products of f, 168 tokens at most (264
// backwards); tile by tile and group by group, where such roundings would become a wrong rate, the smaller of a piece's factor
// and its complement is carried.  An infinite state stays infinite, and NaN comes only where the formula has it.
//
// Bound by memory and by the waits for states.  Measured, bfloat16: 64 rows of 8,192 tokens x 512 forward 412 us with the fill
// of the words, 3.91 TB/s (a copy 4.76); a contig of 1,000,003 x 256 428; 256 rows of 1,024 x 512 forward and backward 524.
// Vector issue is busy 0.41 of the time forward and 0.44 backward.  float32, 300 rows x 203: 1723, 2.5 TB/s of the bytes: a
// slab's piece of a token, 256 bytes, does not begin on a line.
#include "lm_common.hpp"

#include <algorithm>

namespace dnatok {

constexpr uint64_t kNoWord = ~0ull;
constexpr int kGroup = 16;                        // tiles of a group, and groups that a tile looks back
constexpr int kCounterStride = 32;                // (a 128-byte line to a counter)

__global__ __launch_bounds__(256) void fill_words_kernel(uint64_t *words, int64_t n, int64_t n_counters)
{
    typedef uint64_t two __attribute__((ext_vector_type(2)));         // (n is a multiple of 16, a counter 16 words)
    const int64_t all = n + n_counters * kCounterStride / 2;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 2; i < all; i += (int64_t)gridDim.x * 512) {
        const uint64_t v = i < n ? kNoWord : 0;
        *reinterpret_cast<two *>(words + i) = two{v, v};
    }
}

template <typename T>
struct ScanArgs {
    const T *x, *gate;
    int64_t x_stride, gate_stride;
    Rows rows;
    int64_t dim, n_tiles;
    uint32_t n_slabs;
    const float *h0;
    float *states;                                // [waves' pieces, dim] or NULL: the state in front of each piece
    uint64_t *tile_words, *group_words;           // [n_tiles, dim], [n_groups, dim]
    uint32_t *counters;                           // [n_slabs], kCounterStride apart: tiles that have been taken
    T *y;
    float *last;
    // the backward pass
    const T *dy;
    int64_t dy_stride;
    const float *dlast;
    T *dx, *dgate;
    float *dh0;
};

// V channels of one token as they lie in memory.
template <typename T, int V> struct Cell { T v[V]; };

// A number that was there before, and what was found out about it is not kept with it.
__device__ __forceinline__ float once_more(float m)
{
    asm volatile("" : "+v"(m));
    return m;
}

// step(i, look) for the S tokens of a wave, forwards or backwards, PART at a time: look is a true_type where one of a part has a bit in
// `looks`.  (The compiler keeps room for both kinds of a part at once, so parts are as long as the registers allow: states 4 tokens
// with two channels to a lane, 8 with one; gradients and outputs 12.  300 rows x 203 in float32 1730 us, with parts of 4 throughout 1770;
// 256 x 1024 x 512 526, 541.)
template <int S, int PART, typename Fn>
__device__ __forceinline__ void by_parts(uint64_t looks, Fn step)
{
    static_assert(S % PART == 0, "whole parts");
#pragma unroll
    for (int from = 0; from < S; from += PART) {
        if (looks >> from & ((1 << PART) - 1)) {
#pragma unroll
            for (int i = from; i < from + PART; ++i) step(i, std::true_type{});
        } else {
#pragma unroll
            for (int i = from; i < from + PART; ++i) step(i, std::false_type{});
        }
    }
}
template <int S, int PART, typename Fn>
__device__ __forceinline__ void by_parts_back(uint64_t looks, Fn step)
{
#pragma unroll
    for (int from = S - PART; from >= 0; from -= PART) {
        if (looks >> from & ((1 << PART) - 1)) {
#pragma unroll
            for (int i = from + PART - 1; i >= from; --i) step(i, std::true_type{});
        } else {
#pragma unroll
            for (int i = from + PART - 1; i >= from; --i) step(i, std::false_type{});
        }
    }
}
template <int V>
__device__ __forceinline__ void clear_floats(float (&to)[V])
{
#pragma unroll
    for (int v = 0; v < V; ++v) to[v] = 0.0f;
}
// Channels from c on of one row of an array [rows, dim]; zeros without an array, or where there is no row (-1).
template <int V>
__device__ __forceinline__ void load_row(float (&to)[V], const float *array, int64_t row, int64_t dim, uint32_t c)
{
    clear_floats<V>(to);
    if (array && row >= 0)
#pragma unroll
        for (int v = 0; v < V; ++v) to[v] = array[row * dim + c + v];
}
template <int V>
__device__ __forceinline__ void store_floats(float *p, const float (&v)[V])
{
#pragma unroll
    for (int j = 0; j < V; ++j) p[j] = v[j];
}

// The packed axis in the order of the recurrence: position p is token p, or token total - 1 - p where rows run
// backwards; span j in this order ends where span j + 1 starts.
template <bool REV>
struct Axis {
    Rows r;
    __device__ __forceinline__ int64_t count() const { return r.count(); }
    __device__ __forceinline__ int64_t at(int64_t j) const { return REV ? r.total - r.at(r.count() - j) : r.at(j); }
    __device__ __forceinline__ int64_t row(int64_t j) const { return r.row(REV ? r.count() - 1 - j : j); }
    __device__ __forceinline__ int64_t token(int64_t p) const { return REV ? r.total - 1 - p : p; }

    // The first j with at(j) >= p, or with offsets the last but one if there is none before: every lane of the wave looks at one
    // place of the range that is left.
    __device__ __forceinline__ int64_t first_from(int64_t p, int lane) const
    {
        if (!r.offsets) return (p + r.length - 1) / r.length;
        if (p <= 0) return 0;
        int64_t lo = 1, hi = r.n + 1;                                  // (a place to each row's start, and one round for 64 rows)
        while (hi > lo) {
            const int64_t step = (hi - lo + 63) >> 6, i = lo + lane * step;
            const int before = __popcll(__ballot(i < hi && at(i) < p));
            const int64_t next = lo + before * step;
            if (before) lo += (before - 1) * step + 1;
            hi = next < hi ? next : hi;
        }
        return lo;
    }
};

// Where spans start and end among a wave's positions p0 .. p0 + n: the spans' rows, -1 for tokens in no row, kNoEdge where there is no
// edge.
constexpr int32_t kNoEdge = -2;
template <int S>
struct Edges {
    int32_t start[S + 1], end[S + 1];             // [i]: that whose first position is p0 + i / whose last is p0 + i - 1
};

// Fills `e` and returns the bits of e.start and e.end that are set, and whether the first or the last span may be here.  empty(row)
// is called by the whole wave for each row without tokens that lies here.
template <int S, bool REV, typename Fn>
__device__ __forceinline__ bool find_edges(const Axis<REV> &axis, int64_t p0, int n, int lane, Edges<S> &e,
                                           uint64_t &starts, uint64_t &ends, Fn empty)
{
    static_assert(S + 1 <= 64, "a lane to a position");
    if (lane <= S) e.start[lane] = e.end[lane] = kNoEdge;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    bool rim = false;
    if (n > 0) {
        const int64_t first = axis.first_from(p0, lane);
        rim = first <= 1;
        for (int64_t base = first;; base += 64) {
            const int64_t j = base + lane;
            int64_t p = INT64_MAX;
            bool is_empty = false;
            if (j <= axis.count()) {
                const int64_t at = axis.at(j);
                p = at - p0;
                if (p >= 0 && p <= n) {
                    if (j > 0 && p > 0 && axis.at(j - 1) < at) e.end[p] = (int32_t)axis.row(j - 1);
                    if (j < axis.count()) {
                        const bool none = axis.at(j + 1) == at;
                        if (!none && p < n) e.start[p] = (int32_t)axis.row(j);
                        is_empty = none && (p < n || at == axis.r.total);
                    }
                }
            }
            for (uint64_t left = __ballot(is_empty); left; left &= left - 1) {
                const int64_t row = axis.row(base + __builtin_ctzll(left));
                if (row >= 0) empty(row);
            }
            rim = rim || __ballot(j + 1 >= axis.count() && p <= n);
            if (__ballot(p <= n) != ~0ull) break;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int i = lane <= S ? lane : S;
    starts = __ballot(lane <= S && e.start[i] != kNoEdge);
    ends = __ballot(lane <= S && e.end[i] != kNoEdge);
    return rim;
}

// Whether some of a wave's positions are in no row, and which are not: bit i of `outside`.  Such tokens give zeros: their span
// starts from zero, and their cells become zeros.
template <int S, bool REV>
__device__ __forceinline__ uint64_t outside_rows(const Axis<REV> &axis, int64_t p0, int n)
{
    if (!axis.r.offsets) return 0;
    const int64_t lo = axis.at(1) - p0, hi = axis.at(axis.count() - 1) - p0;
    const uint64_t all = (1ull << n) - 1, front = lo >= n ? all : lo > 0 ? (1ull << lo) - 1 : 0;
    const uint64_t back = hi >= n ? 0 : hi > 0 ? all & ~((1ull << hi) - 1) : all;
    return front | back;
}
template <typename T, int V, int S>
__device__ __forceinline__ void clear_cells(Cell<T, V> (&c)[S], uint64_t which)
{
#pragma unroll
    for (int i = 0; i < S; ++i) {
        typename std::conditional<V * sizeof(T) == 4, uint32_t, uint16_t>::type w;
        __builtin_memcpy(&w, &c[i], sizeof(w));
        w = which >> i & 1 ? 0 : w;
        __builtin_memcpy(&c[i], &w, sizeof(w));
    }
}

// What a run of tokens makes of the state in front of it, c -> a c + h, with b = 1 - a beside a: a rounded product of factors next to 1
// would lose what slow channels forget, always in the same direction where the gate is constant, and what is left of 1 - b would
// lose a small a.  An infinite state stays one whatever is forgotten: no a is 0.
__device__ __forceinline__ float not_zero(float a) { return fmaxf(a, FLT_MIN); }      // (of a NaN as well: then h is one)

template <int V>
struct Run {
    float a[V], b[V], h[V];
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] = 1.0f, b[v] = h[v] = 0.0f;
    }
    __device__ __forceinline__ void factor(int v, const Gate &g)
    {
        b[v] = fmaf(g.k, a[v], b[v]);
        a[v] *= g.f;
    }
    __device__ __forceinline__ void then(const Run &r)
    {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            h[v] = fmaf(r.a[v], h[v], r.h[v]);
            b[v] = fmaf(a[v], r.b[v], b[v]);
            a[v] = not_zero(a[v] * r.a[v]);
        }
    }
};

// The same of a tile or a group in a word: of a and b the one that is at most 1/2, t >= 0 is b, t < 0 is -a.
// Where a row begins inside (or ends, for what flows backwards) it is a reset: h comes out, and nothing of what comes in,
// be it infinite.
constexpr float kReset = 2.0f;

__device__ __forceinline__ bool is_b(float t) { return t >= 0.0f; }
__device__ __forceinline__ float carry_through(float t, float h, float c)
{
    return t == kReset ? h : (__builtin_isinf(c) ? c : fmaf(-t, c, is_b(t) ? c : 0.0f)) + h;
}

template <int V>
struct Piece {
    float t[V], h[V];
    __device__ __forceinline__ Piece(const Run<V> &r, bool reset)
    {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            t[v] = reset ? kReset : r.b[v] <= 0.5f ? r.b[v] : -r.a[v];
            h[v] = r.h[v];
        }
    }
    __device__ __forceinline__ bool is_reset() const { return t[0] == kReset; }        // (of all channels at once)
    __device__ __forceinline__ void through(float (&c)[V]) const
    {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = carry_through(t[v], h[v], c[v]);
    }
};

// A word of the tiles: low t, high h.  (t is never the NaN of an absent word.)
template <int V>
__device__ __forceinline__ void put_words(uint64_t *to, const Piece<V> &p)
{
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float t = p.t[v] == p.t[v] ? p.t[v] : __builtin_nanf("");
        __hip_atomic_store(to + v, (uint64_t)__float_as_uint(p.h[v]) << 32 | __float_as_uint(t), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    }
}
// The word of a tile whose end state is known.
template <int V>
__device__ __forceinline__ void put_states(uint64_t *to, const float (&h)[V])
{
#pragma unroll
    for (int v = 0; v < V; ++v)
        __hip_atomic_store(to + v, (uint64_t)__float_as_uint(h[v]) << 32 | __float_as_uint(kReset), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t get_word(const uint64_t *p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float word_t(uint64_t w) { return __uint_as_float((uint32_t)w); }
__device__ __forceinline__ float word_h(uint64_t w) { return __uint_as_float((uint32_t)(w >> 32)); }
// The word of a tile that is no reset, as a run again.
template <int V>
__device__ __forceinline__ Run<V> run_of(const uint64_t (&words)[V][64], int lane)
{
    Run<V> r;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float t = word_t(words[v][lane]);
        r.a[v] = is_b(t) ? 1.0f - t : -t;
        r.b[v] = is_b(t) ? t : 1.0f + t;
        r.h[v] = word_h(words[v][lane]);
    }
    return r;
}
__device__ __forceinline__ bool is_there(uint64_t w) { return (uint32_t)w != 0xFFFFFFFFu; }

// The first n waves of a tile, in the order of the recurrence, as one run.  reset: a row starts (ends) in one of them, and the
// run is what follows it.
template <int V>
struct Front {
    Run<V> run;
    bool reset;
    __device__ __forceinline__ Piece<V> piece() const { return Piece<V>(run, reset); }
};

// One wave: what reaches the tile that is the `at`-th in order, at > 0, from the tiles in front of it.  own() waits for what the
// tile itself does and returns it; where the tile is the last of its group the group's word and then its state are left here
// (unless the tile starts a row: then it has left the state), or true is returned: a row starts in the group, and its state is what
// the tile makes of the carry.  The state of a group without a row's start is the
// one in front of it run through the group's piece, as a tile does that finds only the piece: one rounding, whichever it
// finds.
// Every wait ends.  Tiles are taken in order by workgroups that run, and each leaves its word, and its group's piece, before it
// waits for a state; the first tile of all has its word as a reset, whatever the offsets are, so the first group's state needs
// no other group's, and each further one only those in front of it.
template <int V, typename Own>
__device__ __forceinline__ bool find_carry(uint64_t (&window)[kGroup][V][64], const uint64_t *tile_words,
                                           uint64_t *group_words, int64_t dim, uint32_t at, uint32_t slab0, uint32_t c,
                                           Own own, int lane, float (&carry)[V])
{
    const int pos = (int)(at % kGroup), n_groups = (int)(at / kGroup < kGroup ? at / kGroup : kGroup);
    const uint64_t *tiles = tile_words + (int64_t)at * dim;
    uint64_t *groups = group_words + (int64_t)(at / kGroup) * dim;
    // what one channel's words say: lanes 0 .. look at the tiles of the group in front, lanes kGroup .. at the groups
    const bool group = lane >= kGroup;
    const int back = (lane & (kGroup - 1)) + 1;
    const bool wanted = group ? lane < 2 * kGroup && back <= n_groups : back <= pos;
    const uint64_t *const mine = (group ? groups : tiles) - back * dim + slab0;
    int need, nearest;                                                 // tiles that count; the nearest group with a state, or -1
    const auto look = [&] {
        const uint64_t w = wanted ? get_word(mine) : kNoWord;
        const uint64_t there = __ballot(is_there(w)), resets = __ballot(word_t(w) == kReset);
        const uint32_t t = (uint32_t)resets & ((1u << kGroup) - 1), g = (uint32_t)(resets >> kGroup);
        need = t ? __builtin_ctz(t) + 1 : pos;
        nearest = g ? __builtin_ctz(g) : -1;
        if (g && (~(uint32_t)(there >> kGroup) & ((1u << nearest) - 1))) nearest = -1;
        return (~(uint32_t)there & ((1u << need) - 1)) == 0;
    };
    clear_floats<V>(carry);
    for (bool ok = false; !ok;) {
        while (!look()) __builtin_amdgcn_s_sleep(1);
        ok = true;
        for (int e0 = 0; e0 < need; e0 += 8) {
            uint64_t q[8][V];
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) q[k][v] = e0 + k < need ? get_word(tiles - (e0 + k + 1) * dim + c + v) : 0;
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    ok = ok && is_there(q[k][v]);
                    if (e0 + k < kGroup) window[e0 + k][v][lane] = q[k][v];
                }
        }
        ok = __all(ok);
    }
    const bool reset = need > 0 && word_t(window[need > 0 ? need - 1 : 0][0][lane]) == kReset;     // (of all channels at once)
    const bool group_end = pos == kGroup - 1;
    Run<V> sum;
    sum.clear();
    bool leave_state = false;                                          // (otherwise the tile has left it)
    if (group_end && !reset) {
        const Front<V> last = own();
        leave_state = !last.reset;
        if (leave_state) {
#pragma unroll 3
            for (int e = need - 1; e >= 0; --e) sum.then(run_of<V>(window[e], lane));
            sum.then(last.run);
            put_words<V>(groups + c, Piece<V>(sum, false));
        }
    }
    for (bool ok = reset; !ok;) {
        while (nearest < 0) {
            __builtin_amdgcn_s_sleep(1);
            look();
        }
        ok = true;
        for (int far = nearest; far >= 0; far -= 4) {
            uint64_t q[4][V];
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) q[k][v] = far >= k ? get_word(groups - (far - k + 1) * dim + c + v) : 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (far < k) continue;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float t = word_t(q[k][v]);
                    ok = ok && is_there(q[k][v]) && (t == kReset || far - k < nearest);
                    carry[v] = carry_through(t, word_h(q[k][v]), carry[v]);
                }
            }
        }
        ok = __all(ok);
        if (!ok) nearest = -1;
    }
    if (leave_state) {
        float end[V];
#pragma unroll
        for (int v = 0; v < V; ++v) end[v] = carry[v];
        Piece<V>(sum, false).through(end);
        put_states<V>(groups + c, end);
    }
    // (for this tile alone: what each of at most fifteen tiles keeps may be rounded)
    if (reset)
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = word_h(window[need - 1][v][lane]);
#pragma unroll 4
    for (int e = need - 1 - reset; e >= 0; --e) {
        const Run<V> r = run_of<V>(window[e], lane);
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = fmaf(r.a[v], carry[v], r.h[v]);
    }
    return group_end && reset;
}

template <int S, int W, int V>
struct ScanShared {
    float a[W][V][64], b[W][V][64], h[W][V][64];  // the waves' runs, in order: of states forwards, gradients backwards
    uint64_t window[kGroup][V][64];
    float carry[V][64];
    uint32_t tile;
    uint32_t arrived;                             // how many waves' runs are there, and from bit 8 on which hold a reset
    Edges<S> edges[W];
    static_assert(W <= 24, "a bit to a wave");

    // A wave's run is there.  True for the last of the waves.
    __device__ __forceinline__ bool arrive(int nth, int lane, const Run<V> &r, bool reset)
    {
#pragma unroll
        for (int v = 0; v < V; ++v) a[nth][v][lane] = not_zero(r.a[v]), b[nth][v][lane] = r.b[v], h[nth][v][lane] = r.h[v];
        uint32_t before = 0;
        if (lane == 0)
            before = __hip_atomic_fetch_add(&arrived, 1u + (reset ? 256u << nth : 0u), __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_WORKGROUP);
        return (__builtin_amdgcn_readfirstlane(before) & 255) == W - 1;
    }
    // The first n of the waves, n > 0, once all are there.
    __device__ __forceinline__ Front<V> front(int n, int lane) const
    {
        uint32_t now;
        while (((now = __hip_atomic_load(&arrived, __ATOMIC_ACQUIRE, __HIP_MEMORY_SCOPE_WORKGROUP)) & 255) < W)
            __builtin_amdgcn_s_sleep(1);
        const uint32_t resets = __builtin_amdgcn_readfirstlane(now) >> 8 & ((1u << n) - 1);
        const int first = resets ? 31 - __builtin_clz(resets) : 0;
        const auto get = [&](int w) {
            Run<V> r;
#pragma unroll
            for (int v = 0; v < V; ++v) r.a[v] = a[w][v][lane], r.b[v] = b[w][v][lane], r.h[v] = h[w][v][lane];
            return r;
        };
        Front<V> f{get(first), resets != 0};
#pragma unroll 3
        for (int w = first + 1; w < n; ++w) f.run.then(get(w));
        return f;
    }
};

// A wave's share of the axis: positions p0 .. p0 + n, its lanes V channels each.  Lanes behind the last channel take the
// last ones once more and write the same values to the same places.
template <int V, int S, int W, bool REV>
struct Span {
    int64_t p0, lowest;                           // lowest: the first in memory of the tokens
    uint32_t c, slab0;
    int n;
    __device__ __forceinline__ Span(const Rows &rows, int64_t dim, int64_t tile, uint32_t slab, int wave, int lane)
    {
        p0 = (tile * W + wave) * S;
        n = rows.total - p0 < S ? (rows.total > p0 ? (int)(rows.total - p0) : 0) : S;
        lowest = n == 0 ? rows.total - 1 : REV ? rows.total - p0 - n : p0;
        slab0 = slab * 64 * V;
        const uint32_t first = slab0 + lane * V;
        c = first < dim ? first : (uint32_t)dim - V;
    }
};

// The tokens of a span in one array: a buffer resource and one 32-bit offset in the lanes, the token's offset from
// the span's lowest in a scalar, so that a cell costs no address arithmetic in the lanes.
template <typename T, int V, int S, bool REV>
struct Strip {
    __amdgpu_buffer_rsrc_t rsrc;
    int lane_bytes, token_bytes, n;
    template <int W>
    __device__ __forceinline__ Strip(const T *base, int64_t stride, const Span<V, S, W, REV> &span, int64_t dim)
    {
        n = span.n > 0 ? span.n : 1;
        lane_bytes = (int)(span.c * sizeof(T));
        token_bytes = (int)(stride * sizeof(T));
        rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)(base + span.lowest * stride), 0,
                                                 (n - 1) * token_bytes + (int)(dim * sizeof(T)), 0x00020000);
    }
    // No array: loads give zeros, since they lie behind the end of a buffer of no bytes (at its first token, so that no offset
    // of a token is taken off those none).
    __device__ __forceinline__ void empty()
    {
        n = 1;
        rsrc = __builtin_amdgcn_make_buffer_rsrc(nullptr, 0, 0, 0x00020000);
    }
    __device__ __forceinline__ int offset(int i) const                 // (positions behind the last one: the last one)
    {
        const int k = i < n ? i : n - 1;
        return (REV ? n - 1 - k : k) * token_bytes;
    }
    __device__ __forceinline__ Cell<T, V> load(int i) const
    {
        Cell<T, V> c;
        if constexpr (V * sizeof(T) == 4) {
            const uint32_t w = __builtin_amdgcn_raw_buffer_load_b32(rsrc, lane_bytes, offset(i), 0);
            __builtin_memcpy(&c, &w, 4);
        } else {
            const uint16_t w = __builtin_amdgcn_raw_buffer_load_b16(rsrc, lane_bytes, offset(i), 0);
            __builtin_memcpy(&c, &w, 2);
        }
        return c;
    }
    __device__ __forceinline__ void store(int i, const float (&v)[V]) const
    {
        Cell<T, V> c;
#pragma unroll
        for (int j = 0; j < V; ++j) c.v[j] = from_float<T>(v[j]);
        if constexpr (V * sizeof(T) == 4) {
            uint32_t w;
            __builtin_memcpy(&w, &c, 4);
            // (2: streamed, not kept in the caches.  64 x 8192 x 512 434 -> 400 us, a training step's backward 342 -> 322, both in
            // an earlier form.  For 32 bits between 3 % less and, with rows of 203 floats, whose ends share lines, 5 % more: not used.  Loads
            // gain less.)
            __builtin_amdgcn_raw_buffer_store_b32(w, rsrc, lane_bytes, offset(i), sizeof(T) == 2 ? 2 : 0);
        } else {
            uint16_t w;
            __builtin_memcpy(&w, &c, 2);
            __builtin_amdgcn_raw_buffer_store_b16(w, rsrc, lane_bytes, offset(i), 0);
        }
    }
};

__device__ __forceinline__ int32_t one_row(int32_t row) { return __builtin_amdgcn_readfirstlane(row); }

// The channels of a workgroup.  Workgroups go to the eight XCDs in turn, each with an L2 of its own; eight neighbours take
// the same channels of eight tiles, so that a tile's slabs, which share the lines that they meet in, meet in one L2.
__device__ __forceinline__ uint32_t slab_of(uint32_t n_slabs, bool only_one)
{
    return (only_one ? blockIdx.x : blockIdx.x >> 3) % n_slabs;
}

// The next tile of a slab, one to each workgroup in the order of their arrival: a tile waits for tiles that running
// workgroups hold, the first of which waits for none, so every wait ends.
template <int S, int W, int V>
__device__ __forceinline__ uint32_t take_tile(ScanShared<S, W, V> &sh, uint32_t *counters, uint32_t slab, bool only_one)
{
    if (threadIdx.x == 0) {
        sh.arrived = 0;
        sh.tile = only_one ? 0 : atomicAdd(counters + slab * kCounterStride, 1u);
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(sh.tile);
}

// The last wave of a workgroup looks for the carry while the others, W, compute; `nth`: the tile's place in the order of the
// launch.  (Also where a row starts, or ends, at the tile's edge and nothing comes in: so it is no matter of the offsets whether a
// group's word is left.)
template <int S, int W, int V, typename T, typename Own>
__device__ __forceinline__ void carry_wave(ScanShared<S, W, V> &sh, const ScanArgs<T> &a, uint32_t nth, uint32_t slab0,
                                           uint32_t c, Own own, int lane)
{
    float carry[V];
    clear_floats<V>(carry);
    const bool leave_state = nth > 0 && find_carry<V>(sh.window, a.tile_words, a.group_words, a.dim, nth, slab0, c, own, lane, carry);
#pragma unroll
    for (int v = 0; v < V; ++v) sh.carry[v][lane] = carry[v];
    __syncthreads();
    if (leave_state) {
        const Front<V> f = own();
        if (!f.reset) {                                                // (otherwise the tile has left it)
            f.piece().through(carry);
            put_states<V>(a.group_words + (int64_t)(nth / kGroup) * a.dim + c, carry);
        }
    }
}

// The word of a tile, and that of its group if the tile is the last of it and a row starts (ends) inside: then the state
// at the end is known at once.
template <int V, typename T>
__device__ __forceinline__ void put_tile(const ScanArgs<T> &a, uint32_t nth, uint32_t c, const Piece<V> &p)
{
    put_words<V>(a.tile_words + (int64_t)nth * a.dim + c, p);
    if (nth % kGroup == kGroup - 1 && p.is_reset())
        put_states<V>(a.group_words + (int64_t)(nth / kGroup) * a.dim + c, p.h);
}

// (Two workgroups on a CU, three with one channel to a lane: with two registers more than the 128 of that it was one, 568 us
// instead of 413 for 64 x 8192 x 512.)
template <typename T, int V, int S, int W, bool REV>
__global__ __launch_bounds__(64 * (W + 1)) __attribute__((amdgpu_waves_per_eu(V == 1 ? 6 : 4))) void gated_scan_kernel(ScanArgs<T> a)
{
    __shared__ ScanShared<S, W, V> sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t slab = slab_of(a.n_slabs, a.n_tiles == 1), tile = take_tile(sh, a.counters, slab, a.n_tiles == 1);
    if (tile >= a.n_tiles) return;
    const Axis<REV> axis{a.rows};
    const Span<V, S, W, REV> span(a.rows, a.dim, tile, slab, wave, lane);
    const uint32_t c = span.c;
    if (wave == W) {
        carry_wave<S, W, V>(sh, a, tile, span.slab0, c, [&] { return sh.front(W, lane); }, lane);
        return;
    }
    const int n = span.n;
    typedef Strip<T, V, S, REV> strip;
    const strip xs(a.x, a.x_stride, span, a.dim), gs(a.gate, a.gate_stride, span, a.dim);
    Cell<T, V> x[S], g[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
        x[i] = xs.load(i);
        g[i] = gs.load(i);
    }
    Edges<S> &edges = sh.edges[wave];
    uint64_t starts, ends;
    const bool rim = find_edges<S, REV>(axis, span.p0, n, lane, edges, starts, ends, [&](int64_t row) {
        float h[V];
        load_row<V>(h, a.h0, row, a.dim, c);
        if (a.last) store_floats<V>(a.last + row * a.dim + c, h);
    });
    if (const uint64_t outside = rim ? outside_rows<S, REV>(axis, span.p0, n) : 0) {
        clear_cells<T, V, S>(x, outside);
        clear_cells<T, V, S>(g, outside);
    }
    const uint64_t looks = starts | ends >> 1 | ~0ull << n;            // positions at which a step has to look

    // What the tokens up to each make of zero, and the factor of what comes in: state = A c + H.  (24 roundings of f at most: it is
    // between the tiles that an f next to 1 must not be rounded, and there its b is at hand.)
    float A[S][V], H[S][V];
    Run<V> own;
    own.clear();
    by_parts<S, V == 1 ? 8 : 4>(looks, [&](int i, auto look) {
        if (look && i >= n) return;
        if (look && (starts >> i & 1)) {
            own.clear();
            load_row<V>(own.h, a.h0, one_row(edges.start[i]), a.dim, c);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Gate gate = gate_of(to_float(g[i].v[v]));
            own.h[v] = fmaf(gate.f, own.h[v], gate.k * to_float(x[i].v[v]));
            own.factor(v, gate);
            A[i][v] = own.a[v] = not_zero(own.a[v]);
            H[i][v] = own.h[v];
        }
    });
    // (the axis' first token starts a span, were the offsets wrong)
    if (sh.arrive(wave, lane, own, starts != 0 || span.p0 == 0) && a.n_tiles > 1) put_tile<V>(a, tile, c, sh.front(W, lane).piece());
    Front<V> front;                                                    // the tile's waves in front of this one
    if (wave > 0) front = sh.front(wave, lane);
    __syncthreads();
    float c0[V];
#pragma unroll
    for (int v = 0; v < V; ++v) c0[v] = sh.carry[v][lane];
    if (wave > 0) front.piece().through(c0);
    if (a.states && n > 0) store_floats<V>(a.states + span.p0 / S * a.dim + c, c0);
    const strip ys(a.y, a.dim, span, a.dim);
    by_parts<S, 12>(looks, [&](int i, auto look) {
        if (look && i >= n) return;
        if (look && (starts >> i & 1)) clear_floats<V>(c0);
        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = fmaf(A[i][v], c0[v], H[i][v]);
        ys.store(i, h);
        if (look && (ends >> (i + 1) & 1) && a.last) {
            const int32_t row = one_row(edges.end[i + 1]);
            if (row >= 0) store_floats<V>(a.last + row * a.dim + c, h);
        }
    });
}

//   dh_t = dy_t + f_(t+1) dh_(t+1),  dx_t = (1 - f_t) dh_t,  dgate_t = dh_t (h_(t-1) - x_t) f_t (1 - f_t)
template <typename T, int V, int S, int W, bool REV>
__global__ __launch_bounds__(64 * (W + 1)) void gated_scan_backward_kernel(ScanArgs<T> a)
{
    __shared__ ScanShared<S, W, V> sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t slab = slab_of(a.n_slabs, a.n_tiles == 1), nth = take_tile(sh, a.counters, slab, a.n_tiles == 1);
    if (nth >= a.n_tiles) return;
    const uint32_t tile = (uint32_t)a.n_tiles - 1 - nth;
    const Axis<REV> axis{a.rows};
    const Span<V, S, W, REV> span(a.rows, a.dim, tile, slab, wave, lane);
    const uint32_t c = span.c;
    if (wave == W) {
        carry_wave<S, W, V>(sh, a, nth, span.slab0, c, [&] { return sh.front(W, lane); }, lane);
        return;
    }
    const int n = span.n, order = W - 1 - wave;
    typedef Strip<T, V, S, REV> strip;
    const strip xs(a.x, a.x_stride, span, a.dim), gs(a.gate, a.gate_stride, span, a.dim);
    Cell<T, V> x[S], g[S], dy[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
        x[i] = xs.load(i);
        g[i] = gs.load(i);
    }
    strip ds(a.dy, a.dy_stride, span, a.dim);
    if (!a.dy) ds.empty();
#pragma unroll
    for (int i = 0; i < S; ++i) dy[i] = ds.load(i);
    Edges<S> &edges = sh.edges[wave];
    uint64_t starts, ends;
    const bool rim = find_edges<S, REV>(axis, span.p0, n, lane, edges, starts, ends, [&](int64_t row) {
        float d[V];
        load_row<V>(d, a.dlast, row, a.dim, c);
        if (a.dh0) store_floats<V>(a.dh0 + row * a.dim + c, d);
    });
    if (const uint64_t outside = rim ? outside_rows<S, REV>(axis, span.p0, n) : 0) {
        clear_cells<T, V, S>(x, outside);
        clear_cells<T, V, S>(g, outside);
        clear_cells<T, V, S>(dy, outside);
    }
    const uint64_t looks = starts | ends >> 1 | ~0ull << n;            // positions at which a step has to look
    const auto final_grad = [&](int i, float (&to)[V]) {
        load_row<V>(to, a.dlast, one_row(edges.end[i + 1]), a.dim, c);
    };

    // The gates, both numbers of each where there are registers for them: with one channel to a lane.
    constexpr bool kBoth = V == 1;
    float m[S][V], fs[kBoth ? S : 1][V];
    const auto gate_at = [&](int i, int v) { return kBoth ? Gate{fs[kBoth ? i : 0][v], m[i][v]} : gate_from(once_more(m[i][v])); };
    Run<V> own;
    own.clear();
    by_parts_back<S, 12>(looks, [&](int i, auto look) {
        if (look && i >= n) return;
        if (look && (ends >> (i + 1) & 1)) {
            own.clear();
            final_grad(i, own.h);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Gate gate = gate_of(to_float(g[i].v[v]));
            m[i][v] = kBoth ? gate.k : one_number(gate);
            if (kBoth) fs[kBoth ? i : 0][v] = gate.f;
            own.h[v] = gate.f * (own.h[v] + to_float(dy[i].v[v]));
            own.factor(v, gate);
        }
    });
    // (the axis' last token ends a span, were the offsets wrong)
    const bool reset = ends != 0 || (n > 0 && span.p0 + n == a.rows.total);
    if (sh.arrive(order, lane, own, reset) && a.n_tiles > 1) put_tile<V>(a, nth, c, sh.front(W, lane).piece());
    Front<V> behind;                                                   // the tile's waves behind this one
    if (order > 0) behind = sh.front(order, lane);
    float h[V];                                                        // the state in front of the wave's first token
    load_row<V>(h, a.states, n > 0 ? span.p0 / S : -1, a.dim, c);
    __syncthreads();
    float carry[V];
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = sh.carry[v][lane];
    if (order > 0) behind.piece().through(carry);
    const strip dxs(a.dx, a.dim, span, a.dim), dgs(a.dgate, a.dim, span, a.dim);
    float from_x[S][V];                                                // h_(t-1) - x_t
    by_parts<S, V == 1 ? 8 : 4>(looks, [&](int i, auto look) {
        if (look && i >= n) return;
        if (look && (starts >> i & 1)) load_row<V>(h, a.h0, one_row(edges.start[i]), a.dim, c);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Gate gate = gate_at(i, v);
            const float xv = to_float(x[i].v[v]);
            from_x[i][v] = h[v] - xv;
            h[v] = fmaf(gate.f, h[v], gate.k * xv);
        }
    });
    by_parts_back<S, 12>(looks, [&](int i, auto look) {
        if (look && i >= n) return;
        if (look && (ends >> (i + 1) & 1)) final_grad(i, carry);
        float dx[V], dg[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Gate gate = gate_at(i, v);
            const float dh = to_float(dy[i].v[v]) + carry[v];
            dx[v] = gate.k * dh;
            dg[v] = dh * from_x[i][v] * (gate.f * gate.k);
            carry[v] = gate.f * dh;
        }
        dxs.store(i, dx);
        dgs.store(i, dg);
        if (look && (starts >> i & 1) && a.dh0) {
            const int32_t row = one_row(edges.start[i]);
            if (row >= 0) store_floats<V>(a.dh0 + row * a.dim + c, carry);
        }
    });
}

// Rows that are all empty have no tile: their states go straight through.
__global__ __launch_bounds__(256) void copy_states_kernel(const float *from, float *to, int64_t n)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) to[i] = from ? from[i] : 0.0f;
}

// One token of every row: a thread to a channel.  1000 x 1024 float16: 4.9 us (its bytes take 3.0); 1 x 512: 2.2 us, a launch.
template <typename T>
__global__ __launch_bounds__(256) void gated_step_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ gate, int64_t gate_stride, const float *state,
    int64_t n_rows, int64_t dim, T *__restrict__ y, float *new_state)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n_rows * dim) return;
    const int64_t b = i / dim, c = i - b * dim;
    const Gate g = gate_of(to_float(gate[b * gate_stride + c]));
    const float h = next_state(g, state ? state[i] : 0.0f, to_float(x[b * x_stride + c]));
    y[i] = from_float<T>(h);
    new_state[i] = h;
}

}  // namespace dnatok

using namespace dnatok;

#define SCAN_REQUIRE(cond, text) DNATOK_REQUIRE(cond, DNATOK_E_INVALID, "%s: " text, who)

namespace {

constexpr int kSteps = 24;                        // tokens that a wave holds in registers
// Waves to a tile beside the one that looks for the carry.  On 64 rows of 8,192 tokens x 512 (bfloat16), us forward and
// backward: 24 tokens x 7 waves 411, 691; x 11 432, 632; 16 tokens x 15 476, 651; x 7 506, 724; 32 tokens x 7 472, 691
// (all in an earlier form).
// Small batches differ by 1 us in 15.
constexpr int kForwardWaves = 7, kBackwardWaves = 11;

// A launch's words, those of the tiles and of the groups, and its counters: each starting on a line of its own.
struct Layout {
    int64_t tiles = 0, words = 0, counters = 0;   // tiles; 64-bit words of tiles and groups; counters
    size_t bytes = 0;                             // 0 where one tile holds all
    Layout(int64_t total, int64_t dim, int waves)
    {
        if (total <= 0 || dim <= 0) return;
        tiles = (total + kSteps * waves - 1) / (kSteps * waves);
        if (tiles == 1) return;
        words = (tiles + (tiles + kGroup - 1) / kGroup) * dim;
        words += -words & 15;
        counters = (dim + 63) / 64;
        bytes = (size_t)words * 8 + (size_t)counters * kCounterStride * 4;
    }
};

// The states that the backward pass starts its pieces from.
size_t states_bytes(int64_t total, int64_t dim)
{
    return total > 0 && dim > 0 ? (size_t)((total + kSteps - 1) / kSteps) * (size_t)dim * 4 : 0;
}

int check_rows(const char *who, int32_t dtype, int64_t n_rows, int64_t total, int64_t dim, const int64_t *offsets)
{
    SCAN_REQUIRE(dtype == DNATOK_F32 || dtype == DNATOK_BF16 || dtype == DNATOK_F16, "unknown element type");
    SCAN_REQUIRE(n_rows >= 0 && total >= 0 && dim > 0 && (n_rows > 0 || total == 0), "bad size");
    SCAN_REQUIRE(offsets || n_rows == 0 || total % n_rows == 0, "rows without offsets must be of one length");
    DNATOK_REQUIRE(n_rows < (1ll << 31) - 2 && dim < (1ll << 30), DNATOK_E_TOO_LARGE, "%s: fewer than 2^31 - 2 rows of 2^30 channels",
                   who);                                               // (two more spans than rows)
    return DNATOK_OK;
}

template <typename T>
int fill_words(ScanArgs<T> &a, const Layout &l, void *at, hipStream_t s)
{
    const int64_t blocks = (l.words + 1023) / 1024;
    a.tile_words = (uint64_t *)at;
    a.group_words = a.tile_words + l.tiles * a.dim;
    a.counters = (uint32_t *)(a.tile_words + l.words);
    fill_words_kernel<<<(unsigned)std::min<int64_t>(blocks, 2048), 256, 0, s>>>(a.tile_words, l.words, l.counters);
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

int copy_states(const float *from, float *to, int64_t n, hipStream_t s)
{
    if (!to || n == 0) return DNATOK_OK;
    const int64_t blocks = (n + 255) / 256;
    copy_states_kernel<<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>(from, to, n);
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

// Two channels of a 16-bit type to a lane where every row begins on a multiple of four bytes and there are more
// channels than lanes.
template <typename T>
bool paired(const ScanArgs<T> &a)
{
    const uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.gate | (uintptr_t)a.dy | (uintptr_t)a.y | (uintptr_t)a.dx |
                           (uintptr_t)a.dgate;
    return sizeof(T) == 2 && a.dim > 64 && (bits & 3) == 0 &&
           ((a.dim | a.x_stride | a.gate_stride | a.dy_stride) & 1) == 0;
}

// (everything that is refused is refused before the first launch, that of the words)
template <typename T, int V>
int launch_scan(const char *who, ScanArgs<T> a, const Layout &l, void *work, bool backward, bool reverse, hipStream_t s)
{
    a.n_slabs = (uint32_t)((a.dim + 64 * V - 1) / (64 * V));
    // (a wave's tokens in 32 bits)
    const int64_t widest = std::max({a.x_stride, a.gate_stride, a.dy_stride, a.dim});
    DNATOK_REQUIRE(widest <= ((1ll << 31) - 1) / (int64_t)(sizeof(T) * (kSteps + 1)), DNATOK_E_TOO_LARGE, "%s: tokens too far apart", who);
    // (eight workgroups of a slab at a time: some find no tile left)
    const int64_t blocks = a.n_slabs * (a.n_tiles == 1 ? 1 : (a.n_tiles + 7) & ~7ll);
    const unsigned threads = 64 * ((backward ? kBackwardWaves : kForwardWaves) + 1);
    DNATOK_REQUIRE(blocks * threads < (1ll << 32), DNATOK_E_TOO_LARGE, "%s: more cells than one launch takes", who);
    const unsigned grid = (unsigned)blocks;
    if (l.bytes)
        if (int rc = fill_words(a, l, work, s)) return rc;
    if (backward) {
        if (reverse) gated_scan_backward_kernel<T, V, kSteps, kBackwardWaves, true><<<grid, threads, 0, s>>>(a);
        else gated_scan_backward_kernel<T, V, kSteps, kBackwardWaves, false><<<grid, threads, 0, s>>>(a);
    } else {
        if (reverse) gated_scan_kernel<T, V, kSteps, kForwardWaves, true><<<grid, threads, 0, s>>>(a);
        else gated_scan_kernel<T, V, kSteps, kForwardWaves, false><<<grid, threads, 0, s>>>(a);
    }
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

template <typename T>
int run_scan(const char *who, const ScanArgs<T> &a, const Layout &l, void *work, bool backward, bool reverse, hipStream_t s)
{
    if constexpr (sizeof(T) == 2)
        if (paired(a)) return launch_scan<T, 2>(who, a, l, work, backward, reverse, s);
    return launch_scan<T, 1>(who, a, l, work, backward, reverse, s);
}

}  // namespace

extern "C" size_t dnatok_gated_scan_states_bytes(int64_t total, int64_t dim)
{
    return states_bytes(total, dim);
}

extern "C" size_t dnatok_gated_scan_work_bytes(int64_t total, int64_t dim)
{
    return std::max(Layout(total, dim, kForwardWaves).bytes, Layout(total, dim, kBackwardWaves).bytes);
}

extern "C" int dnatok_gated_scan(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride, int32_t dtype,
                                 const int64_t *offsets, int64_t n_rows, int64_t total, int64_t dim, int reverse,
                                 const float *h0, void *y, float *last, float *states, void *work, size_t work_bytes,
                                 void *stream)
{
    static const char *who = "dnatok_gated_scan";
    if (int rc = check_rows(who, dtype, n_rows, total, dim, offsets)) return rc;
    if (n_rows == 0) return DNATOK_OK;
    hipStream_t s = (hipStream_t)stream;
    if (total == 0) return copy_states(h0, last, n_rows * dim, s);
    SCAN_REQUIRE(x && gate && y, "null buffer");
    SCAN_REQUIRE(x_stride >= 0 && gate_stride >= 0, "negative stride");
    const Layout l(total, dim, kForwardWaves);
    DNATOK_REQUIRE(l.bytes == 0 || (work && work_bytes >= l.bytes), DNATOK_E_SCRATCH, "%s: the work space needs %zu bytes",
                   who, l.bytes);
    SCAN_REQUIRE(((uintptr_t)work & 15) == 0, "the work space must be 16-byte aligned");
    int rc = DNATOK_OK;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        ScanArgs<T> a{};
        a.x = (const T *)x, a.x_stride = x_stride, a.gate = (const T *)gate, a.gate_stride = gate_stride;
        a.rows = Rows{offsets, n_rows, total, total / n_rows};
        a.dim = dim, a.n_tiles = l.tiles, a.h0 = h0, a.states = states;
        a.y = (T *)y, a.last = last;
        rc = run_scan<T>(who, a, l, work, false, reverse != 0, s);
    });
    return rc;
}

extern "C" int dnatok_gated_scan_backward(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride,
                                          int32_t dtype, const int64_t *offsets, int64_t n_rows, int64_t total,
                                          int64_t dim, int reverse, const float *h0, const void *dy, int64_t dy_stride,
                                          const float *dlast, const float *states, void *dx, void *dgate, float *dh0,
                                          void *work, size_t work_bytes, void *stream)
{
    static const char *who = "dnatok_gated_scan_backward";
    if (int rc = check_rows(who, dtype, n_rows, total, dim, offsets)) return rc;
    if (n_rows == 0) return DNATOK_OK;
    hipStream_t s = (hipStream_t)stream;
    if (total == 0) return copy_states(dlast, dh0, n_rows * dim, s);
    SCAN_REQUIRE(x && gate && states && dx && dgate, "null buffer");
    SCAN_REQUIRE(x_stride >= 0 && gate_stride >= 0 && (!dy || dy_stride >= 0), "negative stride");
    const Layout l(total, dim, kBackwardWaves);
    DNATOK_REQUIRE(l.bytes == 0 || (work && work_bytes >= l.bytes), DNATOK_E_SCRATCH, "%s: the work space needs %zu bytes",
                   who, l.bytes);
    SCAN_REQUIRE(((uintptr_t)work & 15) == 0, "the work space must be 16-byte aligned");
    int rc = DNATOK_OK;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        ScanArgs<T> a{};
        a.x = (const T *)x, a.x_stride = x_stride, a.gate = (const T *)gate, a.gate_stride = gate_stride;
        a.rows = Rows{offsets, n_rows, total, total / n_rows};
        a.dim = dim, a.n_tiles = l.tiles, a.h0 = h0, a.states = const_cast<float *>(states);
        a.dy = (const T *)dy, a.dy_stride = dy ? dy_stride : 0, a.dlast = dlast;
        a.dx = (T *)dx, a.dgate = (T *)dgate, a.dh0 = dh0;
        rc = run_scan<T>(who, a, l, work, true, reverse != 0, s);
    });
    return rc;
}

extern "C" int dnatok_gated_step(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride, int32_t dtype,
                                 const float *state, int64_t n_rows, int64_t dim, void *y, float *new_state, void *stream)
{
    static const char *who = "dnatok_gated_step";
    if (int rc = check_rows(who, dtype, n_rows, n_rows, dim, nullptr)) return rc;
    if (n_rows == 0) return DNATOK_OK;
    SCAN_REQUIRE(x && gate && y && new_state, "null buffer");
    SCAN_REQUIRE(x_stride >= 0 && gate_stride >= 0, "negative stride");
    const int64_t blocks = (n_rows * dim + 255) / 256;
    DNATOK_REQUIRE(blocks < (1ll << 31), DNATOK_E_TOO_LARGE, "%s: more cells than one launch takes", who);
    hipStream_t s = (hipStream_t)stream;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        gated_step_kernel<T><<<(unsigned)blocks, 256, 0, s>>>((const T *)x, x_stride, (const T *)gate, gate_stride, state,
                                                              n_rows, dim, (T *)y, new_state);
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
