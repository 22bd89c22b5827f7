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
// with what flows towards earlier tokens, and runs the states of its tile again from the one that the forward pass
// left at the end of the tile in front, which costs a 64-bit word per tile and channel instead of a state per token.
//
// The tiles in front: a 64-bit word per tile and channel holds (A, H) once its tile knows them and the state h at its end
// (marked) once it knows that.  A word says by itself whether it is there (a fill kernel has put a pattern that none has), so
// nothing has to be ordered by a fence.  A tile looks at the 64 words in front of it until they hold a state with
// nothing missing behind it, and runs that state through the tiles between one by one.  The result is
// therefore the same to the last bit, wherever the state is found and whoever came first.  A wait ends after
// a bounded number of looks; then the workgroup runs the row from its start itself, by the same steps.
#include "lm_common.hpp"

namespace dnatok {

constexpr uint64_t kNoWord = ~0ull;
constexpr int kLooks = 1 << 14;

__global__ __launch_bounds__(256) void fill_words_kernel(uint64_t *words, int64_t n)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) words[i] = kNoWord;
}

template <typename T>
struct ScanArgs {
    const T *x, *gate;
    int64_t x_stride, gate_stride;
    Rows rows;
    int64_t dim, n_tiles;
    uint32_t n_slabs;
    const float *h0;
    uint64_t *words;                              // [n_tiles, dim]: states at the tiles' ends
    int looks;
    T *y;
    float *last;
    // the backward pass
    const T *dy;
    int64_t dy_stride;
    const float *dlast;
    T *dx, *dgate;
    float *dh0;
    uint64_t *back_words;                         // [n_tiles, dim]: what flows from a tile to the tile in front of it
};

// V channels of one token as they lie in memory.
template <typename T, int V> struct Cell { T v[V]; };
template <typename T, int V>
__device__ __forceinline__ Cell<T, V> load_cell(const T *p)
{
    Cell<T, V> c;
    if constexpr (V * sizeof(T) == 4) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(p);
        __builtin_memcpy(&c, &w, 4);
    } else {
        c.v[0] = p[0];
    }
    return c;
}
template <typename T, int V>
__device__ __forceinline__ void store_cell(T *p, const float *v)
{
    Cell<T, V> c;
#pragma unroll
    for (int j = 0; j < V; ++j) c.v[j] = from_float<T>(v[j]);
    if constexpr (V * sizeof(T) == 4) {
        uint32_t w;
        __builtin_memcpy(&w, &c, 4);
        *reinterpret_cast<uint32_t *>(p) = w;
    } else {
        p[0] = c.v[0];
    }
}
template <int V>
__device__ __forceinline__ void load_floats(float (&to)[V], const float *p)       // (zeros without an array)
{
#pragma unroll
    for (int v = 0; v < V; ++v) to[v] = p ? p[v] : 0.0f;
}
template <int V>
__device__ __forceinline__ void store_floats(float *p, const float (&v)[V])
{
#pragma unroll
    for (int j = 0; j < V; ++j) p[j] = v[j];
}

// The packed rows along the axis in the order of the recurrence: position p is token p, or token total - 1 - p
// where rows run backwards; row j in this order ends where row j + 1 starts.
template <bool REV>
struct Axis {
    Rows r;
    __device__ __forceinline__ int64_t at(int64_t j) const { return REV ? r.total - r.at(r.n - j) : r.at(j); }
    __device__ __forceinline__ int64_t row(int64_t j) const { return REV ? r.n - 1 - j : j; }
    __device__ __forceinline__ int64_t token(int64_t p) const { return REV ? r.total - 1 - p : p; }

    // The first j with at(j) >= p: every lane of the wave looks at one place of the range that is left.
    __device__ __forceinline__ int64_t first_from(int64_t p, int lane) const
    {
        if (!r.offsets) return (p + r.length - 1) / r.length;
        int64_t lo = 0, hi = r.n;
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

// Where rows start and end among a wave's positions p0 .. p0 + n: rows (in the axis' order), -1 where there is none.
template <int S>
struct Edges {
    int32_t start[S + 1], end[S + 1];             // [i]: the row whose first position is p0 + i / whose last is p0 + i - 1
};

// Fills `e` and returns the bits of e.start and e.end that are set.  empty(row) is called by the whole wave for each row
// without tokens that lies here.
template <int S, bool REV, typename Fn>
__device__ __forceinline__ void find_edges(const Axis<REV> &axis, int64_t p0, int n, int lane, Edges<S> &e,
                                           uint64_t &starts, uint64_t &ends, Fn empty)
{
    static_assert(S + 1 <= 64, "a lane to a position");
    if (lane <= S) e.start[lane] = e.end[lane] = -1;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (n > 0) {
        for (int64_t base = axis.first_from(p0, lane);; base += 64) {
            const int64_t j = base + lane;
            int64_t p = INT64_MAX;
            bool is_empty = false;
            if (j <= axis.r.n) {
                const int64_t at = axis.at(j);
                p = at - p0;
                if (p >= 0 && p <= n) {
                    if (j > 0 && p > 0 && axis.at(j - 1) < at) e.end[p] = (int32_t)(j - 1);
                    if (j < axis.r.n) {
                        const bool none = axis.at(j + 1) == at;
                        if (!none && p < n) e.start[p] = (int32_t)j;
                        is_empty = none && (p < n || at == axis.r.total);
                    }
                }
            }
            for (uint64_t left = __ballot(is_empty); left; left &= left - 1)
                empty(axis.row(base + __builtin_ctzll(left)));
            if (__ballot(p <= n) != ~0ull) break;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int i = lane <= S ? lane : S;
    starts = __ballot(lane <= S && e.start[i] >= 0);
    ends = __ballot(lane <= S && e.end[i] >= 0);
}

// A piece of the axis: c -> a c + h in every channel, with b = 1 - a beside a, each multiplied up on its own: a rounded
// product of factors next to 1 would lose what slow channels forget (always in the same direction where the gate is
// constant).  Where a row begins inside (or ends, for what flows backwards) the piece is a reset: h comes out, and nothing
// of what comes in, be it infinite.
constexpr float kReset = 2.0f;

__device__ __forceinline__ float carry_through(float s, float h, float c)          // s: kReset, b, or -a where a < 1/2
{
    const float f = mostly_kept(s) ? fmaf(-s, c, c) + h : fmaf(-s, c, h);
    return s == kReset ? h : f;
}

template <int V>
struct Piece {
    float a[V], b[V], h[V];
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] = 1.0f, b[v] = h[v] = 0.0f;
    }
    __device__ __forceinline__ void factor(int v, float share)
    {
        b[v] = next_state(share, b[v], 1.0f);
        a[v] = forget(share, a[v]);
    }
    __device__ __forceinline__ void close(bool edge)
    {
#pragma unroll
        for (int v = 0; v < V; ++v) b[v] = edge ? kReset : b[v];
    }
    __device__ __forceinline__ float small(int v) const { return a[v] < 0.5f && b[v] != kReset ? -a[v] : b[v]; }
    __device__ __forceinline__ void through(float (&c)[V]) const
    {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = carry_through(small(v), h[v], c[v]);
    }
    __device__ __forceinline__ void then(const Piece &p)
    {
        p.through(h);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            b[v] = b[v] == kReset || p.b[v] == kReset ? kReset : fmaf(p.b[v], a[v], b[v]);
            a[v] *= p.a[v];
        }
    }
};

// A word of the tiles: low s of carry_through, high h.  (s is never the NaN of an absent word.)
template <int V>
__device__ __forceinline__ void put_words(uint64_t *to, const Piece<V> &p)
{
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float s = p.small(v);
        if (!(s == s)) s = __builtin_nanf("");
        __hip_atomic_store(to + v, (uint64_t)__float_as_uint(p.h[v]) << 32 | __float_as_uint(s), __ATOMIC_RELAXED,
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
__device__ __forceinline__ float word_s(uint64_t w) { return __uint_as_float((uint32_t)w); }
__device__ __forceinline__ float word_h(uint64_t w) { return __uint_as_float((uint32_t)(w >> 32)); }
__device__ __forceinline__ bool is_there(uint64_t w) { return (uint32_t)w != 0xFFFFFFFFu; }

// One wave: what reaches a tile from the tiles next to it (step = -1: those in front, 1: those behind).  `words` is the
// tile's own place.  False if the words did not come.
template <int V>
__device__ __forceinline__ bool wait_for_carry(const uint64_t *words, int64_t step_words, int64_t n_near, int64_t slab0,
                                               int64_t c, int looks, int lane, float (&carry)[V])
{
    for (int look = 0; look < looks; ++look) {
        // one channel's words say how far the nearest state is (behind the last tile of the axis none is looked for)
        const uint64_t w = lane < n_near ? get_word(words + step_words * (lane + 1) + slab0) : kNoWord;
        const uint64_t there = __ballot(is_there(w)), states = __ballot(word_s(w) == kReset);
        const int d = states ? __builtin_ctzll(states) : 63;
        if (!states || (~there & ((1ull << d) - 1))) {
            __builtin_amdgcn_s_sleep(2);
            continue;
        }
        bool ok = true;
        for (int far = d; far >= 0; far -= 4) {
            uint64_t q[4][V];
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) q[k][v] = far >= k ? get_word(words + step_words * (far - k + 1) + c + v) : 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (far < k) continue;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float s = word_s(q[k][v]);
                    ok = ok && is_there(q[k][v]) && (s == kReset || far - k < d);
                    carry[v] = carry_through(s, word_h(q[k][v]), carry[v]);
                }
            }
        }
        if (__all(ok)) return true;
    }
    return false;
}

// The pieces of a tile's waves, in LDS (array by array: lanes read neighbouring words).
template <int W, int V>
struct Pieces {
    float a[W][V][64], b[W][V][64], h[W][V][64];
    __device__ __forceinline__ void put(int wave, int lane, const Piece<V> &p)
    {
#pragma unroll
        for (int v = 0; v < V; ++v) a[wave][v][lane] = p.a[v], b[wave][v][lane] = p.b[v], h[wave][v][lane] = p.h[v];
    }
    __device__ __forceinline__ Piece<V> get(int wave, int lane) const
    {
        Piece<V> p;
#pragma unroll
        for (int v = 0; v < V; ++v) p.a[v] = a[wave][v][lane], p.b[v] = b[wave][v][lane], p.h[v] = h[wave][v][lane];
        return p;
    }
};

template <int S, int W, int V>
struct ScanShared {
    Pieces<W, V> parts;
    float carry[V][64];
    int inside;                                   // a row starts (backward: ends) in the tile
    Edges<S> edges[W];
};

// A wave's share of the axis: positions p0 .. p0 + n, its lanes V channels each.  Lanes behind the last channel take the
// last ones once more and write the same values to the same places.
template <int V, int S, int W, bool REV>
struct Span {
    int64_t p0;
    uint32_t c, slab0;
    int n;
    __device__ __forceinline__ Span(const Rows &rows, int64_t dim, int64_t tile, uint32_t slab, int wave, int lane)
    {
        p0 = (tile * W + wave) * S;
        n = rows.total - p0 < S ? (rows.total > p0 ? (int)(rows.total - p0) : 0) : S;
        slab0 = slab * 64 * V;
        const uint32_t first = slab0 + lane * V;
        c = first < dim ? first : (uint32_t)dim - V;
    }
    // base + the token of position p0 + i; of the last one there is for positions behind it
    template <typename T>
    __device__ __forceinline__ T *at(T *base, int64_t stride, int64_t total, int i) const
    {
        const int64_t from = n > 0 ? p0 : total - 1, step = i < n ? i : n > 0 ? n - 1 : 0;
        return base + (REV ? total - 1 - from : from) * stride + (REV ? -step : step) * stride;
    }
};

__device__ __forceinline__ int32_t one_row(int32_t row) { return __builtin_amdgcn_readfirstlane(row); }

// The state in front of position p0, from the start of the row that p0 lies in: tile by tile, as the tiles' own
// workgroups run it, so with the same bits.  One wave; `e` is written over.
template <typename T, int V, int S, int W, bool REV>
__device__ __forceinline__ void run_from_row_start(const ScanArgs<T> &a, const Axis<REV> &axis, int64_t p0, int64_t c, int lane,
                                                Edges<S> &e, float (&state)[V])
{
    const int64_t j = axis.first_from(p0, lane);                       // (p0 is inside row j - 1)
    for (int64_t q = axis.at(j > 0 ? j - 1 : 0) / (S * W) * (S * W); q < p0; q += S * W) {
        Piece<V> tile;
#pragma unroll 1
        for (int w = 0; w < W; ++w) {
            uint64_t starts, ends;
            find_edges<S, REV>(axis, q + w * S, S, lane, e, starts, ends, [](int64_t) {});
            Piece<V> p;
            p.clear();
#pragma unroll 1
            for (int i = 0; i < S; ++i) {
                if (starts >> i & 1) load_floats<V>(p.h, a.h0 ? a.h0 + axis.row(e.start[i]) * a.dim + c : nullptr);
                const int64_t t = axis.token(q + w * S + i);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float share = gate_share(to_float(a.gate[t * a.gate_stride + c + v]));
                    p.h[v] = next_state(share, p.h[v], to_float(a.x[t * a.x_stride + c + v]));
                    p.factor(v, share);
                }
            }
            p.close(starts != 0);
            if (w == 0) tile = p;
            else tile.then(p);
        }
        tile.through(state);
    }
}

// What flows to the position in front of p1 from the end of the row that it lies in, in the same way.
template <typename T, int V, int S, int W, bool REV>
__device__ __forceinline__ void run_from_row_end(const ScanArgs<T> &a, const Axis<REV> &axis, int64_t p1, int64_t c, int lane,
                                              Edges<S> &e, float (&carry)[V])
{
    const int64_t total = a.rows.total, last = axis.at(axis.first_from(p1, lane)) - 1;   // (p1 is inside the row)
    for (int64_t q = last / (S * W) * (S * W); q >= p1; q -= S * W) {
        Piece<V> tile;
#pragma unroll 1
        for (int w = W - 1; w >= 0; --w) {
            const int64_t p0 = q + w * S;
            const int n = total - p0 < S ? (total > p0 ? (int)(total - p0) : 0) : S;
            uint64_t starts, ends;
            find_edges<S, REV>(axis, p0, n, lane, e, starts, ends, [](int64_t) {});
            Piece<V> p;
            p.clear();
#pragma unroll 1
            for (int i = 0; i < n; ++i)                                // (the factors in the order of the tile's own wave)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    p.factor(v, gate_share(to_float(a.gate[axis.token(p0 + i) * a.gate_stride + c + v])));
#pragma unroll 1
            for (int i = n - 1; i >= 0; --i) {
                if (ends >> (i + 1) & 1)
                    load_floats<V>(p.h, a.dlast ? a.dlast + axis.row(e.end[i + 1]) * a.dim + c : nullptr);
                const int64_t t = axis.token(p0 + i);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float share = gate_share(to_float(a.gate[t * a.gate_stride + c + v]));
                    p.h[v] = forget(share, p.h[v] + (a.dy ? to_float(a.dy[t * a.dy_stride + c + v]) : 0.0f));
                }
            }
            p.close(ends != 0);
            if (w == W - 1) tile = p;
            else tile.then(p);
        }
        tile.through(carry);
    }
}

template <typename T, int V, int S, int W, bool REV>
__global__ __launch_bounds__(64 * W) void gated_scan_kernel(ScanArgs<T> a)
{
    __shared__ ScanShared<S, W, V> sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tile = blockIdx.x / a.n_slabs, slab = blockIdx.x - tile * a.n_slabs;
    const Axis<REV> axis{a.rows};
    const int64_t total = a.rows.total;
    const Span<V, S, W, REV> span(a.rows, a.dim, tile, slab, wave, lane);
    const uint32_t c = span.c;
    const int n = span.n;

    Cell<T, V> x[S], g[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
        x[i] = load_cell<T, V>(span.at(a.x, a.x_stride, total, i) + c);
        g[i] = load_cell<T, V>(span.at(a.gate, a.gate_stride, total, i) + c);
    }
    if (threadIdx.x == 0) sh.inside = 0;
    Edges<S> &edges = sh.edges[wave];
    uint64_t starts, ends;
    find_edges<S, REV>(axis, span.p0, n, lane, edges, starts, ends, [&](int64_t row) {
        float h[V];
        load_floats<V>(h, a.h0 ? a.h0 + row * a.dim + c : nullptr);
        if (a.last) store_floats<V>(a.last + row * a.dim + c, h);
    });
    const bool plain = n == S && (starts | ends) == 0;                 // no row starts or ends here: no step has to look
    const auto initial = [&](int i) { return a.h0 ? a.h0 + axis.row(one_row(edges.start[i])) * a.dim + c : nullptr; };

    float share[S][V];
    Piece<V> own;
    own.clear();
    const auto first_pass = [&](auto with_edges) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
            if (with_edges && i >= n) break;
            if (with_edges && (starts >> i & 1)) load_floats<V>(own.h, initial(i));
#pragma unroll
            for (int v = 0; v < V; ++v) {
                share[i][v] = gate_share(to_float(g[i].v[v]));
                own.h[v] = next_state(share[i][v], own.h[v], to_float(x[i].v[v]));
                own.factor(v, share[i][v]);
            }
        }
    };
    if (plain) first_pass(std::false_type{});
    else first_pass(std::true_type{});
    own.close(starts != 0);
    sh.parts.put(wave, lane, own);
    __syncthreads();
    if (starts && lane == 0) sh.inside = 1;
    Piece<V> front;                                                    // the tile's waves in front of this one
    if (wave > 0) {
        front = sh.parts.get(0, lane);
        for (int w = 1; w < wave; ++w) front.then(sh.parts.get(w, lane));
    }
    uint64_t *const words = a.words + (int64_t)tile * a.dim;
    if (wave == W - 1 && a.n_tiles > 1) {
        Piece<V> all = front;
        all.then(own);
        put_words<V>(words + c, all);
    }
    const bool at_row = sh.edges[0].start[0] >= 0;                     // the tile's first position starts a row
    __syncthreads();
    float h[V];
    load_floats<V>(h, nullptr);
    if (!at_row) {
        if (wave == 0) {
            if (!wait_for_carry<V>(words, -a.dim, tile, span.slab0, c, a.looks, lane, h)) {
                load_floats<V>(h, nullptr);
                run_from_row_start<T, V, S, W, REV>(a, axis, span.p0, c, lane, edges, h);
                find_edges<S, REV>(axis, span.p0, n, lane, edges, starts, ends, [](int64_t) {});
            }
#pragma unroll
            for (int v = 0; v < V; ++v) sh.carry[v][lane] = h[v];
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = sh.carry[v][lane];
        if (wave == W - 1 && !sh.inside) {
            Piece<V> all = front;
            all.then(own);
            float state[V];
#pragma unroll
            for (int v = 0; v < V; ++v) state[v] = h[v];
            all.through(state);
            put_states<V>(words + c, state);
        }
    }
    if (wave > 0) front.through(h);
    const auto second_pass = [&](auto with_edges) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
            if (with_edges && i >= n) break;
            if (with_edges && (starts >> i & 1)) load_floats<V>(h, initial(i));
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = next_state(share[i][v], h[v], to_float(x[i].v[v]));
            store_cell<T, V>(span.at(a.y, a.dim, total, i) + c, h);
            if (with_edges && (ends >> (i + 1) & 1) && a.last)
                store_floats<V>(a.last + axis.row(one_row(edges.end[i + 1])) * a.dim + c, h);
        }
    };
    if (plain) second_pass(std::false_type{});
    else second_pass(std::true_type{});
}

//   dh_t = dy_t + f_(t+1) dh_(t+1),  dx_t = (1 - f_t) dh_t,  dgate_t = dh_t (h_(t-1) - x_t) f_t (1 - f_t)
template <typename T, int V, int S, int W, bool REV>
__global__ __launch_bounds__(64 * W) void gated_scan_backward_kernel(ScanArgs<T> a)
{
    __shared__ ScanShared<S, W, V> sh;
    __shared__ float back_h[W][V][64];            // (a wave's factors are those of its forward piece)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t nth = blockIdx.x / a.n_slabs, slab = blockIdx.x - nth * a.n_slabs, tile = (uint32_t)a.n_tiles - 1 - nth;
    const Axis<REV> axis{a.rows};
    const int64_t total = a.rows.total;
    const Span<V, S, W, REV> span(a.rows, a.dim, tile, slab, wave, lane);
    const uint32_t c = span.c;
    const int n = span.n;

    Cell<T, V> x[S], g[S], dy[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
        x[i] = load_cell<T, V>(span.at(a.x, a.x_stride, total, i) + c);
        g[i] = load_cell<T, V>(span.at(a.gate, a.gate_stride, total, i) + c);
        if (a.dy) dy[i] = load_cell<T, V>(span.at(a.dy, a.dy_stride, total, i) + c);
        else dy[i] = Cell<T, V>{};
    }
    float h[V];                                                        // the state in front of the tile
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = tile > 0 ? word_h(a.words[((int64_t)tile - 1) * a.dim + c + v]) : 0.0f;
    if (threadIdx.x == 0) sh.inside = 0;
    Edges<S> &edges = sh.edges[wave];
    uint64_t starts, ends;
    find_edges<S, REV>(axis, span.p0, n, lane, edges, starts, ends, [&](int64_t row) {
        float d[V];
        load_floats<V>(d, a.dlast ? a.dlast + row * a.dim + c : nullptr);
        if (a.dh0) store_floats<V>(a.dh0 + row * a.dim + c, d);
    });
    const bool plain = n == S && (starts | ends) == 0;
    const auto initial = [&](int i) { return a.h0 ? a.h0 + axis.row(one_row(edges.start[i])) * a.dim + c : nullptr; };
    const auto final_grad = [&](int i) {
        return a.dlast ? a.dlast + axis.row(one_row(edges.end[i + 1])) * a.dim + c : nullptr;
    };

    float share[S][V];
    Piece<V> own, back;
    own.clear();
    load_floats<V>(back.h, nullptr);
    const auto first_pass = [&](auto with_edges) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
            if (with_edges && i >= n) break;
            if (with_edges && (starts >> i & 1)) load_floats<V>(own.h, initial(i));
#pragma unroll
            for (int v = 0; v < V; ++v) {
                share[i][v] = gate_share(to_float(g[i].v[v]));
                own.h[v] = next_state(share[i][v], own.h[v], to_float(x[i].v[v]));
                own.factor(v, share[i][v]);
            }
        }
#pragma unroll
        for (int i = S - 1; i >= 0; --i) {
            if (with_edges && i >= n) continue;
            if (with_edges && (ends >> (i + 1) & 1)) load_floats<V>(back.h, final_grad(i));
#pragma unroll
            for (int v = 0; v < V; ++v) back.h[v] = forget(share[i][v], back.h[v] + to_float(dy[i].v[v]));
        }
    };
    if (plain) first_pass(std::false_type{});
    else first_pass(std::true_type{});
#pragma unroll
    for (int v = 0; v < V; ++v) back.a[v] = own.a[v], back.b[v] = own.b[v], back_h[wave][v][lane] = back.h[v];
    sh.parts.put(wave, lane, own);
    own.close(starts != 0);
    back.close(ends != 0);
    __shared__ uint8_t resets[W][2];              // the wave's piece is one forwards, backwards
    if (lane == 0) resets[wave][0] = starts != 0, resets[wave][1] = ends != 0;
    __syncthreads();
    if (ends && lane == 0) sh.inside = 1;
    if (wave > 0) {
        Piece<V> front = sh.parts.get(0, lane);
        front.close(resets[0][0]);
        for (int w = 1; w < wave; ++w) {
            Piece<V> p = sh.parts.get(w, lane);
            p.close(resets[w][0]);
            front.then(p);
        }
        front.through(h);
    }
    Piece<V> behind;                                                   // the tile's waves behind this one
    const auto back_piece = [&](int w) {
        Piece<V> p = sh.parts.get(w, lane);
#pragma unroll
        for (int v = 0; v < V; ++v) p.h[v] = back_h[w][v][lane];
        p.close(resets[w][1]);
        return p;
    };
    if (wave < W - 1) {
        behind = back_piece(W - 1);
        for (int w = W - 2; w > wave; --w) behind.then(back_piece(w));
    }
    uint64_t *const words = a.back_words + (int64_t)tile * a.dim;
    if (wave == 0 && a.n_tiles > 1) {
        Piece<V> all = behind;
        all.then(back);
        put_words<V>(words + c, all);
    }
    const bool at_end = tile == (uint32_t)a.n_tiles - 1 || sh.edges[W - 1].end[S] >= 0;      // the tile's last position ends a row
    __syncthreads();
    float carry[V];
    load_floats<V>(carry, nullptr);
    if (!at_end) {
        if (wave == W - 1) {
            if (!wait_for_carry<V>(words, a.dim, a.n_tiles - 1 - tile, span.slab0, c, a.looks, lane, carry)) {
                load_floats<V>(carry, nullptr);
                run_from_row_end<T, V, S, W, REV>(a, axis, span.p0 + S, c, lane, edges, carry);
                find_edges<S, REV>(axis, span.p0, n, lane, edges, starts, ends, [](int64_t) {});
            }
#pragma unroll
            for (int v = 0; v < V; ++v) sh.carry[v][lane] = carry[v];
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = sh.carry[v][lane];
        if (wave == 0 && !sh.inside) {
            Piece<V> all = behind;
            all.then(back);
            float out[V];
#pragma unroll
            for (int v = 0; v < V; ++v) out[v] = carry[v];
            all.through(out);
            put_states<V>(words + c, out);
        }
    }
    if (wave < W - 1) behind.through(carry);
    const auto second_pass = [&](auto with_edges) {
        float from_x[S][V];                                            // h_(t-1) - x_t
#pragma unroll
        for (int i = 0; i < S; ++i) {
            if (with_edges && i >= n) break;
            if (with_edges && (starts >> i & 1)) load_floats<V>(h, initial(i));
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float xv = to_float(x[i].v[v]);
                from_x[i][v] = h[v] - xv;
                h[v] = next_state(share[i][v], h[v], xv);
            }
        }
#pragma unroll
        for (int i = S - 1; i >= 0; --i) {
            if (with_edges && i >= n) continue;
            if (with_edges && (ends >> (i + 1) & 1)) load_floats<V>(carry, final_grad(i));
            float dx[V], dg[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float dh = to_float(dy[i].v[v]) + carry[v];
                dx[v] = taken(share[i][v]) * dh;
                dg[v] = dh * from_x[i][v] * slope(share[i][v]);
                carry[v] = forget(share[i][v], dh);
            }
            store_cell<T, V>(span.at(a.dx, a.dim, total, i) + c, dx);
            store_cell<T, V>(span.at(a.dgate, a.dim, total, i) + c, dg);
            if (with_edges && (starts >> i & 1) && a.dh0)
                store_floats<V>(a.dh0 + axis.row(one_row(edges.start[i])) * a.dim + c, carry);
        }
    };
    if (plain) second_pass(std::false_type{});
    else second_pass(std::true_type{});
}

// Rows that are all empty have no tile: their states go straight through.
__global__ __launch_bounds__(256) void copy_states_kernel(const float *from, float *to, int64_t n)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) to[i] = from ? from[i] : 0.0f;
}

template <typename T>
__global__ __launch_bounds__(256) void gated_step_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ gate, int64_t gate_stride, const float *state,
    int64_t n_rows, int64_t dim, T *__restrict__ y, float *new_state)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n_rows * dim) return;
    const int64_t b = i / dim, c = i - b * dim;
    const float share = gate_share(to_float(gate[b * gate_stride + c]));
    const float h = next_state(share, state ? state[i] : 0.0f, to_float(x[b * x_stride + c]));
    y[i] = from_float<T>(h);
    new_state[i] = h;
}

}  // namespace dnatok

using namespace dnatok;

#define SCAN_REQUIRE(cond, text) DNATOK_REQUIRE(cond, DNATOK_E_INVALID, "%s: " text, who)

namespace {

constexpr int kSteps = 16;                        // tokens that a wave holds in registers

// Waves to a tile: 16, or 4 where the batch would not give the chip's 256 CUs a tile each.  By sizes alone: the forward
// call's tiles are the backward call's.
int waves_of(int64_t total, int64_t dim, int32_t dtype)
{
    const int64_t channels = dtype == DNATOK_F32 ? 64 : 128;
    return ((total + 255) / 256) * ((dim + channels - 1) / channels) >= 256 ? 16 : 4;
}

int64_t tiles_of(int64_t total, int64_t dim, int32_t dtype)
{
    const int64_t tile = (int64_t)kSteps * waves_of(total, dim, dtype);
    return (total + tile - 1) / tile;
}

size_t words_bytes(int64_t total, int64_t dim, int32_t dtype)
{
    if (total <= 0 || dim <= 0) return 0;
    const int64_t tiles = tiles_of(total, dim, dtype);
    return tiles > 1 ? (size_t)tiles * (size_t)dim * 8 : 0;
}

int check_rows(const char *who, int32_t dtype, int64_t n_rows, int64_t total, int64_t dim, const int64_t *offsets)
{
    SCAN_REQUIRE(dtype == DNATOK_F32 || dtype == DNATOK_BF16 || dtype == DNATOK_F16, "unknown element type");
    SCAN_REQUIRE(n_rows >= 0 && total >= 0 && dim > 0 && (n_rows > 0 || total == 0), "bad size");
    SCAN_REQUIRE(offsets || n_rows == 0 || total % n_rows == 0, "rows without offsets must be of one length");
    DNATOK_REQUIRE(n_rows < (1ll << 31) && dim < (1ll << 30), DNATOK_E_TOO_LARGE, "%s: at most 2^31 rows of 2^30 channels", who);
    return DNATOK_OK;
}

int fill_words(void *words, size_t bytes, hipStream_t s)
{
    const int64_t n = (int64_t)(bytes / 8), blocks = (n + 255) / 256;
    fill_words_kernel<<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>((uint64_t *)words, n);
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

template <typename T, int V, int W>
int launch_scan(const char *who, ScanArgs<T> a, bool backward, bool reverse, hipStream_t s)
{
    a.n_slabs = (uint32_t)((a.dim + 64 * V - 1) / (64 * V));
    const int64_t blocks = a.n_slabs * a.n_tiles;
    DNATOK_REQUIRE(blocks * 64 * W < (1ll << 32), DNATOK_E_TOO_LARGE, "%s: more cells than one launch takes", who);
    const unsigned grid = (unsigned)blocks;
    if (backward) {
        if (reverse) gated_scan_backward_kernel<T, V, kSteps, W, true><<<grid, 64 * W, 0, s>>>(a);
        else gated_scan_backward_kernel<T, V, kSteps, W, false><<<grid, 64 * W, 0, s>>>(a);
    } else {
        if (reverse) gated_scan_kernel<T, V, kSteps, W, true><<<grid, 64 * W, 0, s>>>(a);
        else gated_scan_kernel<T, V, kSteps, W, false><<<grid, 64 * W, 0, s>>>(a);
    }
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

template <typename T>
int run_scan(const char *who, const ScanArgs<T> &a, int32_t dtype, bool backward, bool reverse, hipStream_t s)
{
    const bool wide = waves_of(a.rows.total, a.dim, dtype) == 16;
    if constexpr (sizeof(T) == 2)
        if (paired(a))
            return wide ? launch_scan<T, 2, 16>(who, a, backward, reverse, s) : launch_scan<T, 2, 4>(who, a, backward, reverse, s);
    return wide ? launch_scan<T, 1, 16>(who, a, backward, reverse, s) : launch_scan<T, 1, 4>(who, a, backward, reverse, s);
}

}  // namespace

extern "C" size_t dnatok_gated_scan_states_bytes(int64_t total, int64_t dim, int32_t dtype)
{
    return words_bytes(total, dim, dtype);
}

extern "C" size_t dnatok_gated_scan_work_bytes(int64_t total, int64_t dim, int32_t dtype)
{
    return words_bytes(total, dim, dtype);
}

extern "C" int dnatok_gated_scan(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride, int32_t dtype,
                                 const int64_t *offsets, int64_t n_rows, int64_t total, int64_t dim, int flags,
                                 const float *h0, void *y, float *last, void *states, size_t states_bytes, void *stream)
{
    static const char *who = "dnatok_gated_scan";
    if (int rc = check_rows(who, dtype, n_rows, total, dim, offsets)) return rc;
    if (n_rows == 0) return DNATOK_OK;
    hipStream_t s = (hipStream_t)stream;
    if (total == 0) return copy_states(h0, last, n_rows * dim, s);
    SCAN_REQUIRE(x && gate && y, "null buffer");
    const size_t need = words_bytes(total, dim, dtype);
    DNATOK_REQUIRE(need == 0 || (states && states_bytes >= need), DNATOK_E_SCRATCH, "%s: the states need %zu bytes", who, need);
    if (need)
        if (int rc = fill_words(states, need, s)) return rc;
    int rc = DNATOK_OK;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        ScanArgs<T> a{};
        a.x = (const T *)x, a.x_stride = x_stride, a.gate = (const T *)gate, a.gate_stride = gate_stride;
        a.rows = Rows{offsets, n_rows, total, total / n_rows};
        a.dim = dim, a.n_tiles = tiles_of(total, dim, dtype), a.h0 = h0, a.words = (uint64_t *)states;
        a.looks = flags & DNATOK_SCAN_NO_WAIT ? 0 : kLooks;
        a.y = (T *)y, a.last = last;
        rc = run_scan<T>(who, a, dtype, false, flags & DNATOK_SCAN_REVERSE, s);
    });
    return rc;
}

extern "C" int dnatok_gated_scan_backward(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride,
                                          int32_t dtype, const int64_t *offsets, int64_t n_rows, int64_t total,
                                          int64_t dim, int flags, const float *h0, const void *dy, int64_t dy_stride,
                                          const float *dlast, const void *states, size_t states_bytes, void *dx,
                                          void *dgate, float *dh0, void *work, size_t work_bytes, void *stream)
{
    static const char *who = "dnatok_gated_scan_backward";
    if (int rc = check_rows(who, dtype, n_rows, total, dim, offsets)) return rc;
    if (n_rows == 0) return DNATOK_OK;
    hipStream_t s = (hipStream_t)stream;
    if (total == 0) return copy_states(dlast, dh0, n_rows * dim, s);
    SCAN_REQUIRE(x && gate && dx && dgate, "null buffer");
    const size_t need = words_bytes(total, dim, dtype);
    DNATOK_REQUIRE(need == 0 || (states && states_bytes >= need), DNATOK_E_SCRATCH, "%s: the states need %zu bytes", who, need);
    DNATOK_REQUIRE(need == 0 || (work && work_bytes >= need), DNATOK_E_SCRATCH, "%s: the work space needs %zu bytes", who, need);
    if (need)
        if (int rc = fill_words(work, need, s)) return rc;
    int rc = DNATOK_OK;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        ScanArgs<T> a{};
        a.x = (const T *)x, a.x_stride = x_stride, a.gate = (const T *)gate, a.gate_stride = gate_stride;
        a.rows = Rows{offsets, n_rows, total, total / n_rows};
        a.dim = dim, a.n_tiles = tiles_of(total, dim, dtype), a.h0 = h0, a.words = (uint64_t *)states;
        a.looks = flags & DNATOK_SCAN_NO_WAIT ? 0 : kLooks;
        a.dy = (const T *)dy, a.dy_stride = dy ? dy_stride : 0, a.dlast = dlast;
        a.dx = (T *)dx, a.dgate = (T *)dgate, a.dh0 = dh0, a.back_words = (uint64_t *)work;
        rc = run_scan<T>(who, a, dtype, true, flags & DNATOK_SCAN_REVERSE, s);
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
