// Linear attention with a decay for each head, over packed rows: T_t = g T_(t-1) + k_t v_t^T, y_t = scale q_t T_t.
//
// Every product that the operator and its gradients need is one walk over a row,
//   T_t = D_(t-1) + b_t c_t^T,  D_t = g T_t,  out_t = scale a_t T_t:
// y = walk(q, k, v), dq = walk(dy, v, k), and from the row's other end dv = walk(k, q, dy) and dk = walk(v, dy, q), whose T is the
// gradient of the state.  What is in front of a row's first token (h0, or the gradient of the last state) enters as
// T forwards, so that it decays on its way in, and as D backwards; what is left behind its last token is the same.
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
    float *slots;                                  // states at the cuts [cuts, heads, b.dim, c.dim], as `start` is laid out
    int64_t cut, cuts;                             // tokens from one to the next
};

constexpr int kOutside = 64;                       // workgroups that clear what is in no row

// ---- operands of the matrix cores ---------------------------------------------------------------

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Eight { typedef T type __attribute__((ext_vector_type(8))); };
template <typename T> struct Four { typedef T type __attribute__((ext_vector_type(4))); };

// c + a b, 16 x 16 x 32: a lane has row (column) lane % 16 of a (b) and 8 of the 32, which 8 does not matter as long as it is the
// same ones for a and b; it gets column lane % 16 and rows 4 (lane / 16) .. + 3 of c.
__device__ __forceinline__ f32x4 mma(Eight<__bf16>::type a, Eight<__bf16>::type b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(Eight<_Float16>::type a, Eight<_Float16>::type b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(f32x8 a, f32x8 b, f32x4 c)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

constexpr int kChunk = 64;
constexpr int kSlotThreads = 256;
// A wave to sixteen columns of the state.
constexpr int threads_of(int columns) { return columns * 4; }

// A chunk of an operand in LDS, rows of DIM elements and some room, so that lanes with neighbouring rows meet different banks.
template <typename T, int DIM> struct alignas(16) Tile {
    static constexpr int kPitch = DIM + 16 / sizeof(T);
    T cell[kChunk * kPitch];
    // eight elements of a row from `at` on
    __device__ __forceinline__ typename Eight<T>::type row8(int row, int at) const
    {
        return *reinterpret_cast<const typename Eight<T>::type *>(cell + row * kPitch + at);
    }
    // four from `at` on and four from at + 16 on
    __device__ __forceinline__ typename Eight<T>::type row44(int row, int at) const
    {
        typedef typename Four<T>::type four;
        const four a = *reinterpret_cast<const four *>(cell + row * kPitch + at);
        const four b = *reinterpret_cast<const four *>(cell + row * kPitch + at + 16);
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    // column at + lane % 16 of rows row + 8 (lane / 16) .. + 7
    __device__ __forceinline__ typename Eight<T>::type column8(int row, int at, int lane) const
    {
        typename Eight<T>::type v;
        if constexpr (sizeof(T) == 2) {
            // (sixteen lanes read four rows of sixteen and get a column of four each)
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef s4 __attribute__((address_space(3))) * place;
            const T *p = cell + (row + 8 * (lane >> 4) + (lane >> 2 & 3)) * kPitch + at + 4 * (lane & 3);
            const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)p);
            const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)(p + 4 * kPitch));
            v = __builtin_bit_cast(typename Eight<T>::type, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const T *p = cell + (row + 8 * (lane >> 4)) * kPitch + at + (lane & 15);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = p[j * kPitch];
        }
        return v;
    }
};

// A thread's part of a chunk on its way from memory to LDS: 16 bytes of a row at a time (at any alignment).
template <typename T, int DIM, bool TAIL, int THREADS> struct Stage {
    static constexpr int kVec = 16 / sizeof(T), kPerRow = DIM / kVec, kRows = THREADS / kPerRow, kSteps = kChunk / kRows;
    u32x4 v[kSteps];
    // n tokens from p on, `token` bytes apart (64 of them span less than 2^31); zeros for those behind them, and behind the dim-th
    // element.  Whatever n is there is the same number of loads, so that a later wait counts only what was requested behind them; a lane
    // without a row asks for what is out of the buffer's range, and gets zeros.  TAIL: dim may end within 16 bytes.
    __device__ __forceinline__ void load(const char *p, int64_t token, int dim, int n)
    {
        const int at = threadIdx.x % kPerRow * kVec, row0 = threadIdx.x / kPerRow;
        if constexpr (!TAIL) {
            const __amdgpu_buffer_rsrc_t from =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(p), (short)0, (n - 1) * (int)token + dim * (int)sizeof(T), 0x00020000);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int row = row0 + s * kRows;
                const int place = row < n && at < dim ? row * (int)token + at * (int)sizeof(T) : -16;
                v[s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, place, 0, 0));
            }
        } else {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int row = row0 + s * kRows;
                v[s] = u32x4{0, 0, 0, 0};
                if (row >= n || at >= dim) continue;
                const T *q = reinterpret_cast<const T *>(p + row * token) + at;
                if (at + kVec <= dim) {
                    __builtin_memcpy(&v[s], q, 16);
                } else {
                    T e[kVec];
#pragma unroll
                    for (int i = 0; i < kVec; ++i) e[i] = at + i < dim ? q[i] : (T)0.0f;
                    __builtin_memcpy(&v[s], e, 16);
                }
            }
        }
    }
    // Token r of the chunk is its step r, or n - 1 - r.
    __device__ __forceinline__ void store(Tile<T, DIM> &t, bool reverse, int n) const
    {
        const int at = threadIdx.x % kPerRow * kVec, row0 = threadIdx.x / kPerRow;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int row = row0 + s * kRows;
            *reinterpret_cast<u32x4 *>(t.cell + (reverse && row < n ? n - 1 - row : row) * Tile<T, DIM>::kPitch + at) = v[s];
        }
    }
};

// Numbers of 32 bits as sums of parts of T, each the rounding of what the ones before leave.
template <typename T> constexpr int kParts = std::is_same<T, __bf16>::value ? 3 : std::is_same<T, _Float16>::value ? 2 : 1;
template <typename T, int N, typename V, typename P> __device__ __forceinline__ void split(V v, P (&part)[N])
{
    constexpr int kCount = sizeof(V) / 4;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (std::is_same<T, __bf16>::value) {
            typedef __bf16 two __attribute__((ext_vector_type(2)));
            typedef float f32x2 __attribute__((ext_vector_type(2)));
            typedef uint32_t words __attribute__((ext_vector_type(kCount / 2)));
            words all;
#pragma unroll
            for (int j = 0; j < kCount; j += 2) {
                uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[j], v[j + 1]}), two));
                asm("" : "+v"(w));                 // (or the second of the two is rounded again by itself)
                all[j / 2] = w;
                if (i + 1 < N) {
                    v[j] -= __uint_as_float(w << 16);
                    v[j + 1] -= __uint_as_float(w & 0xFFFF0000u);
                }
            }
            part[i] = __builtin_bit_cast(P, all);
        } else {
            part[i] = __builtin_convertvector(v, P);
            if (i + 1 < N) v -= __builtin_convertvector(part[i], V);
        }
    }
}

__device__ __forceinline__ float finite_size(float v)
{
    const float a = __builtin_fabsf(v);
    return a < INFINITY ? a : 0.0f;
}
// 2^-e and 2^e that bring numbers up to `most` to somewhat below 2^14 (float16 reaches to 2^16, and small parts need room below).
struct Power {
    float down, up;
};
__device__ __forceinline__ Power power_for(float most)
{
    int e = most > 0.0f ? __builtin_amdgcn_frexp_expf(most) - 14 : 0;
    e = e < -100 ? -100 : e > 100 ? 100 : e;
    return Power{__builtin_amdgcn_ldexpf(1.0f, -e), __builtin_amdgcn_ldexpf(1.0f, e)};
}

// Whether any element is an infinity or NaN.
template <typename V> __device__ __forceinline__ uint32_t not_finite(V v)
{
    uint32_t odd = 0;
    if constexpr (sizeof(v) == 32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) odd |= !(__builtin_fabsf(v[j]) < INFINITY);
    } else {
        // (two numbers to a word: one added to an exponent of ones reaches the sign's bit)
        constexpr bool brain = std::is_same<V, Eight<__bf16>::type>::value;
        const u32x4 words = __builtin_bit_cast(u32x4, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) odd |= (words[j] & (brain ? 0x7F807F80u : 0x7C007C00u)) + (brain ? 0x00800080u : 0x04000400u);
        odd &= 0x80008000u;
    }
    return odd;
}

// Four columns of each of 64 rows of `dim`, `pitch` elements apart, of which there are n: columns from `col` on of rows row[0 .. 3].
template <bool TAIL, typename OUT>
__device__ __forceinline__ void put(OUT *rows, int pitch, int dim, int n, int col, const int (&row)[4], const f32x4 (&v)[4])
{
    typedef typename Four<OUT>::type four;
    if constexpr (!TAIL) {                         // (as many stores whatever n is)
        const __amdgpu_buffer_rsrc_t to =
            __builtin_amdgcn_make_buffer_rsrc(rows, (short)0, ((n - 1) * pitch + dim) * (int)sizeof(OUT), 0x00020000);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int place = row[j] >= 0 && col < dim ? (row[j] * pitch + col) * (int)sizeof(OUT) : -16;
            if constexpr (sizeof(OUT) == 4)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v[j]), to, place, 0, 0);
            else
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, __builtin_convertvector(v[j], four)), to, place, 0, 0);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (row[j] >= 0 && col + r < dim) rows[(int64_t)row[j] * pitch + col + r] = (OUT)v[j][r];
    }
}

// Nothing moves past this: what is requested from LDS in front of it is under way while what is behind it is computed.  (Left to
// itself the compiler asks for one operand, waits, and uses it.)
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

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

// What is left of a state after n steps: by the factor, or by 1 - it.  (A factor next to 1, rounded once and multiplied thousands of times,
// would be a wrong rate.)
struct Left {
    float factor, lost;
};
__device__ __forceinline__ Left left_after(float log_decay, float n)
{
    // factor s - lost s: one of them is 0, and the other the more exact one
    const float lost = -expm1f(n * log_decay);
    return lost < 0.5f ? Left{1.0f, lost} : Left{expf(n * log_decay), 0.0f};
}
__device__ __forceinline__ float decayed(float s, const Left &l) { return fmaf(-l.lost, s, l.factor * s); }

__device__ __forceinline__ float log_decay_of(const WalkArgs &w, int head)
{
    return __builtin_elementwise_maximum(w.log_decay[head], -1e30f);    // (so that -inf times no step at all is 0; keeps a NaN)
}

// ---- the walk ----------------------------------------------------------------------------------------

// What a workgroup holds in LDS.
template <typename T, int KD, int CD> struct alignas(16) WalkTiles {
    static constexpr int kSplits = sizeof(T) == 2 ? 2 : 1;             // parts of a score
    Tile<T, KD> a, b;
    Tile<T, CD> c;
    Tile<T, kChunk> p[kSplits];                                        // scores times decay, [step][earlier step]
    float power[kChunk + 1];                                           // decays of 0, 1, 2 .. steps
    float up[2][kChunk];                                               // float16: what each row's scores were divided by (with 32 steps each)
};

template <typename T, int KD, int CD> struct alignas(16) PieceTiles {
    Tile<T, KD> b;
    Tile<T, CD> c;
    float power[kChunk + 1];
};

// The decays from a lane's eight steps of 32 to the end of those, and of 32 steps.
struct Decays {
    float to_end[8], over32;
};
__device__ __forceinline__ Decays decays_of(float log_decay, int late, int lane)
{
    Decays d;
#pragma unroll
    for (int j = 0; j < 8; ++j) d.to_end[j] = expf((float)(31 - 8 * (lane >> 4) - j + late) * log_decay);
    d.over32 = expf(32.0f * log_decay);
    return d;
}

// Adds b_s c_s^T, decayed to the chunk's end, to what is left of the state: `c8` is sixteen of the wave's columns of the chunk, two times
// 32 steps.  power[i] is the decay over i steps.
template <typename T, int KD>
__device__ __forceinline__ void add_chunk(f32x4 (&state)[KD / 16], const Tile<T, KD> &b, const typename Eight<T>::type (&c8)[2],
                                          const Decays &decays, const float *power, int n, int late, const Left &left, int lane)
{
    typedef typename Eight<T>::type eight;
    constexpr int N = kParts<T>;
    constexpr bool scaled = std::is_same<T, _Float16>::value;
    eight part[2][N];
    Power size{1.0f, 1.0f};
    f32x8 v[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) v[ks] = __builtin_convertvector(c8[ks], f32x8);
    if (n == kChunk) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[0][j] *= decays.to_end[j] * decays.over32;
            v[1][j] *= decays.to_end[j];
        }
    } else {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int behind = n - 1 - (32 * ks + 8 * (lane >> 4) + j);
                v[ks][j] *= power[(behind < 0 ? 0 : behind) + late];
            }
    }
    if constexpr (scaled) {                        // (a column's parts must not fall below the smallest number)
        float most = 0.0f;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, finite_size(v[ks][j]));
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        size = power_for(most);
        v[0] *= size.down;
        v[1] *= size.down;
    }
    eight b8[2][2];
    const auto fetch = [&](int kt) {
        b8[kt & 1][0] = b.column8(0, 16 * kt, lane);
        b8[kt & 1][1] = b.column8(32, 16 * kt, lane);
    };
    fetch(0);
    in_order();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) split<T>(v[ks], part[ks]);
    if (left.lost != 0.0f) {
#pragma unroll
        for (int kt = 0; kt < KD / 16; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) state[kt][r] = fmaf(-left.lost, state[kt][r], state[kt][r]);
    } else {
#pragma unroll
        for (int kt = 0; kt < KD / 16; ++kt) state[kt] *= left.factor;
    }
#pragma unroll
    for (int kt = 0; kt < KD / 16; ++kt) {
        if (kt + 1 < KD / 16) fetch(kt + 1);
        in_order();
        f32x4 sum = scaled ? f32x4{0, 0, 0, 0} : state[kt];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sum = mma(b8[kt & 1][0], part[0][i], sum);
            sum = mma(b8[kt & 1][1], part[1][i], sum);
        }
        if constexpr (scaled) {
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[r] = fmaf(sum[r], size.up, state[kt][r]);
        }
        state[kt] = sum;
    }
}

// A state [db, dc] in memory, or its transpose: a lane's column and rows of it.
template <int KD, typename Fn> __device__ __forceinline__ void each_cell(const WalkArgs &w, int column, int lane, bool transposed, Fn fn)
{
    const int db = w.b.dim, dc = w.c.dim, n = column + (lane & 15);
#pragma unroll
    for (int kt = 0; kt < KD / 16; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int m = 16 * kt + 4 * (lane >> 4) + r;
            if (m < db && n < dc) fn(kt, r, transposed ? n * db + m : m * dc + n);
        }
}

__device__ __forceinline__ const char *base_of(const Operand &o, int head, int size)
{
    return (const char *)o.p + head / o.shared * o.head * size;
}

// One workgroup to a piece of a row and a head.  Its four waves have a quarter of the state's columns each, which no other wave
// needs; scores are shared.
template <typename T, int KD, int CD, bool TAIL>
__global__ __launch_bounds__(threads_of(CD), sizeof(T) == 2 || KD + CD == 128 ? 2 : 1) void walk_kernel(WalkArgs w)
{
    typedef typename Eight<T>::type eight;
    typedef typename Four<T>::type four;
    // (scores: two or one of the waves to sixteen steps, each with half or all of the steps before them)
    constexpr int KT = KD / 16, SP = WalkTiles<T, KD, CD>::kSplits, kThreads = threads_of(CD), kScores = 16 / (CD / 16);
    constexpr bool scaled = std::is_same<T, _Float16>::value;
    __shared__ WalkTiles<T, KD, CD> lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, l16 = lane & 15;
    const int column = wave * 16, dc = w.c.dim;
    const int head = blockIdx.x % w.heads;
    const int64_t item = blockIdx.x / w.heads;
    if (item >= w.n_rows + w.cuts) {               // tokens in no row
        const int64_t front = row_at(w, 0), back = row_at(w, w.n_rows), waves = CD / 16, first = (item - w.n_rows - w.cuts) * waves + wave;
        const auto clear = [&](int64_t t) {
            for (int i = lane; i < dc; i += 64) {
                const int64_t at = (t * w.heads + head) * dc + i;
                if (w.out32) ((float *)w.out)[at] = 0.0f;
                else ((T *)w.out)[at] = (T)0.0f;
            }
        };
        for (int64_t t = first; t < front; t += kOutside * waves) clear(t);
        for (int64_t t = (back > front ? back : front) + first; t < w.total; t += kOutside * waves) clear(t);
        return;
    }
    const Piece p = piece_of(w, item);
    if (p.none) return;
    const float ld = log_decay_of(w, head);
    const int late = w.decayed ? 1 : 0;
    const bool reverse = w.reverse;
    const int64_t length = p.hi - p.lo;
    const bool starts = reverse ? p.back : p.front, ends = reverse ? p.front : p.back;
    const int64_t cells = (int64_t)w.b.dim * w.c.dim;

    // what is in front of the piece
    f32x4 state[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) state[kt] = f32x4{0, 0, 0, 0};
    if (starts ? w.start != nullptr : true) {
        const int64_t slot = (reverse ? p.hi : p.lo) / w.cut;
        const float *from = starts ? w.start + (p.row * w.heads + head) * cells : w.slots + ((slot - 1) * w.heads + head) * cells;
        const float scale = starts ? w.start_scale : 1.0f;
        each_cell<KD>(w, column, lane, w.transposed, [&](int kt, int r, int at) { state[kt][r] = scale * from[at]; });
    }

    for (int i = threadIdx.x; i <= kChunk; i += kThreads) lds.power[i] = expf((float)i * ld);
    // scores of sixteen steps with those before them, and the state's share of a step
    const int score_tile = wave * kScores / 4, first_score = wave * kScores % 4;
    float within[kScores][4], share[4];
#pragma unroll
    for (int j = 0; j < kScores; ++j) {
        const int t = 16 * score_tile + l16;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int s = 16 * (first_score + j) + 4 * g + r;
            within[j][r] = s <= t ? w.scale * expf((float)(t - s) * ld) : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) share[j] = w.scale * expf((float)(16 * j + l16 + 1 - late) * ld);
    Left left = left_after(ld, kChunk);
    const Decays decays = decays_of(ld, late, lane);

    const int64_t ta = w.a.token * sizeof(T), tb = w.b.token * sizeof(T), tc = w.c.token * sizeof(T);
    const char *pa = base_of(w.a, head, sizeof(T)), *pb = base_of(w.b, head, sizeof(T)), *pc = base_of(w.c, head, sizeof(T));
    const int da = w.a.dim, db = w.b.dim;
    Stage<T, KD, TAIL, threads_of(CD)> sa, sb;
    Stage<T, CD, TAIL, threads_of(CD)> sc;
    // the chunk that begins `done` steps into the piece: its first token, and how many
    const auto first_of = [&](int64_t done, int n) { return reverse ? p.hi - done - n : p.lo + done; };
    const auto count_of = [&](int64_t done) { return length - done < kChunk ? (int)(length - done) : kChunk; };
    const int row_cells = w.heads * dc;
    const auto fetch = [&](int64_t done) {
        const int n = count_of(done);
        const int64_t first = first_of(done, n);
        sa.load(pa + first * ta, ta, da, n);
        sb.load(pb + first * tb, tb, db, n);
        sc.load(pc + first * tc, tc, dc, n);
    };
    if (length) fetch(0);
    for (int64_t done = 0; done < length; done += kChunk) {
        const int n = count_of(done);
        if (n < kChunk) left = left_after(ld, (float)n);
        __syncthreads();
        sa.store(lds.a, reverse, n);
        sb.store(lds.b, reverse, n);
        sc.store(lds.c, reverse, n);
        __syncthreads();
        if (done + kChunk < length) fetch(done + kChunk);

        // scores, transposed: a lane has one step and four earlier ones at a time
        {
            eight a8[2], b8[2][kScores];
            const auto request = [&](int ks) {
                a8[ks & 1] = lds.a.row8(16 * score_tile + l16, 32 * ks + 8 * g);
#pragma unroll
                for (int j = 0; j < kScores; ++j) b8[ks & 1][j] = lds.b.row8(16 * (first_score + j) + l16, 32 * ks + 8 * g);
            };
            f32x4 score[kScores];
#pragma unroll
            for (int j = 0; j < kScores; ++j) score[j] = f32x4{0, 0, 0, 0};
            request(0);
#pragma unroll
            for (int ks = 0; ks < KD / 32; ++ks) {
                if (ks + 1 < KD / 32) request(ks + 1);
                in_order();
#pragma unroll
                for (int j = 0; j < kScores; ++j) score[j] = mma(b8[ks & 1][j], a8[ks & 1], score[j]);
            }
#pragma unroll
            for (int half = 0; half < kScores / 2; ++half) {
                float most = 0.0f;
#pragma unroll
                for (int j = 2 * half; j < 2 * half + 2; ++j) {
                    if (first_score + j < score_tile) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) score[j][r] *= within[j][r];
                    } else if (first_score + j == score_tile) {        // (a step behind may be NaN)
#pragma unroll
                        for (int r = 0; r < 4; ++r) score[j][r] = 4 * g + r <= l16 ? score[j][r] * within[j][r] : 0.0f;
                    } else {
                        score[j] = f32x4{0, 0, 0, 0};
                    }
                    if constexpr (scaled) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) most = fmaxf(most, finite_size(score[j][r]));
                    }
                }
                Power size{1.0f, 1.0f};
                if constexpr (scaled) {
                    most = fmaxf(most, __shfl_xor(most, 16));
                    most = fmaxf(most, __shfl_xor(most, 32));
                    size = power_for(most);
                    if (g == 0) lds.up[first_score / 2 + half][16 * score_tile + l16] = size.up;
                }
                // (in pairs of sixteen: products take 32 steps at a time)
                if (first_score + 2 * half <= score_tile) {
#pragma unroll
                    for (int j = 2 * half; j < 2 * half + 2; ++j) {
                        f32x4 v = score[j];
                        if (scaled) v *= size.down;
                        four part[SP];
                        split<T>(v, part);
#pragma unroll
                        for (int q = 0; q < SP; ++q)
                            *reinterpret_cast<four *>(lds.p[q].cell + (16 * score_tile + l16) * Tile<T, kChunk>::kPitch +
                                                      16 * (first_score + j) + 4 * g) = part[q];
                    }
                }
            }
        }
        Power size{1.0f, 1.0f};
        if constexpr (scaled) {
            float most = 0.0f;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) most = fmaxf(most, finite_size(state[kt][r]));
#pragma unroll
            for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
            size = power_for(most);
        }
        __syncthreads();

        eight c8[2];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) c8[ks] = lds.c.column8(32 * ks, column, lane);
        // a T in front of the chunk, transposed: a lane has one step and four columns at a time
        f32x4 out[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = f32x4{0, 0, 0, 0};
        eight a8[2][4], s8[SP], p8[SP][4];
        const auto request = [&](int ks) {
#pragma unroll
            for (int j = 0; j < 4; ++j) a8[ks & 1][j] = lds.a.row44(16 * j + l16, 32 * ks + 4 * g);
        };
        request(0);
        in_order();
        // whether any of the columns' cells is no finite number: 0 times it would reach the steps in front of it, so those are left
        // out at first, and then added to the steps from theirs on
        uint32_t odd = not_finite(c8[0]) | not_finite(c8[1]);
        const bool any_odd = __builtin_amdgcn_ballot_w64(odd != 0) != 0;
        if (__builtin_expect(any_odd, false)) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!(__builtin_fabsf((float)c8[ks][e]) < INFINITY)) c8[ks][e] = (T)0.0f;
        }
#pragma unroll
        for (int ks = 0; ks < KD / 32; ++ks) {
            f32x8 v = __builtin_shufflevector(state[2 * ks], state[2 * ks + 1], 0, 1, 2, 3, 4, 5, 6, 7);
            if (scaled) v *= size.down;
            split<T>(v, s8);
            if (ks + 1 < KD / 32) {
                request(ks + 1);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) p8[0][j] = lds.p[0].row8(16 * j + l16, 8 * g);
            }
            in_order();
#pragma unroll
            for (int q = 0; q < SP; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) out[j] = mma(s8[q], a8[ks & 1][j], out[j]);
        }
#pragma unroll
        for (int q = 1; q < SP; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) p8[q][j] = lds.p[q].row8(16 * j + l16, 8 * g);
        in_order();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float by = share[j];
            if constexpr (scaled) by = by * size.up / lds.up[0][16 * j + l16];
            out[j] *= by;
        }
        // the chunk's own steps
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = mma(c8[0], p8[0][j], out[j]);
        eight later[SP][2];
#pragma unroll
        for (int q = 0; q < SP; ++q)
#pragma unroll
            for (int j = 0; j < 2; ++j) later[q][j] = lds.p[q].row8(16 * j + 32 + l16, 32 + 8 * g);
        in_order();
#pragma unroll
        for (int q = 1; q < SP; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = mma(c8[0], p8[q][j], out[j]);
        if constexpr (scaled) {
#pragma unroll
            for (int j = 2; j < 4; ++j) out[j] *= lds.up[0][16 * j + l16] / lds.up[1][16 * j + l16];
        }
#pragma unroll
        for (int q = 0; q < SP; ++q)
#pragma unroll
            for (int j = 0; j < 2; ++j) out[2 + j] = mma(c8[1], later[q][j], out[2 + j]);
        if constexpr (scaled) {
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] *= lds.up[j / 2][16 * j + l16];
        }
        if (__builtin_expect(any_odd, false)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int last = 16 * j + l16;
                for (int s = 0; s <= last; ++s) {
                    float score = 0.0f;
                    for (int q = 0; q < SP; ++q) score += (float)lds.p[q].cell[last * Tile<T, kChunk>::kPitch + s];
                    if constexpr (scaled) score *= lds.up[s / 32][last];
                    for (int r = 0; r < 4; ++r) {
                        const float v = (float)lds.c.cell[s * Tile<T, CD>::kPitch + column + 4 * g + r];
                        if (!(__builtin_fabsf(v) < INFINITY)) out[j][r] += score * v;
                    }
                }
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) c8[ks] = lds.c.column8(32 * ks, column, lane);
        }
        const int64_t cell = (first_of(done, n) * w.heads + head) * dc;
        int row[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = 16 * j + l16;
            row[j] = at >= n ? -1 : reverse ? n - 1 - at : at;
        }
        if (w.out32) put<TAIL>((float *)w.out + cell, row_cells, dc, n, column + 4 * g, row, out);
        else put<TAIL>((T *)w.out + cell, row_cells, dc, n, column + 4 * g, row, out);
        add_chunk<T, KD>(state, lds.b, c8, decays, lds.power, n, late, left, lane);
    }
    if (ends && w.end) {
        float *to = w.end + (p.row * w.heads + head) * cells;
        each_cell<KD>(w, column, lane, false, [&](int kt, int r, int at) { to[at] = w.end_scale * state[kt][r]; });
    }
}

// What each piece that does not end its row adds to the state: into the slot of the cut behind it.
template <typename T, int KD, int CD, bool TAIL>
__global__ __launch_bounds__(threads_of(CD), sizeof(T) == 2 ? 2 : 1) void piece_kernel(WalkArgs w)
{
    typedef typename Eight<T>::type eight;
    constexpr int KT = KD / 16, kThreads = threads_of(CD);
    __shared__ PieceTiles<T, KD, CD> lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), column = wave * 16;
    const int head = blockIdx.x % w.heads;
    const Piece p = piece_of(w, blockIdx.x / w.heads);
    if (p.none || (w.reverse ? p.front : p.back)) return;
    const float ld = log_decay_of(w, head);
    const int late = w.decayed ? 1 : 0;
    const bool reverse = w.reverse;
    const int64_t length = p.hi - p.lo;
    f32x4 state[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) state[kt] = f32x4{0, 0, 0, 0};
    for (int i = threadIdx.x; i <= kChunk; i += kThreads) lds.power[i] = expf((float)i * ld);
    Left left = left_after(ld, kChunk);
    const Decays decays = decays_of(ld, late, lane);
    const int64_t tb = w.b.token * sizeof(T), tc = w.c.token * sizeof(T);
    const char *pb = base_of(w.b, head, sizeof(T)), *pc = base_of(w.c, head, sizeof(T));
    const int db = w.b.dim, dc = w.c.dim;
    Stage<T, KD, TAIL, threads_of(CD)> sb;
    Stage<T, CD, TAIL, threads_of(CD)> sc;
    const auto count_of = [&](int64_t done) { return length - done < kChunk ? (int)(length - done) : kChunk; };
    const auto fetch = [&](int64_t done) {
        const int n = count_of(done);
        const int64_t first = reverse ? p.hi - done - n : p.lo + done;
        sb.load(pb + first * tb, tb, db, n);
        sc.load(pc + first * tc, tc, dc, n);
    };
    if (length) fetch(0);
    for (int64_t done = 0; done < length; done += kChunk) {
        const int n = count_of(done);
        if (n < kChunk) left = left_after(ld, (float)n);
        __syncthreads();
        sb.store(lds.b, reverse, n);
        sc.store(lds.c, reverse, n);
        __syncthreads();
        if (done + kChunk < length) fetch(done + kChunk);
        eight c8[2];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) c8[ks] = lds.c.column8(32 * ks, column, lane);
        add_chunk<T, KD>(state, lds.b, c8, decays, lds.power, n, late, left, lane);
    }
    const int64_t slot = (reverse ? p.lo : p.hi) / w.cut;
    float *to = w.slots + ((slot - 1) * w.heads + head) * (int64_t)db * dc;
    each_cell<KD>(w, column, lane, false, [&](int kt, int r, int at) { to[at] = state[kt][r]; });
}

// The slots' states from what the pieces add: a thread has one cell of a head's state and runs through a row's cuts.  What comes next is
// requested before what is done is stored (a wait for a load is one for the stores in front of it).
__global__ __launch_bounds__(kSlotThreads) void slots_kernel(WalkArgs w)
{
    constexpr int kAhead = 16;
    const int head = blockIdx.y;
    const int64_t cells = (int64_t)w.b.dim * w.c.dim, cut = blockIdx.x + 1, at = cut * w.cut;
    const int64_t row = uniform(last_row(w.n_rows, at, [&](int64_t r) { return row_at(w, r); }));
    if (row < 0) return;
    const int64_t lo = uniform(row_at(w, row)), hi = uniform(row_at(w, row + 1));
    if (at <= lo || at >= hi) return;
    const int64_t first = lo / w.cut + 1, last = (hi - 1) / w.cut, n = last - first + 1;
    if (cut != (w.reverse ? last : first)) return;
    const int64_t i = (int64_t)blockIdx.z * kSlotThreads + threadIdx.x;
    if (i >= cells) return;
    const float ld = log_decay_of(w, head);
    float state = w.start ? w.start_scale * w.start[(row * w.heads + head) * cells + i] : 0.0f;
    const int64_t outer = w.reverse ? hi - last * w.cut : first * w.cut - lo;
    const Left left = left_after(ld, (float)w.cut);
    state = decayed(state, left_after(ld, (float)outer));
    float *slot = w.slots + ((w.reverse ? last : first) - 1) * w.heads * cells + head * cells + i;
    const int64_t next = (w.reverse ? -1 : 1) * w.heads * cells;
    float added[kAhead], coming[kAhead];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) added[e] = e < n ? slot[e * next] : 0.0f;
    for (int64_t j = 0; j < n; j += kAhead) {
#pragma unroll
        for (int e = 0; e < kAhead; ++e) coming[e] = j + kAhead + e < n ? slot[(kAhead + e) * next] : 0.0f;
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            state += added[e];
            if (j + e < n) slot[e * next] = state;
            state = decayed(state, left);
            added[e] = coming[e];
        }
        slot += kAhead * next;
    }
}

// Gradients of keys and values that several heads share: the heads' parts, 32-bit [total, heads, dim], added up.
template <typename T>
__global__ __launch_bounds__(256) void shared_sum_kernel(const float *parts, T *out, int64_t cells, int32_t shared, int32_t dim)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (int64_t)gridDim.x * 256) {
        const int64_t head = i / dim, at = i % dim;
        float sum = 0.0f;
        for (int j = 0; j < shared; ++j) sum += parts[(head * shared + j) * dim + at];
        out[i] = from_float<T>(sum);
    }
}

// One token of each row: a workgroup has a head's state, a thread every few rows of VEC of its columns.  The state is
// read and written once; nothing else weighs anything.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void linear_step_kernel(Operand q, Operand k, Operand v, const float *log_decay, float scale,
                                                          const float *state, T *y, float *new_state)
{
    typedef float vec __attribute__((ext_vector_type(VEC)));
    __shared__ float qk[2][128];
    __shared__ float part[256 * VEC];
    const int64_t row = blockIdx.y;
    const int head = blockIdx.x, heads = gridDim.x, dk = q.dim, dv = v.dim, cols = dv / VEC;
    const T *qp = (const T *)q.p + row * q.token + head * q.head;
    const T *kp = (const T *)k.p + row * k.token + head / k.shared * k.head;
    const T *vp = (const T *)v.p + row * v.token + head / v.shared * v.head;
    for (int i = threadIdx.x; i < dk; i += 256) {
        qk[0][i] = to_float(qp[i]);
        qk[1][i] = to_float(kp[i]);
    }
    const float g = expf(log_decay[head]);
    const int per = 256 / cols, col = threadIdx.x % cols, first = threadIdx.x / cols;      // (threads behind the last whole row have none)
    const int64_t at = (row * heads + head) * dk * dv;
    vec sum{}, value{};
    if (first < per)
#pragma unroll
        for (int e = 0; e < VEC; ++e) value[e] = to_float(vp[col * VEC + e]);
    __syncthreads();
    if (first < per) {
        for (int m = first; m < dk; m += per) {
            vec s{};
            if (state) s = *reinterpret_cast<const vec *>(state + at + m * dv + col * VEC);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                s[e] = (state ? g * s[e] : 0.0f) + qk[1][m] * value[e];
                sum[e] += qk[0][m] * s[e];
            }
            *reinterpret_cast<vec *>(new_state + at + m * dv + col * VEC) = s;
        }
    }
    *reinterpret_cast<vec *>(part + threadIdx.x * VEC) = sum;
    __syncthreads();
    for (int i = threadIdx.x; i < dv; i += 256) {
        float all = 0.0f;
        for (int j = 0; j < per; ++j) all += part[j * dv + i];
        y[(row * heads + head) * dv + i] = from_float<T>(scale * all);
    }
}

}  // namespace dnatok

using namespace dnatok;

#define LINEAR_REQUIRE(cond, text) DNATOK_REQUIRE(cond, DNATOK_E_INVALID, "%s: " text, who)

static int check_shape(const char *who, const dnatok_linear_shape *s)
{
    LINEAR_REQUIRE(s, "null shape");
    LINEAR_REQUIRE(s->dtype == DNATOK_F32 || s->dtype == DNATOK_BF16 || s->dtype == DNATOK_F16, "unknown element type");
    LINEAR_REQUIRE(s->n_rows >= 0 && s->total >= 0 && s->heads > 0 && s->kv_heads > 0 && s->dim_k > 0 && s->dim_v > 0, "bad size");
    LINEAR_REQUIRE(s->heads % s->kv_heads == 0, "the heads must be a multiple of those of the keys and values");
    LINEAR_REQUIRE(s->scale != 0.0f && __builtin_isfinite(s->scale), "the scale must be a finite number other than 0");
    LINEAR_REQUIRE(s->q_token >= 0 && s->q_head >= 0 && s->k_token >= 0 && s->k_head >= 0 && s->v_token >= 0 && s->v_head >= 0 &&
                       s->dy_token >= 0 && s->dy_head >= 0, "negative stride");
    constexpr int64_t kFar = (1ll << 31) / 64 / 4;
    DNATOK_REQUIRE(s->q_token < kFar && s->k_token < kFar && s->v_token < kFar && s->dy_token < kFar && (int64_t)s->heads * 128 < kFar,
                   DNATOK_E_TOO_LARGE, "%s: tokens must lie less than 2^23 elements apart", who);
    DNATOK_REQUIRE(s->dim_k <= 128 && s->dim_v <= 128 && s->heads <= 65535 && s->total < (1ll << 40) && s->n_rows < (1ll << 30),
                   DNATOK_E_TOO_LARGE, "%s: at most 65535 heads of 128 x 128", who);
    return DNATOK_OK;
}

static int check_call(const char *who, const dnatok_linear_shape &s, const int64_t *offsets)
{
    LINEAR_REQUIRE(!offsets == !s.with_offsets, "the shape must say whether there are offsets");
    LINEAR_REQUIRE(s.n_rows > 0 || s.total == 0, "tokens without rows");
    LINEAR_REQUIRE(offsets || s.n_rows == 0 || s.total % s.n_rows == 0, "rows of one length must fill the axis");
    DNATOK_REQUIRE((s.n_rows + (s.total >> 9) + kOutside) < (1ll << 24) / s.heads, DNATOK_E_TOO_LARGE,
                   "%s: at most 2^24 rows and pieces of rows times heads", who);
    return DNATOK_OK;
}

static Operand operand(const void *p, int64_t token, int64_t head, int32_t shared, int32_t dim)
{
    return Operand{p, token, head, shared, dim};
}
static Operand q_of(const dnatok_linear_shape *s, const void *q) { return operand(q, s->q_token, s->q_head, 1, s->dim_k); }
static Operand k_of(const dnatok_linear_shape *s, const void *k)
{
    return operand(k, s->k_token, s->k_head, s->heads / s->kv_heads, s->dim_k);
}
static Operand v_of(const dnatok_linear_shape *s, const void *v)
{
    return operand(v, s->v_token, s->v_head, s->heads / s->kv_heads, s->dim_v);
}

static unsigned sum_grid(int64_t cells) { return (unsigned)(cells < 65536 * 256 ? (cells + 255) / 256 : 65536); }

static size_t slots_bytes(const dnatok_linear_shape *s, int64_t cuts) { return (size_t)cuts * s->heads * s->dim_k * s->dim_v * 4; }

// Where rows are cut, so that one long row has many workgroups: at multiples of `cut` tokens, which leave as many pieces as run at
// once (two workgroups on each of 256 CUs), the rows' own beginnings among them; where those alone are more than half of that, some
// 512 more.  512 tokens at least.  Rows of one length that are half of what runs at once are not cut.
constexpr int64_t kRunning = 512;
struct Cuts {
    int64_t cut, cuts;
};
static Cuts cuts_of(const dnatok_linear_shape *s)
{
    const int64_t rows = s->n_rows * s->heads, room = rows <= kRunning / 2 ? kRunning - rows : kRunning;
    int64_t cut = (s->total * s->heads + room - 1) / room;
    cut = cut < 512 ? 512 : (cut + kChunk - 1) / kChunk * kChunk;
    if (s->total == 0 || (!s->with_offsets && rows >= kRunning / 2)) return Cuts{cut, 0};
    return Cuts{cut, (s->total - 1) / cut};
}

template <typename T, typename Fn> static void with_tiles(int32_t db, int32_t dc, Fn fn)
{
    typedef std::integral_constant<int, 64> Small;
    typedef std::integral_constant<int, 128> Large;
    const auto sized = [&](auto tail) {
        if (db <= 64) {
            if (dc <= 64) fn(Small{}, Small{}, tail);
            else fn(Small{}, Large{}, tail);
        } else {
            if (dc <= 64) fn(Large{}, Small{}, tail);
            else fn(Large{}, Large{}, tail);
        }
    };
    constexpr int kVec = 16 / sizeof(T);
    if (db % kVec || dc % kVec) sized(std::true_type{});
    else sized(std::false_type{});
}
// The states at the cuts, then.
template <typename T> static void fill_slots(const WalkArgs &w, hipStream_t s)
{
    if (!w.cuts) return;
    with_tiles<T>(w.b.dim, w.c.dim, [&](auto kd, auto cd, auto tail) {
        piece_kernel<T, kd(), cd(), tail()><<<(unsigned)((w.n_rows + w.cuts) * w.heads), threads_of(cd()), 0, s>>>(w);
    });
    const unsigned parts = (unsigned)((w.b.dim * w.c.dim + kSlotThreads - 1) / kSlotThreads);
    slots_kernel<<<dim3((unsigned)w.cuts, (unsigned)w.heads, parts), kSlotThreads, 0, s>>>(w);
}
template <typename T> static void walk(const WalkArgs &w, hipStream_t s)
{
    const int64_t items = w.n_rows + w.cuts + (w.offsets ? kOutside : 0);
    with_tiles<T>(w.b.dim, w.c.dim, [&](auto kd, auto cd, auto tail) {
        walk_kernel<T, kd(), cd(), tail()><<<(unsigned)(items * w.heads), threads_of(cd()), 0, s>>>(w);
    });
}

extern "C" size_t dnatok_linear_attention_states_bytes(const dnatok_linear_shape *s)
{
    return s && s->heads > 0 ? slots_bytes(s, cuts_of(s).cuts) : 0;
}

extern "C" size_t dnatok_linear_attention_work_bytes(const dnatok_linear_shape *s, int backward)
{
    if (!s || s->heads <= 0) return 0;
    size_t n = slots_bytes(s, cuts_of(s).cuts);
    if (backward && s->kv_heads != s->heads) n += (size_t)s->total * s->heads * (s->dim_k + s->dim_v) * 4;
    return n;
}

extern "C" int dnatok_linear_attention(const dnatok_linear_shape *shape, const void *q, const void *k, const void *v,
                                       const float *log_decay, const int64_t *offsets, const float *h0, void *y, float *last,
                                       float *states, void *work, size_t work_bytes, void *stream)
{
    static const char *who = "dnatok_linear_attention";
    if (int rc = check_shape(who, shape)) return rc;
    const dnatok_linear_shape &s = *shape;
    if (int rc = check_call(who, s, offsets)) return rc;
    LINEAR_REQUIRE(log_decay && (s.total == 0 || (q && k && v && y)), "null buffer");
    LINEAR_REQUIRE(states || (work_bytes >= dnatok_linear_attention_work_bytes(shape, 0) && (work || !work_bytes)), "work space too small");
    LINEAR_REQUIRE((uintptr_t)work % 16 == 0 && (uintptr_t)states % 16 == 0, "work space must be 16-byte aligned");
    if (s.n_rows == 0) return DNATOK_OK;
    const Cuts cuts = cuts_of(shape);
    with_type(s.dtype, [&](auto t) {
        using T = decltype(t);
        const WalkArgs w{q_of(shape, q), k_of(shape, k), v_of(shape, v), log_decay, offsets, s.n_rows, s.total, s.total / s.n_rows,
                         s.heads, s.reverse != 0, false, s.scale, 1.0f, 1.0f, h0, false, last, y, false,
                         states ? states : (float *)work, cuts.cut, cuts.cuts};
        fill_slots<T>(w, (hipStream_t)stream);
        walk<T>(w, (hipStream_t)stream);
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

extern "C" int dnatok_linear_attention_backward(const dnatok_linear_shape *shape, const void *q, const void *k, const void *v,
                                                const float *log_decay, const int64_t *offsets, const float *h0, const void *dy,
                                                const float *dlast, const float *states, void *dq, void *dk, void *dv, float *dh0,
                                                void *work, size_t work_bytes, void *stream)
{
    static const char *who = "dnatok_linear_attention_backward";
    if (int rc = check_shape(who, shape)) return rc;
    const dnatok_linear_shape &s = *shape;
    if (int rc = check_call(who, s, offsets)) return rc;
    LINEAR_REQUIRE(log_decay && (s.total == 0 || (q && k && v && dy && dq && dk && dv)), "null buffer");
    LINEAR_REQUIRE(states || !dnatok_linear_attention_states_bytes(shape), "the forward pass' states are missing");
    LINEAR_REQUIRE(work_bytes >= dnatok_linear_attention_work_bytes(shape, 1) && (work || !work_bytes), "work space too small");
    LINEAR_REQUIRE((uintptr_t)work % 16 == 0 && (uintptr_t)states % 16 == 0, "work space must be 16-byte aligned");
    if (s.n_rows == 0) return DNATOK_OK;
    hipStream_t stm = (hipStream_t)stream;
    const Operand qo = q_of(shape, q), ko = k_of(shape, k), vo = v_of(shape, v),
                  go = operand(dy, s.dy_token, s.dy_head, 1, s.dim_v);
    const int64_t length = s.total / s.n_rows;
    const Cuts cuts = cuts_of(shape);
    with_type(s.dtype, [&](auto t) {
        using T = decltype(t);
        const bool shared = s.heads != s.kv_heads, rev = s.reverse != 0;
        walk<T>(WalkArgs{go, vo, ko, log_decay, offsets, s.n_rows, s.total, length, s.heads, rev, false, s.scale, 1.0f, 1.0f, h0,
                         true, nullptr, dq, false, const_cast<float *>(states), cuts.cut, cuts.cuts}, stm);
        float *slots = (float *)work, *pk = slots + slots_bytes(shape, cuts.cuts) / 4, *pv = pk + s.total * s.heads * s.dim_k;
        // (a state's gradient without the scale, which all that is made of it gets)
        const float inv = 1.0f / s.scale;
        const WalkArgs wv{ko, qo, go, log_decay, offsets, s.n_rows, s.total, length, s.heads, !rev, true, s.scale, inv, s.scale, dlast,
                          false, dh0, shared ? (void *)pv : dv, shared, slots, cuts.cut, cuts.cuts};
        const WalkArgs wk{vo, go, qo, log_decay, offsets, s.n_rows, s.total, length, s.heads, !rev, true, s.scale, inv, s.scale, dlast,
                          true, nullptr, shared ? (void *)pk : dk, shared, slots, cuts.cut, cuts.cuts};
        fill_slots<T>(wv, stm);
        walk<T>(wv, stm);
        walk<T>(wk, stm);
        if (shared && s.total) {
            const int64_t ck = s.total * s.kv_heads * s.dim_k, cv = s.total * s.kv_heads * s.dim_v;
            shared_sum_kernel<T><<<sum_grid(ck), 256, 0, stm>>>(pk, (T *)dk, ck, s.heads / s.kv_heads, s.dim_k);
            shared_sum_kernel<T><<<sum_grid(cv), 256, 0, stm>>>(pv, (T *)dv, cv, s.heads / s.kv_heads, s.dim_v);
        }
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

extern "C" int dnatok_linear_attention_step(const dnatok_linear_shape *shape, const void *q, const void *k, const void *v,
                                            const float *log_decay, const float *state, void *y, float *new_state, void *stream)
{
    static const char *who = "dnatok_linear_attention_step";
    if (int rc = check_shape(who, shape)) return rc;
    const dnatok_linear_shape &s = *shape;
    if (s.n_rows == 0) return DNATOK_OK;
    LINEAR_REQUIRE(q && k && v && log_decay && y && new_state, "null buffer");
    DNATOK_REQUIRE(s.n_rows <= 65535, DNATOK_E_TOO_LARGE, "%s: at most 65535 rows", who);
    const dim3 grid((unsigned)s.heads, (unsigned)s.n_rows);
    const bool wide = s.dim_v % 4 == 0 && ((uintptr_t)state | (uintptr_t)new_state) % 16 == 0;
    with_type(s.dtype, [&](auto t) {
        using T = decltype(t);
        if (wide)
            linear_step_kernel<T, 4><<<grid, 256, 0, (hipStream_t)stream>>>(q_of(shape, q), k_of(shape, k), v_of(shape, v), log_decay,
                                                                            s.scale, state, (T *)y, new_state);
        else
            linear_step_kernel<T, 1><<<grid, 256, 0, (hipStream_t)stream>>>(q_of(shape, q), k_of(shape, k), v_of(shape, v), log_decay,
                                                                            s.scale, state, (T *)y, new_state);
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
