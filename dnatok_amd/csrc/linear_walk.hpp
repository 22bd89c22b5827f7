// The walk of linear attention on the matrix cores (see linear_common.hpp for the mathematics), for one element type to a file.
//
// 16-bit operands: scores and T are fed to the products as two parts of T's type each (hi + lo, 2^-17 of themselves), what is added
// to the state as three parts of a bfloat16 or two of a float16, so that results are as if computed in 32 bits and rounded once, and
// the states are good to 32 bits.  (With one part, y would be off by 1.4 roundings of its type instead of one.)  float16 has no range for
// scores and states: each row of scores, each column that is added and each wave's part of T is brought near 2^14 by a power of two, and what
// is 2^39 below its largest is lost: next to its rounding a state is off by up to 2^-39 of a chunk's largest b and c.  (That is seen
// only in cells whose last steps add exact zeros while the decay takes them there; y, of 11 bits, is not.)
#pragma once

#include "linear_common.hpp"

namespace dnatok {

// ---- operands of the matrix cores ---------------------------------------------------------------

// Sixteen bytes of an operand: a lane's part of a product of depth kDepth.
template <typename T> struct Frag {
    static constexpr int kCount = 16 / sizeof(T), kDepth = 4 * kCount;
    typedef T type __attribute__((ext_vector_type(kCount)));
    typedef float floats __attribute__((ext_vector_type(kCount)));
};
template <typename T> struct Four { typedef T type __attribute__((ext_vector_type(4))); };

// c + a b: a lane has row (column) lane % 16 of a (b) and kCount of the contraction's kDepth, the same ones of a and b; it gets
// column lane % 16 and rows 4 (lane / 16) .. + 3 of c.
__device__ __forceinline__ f32x4 mma(Frag<__bf16>::type a, Frag<__bf16>::type b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(Frag<_Float16>::type a, Frag<_Float16>::type b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// Which of kDepth steps a lane has as its j-th in a product over steps (chosen so that reading them as columns meets each bank of LDS
// once).
template <typename T> __device__ __forceinline__ constexpr int step_of(int j, int lane)
{
    return sizeof(T) == 2 ? 8 * (lane >> 4) + (j < 4 ? 2 * j : 2 * j - 7) : 4 * (lane >> 4) + j;
}
// Scores [step][earlier step] are kept so that a lane's lie together: where an earlier step's is.
template <typename T> __device__ __forceinline__ constexpr int score_place(int s)
{
    return sizeof(T) == 2 ? (s & ~7) + (s & 1) * 4 + (s >> 1 & 3) : s;
}

// A chunk of an operand in LDS, rows of DIM elements and 16 bytes of room, so that lanes with neighbouring rows meet different banks.
template <typename T, int DIM> struct alignas(16) Tile {
    typedef typename Frag<T>::type frag;
    static constexpr int kPitch = DIM + Frag<T>::kCount;
    T cell[kChunk * kPitch];
    // a lane's part of kDepth elements of a row from `at` on, sixteen bytes in a piece
    __device__ __forceinline__ frag row(int r, int at, int lane) const
    {
        return *reinterpret_cast<const frag *>(cell + r * kPitch + at + Frag<T>::kCount * (lane >> 4));
    }
    // the same elements as those that a lane has of T: four of each sixteen
    __device__ __forceinline__ frag row_as_state(int r, int at, int lane) const
    {
        if constexpr (sizeof(T) == 2) {
            typedef typename Four<T>::type four;
            const T *p = cell + r * kPitch + at + 4 * (lane >> 4);
            return __builtin_shufflevector(*reinterpret_cast<const four *>(p), *reinterpret_cast<const four *>(p + 16), 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return row(r, at, lane);
        }
    }
    // column at + lane % 16 of the lane's of the kDepth rows from `r` on
    __device__ __forceinline__ frag column(int r, int at, int lane) const
    {
        if constexpr (sizeof(T) == 2) {
            // (sixteen lanes read four rows of sixteen and get a column of four each)
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef s4 __attribute__((address_space(3))) * place;
            const T *p = cell + (r + 8 * (lane >> 4) + 2 * (lane >> 2 & 3)) * kPitch + at + 4 * (lane & 3);
            const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)p);
            const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)(p + kPitch));
            return __builtin_bit_cast(frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const T *p = cell + (r + 4 * (lane >> 4)) * kPitch + at + (lane & 15);
            return frag{p[0], p[kPitch], p[2 * kPitch], p[3 * kPitch]};
        }
    }
    // scores of four earlier steps from `from` (a multiple of four) on
    __device__ __forceinline__ void put_scores(int step, int from, typename Four<T>::type v)
    {
        T *p = cell + step * kPitch;
        if constexpr (sizeof(T) == 2) {
            typedef T two __attribute__((ext_vector_type(2)));
            *reinterpret_cast<two *>(p + score_place<T>(from)) = two{v[0], v[2]};
            *reinterpret_cast<two *>(p + score_place<T>(from + 1)) = two{v[1], v[3]};
        } else {
            *reinterpret_cast<typename Four<T>::type *>(p + from) = v;
        }
    }
};

// A thread's part of a chunk on its way from memory to LDS: 16 bytes of a row at a time (at any alignment).
template <typename T, int DIM, bool TAIL, int THREADS> struct Stage {
    static constexpr int kVec = 16 / sizeof(T), kPerRow = DIM / kVec, kAll = kChunk * kPerRow, kSteps = (kAll + THREADS - 1) / THREADS;
    u32x4 v[kSteps];
    // n tokens from p on, `token` bytes apart (64 of them span less than 2^31); zeros for those behind them, and behind the dim-th
    // element.  Whatever n is there is the same number of loads, so that a later wait counts only what was requested behind them; a lane
    // without a row asks for what is out of the buffer's range, and gets zeros.  TAIL: dim may end within 16 bytes.
    __device__ __forceinline__ void load(const char *p, int64_t token, int dim, int n)
    {
        const __amdgpu_buffer_rsrc_t from =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(p), (short)0, (n - 1) * (int)token + dim * (int)sizeof(T), 0x00020000);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int i = threadIdx.x + s * THREADS, row = i / kPerRow, at = i % kPerRow * kVec;
            if constexpr (!TAIL) {
                const int place = row < n && at < dim ? row * (int)token + at * (int)sizeof(T) : -16;
                v[s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, place, 0, 0));
            } else {
                v[s] = u32x4{0, 0, 0, 0};
                if (row >= n || at >= dim) continue;
                const T *q = reinterpret_cast<const T *>(p + row * token) + at;
                if (at + kVec <= dim) {
                    __builtin_memcpy(&v[s], q, 16);
                } else {
                    T e[kVec];
#pragma unroll
                    for (int k = 0; k < kVec; ++k) e[k] = at + k < dim ? q[k] : (T)0.0f;
                    __builtin_memcpy(&v[s], e, 16);
                }
            }
        }
    }
    // Token r of the chunk is its step r, or n - 1 - r.
    __device__ __forceinline__ void store(Tile<T, DIM> &t, bool reverse, int n) const
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int i = threadIdx.x + s * THREADS, row = i / kPerRow, at = i % kPerRow * kVec;
            if (kAll % THREADS && i >= kAll) continue;
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
template <typename T> __device__ __forceinline__ uint32_t not_finite(typename Frag<T>::type v)
{
    uint32_t odd = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) odd |= !(__builtin_fabsf(v[j]) < INFINITY);
    } else {
        // (two numbers to a word: one added to an exponent of ones reaches the sign's bit)
        constexpr bool brain = std::is_same<T, __bf16>::value;
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

// ---- chunks in LDS -----------------------------------------------------------------------------------

// Whether LDS holds two chunks of the operands, so that the next one is there when a chunk is done: where a workgroup has the CU to
// itself.  (256 rows of 1,024 tokens and 4 heads of 128 x 128: 335 us, with one chunk 347; smaller heads have a second workgroup on
// the CU, and want the room: 128 x 64 takes 210, with two 278; 64 rows of 8,192 and 8 heads of 64 x 64 519, with two 550.)
template <typename T, int KD, int CD> constexpr bool kTwoChunks = sizeof(T) == 2 && KD > 64 && CD > 64;

template <typename T, int KD, int CD> struct alignas(16) Chunk {
    Tile<T, KD> a, b;
    Tile<T, CD> c;
};
template <typename T, int KD, int CD> struct alignas(16) WalkTiles {
    static constexpr int kSplits = sizeof(T) == 2 ? 2 : 1;             // parts of a score
    Chunk<T, KD, CD> chunk[kTwoChunks<T, KD, CD> ? 2 : 1];
    Tile<T, kChunk> p[kSplits];
    float power[kChunk + 1];                                           // decays of 0, 1, 2 .. steps
    float up[2][kChunk];                                               // float16: what each row's scores with 32 steps each were divided by
};
template <typename T, int KD, int CD> struct alignas(16) PieceTiles {
    Tile<T, KD> b;
    Tile<T, CD> c;
    float power[kChunk + 1];
};

// The decays from a lane's steps of kDepth to the end of those, and of what lies behind those in the chunk.
template <typename T> struct Decays {
    static constexpr int kBlocks = kChunk / Frag<T>::kDepth;
    float to_end[Frag<T>::kCount], behind[kBlocks];
};
template <typename T> __device__ __forceinline__ Decays<T> decays_of(float log_decay, int late, int lane)
{
    Decays<T> d;
#pragma unroll
    for (int j = 0; j < Frag<T>::kCount; ++j) d.to_end[j] = expf((float)(Frag<T>::kDepth - 1 - step_of<T>(j, lane) + late) * log_decay);
#pragma unroll
    for (int i = 0; i < d.kBlocks; ++i) d.behind[i] = expf((float)(Frag<T>::kDepth * (d.kBlocks - 1 - i)) * log_decay);
    return d;
}

// Adds b_s c_s^T, decayed to the chunk's end, to what is left of the state: `c` is sixteen of the wave's columns of the chunk.
// power[i] is the decay over i steps.  exact: whether a state of 32 bits is asked for (if all that is made of it has 16, two parts of a
// bfloat16 will do).
template <typename T, int KD>
__device__ __forceinline__ void add_chunk(f32x4 (&state)[KD / 16], const Tile<T, KD> &b, const typename Frag<T>::type (&c)[kChunk / Frag<T>::kDepth],
                                          const Decays<T> &decays, const float *power, int n, int late, const Left &left, bool exact, int lane)
{
    typedef typename Frag<T>::type frag;
    typedef typename Frag<T>::floats floats;
    // (KB tiles at a time: two sums that do not wait for each other; 32-bit products take so long that one will do)
    constexpr int N = kParts<T>, KT = KD / 16, KB = sizeof(T) == 2 ? 2 : 1, TS = kChunk / Frag<T>::kDepth, J = Frag<T>::kCount;
    // (apart: what is added is summed from zero and added once.  Rounded sixteen times a chunk, as what the products of 32 bits are added to,
    // states that last for 4,000 tokens are off by 8e-7, apart by 2e-7.  For bfloat16 it is four or six times, and no register is left.)
    constexpr bool scaled = std::is_same<T, _Float16>::value, apart = scaled || sizeof(T) == 4;
    frag b8[2][KB][TS];
    const auto fetch = [&](int kt) {
#pragma unroll
        for (int i = 0; i < KB; ++i)
#pragma unroll
            for (int ts = 0; ts < TS; ++ts) b8[kt / KB & 1][i][ts] = b.column(ts * Frag<T>::kDepth, 16 * (kt + i), lane);
    };
    fetch(0);
    in_order();
    frag part[TS][N];
    Power size{1.0f, 1.0f};
    floats v[TS];
#pragma unroll
    for (int ts = 0; ts < TS; ++ts) v[ts] = __builtin_convertvector(c[ts], floats);
    if (n == kChunk) {
#pragma unroll
        for (int ts = 0; ts < TS; ++ts)
#pragma unroll
            for (int j = 0; j < J; ++j) v[ts][j] *= ts + 1 < TS ? decays.to_end[j] * decays.behind[ts] : decays.to_end[j];
    } else {
#pragma unroll
        for (int ts = 0; ts < TS; ++ts)
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int behind = n - 1 - (ts * Frag<T>::kDepth + step_of<T>(j, lane));
                v[ts][j] *= power[(behind < 0 ? 0 : behind) + late];
            }
    }
    if constexpr (scaled) {                        // (a column's parts must not fall below the smallest number)
        float most = 0.0f;
#pragma unroll
        for (int ts = 0; ts < TS; ++ts)
#pragma unroll
            for (int j = 0; j < J; ++j) most = fmaxf(most, finite_size(v[ts][j]));
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        size = power_for(most);
#pragma unroll
        for (int ts = 0; ts < TS; ++ts) v[ts] *= size.down;
    }
#pragma unroll
    for (int ts = 0; ts < TS; ++ts) split<T>(v[ts], part[ts]);
    if (left.lost != 0.0f) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) state[kt][r] = fmaf(-left.lost, state[kt][r], state[kt][r]);
    } else {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) state[kt] *= left.factor;
    }
#pragma unroll
    for (int kt = 0; kt < KT; kt += KB) {
        if (kt + KB < KT) fetch(kt + KB);
        in_order();
        f32x4 sum[KB];
#pragma unroll
        for (int i = 0; i < KB; ++i) sum[i] = apart ? f32x4{0, 0, 0, 0} : state[kt + i];
#pragma unroll
        for (int q = 0; q < N; ++q) {
            if (q == 2 && !exact) break;
#pragma unroll
            for (int ts = 0; ts < TS; ++ts)
#pragma unroll
                for (int i = 0; i < KB; ++i) sum[i] = mma(b8[kt / KB & 1][i][ts], part[ts][q], sum[i]);
        }
#pragma unroll
        for (int i = 0; i < KB; ++i) {
            if constexpr (apart) {
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[i][r] = scaled ? fmaf(sum[i][r], size.up, state[kt + i][r]) : state[kt + i][r] + sum[i][r];
            }
            state[kt + i] = sum[i];
        }
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

// ---- infinities and NaN ------------------------------------------------------------------------------

// In the products an infinity becomes a NaN at once: its parts are inf and inf - inf, what masks it or has decayed to nothing is 0 times
// it, and terms of the recurrence that are never added there meet.  Such outputs and cells of states are not finite, whatever became
// of them, and no others are touched; so a wave that finds any goes through its piece once more, step by step as the recurrence
// is written, and replaces those.  (An infinite value in each row's first token: 64 rows of 8,192 tokens, 8 heads of 64 x 64,
// 12.0 ms instead of 0.53; one row of 262,147 in 63 pieces, 4 heads of 128 x 128, 8.7 instead of 0.55.)
__device__ __forceinline__ bool is_finite(float v) { return __builtin_fabsf(v) < INFINITY; }
template <int N> __device__ __forceinline__ bool any_not_finite(const f32x4 (&v)[N])
{
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) most = __builtin_elementwise_maximum(most, __builtin_fabsf(v[i][r]));      // (keeps a NaN)
    return __builtin_amdgcn_ballot_w64(!is_finite(most)) != 0;
}

// A number that the compiler knows nothing of: what it would find out (which rows are there), it finds out again, and does not keep it through
// the walk in registers that are needed there.
__device__ __forceinline__ int forgotten(int v)
{
    asm("" : "+v"(v));
    return v;
}

// Another lane's four numbers.
template <typename V> __device__ __forceinline__ V from_lane(V v, int lane)
{
    constexpr int kWords = sizeof(V) / 4;
    typedef int words __attribute__((ext_vector_type(kWords)));
    words w = __builtin_bit_cast(words, v);
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = __shfl(w[i], lane);
    return __builtin_bit_cast(V, w);
}

// The steps of a piece, one at a time: out(step, values) for sixteen steps at a time from the step `quiet` on (OUT), of which a lane has step
// lane % 16 and columns 4 (lane / 16) .. + 3 of the wave's sixteen, and what becomes of the state, of which it has column lane % 16
// and rows 4 (lane / 16) .. + 3 of each sixteen.  Operands are fetched for sixteen steps at once, a lane having one step's, and handed
// round.  Where all of a wave's state is NaN (training that went astray), so is all that follows.
template <typename T, int KD, bool TAIL, bool OUT, typename Fn>
__device__ __forceinline__ void by_steps(const WalkArgs &w, const Piece &p, int head, float log_decay, int column, int lane, f32x4 (&state)[KD / 16],
                                         int64_t quiet, Fn out)
{
    typedef typename Four<T>::type four;
    constexpr int KT = KD / 16;
    const Left left = left_after(log_decay, 1.0f);
    const int g = lane >> 4, l16 = lane & 15, db = w.b.dim, dc = w.c.dim;
    const int64_t length = p.hi - p.lo;
    const T *pa = OUT ? (const T *)base_of(w.a, head, sizeof(T)) : nullptr, *pb = (const T *)base_of(w.b, head, sizeof(T)),
            *pc = (const T *)base_of(w.c, head, sizeof(T));
    const auto four_of = [](const T *row, int m, int dim) {
        four v{};
        if (!TAIL) {
            if (m < dim) __builtin_memcpy(&v, row + m, sizeof(v));
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (m + r < dim) v[r] = row[m + r];
        }
        return v;
    };
    bool lost = false;
    for (int64_t first = 0; first < length; first += 16) {
        const int here = length - first < 16 ? (int)(length - first) : 16;
        const bool puts = OUT && first >= quiet;
        const int64_t mine = first + l16, t = w.reverse ? p.hi - 1 - mine : p.lo + mine;
        f32x4 value = {NAN, NAN, NAN, NAN};
        if (!lost) {
            four a[KT]{}, b[KT]{}, c{};
            if (l16 < here) {
                c = four_of(pc + t * w.c.token + column + 4 * g, 0, dc - column - 4 * g);
                const T *row = pb + t * w.b.token + 4 * g;
                int rows = forgotten(db - 4 * g);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) b[kt] = four_of(row, 16 * kt, rows);
                if (puts) {
                    row = pa + t * w.a.token + 4 * g;
                    rows = forgotten(db - 4 * g);
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) a[kt] = four_of(row, 16 * kt, rows);
                }
            }
#pragma unroll 1
            for (int j = 0; j < here; ++j) {
                const int rows = forgotten(db - 4 * g);
                const four columns = from_lane(c, 16 * (l16 >> 2) + j);
                float mine_of = (float)columns[0], sum = 0.0f;
#pragma unroll
                for (int r = 1; r < 4; ++r) mine_of = (l16 & 3) == r ? (float)columns[r] : mine_of;
                bool all = left.keeps;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    const four bj = from_lane(b[kt], 16 * g + j), aj = puts ? from_lane(a[kt], 16 * g + j) : four{};
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool is = 16 * kt + r < rows;            // (a row that is none times an infinity would be NaN)
                        float s = state[kt][r];
                        if (!w.decayed) s = decayed(s, left);
                        if (is) s = fmaf((float)bj[r], mine_of, s);
                        if (is) sum = fmaf((float)aj[r], s, sum);
                        if (w.decayed) s = decayed(s, left);
                        state[kt][r] = s;
                        all &= !is || column + l16 >= dc || s != s;
                    }
                }
                lost = __builtin_amdgcn_ballot_w64(!all) == 0;
                if (puts) {
                    sum += __shfl_xor(sum, 16);
                    sum += __shfl_xor(sum, 32);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float v = w.scale * __shfl(sum, 4 * g + r);
                        value[r] = l16 == j ? v : value[r];
                    }
                }
                if (lost) break;                   // (the steps behind this one have their NaN)
            }
        }
        if (puts && l16 < here) out(t, value);
    }
}

// ---- the walks ---------------------------------------------------------------------------------------

// One workgroup to a piece of a row and a head.  A wave has sixteen of the state's columns, which no other wave needs; scores are
// shared.  Of 32-bit operands no more than one workgroup of four waves fits beside tiles of 128 x 64.
//
// 64 x 64 of bfloat16, 64 rows of 8,192 tokens, 8 heads: 500 us for 2.15 GB, 4.3 TB/s of the 4.75 that a copy reaches.  128 x 128, 256 rows
// of 1,024 tokens, 4 heads: 340 us for 1.07 GB, bound by the length of a chunk's chain (scores, barrier, two products, state) with
// two waves to a SIMD: matrix instructions busy 0.25, vector 0.40; without the loads it takes 12 % less, without the state's
// products 18 %, with one part of scores and T instead of two 7 %.  (The columns of a head in two workgroups, which each compute all
// scores, took 7 % more.  With 64 x 64, three workgroups to a CU spill registers: 888 us instead of 508.)
// 48 x 40 in 32 bits, 876,000 tokens of long reads, 6 heads: 1,520 us, matrix instructions of 32 bits busy 0.38: the wave with the last
// sixteen steps has four tiles of scores where the first has one, and the fourth has no columns.  (As two float16 each, three products
// instead of one: a training step took 20 % more, with registers spilled.)
template <typename T, int KD, int CD, bool TAIL>
__global__ __launch_bounds__(threads_of(CD), sizeof(T) == 4 && KD > 64 && CD == 64 ? 1 : 2) void walk_kernel(WalkArgs w)
{
    typedef typename Frag<T>::type frag;
    typedef typename Four<T>::type four;
    // (scores: two or one of the waves to sixteen steps, each with half or all of the steps before them)
    constexpr int KT = KD / 16, SP = WalkTiles<T, KD, CD>::kSplits, kThreads = threads_of(CD), kScores = 16 / (CD / 16);
    constexpr int D = Frag<T>::kDepth, KS = KD / D, TS = kChunk / D, kTwo = kTwoChunks<T, KD, CD>;
    constexpr bool scaled = std::is_same<T, _Float16>::value;
    __shared__ WalkTiles<T, KD, CD> lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, l16 = lane & 15;
    const int column = wave * 16, dc = w.c.dim;
    const int head = blockIdx.x % w.heads;
    const int64_t item = w.first_item + blockIdx.x / w.heads;
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
    const float ld = log_decay_of(w.log_decay, head);
    const int late = w.decayed ? 1 : 0;
    const bool reverse = w.reverse;
    const int64_t length = p.hi - p.lo;
    const bool starts = reverse ? p.back : p.front, ends = reverse ? p.front : p.back;
    const int64_t cells = (int64_t)w.b.dim * w.c.dim;

    const int64_t ta = w.a.token * sizeof(T), tb = w.b.token * sizeof(T), tc = w.c.token * sizeof(T);
    const char *pa = base_of(w.a, head, sizeof(T)), *pb = base_of(w.b, head, sizeof(T)), *pc = base_of(w.c, head, sizeof(T));
    const int da = w.a.dim, db = w.b.dim;
    Stage<T, KD, TAIL, kThreads> sa, sb;
    Stage<T, CD, TAIL, kThreads> sc;
    // the chunk that begins `done` steps into the piece: its first token, and how many
    const auto first_of = [&](int64_t done, int n) { return reverse ? p.hi - done - n : p.lo + done; };
    const auto count_of = [&](int64_t done) { return length - done < kChunk ? (int)(length - done) : kChunk; };
    const int row_cells = w.heads * dc;
    const auto fetch = [&](int64_t done) {
        if (done >= length) return;
        const int n = count_of(done);
        const int64_t first = first_of(done, n);
        sa.load(pa + first * ta, ta, da, n);
        sb.load(pb + first * tb, tb, db, n);
        sc.load(pc + first * tc, tc, dc, n);
    };
    const auto keep = [&](int64_t done, Chunk<T, KD, CD> &to) {
        if (done >= length) return;
        const int n = count_of(done);
        sa.store(to.a, reverse, n);
        sb.store(to.b, reverse, n);
        sc.store(to.c, reverse, n);
    };
    fetch(0);

    // what is in front of the piece
    f32x4 state[KT];
    const auto begin = [&](int lane) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) state[kt] = f32x4{0, 0, 0, 0};
        if (starts && !w.start) return;
        const int64_t slot = (reverse ? p.hi : p.lo) / w.cut;
        const float *from = starts ? w.start + (p.row * w.heads + head) * cells : w.slots + ((slot - 1) * w.heads + head) * cells;
        const float scale = starts ? w.start_scale : 1.0f;
        each_cell<KD>(w, column, lane, w.transposed, [&](int kt, int r, int at) { state[kt][r] = scale * from[at]; });
    };
    begin(lane);

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
    const Decays<T> decays = decays_of<T>(ld, late, lane);

    keep(0, lds.chunk[0]);
    fetch(kChunk);
    __syncthreads();
    int turn = 0;
    int64_t odd_from = length;                     // the first chunk of which not all results are finite
    for (int64_t done = 0; done < length; done += kChunk, turn ^= kTwo) {
        const int n = count_of(done);
        const Chunk<T, KD, CD> &chunk = lds.chunk[turn];
        if (n < kChunk) left = left_after(ld, (float)n);

        // scores, transposed: a lane has one step and four earlier ones at a time
        {
            f32x4 score[kScores];
#pragma unroll
            for (int j = 0; j < kScores; ++j) score[j] = f32x4{0, 0, 0, 0};
            if constexpr (sizeof(T) == 2) {
                frag a8[2], b8[2][kScores];
                const auto request = [&](int ks) {
                    a8[ks & 1] = chunk.a.row(16 * score_tile + l16, D * ks, lane);
#pragma unroll
                    for (int j = 0; j < kScores; ++j) b8[ks & 1][j] = chunk.b.row(16 * (first_score + j) + l16, D * ks, lane);
                };
                request(0);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if (ks + 1 < KS) request(ks + 1);
                    in_order();
#pragma unroll
                    for (int j = 0; j < kScores; ++j) score[j] = mma(b8[ks & 1][j], a8[ks & 1], score[j]);
                }
            } else {                               // (products take so long that those that are not needed are left out)
#pragma unroll
                for (int j = 0; j < kScores; ++j) {
                    if (first_score + j > score_tile) break;
                    frag a8[2], b8[2];
                    const auto request = [&](int ks) {
                        a8[ks & 1] = chunk.a.row(16 * score_tile + l16, D * ks, lane);
                        b8[ks & 1] = chunk.b.row(16 * (first_score + j) + l16, D * ks, lane);
                    };
                    request(0);
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        if (ks + 1 < KS) request(ks + 1);
                        in_order();
                        score[j] = mma(b8[ks & 1], a8[ks & 1], score[j]);
                    }
                }
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
                // (in pairs of sixteen: products take up to 32 steps at a time)
                if (first_score + 2 * half <= score_tile) {
#pragma unroll
                    for (int j = 2 * half; j < 2 * half + 2; ++j) {
                        f32x4 v = score[j];
                        if (scaled) v *= size.down;
                        four part[SP];
                        split<T>(v, part);
#pragma unroll
                        for (int q = 0; q < SP; ++q) lds.p[q].put_scores(16 * score_tile + l16, 16 * (first_score + j) + 4 * g, part[q]);
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
        if (kTwo) keep(done + kChunk, lds.chunk[turn ^ 1]);
        __syncthreads();
        if (kTwo) fetch(done + 2 * kChunk);

        if (column < dc) {
            frag c8[TS];
#pragma unroll
            for (int ts = 0; ts < TS; ++ts) c8[ts] = chunk.c.column(D * ts, column, lane);
            // a T in front of the chunk, transposed: a lane has one step and four columns at a time
            f32x4 out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = f32x4{0, 0, 0, 0};
            frag a8[2][4], s8[SP], p8[2][SP][4];
            const auto request = [&](int ks) {
#pragma unroll
                for (int j = 0; j < 4; ++j) a8[ks & 1][j] = chunk.a.row_as_state(16 * j + l16, D * ks, lane);
            };
            // scores with kDepth steps: of those that have any of them behind
            const auto request_scores = [&](int ts) {
#pragma unroll
                for (int q = 0; q < SP; ++q)
#pragma unroll
                    for (int j = ts * D / 16; j < 4; ++j) p8[ts & 1][q][j] = lds.p[q].row(16 * j + l16, D * ts, lane);
            };
            request(0);
            in_order();
            // whether any of the columns' cells is no finite number: 0 times it would reach the steps in front of it, so those are left
            // out, and the steps from theirs on are left to by_steps
            uint32_t odd = 0;
#pragma unroll
            for (int ts = 0; ts < TS; ++ts) odd |= not_finite<T>(c8[ts]);
            const bool any_odd = __builtin_amdgcn_ballot_w64(odd != 0) != 0;
            if (__builtin_expect(any_odd, false)) {
#pragma unroll
                for (int ts = 0; ts < TS; ++ts)
#pragma unroll
                    for (int e = 0; e < Frag<T>::kCount; ++e)
                        if (!is_finite((float)c8[ts][e])) c8[ts][e] = (T)0.0f;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if constexpr (sizeof(T) == 2) {
                    typename Frag<T>::floats v = __builtin_shufflevector(state[2 * ks], state[2 * ks + 1], 0, 1, 2, 3, 4, 5, 6, 7);
                    if (scaled) v *= size.down;
                    split<T>(v, s8);
                } else {
                    s8[0] = state[ks];
                }
                if (ks + 1 < KS) request(ks + 1);
                else request_scores(0);
                in_order();
#pragma unroll
                for (int q = 0; q < SP; ++q)
#pragma unroll
                    for (int j = 0; j < 4; ++j) out[j] = mma(s8[q], a8[ks & 1][j], out[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float by = share[j];
                if constexpr (scaled) by = by * size.up / lds.up[0][16 * j + l16];
                out[j] *= by;
            }
            // the chunk's own steps
#pragma unroll
            for (int ts = 0; ts < TS; ++ts) {
                if (ts + 1 < TS) request_scores(ts + 1);
                in_order();
                if (scaled && ts == 1) {
#pragma unroll
                    for (int j = 2; j < 4; ++j) out[j] *= lds.up[0][16 * j + l16] / lds.up[1][16 * j + l16];
                }
#pragma unroll
                for (int q = 0; q < SP; ++q)
#pragma unroll
                    for (int j = ts * D / 16; j < 4; ++j) out[j] = mma(c8[ts], p8[ts & 1][q][j], out[j]);
            }
            if constexpr (scaled) {
#pragma unroll
                for (int j = 0; j < 4; ++j) out[j] *= lds.up[j / 2][16 * j + l16];
            }
            if (__builtin_expect(any_odd, false)) {
                int from[4] = {kChunk, kChunk, kChunk, kChunk};        // the first step of each column that is left out
                for (int s = kChunk - 1; s >= 0; --s)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!is_finite((float)chunk.c.cell[s * Tile<T, CD>::kPitch + column + 4 * g + r])) from[r] = s;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (16 * j + l16 >= from[r]) out[j][r] = NAN;
#pragma unroll
                for (int ts = 0; ts < TS; ++ts) c8[ts] = chunk.c.column(D * ts, column, lane);
            }
            if (any_not_finite(out) && odd_from > done) odd_from = done;
            const int64_t cell = (first_of(done, n) * w.heads + head) * dc;
            int row[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = 16 * j + l16;
                row[j] = at >= n ? -1 : reverse ? n - 1 - at : at;
            }
            if (w.out32) put<TAIL>((float *)w.out + cell, row_cells, dc, n, column + 4 * g, row, out);
            else put<TAIL>((T *)w.out + cell, row_cells, dc, n, column + 4 * g, row, out);
            add_chunk<T, KD>(state, chunk.b, c8, decays, lds.power, n, late, left, w.exact, lane);
        }
        __syncthreads();
        if (!kTwo) {
            keep(done + kChunk, lds.chunk[0]);
            fetch(done + 2 * kChunk);
            __syncthreads();
        }
    }
    float *end = ends && w.end ? w.end + (p.row * w.heads + head) * cells : nullptr;
    if (end) each_cell<KD>(w, column, lane, false, [&](int kt, int r, int at) { end[at] = w.end_scale * state[kt][r]; });
    if (__builtin_expect(column < dc && length > 0 && (odd_from < length || any_not_finite(state)), false)) {
        const int lane2 = forgotten(lane), g2 = lane2 >> 4;
        begin(lane2);
        // (a lane looks at what it wrote itself)
        by_steps<T, KD, TAIL, true>(w, p, head, ld, column, lane2, state, odd_from, [&](int64_t t, const f32x4 &v) {
            const int64_t at = (t * w.heads + head) * dc + column + 4 * g2;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (column + 4 * g2 + r >= dc) break;
                if (w.out32) {
                    float *place = (float *)w.out + at + r;
                    if (!is_finite(*place)) *place = v[r];
                } else {
                    T *place = (T *)w.out + at + r;
                    if (!is_finite((float)*place)) *place = (T)v[r];
                }
            }
        });
        if (end)
            each_cell<KD>(w, column, lane2, false, [&](int kt, int r, int at) {
                if (!is_finite(end[at])) end[at] = w.end_scale * state[kt][r];
            });
    }
}

// What each piece that does not end its row adds to the state: into the slot of the cut behind it.  One row of 262,147 tokens, 4 heads of
// 128 x 128 of float16: 140 us for 0.54 GB, 30 more for the slots' states, then the walk.
template <typename T, int KD, int CD, bool TAIL>
__global__ __launch_bounds__(threads_of(CD), sizeof(T) == 4 && KD > 64 && CD == 64 ? 1 : sizeof(T) == 4 && KD == 64 ? 3 : 2) void piece_kernel(WalkArgs w)
{
    typedef typename Frag<T>::type frag;
    constexpr int KT = KD / 16, kThreads = threads_of(CD), D = Frag<T>::kDepth, TS = kChunk / D;
    __shared__ PieceTiles<T, KD, CD> lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), column = wave * 16;
    const int head = blockIdx.x % w.heads;
    const Piece p = piece_of(w, w.first_item + blockIdx.x / w.heads);
    if (p.none || (w.reverse ? p.front : p.back)) return;
    const float ld = log_decay_of(w.log_decay, head);
    const int late = w.decayed ? 1 : 0;
    const bool reverse = w.reverse;
    const int64_t length = p.hi - p.lo;
    f32x4 state[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) state[kt] = f32x4{0, 0, 0, 0};
    for (int i = threadIdx.x; i <= kChunk; i += kThreads) lds.power[i] = expf((float)i * ld);
    Left left = left_after(ld, kChunk);
    const Decays<T> decays = decays_of<T>(ld, late, lane);
    const int64_t tb = w.b.token * sizeof(T), tc = w.c.token * sizeof(T);
    const char *pb = base_of(w.b, head, sizeof(T)), *pc = base_of(w.c, head, sizeof(T));
    const int db = w.b.dim, dc = w.c.dim;
    Stage<T, KD, TAIL, kThreads> sb;
    Stage<T, CD, TAIL, kThreads> sc;
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
        if (column < dc) {
            frag c8[TS];
#pragma unroll
            for (int ts = 0; ts < TS; ++ts) c8[ts] = lds.c.column(D * ts, column, lane);
            add_chunk<T, KD>(state, lds.b, c8, decays, lds.power, n, late, left, true, lane);
        }
    }
    const int64_t slot = (reverse ? p.lo : p.hi) / w.cut;
    float *to = w.slots + ((slot - 1) * w.heads + head) * (int64_t)db * dc;
    each_cell<KD>(w, column, lane, false, [&](int kt, int r, int at) { to[at] = state[kt][r]; });
    if (__builtin_expect(column < dc && any_not_finite(state), false)) {
        const int lane2 = forgotten(lane);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) state[kt] = f32x4{0, 0, 0, 0};
        by_steps<T, KD, TAIL, false>(w, p, head, ld, column, lane2, state, 0, [](int64_t, const f32x4 &) {});
        each_cell<KD>(w, column, lane2, false, [&](int kt, int r, int at) {
            if (!is_finite(to[at])) to[at] = state[kt][r];
        });
    }
}

// ---- launches -----------------------------------------------------------------------------------------

// Calls fn with the tiles that hold db x dc, and whether rows end within 16 bytes.  Heads of 32 bits are 32, 48 or 64 deep up to 64 elements
// (a training step on 300 long reads, 6 heads of 48 x 40: 7,290 us, with 64 for 48 8,345); of 65 to 80 and 97 to 112 they pay for
// 96 and 128, as 16-bit ones of 65 to 80 elements pay for 96.
template <typename T, typename Fn> void with_tiles(int32_t db, int32_t dc, Fn fn)
{
    const auto deep = [&](auto kd) {
        const auto wide = [&](auto cd) {
            if (db % Frag<T>::kCount || dc % Frag<T>::kCount) fn(kd, cd, std::true_type{});
            else fn(kd, cd, std::false_type{});
        };
        if (dc <= 64) wide(std::integral_constant<int, 64>{});
        else wide(std::integral_constant<int, 128>{});
    };
    if (db <= 32) deep(std::integral_constant<int, 32>{});
    else if (sizeof(T) == 4 && db <= 48) deep(std::integral_constant<int, sizeof(T) == 4 ? 48 : 32>{});
    else if (db <= 64) deep(std::integral_constant<int, 64>{});
    else if (db <= 96) deep(std::integral_constant<int, 96>{});
    else deep(std::integral_constant<int, 128>{});
}
// Launches of all items, a workgroup to an item and a head: as many to a launch as a grid takes, which has less than 2^32 threads.
template <typename Fn> void in_launches(const WalkArgs &w, int64_t items, Fn fn)
{
    const int64_t most = (1 << 22) / w.heads;
    for (int64_t first = 0; first < items; first += most) {
        WalkArgs part = w;
        part.first_item = first;
        fn(part, (unsigned)((items - first < most ? items - first : most) * w.heads));
    }
}
template <typename T> void launch_pieces(const WalkArgs &w, hipStream_t s)
{
    with_tiles<T>(w.b.dim, w.c.dim, [&](auto kd, auto cd, auto tail) {
        in_launches(w, w.n_rows + w.cuts, [&](const WalkArgs &part, unsigned grid) {
            piece_kernel<T, kd(), cd(), tail()><<<grid, threads_of(cd()), 0, s>>>(part);
        });
    });
}
template <typename T> void launch_walk(const WalkArgs &w, hipStream_t s)
{
    with_tiles<T>(w.b.dim, w.c.dim, [&](auto kd, auto cd, auto tail) {
        in_launches(w, w.n_rows + w.cuts + (w.offsets ? kOutside : 0), [&](const WalkArgs &part, unsigned grid) {
            walk_kernel<T, kd(), cd(), tail()><<<grid, threads_of(cd()), 0, s>>>(part);
        });
    });
}

}  // namespace dnatok
