// y = x W^T + bias for few rows of x, where W[n, k] = (q[n, k] - zero[n, g]) scale[n, g] holds whole numbers q of 4 bits
// and g = k / group.  Eight of them lie in a 32-bit word, the lowest bits first.
//
// What has to move is the weights, half a byte each, so the product is bound by memory as long as a weight costs
// few instructions.  It goes through the matrix cores for any number of rows: D = X W^T with 16 rows of x by 16 rows of W by
// 32 columns to an instruction, so that a weight is unpacked once for 16 rows of x (and for one row as fast as for 16),
// and a lane's part of D has one row of W, so that its scales and zero points are one number a group.
//
// Unpacking: bits 4i and 4i + 16 of a word, masked out together and put into the low bits of the mantissa of two
// 16-bit numbers, give 128 + q (bfloat16) or 1024 + q (float16): 7 instructions for 8 weights.  The pairs are columns
// i and i + 4; the columns of x are put into the same order once.  float16 takes 1024 + zero off again, exactly; bfloat16 has no
// packed subtraction, there the sum over a group of (128 + q) x is corrected by (128 + zero) times the sum of
// x (from the matrix cores as well, with ones for W).  Every product is exact in 32 bits, sums are 32-bit sums; those of
// bfloat16 hold numbers some ten times as large as what the correction leaves, so their rounding weighs as much more: 6e-7 of the
// result at 4096 x 1024 instead of 6e-8, seen where the result has 32 bits.  Sums that are not finite are done again with q - zero.
//
// A workgroup takes TT x 16 rows of W and its eight waves take the columns in slices of KB x 32.  A lane loads four words (32
// columns of one row); four lanes then exchange words, so that an instruction's 32 columns lie next to each other and
// in one group.  The waves' sums meet in LDS.  A wave holds its slice of x in registers (w4_kernel); a single row of x lies in
// LDS, ready to be multiplied (w4_row_kernel).
//
// Measured, us a call: one row, 32000 x 4096 bfloat16 in groups of 64 18.6 (3.77 TB/s; a copy 4.76); 16 rows, 8192 x 8192
// float16 in groups of 32 16.2 (2.5 TB/s); 61 rows, 12301 x 2040 15.4; one row, 4096 x 1024
// 3.9 in the kernel and 8.9 with the host.
#include "lm_common.hpp"

namespace dnatok {

constexpr int kW4Waves = 8;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Frag { typedef T type __attribute__((ext_vector_type(8))); };

__device__ __forceinline__ f32x4 mfma(Frag<__bf16>::type a, Frag<__bf16>::type b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(Frag<_Float16>::type a, Frag<_Float16>::type b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template <typename T>
struct W4Args {
    const T *x;
    int64_t x_stride;
    const uint32_t *w;
    int64_t w_stride;
    const T *scales;
    const uint8_t *zeros;
    int64_t m, n;
    int32_t k, blocks, words, per_group, n_groups;     // columns; 32 of them; words of a row; blocks of a group
    bool x_aligned;                                    // rows of x begin on multiples of 16 bytes
    bool x_in_lines;                                   // and all at the same place of a 128-byte line
    const float *bias;
    void *y;
    int64_t y_stride;
};

// Eight columns of a row of x in the order in which the weights come out of a word.
__device__ __forceinline__ u32x4 in_order(u32x4 v)
{
    u32x4 o;
    o[0] = __builtin_amdgcn_perm(v[2], v[0], 0x05040100);              // columns 0 and 4
    o[1] = __builtin_amdgcn_perm(v[2], v[0], 0x07060302);              // 1 and 5
    o[2] = __builtin_amdgcn_perm(v[3], v[1], 0x05040100);              // 2 and 6
    o[3] = __builtin_amdgcn_perm(v[3], v[1], 0x07060302);              // 3 and 7
    return o;
}
// Columns k .. k + 7 of a row, zeros behind the last one.
template <typename T>
__device__ __forceinline__ u32x4 load_x(const W4Args<T> &a, const T *row, int32_t k)
{
    u32x4 v = {0, 0, 0, 0};
    if (a.x_aligned && k + 8 <= a.k) {
        v = *reinterpret_cast<const u32x4 *>(row + k);
    } else {
        uint16_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = k + i < a.k ? __builtin_bit_cast(uint16_t, row[k + i]) : (uint16_t)0;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (uint32_t)e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
    }
    return v;
}

// The weights of a word: 128 + q, or q - zero (`minus`: -1024 - zero, twice).
template <typename T>
__device__ __forceinline__ typename Frag<T>::type unpack(uint32_t q, uint32_t minus)
{
    constexpr bool half = std::is_same<T, _Float16>::value;
    constexpr uint32_t magic = half ? 0x64006400u : 0x43004300u;
    // (constants in registers: an instruction takes one literal, and `and` with `or` would be two)
    uint32_t low = 0x000F000Fu, high = magic;
    asm("" : "+s"(low));
    asm("" : "+v"(high));
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (q >> (4 * i) & low) | high;
    auto f = __builtin_bit_cast(typename Frag<T>::type, o);
    if constexpr (half) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 z = __builtin_bit_cast(h2, minus);
        f += __builtin_shufflevector(z, z, 0, 1, 0, 1, 0, 1, 0, 1);
    }
    return f;
}

// The same for bfloat16 as q - zero, exactly, by way of 32 bits: three times the instructions.
__device__ __forceinline__ Frag<__bf16>::type unpack_exact(uint32_t q, float zero)
{
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {                                      // (whole numbers below 2^8: the low halves are zeros)
        const uint32_t low = __float_as_uint((float)(q >> (4 * i) & 15) - zero);
        const uint32_t high = __float_as_uint((float)(q >> (4 * i + 16) & 15) - zero);
        o[i] = __builtin_amdgcn_perm(high, low, 0x07060302);
    }
    return __builtin_bit_cast(Frag<__bf16>::type, o);
}

// Words j of four lanes sixteen apart, which hold blocks 0 .. 3 of the columns: to word j of block i in register i of
// lane j.
__device__ __forceinline__ u32x4 exchange(u32x4 q)
{
    auto a = __builtin_amdgcn_permlane32_swap(q[0], q[2], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(q[1], q[3], false, false);
    auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u32x4{c[0], c[1], d[0], d[1]};
}

// A tile's words, scales and zero points of one slice, as a lane holds them.
template <int KB, int SEGS>
struct Slice {
    u32x4 q[KB / 4];
    uint16_t scale[SEGS];
    uint8_t zero[SEGS];
};

// A workgroup's rows of weights: a buffer resource that ends with the matrix (rows and words behind the last one read as
// zeros; words behind a row's last one are the next row's, and multiplied by zeros of x).
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_from(const W4Args<T> &a, int64_t n0)
{
    const int64_t bytes = ((a.n - n0 - 1) * a.w_stride + a.words) * 4;
    return __builtin_amdgcn_make_buffer_rsrc((void *)(a.w + n0 * a.w_stride), 0, (int)(bytes < 0x7FFFFFFF ? bytes : 0x7FFFFFFF),
                                             0x00020000);
}

// Row n0 + local, slice from block b0 on.  GB: blocks with one scale, 1, 2 or 4; groups may be larger.
template <typename T, int KB, int GB>
__device__ __forceinline__ void load_slice(const W4Args<T> &a, __amdgpu_buffer_rsrc_t rows, int64_t n0, int local, int32_t b0,
                                           int kq, Slice<KB, KB / GB> &s)
{
    constexpr int SEGS = KB / GB;
    const int lane_bytes = local * (int)a.w_stride * 4 + kq * 16;      // (a workgroup's rows are less than 2^31 bytes)
#pragma unroll
    for (int h = 0; h < KB / 4; ++h) s.q[h] = __builtin_amdgcn_raw_buffer_load_b128(rows, lane_bytes + h * 64, b0 * 16, 0);
    const int64_t row = n0 + local < a.n ? n0 + local : a.n - 1;
    const T *scales = a.scales + row * a.n_groups;
    const uint8_t *zeros = a.zeros + row * a.n_groups;
    if (a.per_group == GB && b0 / GB + SEGS <= a.n_groups) {
        __builtin_memcpy(s.scale, scales + b0 / GB, 2 * SEGS);
        if (a.zeros) __builtin_memcpy(s.zero, zeros + b0 / GB, SEGS);
    } else {
#pragma unroll
        for (int i = 0; i < SEGS; ++i) {
            const int32_t g = (b0 + i * GB) / a.per_group, at = g < a.n_groups ? g : a.n_groups - 1;
            s.scale[i] = __builtin_bit_cast(uint16_t, scales[at]);
            if (a.zeros) s.zero[i] = zeros[at];
        }
    }
    if (!a.zeros)
#pragma unroll
        for (int i = 0; i < SEGS; ++i) s.zero[i] = 8;
}

// acc += x times a slice of a tile, blocks b0 .. of which a.blocks bounds the last.  x(b, i): columns of block b of the
// slice, i-th sixteen rows; sum(seg, i): their sum over a segment, where the type needs it.  EXACT: with q - zero in bfloat16 too.
template <typename T, int MT, int KB, int GB, bool EXACT, typename X, typename Sum>
__device__ __forceinline__ void multiply(const W4Args<T> &a, const Slice<KB, KB / GB> &s, int32_t b0, X x, Sum sum,
                                         f32x4 (&acc)[MT])
{
    constexpr bool half = std::is_same<T, _Float16>::value;
    const f32x4 zero4 = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 c[MT];
#pragma unroll
    for (int h = 0; h < KB / 4; ++h) {
        const u32x4 q = exchange(s.q[h]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int b = h * 4 + j, seg = b / GB;
            if (b0 + seg * GB >= a.blocks) break;                      // (uniform: nothing but padding from here on)
            uint32_t minus = 0;
            if constexpr (half) {
                minus = 0xE400u + s.zero[seg];                         // -1024 - zero
                minus |= minus << 16;
            }
            typename Frag<T>::type w;
            if constexpr (EXACT && !half) w = unpack_exact(q[j], (float)s.zero[seg]);
            else w = unpack<T>(q[j], minus);
#pragma unroll
            for (int i = 0; i < MT; ++i) c[i] = mfma(x(b, i), w, b % GB == 0 ? zero4 : c[i]);
            if ((b + 1) % GB == 0) {
                const float scale = to_float(__builtin_bit_cast(T, s.scale[seg]));
                const float off = -128.0f - (float)s.zero[seg];
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    if constexpr (!half && !EXACT) {
                        const f32x4 xs = sum(seg, i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[i][e] = fmaf(off, xs[e], c[i][e]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][e] = fmaf(scale, c[i][e], acc[i][e]);
                }
            }
        }
    }
}

// bfloat16: (128 + q) x and the sum of x are infinities, and their difference no number, where x holds one or is so large that
// 2^8 times it passes the largest number.  A wave whose sums are not all finite therefore does its slices once more with q - zero,
// and takes those for the sums that are not: an infinity where the formula has one, and no other row is touched.  The first
// pass pays one comparison at its end for that.
__device__ __forceinline__ bool all_finite(f32x4 acc)
{
    bool ok = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) ok = ok && __builtin_isfinite(acc[e]);
    return __all(ok);
}
__device__ __forceinline__ void take_where_not_finite(f32x4 &acc, f32x4 exact)
{
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = __builtin_isfinite(acc[e]) ? acc[e] : exact[e];
}

// The waves' sums meet, RT tiles of sixteen rows of W at a time, and go to y.  `sums`: [kW4Waves][RT][MT][64].
template <typename T, typename OUT, int MT, int TT, int RT>
__device__ __forceinline__ void write_out(const W4Args<T> &a, f32x4 *sums, const f32x4 (&acc)[TT][MT], int64_t n0, int64_t m0,
                                          int wave, int lane)
{
    constexpr int kThreads = 64 * kW4Waves, kOuts = RT * MT * 256, kEach = (kOuts + kThreads - 1) / kThreads;
#pragma unroll
    for (int t0 = 0; t0 < TT; t0 += RT) {
        float bias[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {                              // (on its way while the sums are put down)
            const int64_t n = n0 + (t0 + (e * kThreads + threadIdx.x) / (MT * 256)) * 16 + threadIdx.x % 16;
            bias[e] = a.bias ? a.bias[n < a.n ? n : a.n - 1] : 0.0f;
        }
        if (t0) __syncthreads();
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int i = 0; i < MT; ++i) sums[((wave * RT + t) * MT + i) * 64 + lane] = acc[t0 + t][i];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int o = e * kThreads + threadIdx.x;
            if (kOuts % kThreads && o >= kOuts) break;
            const int t = o / (MT * 256), i = o / 256 % MT, col = o % 16, in = o / 16 % 16;     // 16 rows of W next to each other
            const int64_t n = n0 + (t0 + t) * 16 + col, m = m0 + i * 16 + in;
            if (n < a.n && m < a.m) {
                const float *from = reinterpret_cast<const float *>(sums + (t * MT + i) * 64 + in / 4 * 16 + col) + in % 4;
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kW4Waves; ++w) sum += from[w * RT * MT * 256];
                ((OUT *)a.y)[m * a.y_stride + n] = from_float<OUT>(sum + bias[e]);
            }
        }
    }
}

// One row of x, in LDS; all sixteen rows of an instruction hold it.  A workgroup takes one tile; its waves request their first
// two slices of weights before they look at x, and stay two slices ahead.
template <typename T, typename OUT, int KB, int GB>
__global__ __launch_bounds__(64 * kW4Waves) void w4_row_kernel(W4Args<T> a)
{
    constexpr bool half = std::is_same<T, _Float16>::value;
    constexpr int SEGS = KB / GB, kThreads = 64 * kW4Waves, kStep = kW4Waves * KB;
    typedef typename Frag<T>::type frag;
    __shared__ float sums[kW4Waves][16];
    extern __shared__ __align__(16) uint8_t dynamic[];
    const int32_t units = (a.blocks + KB - 1) / KB * KB * 4;           // of eight columns
    u32x4 *const xs = reinterpret_cast<u32x4 *>(dynamic);              // [units]
    float *const unit_sums = reinterpret_cast<float *>(xs + units);    // [units]
    float *const seg_sums = unit_sums + units;                         // [units / 4 / GB]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, kq = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const __amdgpu_buffer_rsrc_t rows = rows_from(a, n0);
    int32_t b0 = wave * KB;
    Slice<KB, SEGS> even, odd;
    const auto load = [&](Slice<KB, SEGS> &s, int32_t at) {
        if (at < a.blocks) load_slice<T, KB, GB>(a, rows, n0, r, at, kq, s);
    };
    load(even, b0);
    load(odd, b0 + kStep);
    const int64_t n = n0 + r;
    const float bias = a.bias && n < a.n ? a.bias[n] : 0.0f;

    for (int32_t unit = threadIdx.x; unit < units; unit += kThreads) {
        const u32x4 v = load_x<T>(a, a.x, unit * 8);
        xs[unit] = in_order(v);
        if constexpr (!half) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += __uint_as_float(v[i] << 16) + __uint_as_float(v[i] & 0xFFFF0000u);
            unit_sums[unit] = sum;
        }
    }
    __syncthreads();
    if constexpr (!half) {
        for (int32_t o = threadIdx.x; o < units / 4 / GB; o += kThreads) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4 * GB; ++i) sum += unit_sums[o * 4 * GB + i];
            seg_sums[o] = sum;
        }
        __syncthreads();
    }
    f32x4 acc[1] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
    const auto use = [&](const Slice<KB, SEGS> &s, int32_t at, f32x4 (&to)[1], auto exact) {
        const u32x4 *const mine = xs + at * 4 + kq;
        const float *const seg = seg_sums + at / GB;
        multiply<T, 1, KB, GB, exact.value>(a, s, at, [&](int b, int) { return __builtin_bit_cast(frag, mine[b * 4]); },
                                            [&](int i, int) {
                                                const float v = seg[i];
                                                return f32x4{v, v, v, v};
                                            },
                                            to);
    };
    for (; b0 < a.blocks; b0 += 2 * kStep) {
        use(even, b0, acc, std::false_type{});
        load(even, b0 + 2 * kStep);
        if (b0 + kStep >= a.blocks) break;
        use(odd, b0 + kStep, acc, std::false_type{});
        load(odd, b0 + 3 * kStep);
    }
    if constexpr (!half) {
        if (!all_finite(acc[0])) {
            f32x4 exact[1] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
            for (int32_t at = wave * KB; at < a.blocks; at += kStep) {
                load(even, at);
                use(even, at, exact, std::true_type{});
            }
            take_where_not_finite(acc[0], exact[0]);
        }
    }
    if (lane < 16) sums[wave][r] = acc[0][0];
    __syncthreads();
    if (threadIdx.x < 16 && n < a.n) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kW4Waves; ++w) sum += sums[w][threadIdx.x];
        ((OUT *)a.y)[n] = from_float<OUT>(sum + bias);
    }
}

// LINES: rows of x begin at the same place of their lines.  Then the sixteen rows that a load takes 16 bytes of meet in one
// part of the cache's lines, so odd rows fetch the other half of the line, and two loads' results are exchanged.  us without,
// with: 64 x 32000 x 2048 43.5, 38.0; 64 x 8192 x 8192 46.3, 40.1; 16 x 8192 x 8192 20.2, 19.5; 8 x 8192 x 4096 10.1, 9.6.
// Rows at other strides spread by themselves, there it loses: 61 x 12301 x 2040 16.8, 18.7; 16 x 8192 x 4128 15.3, 17.3.  (bfloat16,
// 64 rows, groups of 128 and more: six registers in scratch memory with it, and still 61 x 12301 x 2048 18.9, 17.1.)
template <typename T, typename OUT, int MT, int KB, int TT, int GB, bool LINES>
__global__ __launch_bounds__(64 * kW4Waves) void w4_kernel(W4Args<T> a)
{
    constexpr bool half = std::is_same<T, _Float16>::value;
    constexpr int SEGS = KB / GB;
    typedef typename Frag<T>::type frag;
    // (64 KB at most.  The 16 tiles by 4 at a time instead of 8: 61 x 12301 x 2040 16.7, 16.4 us; 64 x 32000 x 2048 44.4, 43.4; all at
    // once 16.3, 43.2, but 128 KB)
    constexpr int RT = TT * MT <= 8 ? TT : TT / 2;
    __shared__ f32x4 sums[kW4Waves * RT * MT * 64];
    __shared__ f32x4 x_sums[half ? 1 : kW4Waves][SEGS][MT][4];         // of the slice's segments, four rows of x to an entry
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, kq = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * TT), m0 = (int64_t)blockIdx.y * (16 * MT);
    const __amdgpu_buffer_rsrc_t rows = rows_from(a, n0);
    const f32x4 zero4 = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 acc[TT][MT];
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[t][i] = zero4;
    const int odd = LINES ? (r & 1) * 32 : 0;
    const T *x_row[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = m0 + i * 16 + r;
        x_row[i] = a.x + (m < a.m ? m : a.m - 1) * a.x_stride + kq * 8;
    }

    for (int32_t b0 = wave * KB; b0 < a.blocks; b0 += kW4Waves * KB) {
        Slice<KB, SEGS> next;
        load_slice<T, KB, GB>(a, rows, n0, r, b0, kq, next);
        u32x4 raw[KB][MT];
        if (a.x_aligned && (b0 + KB) * 32 <= a.k) {
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    raw[b][i] = *reinterpret_cast<const u32x4 *>(x_row[i] + (b0 + b) * 32 + (b % 2 ? -odd : odd));
            if constexpr (LINES) {
#pragma unroll
                for (int b = 0; b < KB; b += 2)
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t one = raw[b][i][e], two = raw[b + 1][i][e];
                            raw[b][i][e] = odd ? two : one;
                            raw[b + 1][i][e] = odd ? one : two;
                        }
            }
        } else {
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int i = 0; i < MT; ++i) raw[b][i] = load_x<T>(a, x_row[i] - kq * 8, (b0 + b) * 32 + kq * 8);
        }
        frag x[KB][MT];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < MT; ++i) x[b][i] = __builtin_bit_cast(frag, in_order(raw[b][i]));
        if constexpr (!half) {
            frag ones;
#pragma unroll
            for (int i = 0; i < 8; ++i) ones[i] = (T)1.0f;
#pragma unroll
            for (int s = 0; s < SEGS; ++s)
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    f32x4 c = zero4;
#pragma unroll
                    for (int b = 0; b < GB; ++b) c = mfma(x[s * GB + b][i], ones, c);
                    if (r == 0) x_sums[wave][s][i][kq] = c;
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const Slice<KB, SEGS> s = next;
            if (t + 1 < TT) load_slice<T, KB, GB>(a, rows, n0, (t + 1) * 16 + r, b0, kq, next);
            multiply<T, MT, KB, GB, false>(a, s, b0, [&](int b, int i) { return x[b][i]; },
                                           [&](int seg, int i) { return x_sums[wave][seg][i][kq]; }, acc[t]);
        }
        if constexpr (!half) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if constexpr (!half) {
        float none = 0.0f;                                             // (0 times a sum that is not finite is NaN)
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) none = fmaf(acc[t][i][e], 0.0f, none);
        if (!__all(none == 0.0f)) {
            // sixteen rows of x at a time, and their addresses again, which the loop above would otherwise keep in registers
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    if (all_finite(acc[t][i])) continue;
                    int row = threadIdx.x & 15, part = threadIdx.x >> 4 & 3;
                    asm volatile("" : "+v"(row), "+v"(part));
                    const int64_t m = m0 + i * 16 + row;
                    const T *const from = a.x + (m < a.m ? m : a.m - 1) * a.x_stride;
                    f32x4 exact[1] = {zero4};
                    for (int32_t b0 = wave * KB; b0 < a.blocks; b0 += kW4Waves * KB) {
                        Slice<KB, SEGS> s;
                        load_slice<T, KB, GB>(a, rows, n0, t * 16 + row, b0, part, s);
                        multiply<T, 1, KB, GB, true>(
                            a, s, b0,
                            [&](int b, int) {
                                return __builtin_bit_cast(frag, in_order(load_x<T>(a, from, (b0 + b) * 32 + part * 8)));
                            },
                            [&](int, int) { return zero4; }, exact);
                    }
                    take_where_not_finite(acc[t][i], exact[0]);
                }
        }
    }
    write_out<T, OUT, MT, TT, RT>(a, sums, acc, n0, m0, wave, lane);
}

}  // namespace dnatok

using namespace dnatok;

namespace {

template <typename T, typename OUT, int MT, int KB, int TT, bool LINES>
void launch_w4_x(const W4Args<T> &a, hipStream_t s)
{
    const dim3 grid((unsigned)((a.n + 16 * TT - 1) / (16 * TT)), (unsigned)((a.m + 16 * MT - 1) / (16 * MT)));
    if (a.per_group % 4 == 0) w4_kernel<T, OUT, MT, KB, TT, 4, LINES><<<grid, 64 * kW4Waves, 0, s>>>(a);
    else if (a.per_group % 2 == 0) w4_kernel<T, OUT, MT, KB, TT, 2, LINES><<<grid, 64 * kW4Waves, 0, s>>>(a);
    else w4_kernel<T, OUT, MT, KB, TT, 1, LINES><<<grid, 64 * kW4Waves, 0, s>>>(a);
}

template <typename T, typename OUT, int MT, int KB, int TT>
void launch_w4(const W4Args<T> &a, hipStream_t s)
{
    if (a.x_in_lines) launch_w4_x<T, OUT, MT, KB, TT, true>(a, s);
    else launch_w4_x<T, OUT, MT, KB, TT, false>(a, s);
}

// Tiles to a workgroup, so that x is fetched less often: as many as leave about a workgroup for each of the 256 CUs.  us for
// 1, 2, 4 tiles: 8 x 4096 x 4096 8.1, 10.4, 15; 8 x 8192 x 4096 11.3, 9.6, -; 32 x 8192 x 4096 (1,024 tiles) -, 17.6, 15.4.
template <typename T, typename OUT, int KB>
void launch_w4_tiles(const W4Args<T> &a, hipStream_t s)
{
    const int64_t tiles = (a.n + 15) / 16 * ((a.m + 15) / 16);
    if (tiles >= 900) launch_w4<T, OUT, 1, KB, 4>(a, s);
    else if (tiles >= 450) launch_w4<T, OUT, 1, KB, 2>(a, s);
    else launch_w4<T, OUT, 1, KB, 1>(a, s);
}

// Bytes of LDS that one row of x takes, and the most that is given to it: three workgroups on a CU, with their registers.
constexpr int64_t kRowLds = 48 * 1024;
template <typename T>
int64_t row_lds(const W4Args<T> &a)
{
    return (a.blocks + 7) / 8 * 32 * (std::is_same<T, _Float16>::value ? 16 : 16 + 4 + 1);
}

template <typename T, typename OUT>
void run_w4(const W4Args<T> &a, hipStream_t s)
{
    if (a.m == 1 && row_lds(a) <= kRowLds) {
        const unsigned grid = (unsigned)((a.n + 15) / 16), lds = (unsigned)row_lds(a);
        if (a.per_group % 4 == 0) w4_row_kernel<T, OUT, 8, 4><<<grid, 64 * kW4Waves, lds, s>>>(a);
        else if (a.per_group % 2 == 0) w4_row_kernel<T, OUT, 8, 2><<<grid, 64 * kW4Waves, lds, s>>>(a);
        else w4_row_kernel<T, OUT, 8, 1><<<grid, 64 * kW4Waves, lds, s>>>(a);
    } else if (a.m > 32 && (a.n + 63) / 64 * ((a.m + 15) / 16) > 512) {
        // weights unpacked once for 64 rows, where blocks of 16 rows are more workgroups than run at once, two on each of the 256 CUs.
        // us in blocks of 16 rows and of 64, bfloat16 in groups of 128: with one round of the former 33 x 10240 x 2048 11.8, 13.9;
        // 48 x 10240 x 8192 40.6, 43.2; 64 x 8192 x 1024 7.4, 9.7; 64 x 8192 x 8192 40.3, 43.4; with more 33 x 12301 x 1024 10.8,
        // 9.7; 48 x 12301 x 4096 34.9, 24.1; 64 x 10240 x 512 7.3, 7.4; 64 x 10240 x 2048 16.9, 15.0; 64 x 16384 x 8192 76, 49.
        // The depth decides nothing but at its ends: 33 x 32000 x 512 12.7, 14.1.  (Rows of x that begin off a multiple of 16
        // bytes are read number by number, 64 of them as well: 33 x 12301 x 5500 73, 91, but 64 x 12301 x 5500 135, 128.)
        launch_w4<T, OUT, 4, 4, 4>(a, s);
    } else if (a.k > 1024) {
        launch_w4_tiles<T, OUT, 8>(a, s);
    } else {
        launch_w4_tiles<T, OUT, 4>(a, s);                              // (a slice to a wave at most)
    }
}

}  // namespace

extern "C" int dnatok_w4_matvec(const void *x, int64_t x_stride, int32_t dtype, const uint32_t *weights,
                                int64_t weight_stride, const void *scales, const uint8_t *zeros, int64_t m, int64_t n,
                                int64_t k, int32_t group, const float *bias, void *y, int64_t y_stride, int32_t y_dtype,
                                void *stream)
{
    static const char *who = "dnatok_w4_matvec";
#define W4_REQUIRE(cond, text) DNATOK_REQUIRE(cond, DNATOK_E_INVALID, "%s: " text, who)
    W4_REQUIRE(dtype == DNATOK_BF16 || dtype == DNATOK_F16, "x and scales must be bfloat16 or float16");
    W4_REQUIRE(y_dtype == dtype || y_dtype == DNATOK_F32, "y must have x's type or be float32");
    W4_REQUIRE(m >= 0 && n >= 0 && k > 0, "bad size");
    W4_REQUIRE(group > 0 && group % 32 == 0, "group must be a multiple of 32");
    W4_REQUIRE(weight_stride >= (k + 7) / 8, "weight rows overlap");
    if (m == 0 || n == 0) return DNATOK_OK;
    W4_REQUIRE(x && weights && scales && y, "null buffer");
    W4_REQUIRE(x_stride >= 0 && y_stride >= 0, "negative stride");
    DNATOK_REQUIRE(n < (1ll << 31) && m <= 65535 && weight_stride < (1ll << 22), DNATOK_E_TOO_LARGE,
                   "%s: at most 2^31 outputs of 65535 rows, 2^22 words between rows of weights", who);
    hipStream_t s = (hipStream_t)stream;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if constexpr (sizeof(T) == 2) {
            W4Args<T> a{};
            a.x = (const T *)x, a.x_stride = x_stride, a.w = weights, a.w_stride = weight_stride;
            a.scales = (const T *)scales, a.zeros = zeros, a.m = m, a.n = n, a.k = (int32_t)k;
            a.blocks = (int32_t)((k + 31) / 32), a.words = (int32_t)((k + 7) / 8);
            a.per_group = group / 32, a.n_groups = (int32_t)((k + group - 1) / group);
            a.x_aligned = ((uintptr_t)x & 15) == 0 && x_stride % 8 == 0;
            a.x_in_lines = a.x_aligned && x_stride % 64 == 0;
            a.bias = bias, a.y = y, a.y_stride = y_stride;
            if (y_dtype == DNATOK_F32) run_w4<T, float>(a, s);
            else run_w4<T, T>(a, s);
        }
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
