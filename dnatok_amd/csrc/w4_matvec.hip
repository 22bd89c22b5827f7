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
// x (from the matrix cores as well, with ones for W).  Every product is exact in 32 bits, sums are 32-bit sums.
//
// A workgroup takes TT x 16 rows of W and its eight waves take the columns in slices of KB x 32; a wave holds its slice of
// x in registers for all the rows.  A lane loads four words (32 columns of one row); four lanes then exchange words, so
// that an instruction's 32 columns lie next to each other and in one group.  The waves' sums meet in LDS.
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
    const float *bias;
    void *y;
    int64_t y_stride;
};

// Eight columns of a row of x, in the order in which the weights come out of a word.
template <typename T>
__device__ __forceinline__ typename Frag<T>::type load_x(const W4Args<T> &a, int64_t row, int32_t k)
{
    u32x4 v = {0, 0, 0, 0};
    if (row < a.m && k < a.k) {
        const T *p = a.x + row * a.x_stride + k;
        if (a.x_aligned && k + 8 <= a.k) {
            v = *reinterpret_cast<const u32x4 *>(p);
        } else {
            uint16_t e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = k + i < a.k ? __builtin_bit_cast(uint16_t, p[i]) : (uint16_t)0;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (uint32_t)e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
        }
    }
    u32x4 o;
    o[0] = __builtin_amdgcn_perm(v[2], v[0], 0x05040100);              // columns 0 and 4
    o[1] = __builtin_amdgcn_perm(v[2], v[0], 0x07060302);              // 1 and 5
    o[2] = __builtin_amdgcn_perm(v[3], v[1], 0x05040100);              // 2 and 6
    o[3] = __builtin_amdgcn_perm(v[3], v[1], 0x07060302);              // 3 and 7
    return __builtin_bit_cast(typename Frag<T>::type, o);
}

// The weights of a word: 128 + q, or q - zero (`minus`: -1024 - zero, twice).
template <typename T>
__device__ __forceinline__ typename Frag<T>::type unpack(uint32_t q, uint32_t minus)
{
    constexpr bool half = std::is_same<T, _Float16>::value;
    constexpr uint32_t magic = half ? 0x64006400u : 0x43004300u;
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (q >> (4 * i) & 0x000F000Fu) | magic;
    auto f = __builtin_bit_cast(typename Frag<T>::type, o);
    if constexpr (half) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 z = __builtin_bit_cast(h2, minus);
        f += __builtin_shufflevector(z, z, 0, 1, 0, 1, 0, 1, 0, 1);
    }
    return f;
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

// GB: blocks of a group, if 1, 2 or 4; 1 also for groups of other sizes, whose scale is then looked up for each block.
template <typename T, int KB, int GB>
__device__ __forceinline__ void load_slice(const W4Args<T> &a, int64_t row, int32_t b0, int kq, Slice<KB, KB / GB> &s)
{
    constexpr int SEGS = KB / GB;
    const uint32_t *w = a.w + row * a.w_stride;
    const bool whole = (b0 + KB) * 4 <= a.words;
#pragma unroll
    for (int h = 0; h < KB / 4; ++h) {
        const int32_t at = b0 * 4 + h * 16 + kq * 4;
        if (whole) {
            __builtin_memcpy(&s.q[h], w + at, 16);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) s.q[h][j] = at + j < a.words ? w[at + j] : 0;
        }
    }
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

template <typename T, typename OUT, int MT, int KB, int TT, int GB>
__global__ __launch_bounds__(64 * kW4Waves) void w4_kernel(W4Args<T> a)
{
    constexpr bool half = std::is_same<T, _Float16>::value;
    constexpr int SEGS = KB / GB;
    typedef typename Frag<T>::type frag;
    __shared__ f32x4 sums[kW4Waves][MT][64];
    __shared__ f32x4 x_sums[half ? 1 : kW4Waves][SEGS][MT][4];         // of the slice's segments, four rows of x to an entry
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, kq = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * TT), m0 = (int64_t)blockIdx.y * (16 * MT);
    const f32x4 zero4 = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 acc[TT][MT];
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[t][i] = zero4;

    const auto row_of = [&](int t) {
        const int64_t row = n0 + t * 16 + r;
        return row < a.n ? row : a.n - 1;
    };
    for (int32_t b0 = wave * KB; b0 < a.blocks; b0 += kW4Waves * KB) {
        Slice<KB, SEGS> next;
        load_slice<T, KB, GB>(a, row_of(0), b0, kq, next);
        frag x[KB][MT];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < MT; ++i) x[b][i] = load_x<T>(a, m0 + i * 16 + r, (b0 + b) * 32 + kq * 8);
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
            Slice<KB, SEGS> s = next;
            if (t + 1 < TT) load_slice<T, KB, GB>(a, row_of(t + 1), b0, kq, next);
            f32x4 c[MT];
#pragma unroll
            for (int h = 0; h < KB / 4; ++h) {
                const u32x4 q = exchange(s.q[h]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int b = h * 4 + j, seg = b / GB;
                    if (b0 + seg * GB >= a.blocks) break;              // (uniform: nothing but padding from here on)
                    uint32_t minus = 0;
                    if constexpr (half) {
                        minus = 0xE400u + s.zero[seg];                 // -1024 - zero
                        minus |= minus << 16;
                    }
                    const frag w = unpack<T>(q[j], minus);
#pragma unroll
                    for (int i = 0; i < MT; ++i) c[i] = mfma(x[b][i], w, b % GB == 0 ? zero4 : c[i]);
                    if ((b + 1) % GB == 0) {
                        const float scale = to_float(__builtin_bit_cast(T, s.scale[seg]));
                        const float off = -128.0f - (float)s.zero[seg];
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            if constexpr (!half) {
                                const f32x4 sum = x_sums[wave][seg][i][kq];
#pragma unroll
                                for (int e = 0; e < 4; ++e) c[i][e] = fmaf(off, sum[e], c[i][e]);
                            }
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[t][i][e] = fmaf(scale, c[i][e], acc[t][i][e]);
                        }
                    }
                }
            }
        }
        if constexpr (!half) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }

#pragma unroll
    for (int t = 0; t < TT; ++t) {
        if (t) __syncthreads();
#pragma unroll
        for (int i = 0; i < MT; ++i) sums[wave][i][lane] = acc[t][i];
        __syncthreads();
        for (int o = threadIdx.x; o < MT * 256; o += 64 * kW4Waves) {
            const int i = o >> 8, col = o & 15, in = o >> 4 & 15;      // 16 rows of W next to each other, then rows of x
            const int64_t n = n0 + t * 16 + col, m = m0 + i * 16 + in;
            if (n < a.n && m < a.m) {
                const int from = (in >> 2) * 16 + col;
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kW4Waves; ++w) sum += sums[w][i][from][in & 3];
                ((OUT *)a.y)[m * a.y_stride + n] = from_float<OUT>(sum + (a.bias ? a.bias[n] : 0.0f));
            }
        }
    }
}

}  // namespace dnatok

using namespace dnatok;

namespace {

template <typename T, typename OUT, int MT, int KB, int TT>
void launch_w4(const W4Args<T> &a, hipStream_t s)
{
    const dim3 grid((unsigned)((a.n + 16 * TT - 1) / (16 * TT)), (unsigned)((a.m + 16 * MT - 1) / (16 * MT)));
    if (a.per_group == 4) w4_kernel<T, OUT, MT, KB, TT, 4><<<grid, 64 * kW4Waves, 0, s>>>(a);
    else if (a.per_group == 2) w4_kernel<T, OUT, MT, KB, TT, 2><<<grid, 64 * kW4Waves, 0, s>>>(a);
    else w4_kernel<T, OUT, MT, KB, TT, 1><<<grid, 64 * kW4Waves, 0, s>>>(a);
}

// Sixteen-row tiles to a workgroup: as many as leave two workgroups for each of the 256 CUs.
template <typename T, typename OUT, int MT, int KB>
void launch_w4_rows(const W4Args<T> &a, hipStream_t s)
{
    const int64_t groups = (a.n + 15) / 16 * ((a.m + 16 * MT - 1) / (16 * MT));
    if (groups >= 2048) launch_w4<T, OUT, MT, KB, 4>(a, s);
    else if (groups >= 1024) launch_w4<T, OUT, MT, KB, 2>(a, s);
    else launch_w4<T, OUT, MT, KB, 1>(a, s);
}

template <typename T, typename OUT>
void run_w4(const W4Args<T> &a, hipStream_t s)
{
    if (a.m > 32) launch_w4_rows<T, OUT, 4, 4>(a, s);
    else if (a.m > 16) launch_w4_rows<T, OUT, 2, 4>(a, s);
    else if (a.k <= 32 * 4 * kW4Waves) launch_w4_rows<T, OUT, 1, 4>(a, s);
    else launch_w4_rows<T, OUT, 1, 8>(a, s);
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
    DNATOK_REQUIRE(n < (1ll << 31) && m <= 65535 && k < (1ll << 30), DNATOK_E_TOO_LARGE,
                   "%s: at most 2^31 outputs of 65535 rows, 2^30 columns", who);
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
            a.bias = bias, a.y = y, a.y_stride = y_stride;
            if (y_dtype == DNATOK_F32) run_w4<T, float>(a, s);
            else run_w4<T, T>(a, s);
        }
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
