// One step of a beam search: the `width` best of score + log softmax(logits) over a group's beams and the vocabulary, and rows of
// state in the order of the beams that they belong to.
//
// A beam's candidates are in the order of their logits (a softmax does not change it), so each row of logits gives its
// `width` largest, ties to the lowest token, and the logarithm of its sum of exponentials; a group's beams are then
// merged by score + (logit - that), in 64 bits: neighbours among the best are often a part in 10^6 apart, which is the rounding of
// a sum in 32 bits.
#include "lm_common.hpp"

namespace dnatok {

// Numbers in the order of unsigned integers; both zeros are one, NaN is lowest.
__device__ __forceinline__ uint32_t ordered(float v)
{
    if (v != v) return 0u;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u); }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// exp(v - top) for v <= top to an ulp or two: what the difference and its product with log2(e) are rounded off by is multiplied on (a
// difference of 10 is off by up to 8 roundings of a float, and so would the sum be if most of it is such terms; 16-bit numbers have none
// that matters).  (-inf is far enough at -200.)
template <typename T> __device__ __forceinline__ float exp_of(float v, float top)
{
    float d = v - top, off = 0.0f;
    if constexpr (sizeof(T) == 4) {
        const float back = d - v;
        off = (v - (d - back)) - (top + back);
        off = d > -200.0f ? off : 0.0f;            // (and not inf - inf)
    }
    d = fmaxf(d, -200.0f);
    const float e = 1.44269504f * d, rest = fmaf(1.44269504f, off, fmaf(1.92596299e-8f, d, fmaf(1.44269504f, d, -e))),
                power = __builtin_amdgcn_exp2f(e);
    return fmaf(power, 0.693147181f * rest, power);
}

struct Candidate {
    float logit;
    int32_t token;                                 // -1: none
};
struct Part {                                      // of a row's sum of exponentials
    double sum;
    float top;
};

constexpr int kRowThreads = 1024, kRowWaves = kRowThreads / 64;
constexpr int kSlice = 32768;                      // most tokens of a slice: 32 to a thread
constexpr int kListed = 1024;                      // candidates that are ranked against each other

// The largest of the workgroup's values.
template <typename V> __device__ __forceinline__ V workgroup_max(V v, V *room)
{
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const V other = __shfl_xor(v, d);
        v = other > v ? other : v;
    }
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = v;
    __syncthreads();
    v = room[0];
#pragma unroll
    for (int w = 1; w < kRowWaves; ++w) v = room[w] > v ? room[w] : v;
    __syncthreads();
    return v;
}

// Whether any of sixteen bytes' numbers is NaN.
template <typename T, typename V> __device__ __forceinline__ bool any_nan(V v)
{
    if constexpr (sizeof(T) == 4) {
        return v[0] != v[0] || v[1] != v[1] || v[2] != v[2] || v[3] != v[3];
    } else {
        // (two to a word; what is above infinity reaches the sign's bit)
        constexpr bool brain = std::is_same<T, __bf16>::value;
        const u32x4 w = __builtin_bit_cast(u32x4, v);
        uint32_t odd = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) odd |= (w[j] & 0x7FFF7FFFu) + (brain ? 0x007F007Fu : 0x03FF03FFu);
        return (odd & 0x80008000u) != 0;
    }
}

// The width-th largest of `count` numbers in LDS, of which as many are not below it: found by one wave, `count` a multiple of 4.
__device__ __forceinline__ float nth_largest(const float *numbers, int count, int width)
{
    const int lane = threadIdx.x & 63;
    float bound = -INFINITY;
    for (int i = lane; i < count; i += 64) {
        const float mine = numbers[i];
        int in_front = 0;
        for (int j = 0; j < count; j += 4) {
            const float4 four = *reinterpret_cast<const float4 *>(numbers + j);
            in_front += (four.x > mine || (four.x == mine && j < i)) + (four.y > mine || (four.y == mine && j + 1 < i)) +
                        (four.z > mine || (four.z == mine && j + 2 < i)) + (four.w > mine || (four.w == mine && j + 3 < i));
        }
        if (in_front == width - 1) bound = mine;
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) bound = fmaxf(bound, __shfl_xor(bound, d));
    return bound;
}

// A workgroup to a slice of a row, 32 tokens to a thread at most, held in registers.  The width-th largest of the waves' largest is a
// bound that the slice's `width` largest are not below, and few others are above it: those are listed and ranked by counting who is in
// front.  For more than eight, or where not every wave has tokens, it is that of eight lanes each; and where even those are
// hardly more than `width`, that of the threads, found bit by bit.  (A step with 512 rows of 32,000 bfloat16, eight beams: 53.4 us,
// bounds by eight lanes 61.9, by threads 59.7; 256 rows of floats, four beams: 33.5, 36.5 and 35.5.)  Where the
// list does not hold them all (many equal ones), the largest is looked for again and again.  512 rows of 32,000 bfloat16: 19 us for
// 33 MB, two workgroups to a CU: the chain from the reads to the rank, vector issue busy 0.32.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void beam_rows_kernel(const T *logits, int64_t stride, int32_t vocab, int32_t slice,
                                                                int32_t width, Candidate *found, Part *parts)
{
    constexpr int kCount = 16 / sizeof(T), kSteps = kSlice / kRowThreads / kCount, kGroups = kRowThreads / 8;
    typedef T words __attribute__((ext_vector_type(kCount)));
    __shared__ uint64_t list[kListed], best[kRowWaves];
    __shared__ double sums[kRowWaves];
    __shared__ __align__(16) float groups[kGroups], tops[kRowWaves];
    __shared__ uint32_t listed, counts[2][kRowWaves];
    __shared__ float bound_of;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.y, index = row * gridDim.x + blockIdx.x;
    const int32_t first = blockIdx.x * slice, here = vocab - first < slice ? vocab - first : slice;
    const T *z = logits + row * stride + first;
    if (threadIdx.x == 0) listed = 0;
    words v[kSteps];
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
        const int at = (j * kRowThreads + threadIdx.x) * kCount;
        if (at + kCount <= here) {
            __builtin_memcpy(&v[j], z + at, 16);
        } else {
#pragma unroll
            for (int e = 0; e < kCount; ++e) v[j][e] = at + e < here ? z[at + e] : (T)-INFINITY;
        }
    }
    float mine = -INFINITY;
    bool odd = false;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
        odd |= any_nan<T>(v[j]);
#pragma unroll
        for (int e = 0; e < kCount; ++e) mine = fmaxf(mine, (float)v[j][e]);           // (the number, of a number and NaN)
    }
    float most = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        most = fmaxf(most, __shfl_xor(most, d));
        if (d == 4 && (lane & 7) == 0) groups[threadIdx.x >> 3] = most;
    }
    if (lane == 0) tops[wave] = most;
    __syncthreads();
    float top = tops[0];
#pragma unroll
    for (int w = 1; w < kRowWaves; ++w) top = fmaxf(top, tops[w]);
    const bool by_threads = width * 2 > (here < kGroups * 8 * kCount ? here / (8 * kCount) : kGroups);
    if (wave == 0 && !by_threads) {
        const float nth = width <= 8 && here >= kRowThreads * kCount ? nth_largest(tops, kRowWaves, width) : nth_largest(groups, kGroups, width);
        if (lane == 0) bound_of = nth;
    }
    // (in 64 bits from the first term on: in 32 a thread that has the largest one would lose all below 2^-24 of it)
    double all = odd ? NAN : 0.0;
    if (top > -INFINITY) {
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
            if (j * kRowThreads * kCount < here)
#pragma unroll
                for (int e = 0; e < kCount; ++e) all += exp_of<T>((float)v[j][e], top);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) all += __shfl_xor(all, d);
    if (lane == 0) sums[wave] = all;
    __syncthreads();
    float bound = bound_of;
    if (by_threads) {                              // (16 bits of it, from the highest on, as long as `width` threads reach it)
        const uint32_t own = mine > -INFINITY ? ordered(mine) : 0u;
        uint32_t bits = 0;
        for (int bit = 31; bit >= 16; --bit) {
            const uint32_t next = bits | 1u << bit;
            const uint64_t reach = __ballot(own >= next);
            if (lane == 0) counts[bit & 1][wave] = __popcll(reach);
            __syncthreads();
            uint32_t n = 0;
#pragma unroll
            for (int w = 0; w < kRowWaves; ++w) n += counts[bit & 1][w];
            if (n >= (uint32_t)width) bits = next;
        }
        bound = bits > ordered(-INFINITY) ? from_ordered(bits) : -INFINITY;
    }
    const auto key_of = [&](int j, int e) {
        return (uint64_t)ordered((float)v[j][e]) << 32 | (uint32_t)~(first + (j * kRowThreads + threadIdx.x) * kCount + e);
    };
    if (mine >= bound) {
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
#pragma unroll
            for (int e = 0; e < kCount; ++e) {
                const float f = (float)v[j][e];
                if (f >= bound && f > -INFINITY) {                     // (candidates in the order of integers; -inf and NaN are none)
                    const uint32_t at = atomicAdd(&listed, 1u);
                    if (at < kListed) list[at] = key_of(j, e);
                }
            }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kRowWaves; ++w) all += sums[w];
        parts[index] = Part{all, top};
    }
    found += index * width;
    const auto candidate = [](uint64_t key) { return Candidate{from_ordered((uint32_t)(key >> 32)), (int32_t)~(uint32_t)key}; };
    const uint32_t n = listed;
    if (n <= kListed) {
        const uint64_t own = threadIdx.x < n ? list[threadIdx.x] : 0;
        uint32_t rank = 0;
        if (threadIdx.x < n)
            for (uint32_t i = 0; i < n; ++i) rank += list[i] > own;
        if (threadIdx.x < n && rank < (uint32_t)width) found[rank] = candidate(own);
        for (int i = n + threadIdx.x; i < width; i += kRowThreads) found[i] = Candidate{-INFINITY, -1};
        return;
    }
    uint64_t last = ~0ull;
    for (int i = 0; i < width; ++i) {
        uint64_t next = 0;
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
#pragma unroll
            for (int e = 0; e < kCount; ++e) {
                const uint64_t k = (float)v[j][e] > -INFINITY ? key_of(j, e) : 0;
                if (k < last && k > next) next = k;
            }
        last = workgroup_max((unsigned long long)next, (unsigned long long *)best);
        if (threadIdx.x == 0) found[i] = last ? candidate(last) : Candidate{-INFINITY, -1};
    }
}

// The largest of the wave's numbers, none of which is NaN.
template <int CTRL> __device__ __forceinline__ double max_with_dpp(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const double other = __builtin_bit_cast(double, (uint64_t)dpp_u32<CTRL>((uint32_t)(u >> 32)) << 32 | dpp_u32<CTRL>((uint32_t)u));
    return other > v ? other : v;
}
__device__ __forceinline__ double wave_max(double v)
{
    v = max_with_dpp<0xB1>(v);                     // neighbours, pairs, fours and eights of a row of sixteen
    v = max_with_dpp<0x4E>(v);
    v = max_with_dpp<0x141>(v);
    v = max_with_dpp<0x140>(v);
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    double best = -INFINITY;
#pragma unroll
    for (int row = 0; row < 64; row += 16) {
        const uint32_t high = __builtin_amdgcn_readlane((uint32_t)(u >> 32), row), low = __builtin_amdgcn_readlane((uint32_t)u, row);
        const double other = __builtin_bit_cast(double, (uint64_t)high << 32 | low);
        best = other > best ? other : best;
    }
    return best;
}

// A wave to a group: the lists of its beams' slices, each in falling order, merged.  A lane has the best of what is left of its
// lists (list l is lane l % 64's); lists are in the order of beams and tokens.  A chain of `width` steps: 8.7 us for eight of 8 beams, 5.7
// for four of 4.
constexpr int kMergeStaged = 4096;                 // candidates that are read into LDS at once
template <bool STAGED>
__global__ __launch_bounds__(64) void beam_merge_kernel(const Candidate *found, const Part *parts, const float *scores, const uint8_t *finished,
                                                        int32_t eos, int32_t beams, int32_t slices, int32_t width, int32_t *places,
                                                        float *out_scores, int32_t *tokens, int32_t *parents)
{
    __shared__ Candidate held[STAGED ? kMergeStaged : 1];
    __shared__ int32_t taken[STAGED ? kMergeStaged : 1];               // how many of each list (without room here, in places)
    __shared__ double sums[128];
    __shared__ float before[128];
    __shared__ uint8_t ended[128];
    const int lane = threadIdx.x;
    const int64_t group = blockIdx.x;
    const int lists = beams * slices;
    found += group * lists * width;
    parts += group * lists;
    places += group * lists;
    if (STAGED)
        for (int i = lane; i < lists * width; i += 64) held[i] = found[i];
    for (int b = lane; b < beams; b += 64) {
        float top = -INFINITY;
        for (int s = 0; s < slices; ++s) top = fmaxf(top, parts[b * slices + s].top);
        double sum = 0.0;
        for (int s = 0; s < slices; ++s) {
            const Part p = parts[b * slices + s];
            if (p.sum != 0.0) sum += p.sum * exp((double)p.top - (double)top);     // (a NaN stays one)
        }
        sums[b] = (double)top + log(sum);
        before[b] = scores[group * beams + b];
        ended[b] = finished ? finished[group * beams + b] : 0;
    }
    const auto set_taken = [&](int l, int32_t n) {
        if constexpr (STAGED) taken[l] = n;
        else places[l] = n;
    };
    const auto get_taken = [&](int l) {
        if constexpr (STAGED) return taken[l];
        else return places[l];
    };
    for (int l = lane; l < lists; l += 64) set_taken(l, 0);
    __syncthreads();
    const auto value = [&](int l, int at, float *logit, int32_t *token) {
        const int b = l / slices;
        *token = -1;
        *logit = 0.0f;
        if (ended[b]) {
            if (at == 0 && l == b * slices) {
                *token = eos;
                return (double)before[b];
            }
            return -(double)INFINITY;
        }
        if (at >= width) return -(double)INFINITY;
        const Candidate c = STAGED ? held[l * width + at] : found[(int64_t)l * width + at];
        const double sum = sums[b];
        if (c.token < 0 || !(sum < INFINITY && sum > -INFINITY)) return -(double)INFINITY;
        *token = c.token;
        *logit = c.logit;
        return (double)before[b] + ((double)c.logit - sum);
    };
    double mine = -INFINITY;
    float logit = 0.0f;
    int32_t token = -1, list = lists;
    const auto look = [&] {
        mine = -INFINITY;
        list = lists;
        for (int l = lane; l < lists; l += 64) {
            float z;
            int32_t t;
            const double v = value(l, get_taken(l), &z, &t);
            if (v > mine || (v == mine && v > -INFINITY && l / slices == list / slices && z > logit)) {
                mine = v;
                logit = z;
                token = t;
                list = l;
            }
        }
    };
    look();
    for (int i = 0; i < width; ++i) {
        const double best = wave_max(mine);
        if (!(best > -INFINITY)) {
            for (int j = i + lane; j < width; j += 64) {
                out_scores[group * width + j] = -INFINITY;
                tokens[group * width + j] = -1;
                parents[group * width + j] = j % beams;
            }
            return;
        }
        // of equal ones the lowest beam's, of that beam's the one with the largest logit, the lowest list's
        uint64_t equal = __ballot(mine == best);
        int winner = __builtin_ctzll(equal);
        for (equal &= equal - 1; equal; equal &= equal - 1) {
            const int l = __builtin_ctzll(equal);
            const int list_l = __shfl(list, l), list_w = __shfl(list, winner);
            const float z_l = __shfl(logit, l), z_w = __shfl(logit, winner);
            const int beam_l = list_l / slices, beam_w = list_w / slices;
            if (beam_l < beam_w || (beam_l == beam_w && (z_l > z_w || (z_l == z_w && list_l < list_w)))) winner = l;
        }
        if (lane == winner) {
            out_scores[group * width + i] = (float)mine;
            tokens[group * width + i] = token;
            parents[group * width + i] = list / slices;
            set_taken(list, get_taken(list) + 1);
            look();
        }
    }
}

constexpr int kReorderTensors = 16, kReorderBlock = 16384;             // bytes of a row to a workgroup
struct Reorder {
    dnatok_rows t[kReorderTensors];
};

// Row r of a group's `width` is row parents[r] of its `beams`, 16, 4 or 1 bytes to a lane.  512 rows of 135 KB: 24.8 us, 5.6 TB/s.
__global__ __launch_bounds__(256) void reorder_kernel(Reorder all, const int32_t *parents, int64_t rows, int32_t beams, int32_t width)
{
    const dnatok_rows t = all.t[blockIdx.z];
    const int64_t from = (int64_t)blockIdx.x * kReorderBlock;
    if (from >= t.bytes) return;
    const int64_t end = t.bytes - from < kReorderBlock ? t.bytes : from + kReorderBlock;
    const uint64_t places = (uint64_t)t.in | (uint64_t)t.out | (uint64_t)t.bytes | (uint64_t)t.in_stride | (uint64_t)t.out_stride;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const int32_t parent = parents[r];
        const bool known = parent >= 0 && parent < beams;
        const uint8_t *in = (const uint8_t *)t.in + (r / width * beams + (known ? parent : 0)) * t.in_stride;
        uint8_t *out = (uint8_t *)t.out + r * t.out_stride;
        if (places % 16 == 0) {
            u32x4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t at = from + (i * 256 + threadIdx.x) * 16;
                v[i] = u32x4{0, 0, 0, 0};
                if (at < end && known) v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(in + at));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t at = from + (i * 256 + threadIdx.x) * 16;
                if (at < end) __builtin_nontemporal_store(v[i], reinterpret_cast<u32x4 *>(out + at));
            }
        } else if (places % 4 == 0) {
            for (int64_t at = from + threadIdx.x * 4; at < end; at += 1024)
                *reinterpret_cast<uint32_t *>(out + at) = known ? *reinterpret_cast<const uint32_t *>(in + at) : 0u;
        } else {
            for (int64_t at = from + threadIdx.x; at < end; at += 256) out[at] = known ? in[at] : 0;
        }
    }
}

}  // namespace dnatok

using namespace dnatok;

#define BEAM_REQUIRE(cond, text) DNATOK_REQUIRE(cond, DNATOK_E_INVALID, "%s: " text, who)

// Slices of a row: as few as hold it, or as many as make 256 workgroups, of 4,096 tokens and more.
static int64_t slice_of(int64_t rows, int64_t vocab)
{
    const int64_t fewest = (vocab + kSlice - 1) / kSlice, most = (vocab + 4095) / 4096;
    int64_t slices = 256 / rows;
    slices = slices < fewest ? fewest : slices > most ? most : slices;
    return (vocab + slices - 1) / slices;
}

extern "C" size_t dnatok_beam_work_bytes(int64_t groups, int32_t beams, int64_t vocab, int32_t width)
{
    if (groups <= 0 || beams <= 0 || width <= 0 || vocab <= 0) return 0;
    const int64_t rows = groups * beams, slice = slice_of(rows, vocab);
    return (size_t)(rows * ((vocab + slice - 1) / slice)) * (sizeof(Part) + 4 + sizeof(Candidate) * (size_t)width);
}

extern "C" int dnatok_beam_select(const void *logits, int64_t stride, int32_t dtype, int64_t groups, int32_t beams, int64_t vocab,
                                  const float *scores, const uint8_t *finished, int32_t eos, int32_t width, float *out_scores,
                                  int32_t *tokens, int32_t *parents, void *work, size_t work_bytes, void *stream)
{
    static const char *who = "dnatok_beam_select";
    BEAM_REQUIRE(dtype == DNATOK_F32 || dtype == DNATOK_BF16 || dtype == DNATOK_F16, "unknown element type");
    BEAM_REQUIRE(groups >= 0 && beams > 0 && vocab > 0 && width > 0, "bad size");
    BEAM_REQUIRE(stride >= 0, "negative stride");
    BEAM_REQUIRE(!finished || (eos >= 0 && eos < vocab), "finished beams need an end in the vocabulary");
    // (a grid ends at 2^32 threads, and a group has 64)
    DNATOK_REQUIRE(beams <= 128 && width <= 128 && vocab < (1ll << 31) && groups < (1ll << 26) && groups * beams < (1ll << 31),
                   DNATOK_E_TOO_LARGE, "%s: at most 128 beams, before and after, less than 2^26 groups, 2^31 rows and 2^31 tokens", who);
    if (groups == 0) return DNATOK_OK;
    BEAM_REQUIRE(logits && scores && out_scores && tokens && parents, "null buffer");
    BEAM_REQUIRE(work && work_bytes >= dnatok_beam_work_bytes(groups, beams, vocab, width), "work space too small");
    BEAM_REQUIRE((uintptr_t)work % 16 == 0, "work space must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const int64_t rows = groups * beams, slice = slice_of(rows, vocab), slices = (vocab + slice - 1) / slice;
    Part *parts = (Part *)work;
    Candidate *found = (Candidate *)(parts + rows * slices);
    int32_t *places = (int32_t *)(found + rows * slices * width);
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        for (int64_t first = 0; first < rows; first += 65535) {        // (a grid's second dimension ends there)
            const int64_t here = rows - first < 65535 ? rows - first : 65535;
            beam_rows_kernel<T><<<dim3((unsigned)slices, (unsigned)here), kRowThreads, 0, s>>>(
                (const T *)logits + first * stride, stride, (int32_t)vocab, (int32_t)slice, width, found + first * slices * width,
                parts + first * slices);
        }
    });
    if (beams * slices * width <= kMergeStaged)
        beam_merge_kernel<true><<<(unsigned)groups, 64, 0, s>>>(found, parts, scores, finished, eos, beams, (int32_t)slices, width, places,
                                                                 out_scores, tokens, parents);
    else
        beam_merge_kernel<false><<<(unsigned)groups, 64, 0, s>>>(found, parts, scores, finished, eos, beams, (int32_t)slices, width, places,
                                                                  out_scores, tokens, parents);
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

extern "C" int dnatok_reorder_rows(const dnatok_rows *tensors_h, int32_t n, const int32_t *parents, int64_t groups, int32_t beams,
                                   int32_t width, void *stream)
{
    static const char *who = "dnatok_reorder_rows";
    BEAM_REQUIRE(n >= 0 && groups >= 0 && beams > 0 && width > 0, "bad size");
    BEAM_REQUIRE(n == 0 || tensors_h, "null list");
    DNATOK_REQUIRE(groups < (1ll << 31), DNATOK_E_TOO_LARGE, "%s: at most 2^31 groups", who);
    for (int i = 0; i < n; ++i)
        BEAM_REQUIRE(tensors_h[i].bytes >= 0 && tensors_h[i].bytes < (1ll << 37) && tensors_h[i].in_stride >= 0 &&
                         tensors_h[i].out_stride >= 0, "a size or stride is negative or too large");
    const int64_t rows = groups * width;
    if (rows == 0 || n == 0) return DNATOK_OK;
    BEAM_REQUIRE(parents, "null buffer");
    for (int i = 0; i < n; ++i) BEAM_REQUIRE(tensors_h[i].bytes == 0 || (tensors_h[i].in && tensors_h[i].out), "null buffer");
    for (int32_t first = 0; first < n; first += kReorderTensors) {
        Reorder all{};
        const int32_t here = n - first < kReorderTensors ? n - first : kReorderTensors;
        for (int i = 0; i < here; ++i) all.t[i] = tensors_h[first + i];
        int64_t most = 0;
        for (int i = 0; i < here; ++i) most = tensors_h[first + i].bytes > most ? tensors_h[first + i].bytes : most;
        if (most == 0) continue;
        const unsigned blocks = (unsigned)((most + kReorderBlock - 1) / kReorderBlock);
        reorder_kernel<<<dim3(blocks, (unsigned)(rows < 65535 ? rows : 65535), (unsigned)here), 256, 0, (hipStream_t)stream>>>(all, parents, rows,
                                                                                                              beams, width);
    }
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
