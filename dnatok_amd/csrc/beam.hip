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

struct Candidate {
    float logit;
    int32_t token;                                 // -1: none
};

// A workgroup to a row: its sum, then its largest again and again.
template <typename T>
__global__ __launch_bounds__(256) void beam_rows_kernel(const T *logits, int64_t stride, int32_t vocab, int32_t width,
                                                        Candidate *found, double *sums)
{
    __shared__ uint64_t best[4];
    __shared__ double part[4];
    const int64_t row = blockIdx.x;
    const T *z = logits + row * stride;
    uint64_t last = ~0ull;
    float top = 0.0f;
    for (int i = -1; i < width; ++i) {
        uint64_t mine = 0;
        for (int v = threadIdx.x; v < vocab; v += 256) {
            const uint64_t key = (uint64_t)ordered(to_float(z[v])) << 32 | (uint32_t)~v;
            if (key < last && key > mine) mine = key;
        }
        for (int d = 32; d; d >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)mine, d);
            mine = other > mine ? other : mine;
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = mine;
        __syncthreads();
        for (int w = 0; w < 4; ++w) mine = best[w] > mine ? best[w] : mine;
        const float value = from_ordered((uint32_t)(mine >> 32));
        if (i < 0) {
            top = value;
            double sum = 0.0;
            for (int v = threadIdx.x; v < vocab; v += 256) sum += expf(to_float(z[v]) - top);
            for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
            __syncthreads();
            if (threadIdx.x == 0) sums[row] = (double)top + log(part[0] + part[1] + part[2] + part[3]);
            continue;
        }
        if (threadIdx.x == 0) found[row * width + i] = mine ? Candidate{value, (int32_t)~(uint32_t)mine} : Candidate{-INFINITY, -1};
        last = mine;
    }
}

// A wave to a group: the beams' lists merged.
__global__ __launch_bounds__(64) void beam_merge_kernel(const Candidate *found, const double *sums, const float *scores, const uint8_t *finished,
                                                        int32_t eos, int32_t beams, int32_t width, float *out_scores, int32_t *tokens,
                                                        int32_t *parents)
{
    __shared__ int32_t at[128];
    const int64_t group = blockIdx.x;
    for (int b = threadIdx.x; b < beams; b += 64) at[b] = 0;
    __syncthreads();
    for (int i = 0; i < width; ++i) {
        double value = -INFINITY;
        int32_t beam = 0x7FFFFFFF, token = -1;
        for (int b = threadIdx.x; b < beams; b += 64) {
            const int64_t row = group * beams + b;
            double v = -INFINITY;
            int32_t t = -1;
            if (finished && finished[row]) {
                if (at[b] == 0) {
                    v = scores[row];
                    t = eos;
                }
            } else if (at[b] < width) {
                const Candidate c = found[row * width + at[b]];
                const double sum = sums[row];
                if (c.token >= 0 && sum < INFINITY && sum > -INFINITY) {
                    v = (double)scores[row] + ((double)c.logit - sum);
                    t = c.token;
                }
            }
            if (v > value) {
                value = v;
                beam = b;
                token = t;
            }
        }
        for (int d = 32; d; d >>= 1) {
            const double v = __shfl_xor(value, d);
            const int32_t b = __shfl_xor(beam, d), t = __shfl_xor(token, d);
            if (v > value || (v == value && b < beam)) {
                value = v;
                beam = b;
                token = t;
            }
        }
        const bool none = !(value > -INFINITY);
        if (threadIdx.x == 0) {
            out_scores[group * width + i] = none ? -INFINITY : (float)value;
            tokens[group * width + i] = none ? -1 : token;
            parents[group * width + i] = none ? i % beams : beam;
            if (!none) ++at[beam];
        }
        __syncthreads();
    }
}

constexpr int kReorderTensors = 16;
struct Reorder {
    dnatok_rows t[kReorderTensors];
};

// Row r of a group's `width` is row parents[r] of its `beams`.
__global__ __launch_bounds__(256) void reorder_kernel(Reorder all, const int32_t *parents, int64_t rows, int32_t beams, int32_t width)
{
    const dnatok_rows t = all.t[blockIdx.z];
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const int32_t parent = parents[r];
        const bool known = parent >= 0 && parent < beams;
        const uint8_t *in = (const uint8_t *)t.in + (r / width * beams + (known ? parent : 0)) * t.in_stride;
        uint8_t *out = (uint8_t *)t.out + r * t.out_stride;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < t.bytes; i += (int64_t)gridDim.x * 256) out[i] = known ? in[i] : 0;
    }
}

}  // namespace dnatok

using namespace dnatok;

#define BEAM_REQUIRE(cond, text) DNATOK_REQUIRE(cond, DNATOK_E_INVALID, "%s: " text, who)

extern "C" size_t dnatok_beam_work_bytes(int64_t groups, int32_t beams, int64_t vocab, int32_t width)
{
    if (groups <= 0 || beams <= 0 || width <= 0 || vocab <= 0) return 0;
    return (size_t)groups * beams * (8 + 8 * (size_t)width);
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
    DNATOK_REQUIRE(beams <= 128 && width <= 128 && vocab < (1ll << 31) && groups * beams < (1ll << 31), DNATOK_E_TOO_LARGE,
                   "%s: at most 128 beams, before and after, and 2^31 rows of 2^31 tokens", who);
    if (groups == 0) return DNATOK_OK;
    BEAM_REQUIRE(logits && scores && out_scores && tokens && parents, "null buffer");
    BEAM_REQUIRE(work && work_bytes >= dnatok_beam_work_bytes(groups, beams, vocab, width), "work space too small");
    BEAM_REQUIRE((uintptr_t)work % 16 == 0, "work space must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    double *sums = (double *)work;
    Candidate *found = (Candidate *)(sums + groups * beams);
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        beam_rows_kernel<T><<<(unsigned)(groups * beams), 256, 0, s>>>((const T *)logits, stride, (int32_t)vocab, width, found, sums);
    });
    beam_merge_kernel<<<(unsigned)groups, 64, 0, s>>>(found, sums, scores, finished, eos, beams, width, out_scores, tokens, parents);
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
        BEAM_REQUIRE(tensors_h[i].bytes >= 0 && tensors_h[i].in_stride >= 0 && tensors_h[i].out_stride >= 0, "negative size or stride");
    const int64_t rows = groups * width;
    if (rows == 0 || n == 0) return DNATOK_OK;
    BEAM_REQUIRE(parents, "null buffer");
    for (int i = 0; i < n; ++i) BEAM_REQUIRE(tensors_h[i].bytes == 0 || (tensors_h[i].in && tensors_h[i].out), "null buffer");
    for (int32_t first = 0; first < n; first += kReorderTensors) {
        Reorder all{};
        const int32_t here = n - first < kReorderTensors ? n - first : kReorderTensors;
        for (int i = 0; i < here; ++i) all.t[i] = tensors_h[first + i];
        reorder_kernel<<<dim3(16, (unsigned)(rows < 65535 ? rows : 65535), (unsigned)here), 256, 0, (hipStream_t)stream>>>(all, parents, rows,
                                                                                                              beams, width);
    }
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
