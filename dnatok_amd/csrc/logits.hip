// What happens to a row of logits between a model's head and the choice of a token: penalties for tokens that
// the row's history holds, a bias, and a grammar's bit mask.
//
//   z = logit;  seen: z = z > 0 ? z / repetition : z repetition;  z -= presence [c > 0] + frequency c;
//   z += bias;  -inf where the mask forbids the token
//
// (seen: anywhere in the history; c: how often behind the first prompt_length tokens of it.)
#include "lm_common.hpp"

namespace dnatok {

constexpr int kLogitsThreads = 256;
constexpr int kLogitsSlice = 8192;                 // tokens of the vocabulary that a workgroup counts in LDS
constexpr uint32_t kInPrompt = 0x80000000u;        // beside the count of a token: the prompt holds it

struct LogitsArgs {
    int64_t vocab, in_stride, out_stride;
    const int32_t *history;
    const int64_t *history_offsets;
    const int32_t *prompt_lengths;
    const float *repetition, *presence, *frequency, *bias;
    int64_t bias_stride;
    const uint32_t *allowed;
    int64_t allowed_stride, n_states;
    const int32_t *state;
};

template <typename T, typename OUT>
__global__ __launch_bounds__(kLogitsThreads) void logits_kernel(const T *in, OUT *out, LogitsArgs a)
{
    __shared__ uint32_t counts[kLogitsSlice];
    const int64_t row = blockIdx.y, first = (int64_t)blockIdx.x * kLogitsSlice;
    const int here = (int)(a.vocab - first < kLogitsSlice ? a.vocab - first : kLogitsSlice);
    for (int i = threadIdx.x; i < here; i += kLogitsThreads) counts[i] = 0;
    __syncthreads();
    if (a.history) {
        const int64_t lo = a.history_offsets[row], hi = a.history_offsets[row + 1];
        const int64_t generated = lo + (a.prompt_lengths ? a.prompt_lengths[row] : 0);
        for (int64_t i = lo + threadIdx.x; i < hi; i += kLogitsThreads) {
            const int64_t at = (int64_t)a.history[i] - first;
            if (at >= 0 && at < here) {
                if (i < generated) atomicOr(&counts[at], kInPrompt);
                else atomicAdd(&counts[at], 1u);
            }
        }
    }
    __syncthreads();
    const float repetition = a.repetition ? a.repetition[row] : 1.0f;
    const float presence = a.presence ? a.presence[row] : 0.0f, frequency = a.frequency ? a.frequency[row] : 0.0f;
    const int32_t state = a.allowed ? (a.state ? a.state[row] : a.n_states == 1 ? 0 : (int32_t)row) : -1;
    for (int i = threadIdx.x; i < here; i += kLogitsThreads) {
        const int64_t v = first + i;
        float z = to_float(in[row * a.in_stride + v]);
        const uint32_t n = counts[i];
        if (n) {
            z = z > 0.0f ? z / repetition : z * repetition;
            const uint32_t c = n & ~kInPrompt;
            if (c) z -= presence + frequency * (float)c;
        }
        if (a.bias) z += a.bias[row * a.bias_stride + v];
        if (state >= 0) {
            const bool ok = state < a.n_states && (a.allowed[state * a.allowed_stride + (v >> 5)] >> (v & 31) & 1u);
            if (!ok) z = -INFINITY;
        }
        out[row * a.out_stride + v] = from_float<OUT>(z);
    }
}

}  // namespace dnatok

using namespace dnatok;

extern "C" int dnatok_logits_process(const void *logits, int64_t logits_stride, int32_t dtype, int64_t n_rows,
                                     int64_t vocab, const int32_t *history, const int64_t *history_offsets,
                                     const int32_t *prompt_lengths, const float *repetition, const float *presence,
                                     const float *frequency, const float *bias, int64_t bias_stride,
                                     const uint32_t *allowed, int64_t allowed_stride, int64_t n_states,
                                     const int32_t *state, void *out, int64_t out_stride, int32_t out_dtype, void *stream)
{
    static const char *who = "dnatok_logits_process";
#define LOGITS_REQUIRE(cond, text) DNATOK_REQUIRE(cond, DNATOK_E_INVALID, "%s: " text, who)
    LOGITS_REQUIRE(dtype == DNATOK_F32 || dtype == DNATOK_BF16 || dtype == DNATOK_F16, "unknown element type");
    LOGITS_REQUIRE(out_dtype == dtype || out_dtype == DNATOK_F32, "the result must have the logits' type or be float32");
    LOGITS_REQUIRE(n_rows >= 0 && vocab >= 0, "bad size");
    if (n_rows == 0 || vocab == 0) return DNATOK_OK;
    LOGITS_REQUIRE(logits && out, "null buffer");
    LOGITS_REQUIRE(!history == !history_offsets, "a history needs its offsets and the other way round");
    LOGITS_REQUIRE(!allowed || (n_states > 0 && allowed_stride >= (vocab + 31) / 32), "bad mask size");
    LOGITS_REQUIRE(!state || allowed, "states without masks");
    LOGITS_REQUIRE(!allowed || state || n_states == 1 || n_states == n_rows, "masks without states must be one or one a row");
    DNATOK_REQUIRE(n_rows <= 65535 && vocab < (1ll << 31), DNATOK_E_TOO_LARGE, "%s: at most 65535 rows of 2^31 tokens", who);
    const LogitsArgs a{vocab, logits_stride, out_stride, history, history_offsets, prompt_lengths, repetition, presence,
                       frequency, bias, bias_stride, allowed, allowed_stride, n_states, state};
    const dim3 grid((unsigned)((vocab + kLogitsSlice - 1) / kLogitsSlice), (unsigned)n_rows);
    hipStream_t s = (hipStream_t)stream;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        with_type(out_dtype, [&](auto o) {
            using OUT = decltype(o);
            if constexpr (sizeof(OUT) == 4 || std::is_same<T, OUT>::value)
                logits_kernel<T, OUT><<<grid, kLogitsThreads, 0, s>>>((const T *)logits, (OUT *)out, a);
        });
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
