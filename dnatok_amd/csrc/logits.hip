// What happens to a row of logits between a model's head and the choice of a token: penalties for tokens that
// the row's history holds, a bias, and a grammar's bit mask.
//
//   z = logit;  seen: z = z > 0 ? z / repetition : z repetition;  z -= presence [c > 0] + frequency c;
//   z += bias;  -inf where the mask forbids the token
//
// (seen: anywhere in the history; c: how often behind the first prompt_length tokens of it.)
//
// A workgroup takes a slice of one row's tokens: it reads the whole history and counts the ids of its slice in LDS (a
// word a token: whole numbers, so the order of the additions does not matter), then passes over its logits once.  The
// logits are requested before the counting.  With a history of some thousand ids this is a chain of a few
// trips to memory: offsets, ids, the atomics, stores.  256 rows of 32,000 tokens, bfloat16: 16.3 us a call with histories of up to
// 16,000 ids (2.6 TB/s); replayed in a graph 16.8, and 11.4 with histories of at most two.
#include "lm_common.hpp"

namespace dnatok {

constexpr int kLogitsThreads = 1024;
constexpr int kLogitsSlice = 16384;                // most tokens of a slice: 64 KB of counts
constexpr int kLogitsVectors = kLogitsSlice / kLogitsThreads / 4;      // four tokens to a lane and step
constexpr int kIdsAhead = 4;                       // loads of four ids that a lane has under way
constexpr uint32_t kInPrompt = 0x80000000u;        // beside the count of a token: the prompt holds it

struct LogitsArgs {
    int64_t vocab, in_stride, out_stride;
    int32_t slice;                                 // tokens of a slice, a multiple of 32
    const int32_t *history;
    const int64_t *history_offsets;
    const int32_t *prompt_lengths;
    const float *repetition, *presence, *frequency, *bias;
    int64_t bias_stride;
    const uint32_t *allowed;
    int64_t allowed_stride, n_states;
    const int32_t *state;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// HISTORY: whether there is one; without it nothing is counted.  (Two workgroups to a CU: with 69 registers for 32-bit logits
// instead of 64 it is one, 256 rows of 32,000 tokens 22.6 instead of 19.9 us.  That one, from and to 32 bits, then keeps four
// registers in scratch memory; no other does.)
template <typename T, typename OUT, bool HISTORY>
__global__ __launch_bounds__(kLogitsThreads) __attribute__((amdgpu_waves_per_eu(8))) void logits_kernel(const T *in, OUT *out, LogitsArgs a)
{
    extern __shared__ __align__(16) uint32_t counts[];                 // a.slice of them (rounded up to lanes' fours)
    typedef T four __attribute__((ext_vector_type(4)));
    typedef OUT four_out __attribute__((ext_vector_type(4)));
    const int64_t row = blockIdx.y, first = (int64_t)blockIdx.x * a.slice;
    const int here = (int)(a.vocab - first < a.slice ? a.vocab - first : a.slice);
    in += row * a.in_stride + first;
    out += row * a.out_stride + first;

    // everything that does not depend on the counts is requested first
    const float repetition = a.repetition ? a.repetition[row] : 1.0f;
    const float presence = a.presence ? a.presence[row] : 0.0f, frequency = a.frequency ? a.frequency[row] : 0.0f;
    const int32_t state = a.allowed ? (a.state ? a.state[row] : a.n_states == 1 ? 0 : (int32_t)row) : -1;
    const bool masked = state >= 0, known = masked && state < a.n_states;
    const uint32_t *mask = a.allowed + (known ? state * a.allowed_stride + (first >> 5) : 0);
    const float *bias = a.bias ? a.bias + row * a.bias_stride + first : nullptr;
    four z[kLogitsVectors];                                            // (rows begin at any element: loads of any alignment)
    f32x4 b[kLogitsVectors];
    uint32_t bits[kLogitsVectors];
#pragma unroll
    for (int j = 0; j < kLogitsVectors; ++j) {
        const int v = (j * kLogitsThreads + threadIdx.x) * 4;
        const bool whole = v + 4 <= here;
        if (whole) {
            __builtin_memcpy(&z[j], in + v, sizeof(four));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) z[j][e] = v + e < here ? in[v + e] : (T)0.0f;
        }
        b[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (bias) {
            if (whole) {
                __builtin_memcpy(&b[j], bias + v, 16);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) b[j][e] = v + e < here ? bias[v + e] : 0.0f;
            }
        }
        bits[j] = masked ? (known && v < here ? mask[v >> 5] >> (v & 31) : 0u) : 15u;
    }
    if (HISTORY) {
        const int64_t lo = a.history_offsets[row], n = a.history_offsets[row + 1] - lo;
        const int64_t prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
        const int32_t *ids = a.history + lo;
        for (int i = threadIdx.x * 4; i < here; i += kLogitsThreads * 4) *reinterpret_cast<u32x4 *>(counts + i) = u32x4{0, 0, 0, 0};
        __syncthreads();
        const auto count = [&](int32_t id, int64_t i) {
            const uint32_t at = (uint32_t)(id - (int32_t)first);       // (ids below the slice wrap around to beyond it)
            if (id >= 0 && at < (uint32_t)here) {
                if (i < prompt) atomicOr(&counts[at], kInPrompt);
                else atomicAdd(&counts[at], 1u);
            }
        };
        constexpr int kStep = kLogitsThreads * 4;
        int64_t i = 0;
        for (; i + kStep * kIdsAhead <= n; i += kStep * kIdsAhead) {
            u32x4 q[kIdsAhead];
#pragma unroll
            for (int j = 0; j < kIdsAhead; ++j) __builtin_memcpy(&q[j], ids + i + j * kStep + threadIdx.x * 4, 16);
#pragma unroll
            for (int j = 0; j < kIdsAhead; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) count((int32_t)q[j][e], i + j * kStep + threadIdx.x * 4 + e);
        }
        // what is left, less than kIdsAhead steps
        u32x4 q[kIdsAhead];
#pragma unroll
        for (int j = 0; j < kIdsAhead; ++j) {
            const int64_t at = i + j * kStep + threadIdx.x * 4;
            if (at + 4 <= n) {
                __builtin_memcpy(&q[j], ids + at, 16);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) q[j][e] = at + e < n ? (uint32_t)ids[at + e] : 0xFFFFFFFFu;
            }
        }
#pragma unroll
        for (int j = 0; j < kIdsAhead; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) count((int32_t)q[j][e], i + j * kStep + threadIdx.x * 4 + e);
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kLogitsVectors; ++j) {
        const int v = (j * kLogitsThreads + threadIdx.x) * 4;
        if (v >= here) break;
        const bool whole = v + 4 <= here;
        u32x4 n = {0, 0, 0, 0};
        if (HISTORY) n = *reinterpret_cast<const u32x4 *>(counts + v);
        four_out o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float y = to_float(z[j][e]);
            if (HISTORY && n[e]) {
                y = y > 0.0f ? y / repetition : y * repetition;
                const uint32_t c = n[e] & ~kInPrompt;
                if (c) y -= presence + frequency * (float)c;
            }
            if (bias) y += b[j][e];
            o[e] = from_float<OUT>(bits[j] >> e & 1u ? y : -INFINITY);
        }
        if (whole) {
            __builtin_memcpy(out + v, &o, sizeof(o));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v + e < here) out[v + e] = o[e];
        }
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
    LOGITS_REQUIRE(logits_stride >= 0 && out_stride >= 0 && bias_stride >= 0, "negative stride");
    LOGITS_REQUIRE(!history == !history_offsets, "a history needs its offsets and the other way round");
    LOGITS_REQUIRE(!allowed || (n_states > 0 && allowed_stride >= (vocab + 31) / 32), "bad mask size");
    LOGITS_REQUIRE(!state || allowed, "states without masks");
    LOGITS_REQUIRE(!allowed || state || n_states == 1 || n_states == n_rows, "masks without states must be one or one a row");
    DNATOK_REQUIRE(n_rows <= 65535 && vocab < (1ll << 31), DNATOK_E_TOO_LARGE, "%s: at most 65535 rows of 2^31 tokens", who);
    // slices: as few as hold the vocabulary, or as many as give each of the 256 CUs two, of 1024 tokens and more
    const int64_t fewest = (vocab + kLogitsSlice - 1) / kLogitsSlice, most = (vocab + 1023) / 1024;
    int64_t slices = (511 + n_rows) / n_rows;
    slices = slices < fewest ? fewest : slices > most ? most : slices;
    const int32_t slice = (int32_t)(((vocab + slices - 1) / slices + 31) & ~31ll);
    const LogitsArgs a{vocab, logits_stride, out_stride, slice, history, history_offsets, prompt_lengths, repetition,
                       presence, frequency, bias, bias_stride, allowed, allowed_stride, n_states, state};
    const dim3 grid((unsigned)((vocab + slice - 1) / slice), (unsigned)n_rows);
    hipStream_t s = (hipStream_t)stream;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        with_type(out_dtype, [&](auto o) {
            using OUT = decltype(o);
            if constexpr (sizeof(OUT) == 4 || std::is_same<T, OUT>::value) {
                if (history)
                    logits_kernel<T, OUT, true><<<grid, kLogitsThreads, (size_t)slice * 4, s>>>((const T *)logits, (OUT *)out, a);
                else
                    logits_kernel<T, OUT, false><<<grid, kLogitsThreads, 0, s>>>((const T *)logits, (OUT *)out, a);
            }
        });
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
