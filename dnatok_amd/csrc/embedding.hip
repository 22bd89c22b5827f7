// Rows of an embedding for packed ids, y_t = scale W[id_t], and the weights' gradient, dW[v] = scale sum of dy_t over the tokens
// t of id v.  An id outside the table stands for no row: zeros, and no part of a gradient.
#include "lm_common.hpp"

namespace dnatok {

template <typename T, typename ID>
__global__ __launch_bounds__(256) void embed_kernel(const ID *ids, int64_t n, const T *weight, int64_t w_stride, int64_t vocab,
                                                    int64_t dim, float scale, T *y)
{
    for (int64_t t = blockIdx.x; t < n; t += gridDim.x) {
        const int64_t id = ids[t];
        const bool known = id >= 0 && id < vocab;
        for (int64_t c = threadIdx.x; c < dim; c += 256)
            y[t * dim + c] = from_float<T>(known ? scale * to_float(weight[id * w_stride + c]) : 0.0f);
    }
}

// A workgroup to a row of the gradient: it looks through all ids.
template <typename T, typename ID>
__global__ __launch_bounds__(256) void embed_grad_kernel(const ID *ids, int64_t n, const T *dy, int64_t dy_stride, int64_t dim,
                                                         float scale, T *grad)
{
    __shared__ int found[4], list[256];
    const int64_t id = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t c0 = 0; c0 < dim; c0 += 256) {
        const int64_t c = c0 + threadIdx.x;
        float sum = 0.0f;
        for (int64_t t0 = 0; t0 < n; t0 += 256) {
            const bool here = t0 + threadIdx.x < n && (int64_t)ids[t0 + threadIdx.x] == id;
            const uint64_t mask = __ballot(here);
            if (lane == 0) found[wave] = __popcll(mask);
            __syncthreads();
            int at = 0, all = 0;
            for (int w = 0; w < 4; ++w) {
                at += w < wave ? found[w] : 0;
                all += found[w];
            }
            if (here) list[at + __popcll(mask & ((1ull << lane) - 1))] = threadIdx.x;
            __syncthreads();
            if (c < dim)
                for (int i = 0; i < all; ++i) sum += to_float(dy[(t0 + list[i]) * dy_stride + c]);
            __syncthreads();
        }
        if (c < dim) grad[id * dim + c] = from_float<T>(scale * sum);
    }
}

}  // namespace dnatok

using namespace dnatok;

#define EMBED_REQUIRE(cond, text) DNATOK_REQUIRE(cond, DNATOK_E_INVALID, "%s: " text, who)

static int check_embedding(const char *who, int32_t id_bytes, int64_t n, int64_t stride, int32_t dtype, int64_t vocab, int64_t dim)
{
    EMBED_REQUIRE(id_bytes == 4 || id_bytes == 8, "ids must have 4 or 8 bytes");
    EMBED_REQUIRE(dtype == DNATOK_F32 || dtype == DNATOK_BF16 || dtype == DNATOK_F16, "unknown element type");
    EMBED_REQUIRE(n >= 0 && vocab >= 0 && dim >= 0, "bad size");
    EMBED_REQUIRE(stride >= 0, "negative stride");
    DNATOK_REQUIRE(n < (1ll << 31) && vocab < (1ll << 31), DNATOK_E_TOO_LARGE, "%s: at most 2^31 tokens and rows", who);
    return DNATOK_OK;
}

template <typename Fn> static void with_ids(int32_t id_bytes, Fn fn)
{
    if (id_bytes == 4) fn(int32_t{});
    else fn(int64_t{});
}

extern "C" int dnatok_embedding(const void *ids, int32_t id_bytes, int64_t n, const void *weight, int64_t weight_stride, int32_t dtype,
                                int64_t vocab, int64_t dim, const float *scale_h, void *y, void *stream)
{
    static const char *who = "dnatok_embedding";
    if (int rc = check_embedding(who, id_bytes, n, weight_stride, dtype, vocab, dim)) return rc;
    if (n == 0 || dim == 0) return DNATOK_OK;
    EMBED_REQUIRE(ids && (weight || !vocab) && y && scale_h, "null buffer");
    const float scale = *scale_h;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        with_ids(id_bytes, [&](auto i) {
            using ID = decltype(i);
            embed_kernel<T, ID><<<(unsigned)(n < 65536 ? n : 65536), 256, 0, (hipStream_t)stream>>>(
                (const ID *)ids, n, (const T *)weight, weight_stride, vocab, dim, scale, (T *)y);
        });
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

extern "C" size_t dnatok_embedding_work_bytes(int64_t n, int64_t vocab, int64_t dim) { return 0; }

extern "C" int dnatok_embedding_backward(const void *ids, int32_t id_bytes, int64_t n, const void *dy, int64_t dy_stride, int32_t dtype,
                                         int64_t vocab, int64_t dim, const float *scale_h, void *grad, void *work, size_t work_bytes,
                                         void *stream)
{
    static const char *who = "dnatok_embedding_backward";
    if (int rc = check_embedding(who, id_bytes, n, dy_stride, dtype, vocab, dim)) return rc;
    if (vocab == 0 || dim == 0) return DNATOK_OK;
    EMBED_REQUIRE((n == 0 || (ids && dy)) && grad && scale_h, "null buffer");
    EMBED_REQUIRE(work_bytes >= dnatok_embedding_work_bytes(n, vocab, dim) && (work || !work_bytes), "work space too small");
    const float scale = *scale_h;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        with_ids(id_bytes, [&](auto i) {
            using ID = decltype(i);
            embed_grad_kernel<T, ID><<<(unsigned)vocab, 256, 0, (hipStream_t)stream>>>((const ID *)ids, n, (const T *)dy, dy_stride,
                                                                                        dim, scale, (T *)grad);
        });
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
