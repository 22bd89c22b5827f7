// y = x W^T + bias for few rows of x, where W[n, k] = (q[n, k] - zero[n, g]) scale[n, g] holds whole numbers q of 4 bits
// and g = k / group.  Eight of them lie in a 32-bit word, the lowest bits first.
#include "lm_common.hpp"

namespace dnatok {

// One wave per output: the lanes take the words of weight row n in turn.
template <typename T, typename OUT>
__global__ __launch_bounds__(256) void w4_matvec_kernel(
    const T *__restrict__ x, int64_t x_stride, const uint32_t *__restrict__ w, int64_t w_stride,
    const T *__restrict__ scales, const uint8_t *__restrict__ zeros, int64_t n, int64_t k, int32_t group, int64_t n_groups,
    const float *__restrict__ bias, OUT *__restrict__ y, int64_t y_stride)
{
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), m = blockIdx.y;
    if (row >= n) return;
    float sum = 0.0f;
    for (int64_t word = lane; word * 8 < k; word += 64) {
        const uint32_t q = w[row * w_stride + word];
        const int64_t g = word * 8 / group;
        const int zero = zeros ? zeros[row * n_groups + g] : 8;
        float part = 0.0f;
        for (int i = 0; i < 8 && word * 8 + i < k; ++i)
            part = fmaf((float)((int)(q >> (4 * i) & 15u) - zero), to_float(x[m * x_stride + word * 8 + i]), part);
        sum = fmaf(part, to_float(scales[row * n_groups + g]), sum);
    }
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) y[m * y_stride + row] = from_float<OUT>(sum + (bias ? bias[row] : 0.0f));
}

}  // namespace dnatok

using namespace dnatok;

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
    DNATOK_REQUIRE(n < (1ll << 31) && m <= 65535, DNATOK_E_TOO_LARGE, "%s: at most 2^31 outputs of 65535 rows", who);
    const int64_t n_groups = (k + group - 1) / group;
    const dim3 grid((unsigned)((n + 3) / 4), (unsigned)m);
    hipStream_t s = (hipStream_t)stream;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if constexpr (sizeof(T) == 2)
            with_type(y_dtype, [&](auto o) {
                using OUT = decltype(o);
                if constexpr (sizeof(OUT) == 4 || std::is_same<T, OUT>::value)
                    w4_matvec_kernel<T, OUT><<<grid, 256, 0, s>>>((const T *)x, x_stride, weights, weight_stride,
                                                                  (const T *)scales, zeros, n, k, group, n_groups, bias,
                                                                  (OUT *)y, y_stride);
            });
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
