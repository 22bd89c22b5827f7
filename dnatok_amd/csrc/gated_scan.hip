// Gated linear recurrence over packed rows, its backward pass and its single step.
//
//   f_t = sigmoid(gate_t),   h_t = f_t h_(t-1) + (1 - f_t) x_t   in every channel of a row,
//
// from a given state or from zero.  Values, gates and outputs have 16 or 32 bits, states always 32.
#include "lm_common.hpp"

namespace dnatok {

// One thread per row and channel walks the row.  `all` (float [total, dim]) keeps the states for the backward pass.
template <typename T>
__global__ __launch_bounds__(256) void gated_scan_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ gate, int64_t gate_stride, Rows rows, int64_t dim,
    bool reverse, const float *__restrict__ h0, T *__restrict__ y, float *__restrict__ last, float *__restrict__ all)
{
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= dim) return;
    for (int64_t b = blockIdx.y; b < rows.n; b += gridDim.y) {
        const int64_t lo = rows.at(b), hi = rows.at(b + 1);
        float h = h0 ? h0[b * dim + c] : 0.0f;
        for (int64_t i = 0; i < hi - lo; ++i) {
            const int64_t t = reverse ? hi - 1 - i : lo + i;
            const Gate g(to_float(gate[t * gate_stride + c]));
            h = g.next(h, to_float(x[t * x_stride + c]));
            y[t * dim + c] = from_float<T>(h);
            if (all) all[t * dim + c] = h;
        }
        if (last) last[b * dim + c] = h;
    }
}

//   dh_t = dy_t + f_(t+1) dh_(t+1),  dx_t = (1 - f_t) dh_t,  dgate_t = dh_t (h_(t-1) - x_t) f_t (1 - f_t)
template <typename T>
__global__ __launch_bounds__(256) void gated_scan_backward_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ gate, int64_t gate_stride, Rows rows, int64_t dim,
    bool reverse, const float *__restrict__ h0, const T *__restrict__ dy, int64_t dy_stride,
    const float *__restrict__ dlast, const float *__restrict__ all, T *__restrict__ dx, T *__restrict__ dgate,
    float *__restrict__ dh0)
{
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= dim) return;
    for (int64_t b = blockIdx.y; b < rows.n; b += gridDim.y) {
        const int64_t lo = rows.at(b), hi = rows.at(b + 1);
        float carry = dlast ? dlast[b * dim + c] : 0.0f;
        for (int64_t i = hi - lo - 1; i >= 0; --i) {
            const int64_t t = reverse ? hi - 1 - i : lo + i;
            const int64_t before = reverse ? t + 1 : t - 1;
            const Gate g(to_float(gate[t * gate_stride + c]));
            const float h = i > 0 ? all[before * dim + c] : h0 ? h0[b * dim + c] : 0.0f;
            const float dh = carry + (dy ? to_float(dy[t * dy_stride + c]) : 0.0f);
            dx[t * dim + c] = from_float<T>(g.keep() * dh);
            dgate[t * dim + c] = from_float<T>(dh * (h - to_float(x[t * x_stride + c])) * g.slope());
            carry = g.forget(dh);
        }
        if (dh0) dh0[b * dim + c] = carry;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void gated_step_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ gate, int64_t gate_stride, const float *state,
    int64_t n_rows, int64_t dim, T *__restrict__ y, float *new_state)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n_rows * dim) return;
    const int64_t b = i / dim, c = i - b * dim;
    const Gate g(to_float(gate[b * gate_stride + c]));
    const float h = g.next(state ? state[i] : 0.0f, to_float(x[b * x_stride + c]));
    y[i] = from_float<T>(h);
    new_state[i] = h;
}

}  // namespace dnatok

using namespace dnatok;

#define SCAN_REQUIRE(cond, text) DNATOK_REQUIRE(cond, DNATOK_E_INVALID, "%s: " text, who)

static int check_rows(const char *who, int32_t dtype, int64_t n_rows, int64_t total, int64_t dim, const int64_t *offsets)
{
    SCAN_REQUIRE(dtype == DNATOK_F32 || dtype == DNATOK_BF16 || dtype == DNATOK_F16, "unknown element type");
    SCAN_REQUIRE(n_rows >= 0 && total >= 0 && dim > 0 && (n_rows > 0 || total == 0), "bad size");
    SCAN_REQUIRE(offsets || n_rows == 0 || total % n_rows == 0, "rows without offsets must be of one length");
    return DNATOK_OK;
}

extern "C" size_t dnatok_gated_scan_states_bytes(int64_t total, int64_t dim, int32_t dtype)
{
    (void)dtype;
    return total > 0 && dim > 0 ? (size_t)total * (size_t)dim * 4 : 0;
}

extern "C" size_t dnatok_gated_scan_work_bytes(int64_t total, int64_t dim, int32_t dtype)
{
    (void)total; (void)dim; (void)dtype;
    return 0;
}

extern "C" int dnatok_gated_scan(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride, int32_t dtype,
                                 const int64_t *offsets, int64_t n_rows, int64_t total, int64_t dim, int reverse,
                                 const float *h0, void *y, float *last, void *states, size_t states_bytes, void *stream)
{
    static const char *who = "dnatok_gated_scan";
    if (int rc = check_rows(who, dtype, n_rows, total, dim, offsets)) return rc;
    if (n_rows == 0) return DNATOK_OK;
    SCAN_REQUIRE(total == 0 || (x && gate && y), "null buffer");
    DNATOK_REQUIRE(!states || states_bytes >= dnatok_gated_scan_states_bytes(total, dim, dtype), DNATOK_E_SCRATCH,
                   "%s: the states need %zu bytes", who, dnatok_gated_scan_states_bytes(total, dim, dtype));
    const Rows rows{offsets, n_rows, total};
    const dim3 grid((unsigned)((dim + 255) / 256), (unsigned)(n_rows < 65535 ? n_rows : 65535));
    hipStream_t s = (hipStream_t)stream;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        gated_scan_kernel<T><<<grid, 256, 0, s>>>((const T *)x, x_stride, (const T *)gate, gate_stride, rows, dim,
                                                  reverse != 0, h0, (T *)y, last, (float *)states);
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

extern "C" int dnatok_gated_scan_backward(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride,
                                          int32_t dtype, const int64_t *offsets, int64_t n_rows, int64_t total,
                                          int64_t dim, int reverse, const float *h0, const void *dy, int64_t dy_stride,
                                          const float *dlast, const void *states, size_t states_bytes, void *dx,
                                          void *dgate, float *dh0, void *work, size_t work_bytes, void *stream)
{
    static const char *who = "dnatok_gated_scan_backward";
    (void)work; (void)work_bytes;
    if (int rc = check_rows(who, dtype, n_rows, total, dim, offsets)) return rc;
    if (n_rows == 0) return DNATOK_OK;
    SCAN_REQUIRE(total == 0 || (x && gate && dx && dgate && states), "null buffer");
    DNATOK_REQUIRE(states_bytes >= dnatok_gated_scan_states_bytes(total, dim, dtype), DNATOK_E_SCRATCH,
                   "%s: the states need %zu bytes", who, dnatok_gated_scan_states_bytes(total, dim, dtype));
    const Rows rows{offsets, n_rows, total};
    const dim3 grid((unsigned)((dim + 255) / 256), (unsigned)(n_rows < 65535 ? n_rows : 65535));
    hipStream_t s = (hipStream_t)stream;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        gated_scan_backward_kernel<T><<<grid, 256, 0, s>>>((const T *)x, x_stride, (const T *)gate, gate_stride, rows, dim,
                                                           reverse != 0, h0, (const T *)dy, dy_stride, dlast,
                                                           (const float *)states, (T *)dx, (T *)dgate, dh0);
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

extern "C" int dnatok_gated_step(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride, int32_t dtype,
                                 const float *state, int64_t n_rows, int64_t dim, void *y, float *new_state, void *stream)
{
    static const char *who = "dnatok_gated_step";
    if (int rc = check_rows(who, dtype, n_rows, n_rows, dim, nullptr)) return rc;
    if (n_rows == 0) return DNATOK_OK;
    SCAN_REQUIRE(x && gate && y && new_state, "null buffer");
    const int64_t blocks = (n_rows * dim + 255) / 256;
    DNATOK_REQUIRE(blocks < (1ll << 31), DNATOK_E_TOO_LARGE, "%s: more cells than one launch takes", who);
    hipStream_t s = (hipStream_t)stream;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        gated_step_kernel<T><<<(unsigned)blocks, 256, 0, s>>>((const T *)x, x_stride, (const T *)gate, gate_stride, state,
                                                              n_rows, dim, (T *)y, new_state);
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
