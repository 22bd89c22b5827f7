// Linear attention with a decay for each head: the C entries, and the kernels beside the walks over rows (linear_common.hpp has the
// mathematics, linear_walk.hpp the walks): states at cuts, sums over shared heads, one token of each row.
#include "linear_common.hpp"

namespace dnatok {

constexpr int kSlotThreads = 256;
__host__ __device__ __forceinline__ int64_t slot_parts(const WalkArgs &w)
{
    return ((int64_t)w.b.dim * w.c.dim + kSlotThreads - 1) / kSlotThreads;
}

// The slots' states from what the pieces add: a thread has one cell of a head's state and runs through a row's cuts.  What comes next is
// requested before what is done is stored (a wait for a load is one for the stores in front of it).  63 cuts of 4 heads of 128 x 128,
// 33 MB: 35 us, four round trips of sixteen cuts each.
__global__ __launch_bounds__(kSlotThreads) void slots_kernel(WalkArgs w)
{
    constexpr int kAhead = 16;
    const int64_t cells = (int64_t)w.b.dim * w.c.dim, cut = blockIdx.x + 1, at = cut * w.cut;
    const int64_t row = uniform(last_row(w.n_rows, at, [&](int64_t r) { return row_at(w, r); }));
    if (row < 0) return;
    const int64_t lo = uniform(row_at(w, row)), hi = uniform(row_at(w, row + 1));
    if (at <= lo || at >= hi) return;
    const int64_t first = lo / w.cut + 1, last = (hi - 1) / w.cut, n = last - first + 1;
    if (cut != (w.reverse ? last : first)) return;
    const int64_t outer = w.reverse ? hi - last * w.cut : first * w.cut - lo;
    const int64_t next = (w.reverse ? -1 : 1) * w.heads * cells;
    for (int64_t at_once = blockIdx.y; at_once < slot_parts(w) * w.heads; at_once += gridDim.y) {
        const int head = (int)(at_once % w.heads);
        const int64_t i = at_once / w.heads * kSlotThreads + threadIdx.x;
        if (i >= cells) continue;
        const float ld = log_decay_of(w.log_decay, head);
        float state = w.start ? w.start_scale * w.start[(row * w.heads + head) * cells + i] : 0.0f;
        const Left left = left_after(ld, (float)w.cut);
        state = decayed(state, left_after(ld, (float)outer));
        float *slot = w.slots + ((w.reverse ? last : first) - 1) * w.heads * cells + head * cells + i;
        float added[kAhead], coming[kAhead];
#pragma unroll
        for (int e = 0; e < kAhead; ++e) added[e] = e < n ? slot[e * next] : 0.0f;
        for (int64_t j = 0; j < n; j += kAhead) {
#pragma unroll
            for (int e = 0; e < kAhead; ++e) coming[e] = j + kAhead + e < n ? slot[(kAhead + e) * next] : 0.0f;
#pragma unroll
            for (int e = 0; e < kAhead; ++e) {
                state += added[e];
                if (j + e < n) slot[e * next] = state;
                state = decayed(state, left);
                added[e] = coming[e];
            }
            slot += kAhead * next;
        }
    }
}

// Gradients of keys and values that several heads share: the heads' parts, 32-bit [total, heads, dim], added up.  (876,000 tokens, 6 heads
// of 48 for 2 of them: 1.34 GB in 306 us, 4.4 TB/s.)
template <typename T>
__global__ __launch_bounds__(256) void shared_sum_kernel(const float *parts, T *out, int64_t cells, int32_t shared, int32_t dim)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (int64_t)gridDim.x * 256) {
        const int64_t head = i / dim, at = i % dim;
        float sum = 0.0f;
        for (int j = 0; j < shared; ++j) sum += parts[(head * shared + j) * dim + at];
        out[i] = from_float<T>(sum);
    }
}

// One token of each row: a workgroup has a head's state, a thread every few rows of VEC of its columns.  The state is
// read and written once; nothing else weighs anything.  250 rows, 8 heads of 128 x 128: 48 us for 262 MB, 5.5 TB/s; one row, 8 heads
// of 64 x 64: 4.8 us, a call with its allocations 11.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void linear_step_kernel(Operand q, Operand k, Operand v, const float *log_decay, float scale,
                                                          const float *state, T *y, float *new_state)
{
    typedef float vec __attribute__((ext_vector_type(VEC)));
    __shared__ float qk[2][128];
    __shared__ float part[256 * VEC];
    const int64_t row = blockIdx.y;
    const int head = blockIdx.x, heads = gridDim.x, dk = q.dim, dv = v.dim, cols = dv / VEC;
    const T *qp = (const T *)q.p + row * q.token + head * q.head;
    const T *kp = (const T *)k.p + row * k.token + head / k.shared * k.head;
    const T *vp = (const T *)v.p + row * v.token + head / v.shared * v.head;
    for (int i = threadIdx.x; i < dk; i += 256) {
        qk[0][i] = to_float(qp[i]);
        qk[1][i] = to_float(kp[i]);
    }
    const Left left = left_after(log_decay_of(log_decay, head), 1.0f);
    const int per = 256 / cols, col = threadIdx.x % cols, first = threadIdx.x / cols;      // (threads behind the last whole row have none)
    const int64_t at = (row * heads + head) * dk * dv;
    vec sum{}, value{};
    if (first < per)
#pragma unroll
        for (int e = 0; e < VEC; ++e) value[e] = to_float(vp[col * VEC + e]);
    __syncthreads();
    if (first < per) {
        for (int m = first; m < dk; m += per) {
            vec s{};
            if (state) s = *reinterpret_cast<const vec *>(state + at + m * dv + col * VEC);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                s[e] = fmaf(qk[1][m], value[e], decayed(s[e], left));
                sum[e] = fmaf(qk[0][m], s[e], sum[e]);
            }
            *reinterpret_cast<vec *>(new_state + at + m * dv + col * VEC) = s;
        }
    }
    *reinterpret_cast<vec *>(part + threadIdx.x * VEC) = sum;
    __syncthreads();
    for (int i = threadIdx.x; i < dv; i += 256) {
        float all = 0.0f;
        for (int j = 0; j < per; ++j) all += part[j * dv + i];
        y[(row * heads + head) * dv + i] = from_float<T>(scale * all);
    }
}

}  // namespace dnatok

using namespace dnatok;

#define LINEAR_REQUIRE(cond, text) DNATOK_REQUIRE(cond, DNATOK_E_INVALID, "%s: " text, who)

// Checks a shape of `tokens` tokens, and leaves it in `call` as the kernels take it: where there is one token at most, the distance to the
// next is that of no address, whatever it says (an axis of size one may have any stride).
static int check_shape(const char *who, const dnatok_linear_shape *given, int64_t dnatok_linear_shape::*tokens, dnatok_linear_shape *call)
{
    LINEAR_REQUIRE(given, "null shape");
    const dnatok_linear_shape *s = given;
    LINEAR_REQUIRE(s->dtype == DNATOK_F32 || s->dtype == DNATOK_BF16 || s->dtype == DNATOK_F16, "unknown element type");
    LINEAR_REQUIRE(s->n_rows >= 0 && s->total >= 0 && s->heads > 0 && s->kv_heads > 0 && s->dim_k > 0 && s->dim_v > 0, "bad size");
    LINEAR_REQUIRE(s->heads % s->kv_heads == 0, "the heads must be a multiple of those of the keys and values");
    constexpr float kFarScale = 1099511627776.0f;  // (gradients of states are held divided by it)
    LINEAR_REQUIRE(__builtin_fabsf(s->scale) >= 1.0f / kFarScale && __builtin_fabsf(s->scale) <= kFarScale,
                   "the scale must be 2^-40 to 2^40 in size");
    LINEAR_REQUIRE(s->q_token >= 0 && s->q_head >= 0 && s->k_token >= 0 && s->k_head >= 0 && s->v_token >= 0 && s->v_head >= 0 &&
                       s->dy_token >= 0 && s->dy_head >= 0, "negative stride");
    *call = *given;
    if (given->*tokens <= 1) call->q_token = call->k_token = call->v_token = call->dy_token = 0;
    s = call;
    constexpr int64_t kFar = (1ll << 31) / 64 / 4;
    DNATOK_REQUIRE(s->q_token < kFar && s->k_token < kFar && s->v_token < kFar && s->dy_token < kFar && (int64_t)s->heads * 128 < kFar,
                   DNATOK_E_TOO_LARGE, "%s: tokens must lie less than 2^23 elements apart", who);
    DNATOK_REQUIRE(s->dim_k <= 128 && s->dim_v <= 128 && s->heads <= 65535 && s->total < (1ll << 40) && s->n_rows < (1ll << 30),
                   DNATOK_E_TOO_LARGE, "%s: at most 65535 heads of 128 x 128", who);
    return DNATOK_OK;
}

static int check_call(const char *who, const dnatok_linear_shape &s, const int64_t *offsets)
{
    LINEAR_REQUIRE(!offsets == !s.with_offsets, "the shape must say whether there are offsets");
    LINEAR_REQUIRE(s.n_rows > 0 || s.total == 0, "tokens without rows");
    LINEAR_REQUIRE(offsets || s.n_rows == 0 || s.total % s.n_rows == 0, "rows of one length must fill the axis");
    // (the cuts are a grid's first dimension, which ends at 2^32 threads; rows and pieces go over several launches)
    DNATOK_REQUIRE(s.n_rows + (s.total >> 9) + kOutside < (1ll << 23), DNATOK_E_TOO_LARGE,
                   "%s: less than 2^23 rows and pieces of 512 tokens", who);
    return DNATOK_OK;
}

static Operand operand(const void *p, int64_t token, int64_t head, int32_t shared, int32_t dim)
{
    return Operand{p, token, head, shared, dim};
}
static Operand q_of(const dnatok_linear_shape *s, const void *q) { return operand(q, s->q_token, s->q_head, 1, s->dim_k); }
static Operand k_of(const dnatok_linear_shape *s, const void *k)
{
    return operand(k, s->k_token, s->k_head, s->heads / s->kv_heads, s->dim_k);
}
static Operand v_of(const dnatok_linear_shape *s, const void *v)
{
    return operand(v, s->v_token, s->v_head, s->heads / s->kv_heads, s->dim_v);
}

static unsigned sum_grid(int64_t cells) { return (unsigned)(cells < 65536 * 256 ? (cells + 255) / 256 : 65536); }

static size_t slots_bytes(const dnatok_linear_shape *s, int64_t cuts) { return (size_t)cuts * s->heads * s->dim_k * s->dim_v * 4; }

// Where rows are cut, so that one long row has many workgroups: at multiples of `cut` tokens.  What runs at once is two workgroups of
// four waves on each of 256 CUs, or one of eight.  Rows (of all heads) that are fewer are cut into as many pieces as run at
// once; more than that are cut where they are longer than about half of a CU's share, so that no long one is left running alone.  A
// multiple or a whole part of the mean length, 512 tokens at least, so that rows of one length are cut into equal pieces or not at all.
// (bfloat16, forward.  1 x 262,147 tokens, 4 heads of 128 x 128: 475 us, half as many pieces 784, twice as many 530; 64 x 8,192, 8 heads
// of 64 x 64: 520, 518 and 835.  Long reads, median 2,000 tokens: 1,500 rows, 2 heads of 64 x 64 1,558 us, cut at a quarter of the
// share 1,642, at the share 1,894, uncut 2,314; 300 rows, 6 heads of 64 x 64 934, 1,005, 1,141 and 1,053, 4 heads of 128 x 128 1,788,
// 1,965, 2,043 and 1,695.)
struct Cuts {
    int64_t cut, cuts;
};
static Cuts cuts_of(const dnatok_linear_shape *s)
{
    const int64_t rows = s->n_rows * s->heads, running = s->dim_k <= 64 && s->dim_v <= 64 ? 512 : 256;
    if (s->total == 0 || s->n_rows == 0 || (!s->with_offsets && rows > running / 2)) return Cuts{512, 0};
    const int64_t mean = (s->total + s->n_rows - 1) / s->n_rows, pieces = running / rows, share = (rows + running) / (2 * running);
    int64_t cut = rows <= running ? (mean + pieces - 1) / pieces : mean * (share < 1 ? 1 : share);
    if (cut < 512) {
        const int64_t whole = mean / 512;
        cut = whole ? (mean + whole - 1) / whole : (511 + mean) / mean * mean;
    }
    return Cuts{cut, (s->total - 1) / cut};
}

// The states at the cuts, then.
template <typename T> static void fill_slots(const WalkArgs &w, hipStream_t s)
{
    if (!w.cuts) return;
    launch_pieces<T>(w, s);
    // about 8,192 workgroups: most cuts begin no row's slots and leave at once, but one row's may be all that there is (the whole call, 4
    // heads of 128 x 128: 256 rows of 1,024 tokens 368 us, a workgroup to each part 377, 1,024 workgroups 366; one row of 262,147 524, 528 and 602)
    const int64_t all = slot_parts(w) * w.heads, some = 8192 / w.cuts + 1;
    slots_kernel<<<dim3((unsigned)w.cuts, (unsigned)(all < some ? all : some)), kSlotThreads, 0, s>>>(w);
}

extern "C" size_t dnatok_linear_attention_states_bytes(const dnatok_linear_shape *s)
{
    return s && s->heads > 0 ? slots_bytes(s, cuts_of(s).cuts) : 0;
}

extern "C" size_t dnatok_linear_attention_work_bytes(const dnatok_linear_shape *s, int backward)
{
    if (!s || s->heads <= 0) return 0;
    size_t n = slots_bytes(s, cuts_of(s).cuts);
    if (backward && s->kv_heads != s->heads) n += (size_t)s->total * s->heads * (s->dim_k + s->dim_v) * 4;
    return n;
}

extern "C" int dnatok_linear_attention(const dnatok_linear_shape *shape, const void *q, const void *k, const void *v,
                                       const float *log_decay, const int64_t *offsets, const float *h0, void *y, float *last,
                                       float *states, void *work, size_t work_bytes, void *stream)
{
    static const char *who = "dnatok_linear_attention";
    dnatok_linear_shape s;
    if (int rc = check_shape(who, shape, &dnatok_linear_shape::total, &s)) return rc;
    shape = &s;
    if (int rc = check_call(who, s, offsets)) return rc;
    LINEAR_REQUIRE(log_decay && (s.total == 0 || (q && k && v && y)), "null buffer");
    LINEAR_REQUIRE(states || (work_bytes >= dnatok_linear_attention_work_bytes(shape, 0) && (work || !work_bytes)), "work space too small");
    LINEAR_REQUIRE((uintptr_t)work % 16 == 0 && (uintptr_t)states % 16 == 0, "work space must be 16-byte aligned");
    if (s.n_rows == 0) return DNATOK_OK;
    const Cuts cuts = cuts_of(shape);
    with_type(s.dtype, [&](auto t) {
        using T = decltype(t);
        const WalkArgs w{q_of(shape, q), k_of(shape, k), v_of(shape, v), log_decay, offsets, s.n_rows, s.total, s.total / s.n_rows,
                         s.heads, s.reverse != 0, false, s.scale, 1.0f, 1.0f, h0, false, last, y, false, true,
                         states ? states : (float *)work, cuts.cut, cuts.cuts};
        fill_slots<T>(w, (hipStream_t)stream);
        launch_walk<T>(w, (hipStream_t)stream);
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

extern "C" int dnatok_linear_attention_backward(const dnatok_linear_shape *shape, const void *q, const void *k, const void *v,
                                                const float *log_decay, const int64_t *offsets, const float *h0, const void *dy,
                                                const float *dlast, const float *states, void *dq, void *dk, void *dv, float *dh0,
                                                void *work, size_t work_bytes, void *stream)
{
    static const char *who = "dnatok_linear_attention_backward";
    dnatok_linear_shape s;
    if (int rc = check_shape(who, shape, &dnatok_linear_shape::total, &s)) return rc;
    shape = &s;
    if (int rc = check_call(who, s, offsets)) return rc;
    LINEAR_REQUIRE(log_decay && (s.total == 0 || (q && k && v && dy && dq && dk && dv)), "null buffer");
    LINEAR_REQUIRE(states || !dnatok_linear_attention_states_bytes(shape), "the forward pass' states are missing");
    LINEAR_REQUIRE(work_bytes >= dnatok_linear_attention_work_bytes(shape, 1) && (work || !work_bytes), "work space too small");
    LINEAR_REQUIRE((uintptr_t)work % 16 == 0 && (uintptr_t)states % 16 == 0, "work space must be 16-byte aligned");
    if (s.n_rows == 0) return DNATOK_OK;
    hipStream_t stm = (hipStream_t)stream;
    const Operand qo = q_of(shape, q), ko = k_of(shape, k), vo = v_of(shape, v),
                  go = operand(dy, s.dy_token, s.dy_head, 1, s.dim_v);
    const int64_t length = s.total / s.n_rows;
    const Cuts cuts = cuts_of(shape);
    with_type(s.dtype, [&](auto t) {
        using T = decltype(t);
        const bool shared = s.heads != s.kv_heads, rev = s.reverse != 0;
        launch_walk<T>(WalkArgs{go, vo, ko, log_decay, offsets, s.n_rows, s.total, length, s.heads, rev, false, s.scale, 1.0f, 1.0f, h0,
                         true, nullptr, dq, false, false, const_cast<float *>(states), cuts.cut, cuts.cuts}, stm);
        float *slots = (float *)work, *pk = slots + slots_bytes(shape, cuts.cuts) / 4, *pv = pk + s.total * s.heads * s.dim_k;
        // (a state's gradient without the scale, which all that is made of it gets)
        const float inv = 1.0f / s.scale;
        const WalkArgs wv{ko, qo, go, log_decay, offsets, s.n_rows, s.total, length, s.heads, !rev, true, s.scale, inv, s.scale, dlast,
                          false, dh0, shared ? (void *)pv : dv, shared, true, slots, cuts.cut, cuts.cuts};
        const WalkArgs wk{vo, go, qo, log_decay, offsets, s.n_rows, s.total, length, s.heads, !rev, true, s.scale, inv, s.scale, dlast,
                          true, nullptr, shared ? (void *)pk : dk, shared, false, slots, cuts.cut, cuts.cuts};
        fill_slots<T>(wv, stm);
        launch_walk<T>(wv, stm);
        launch_walk<T>(wk, stm);
        if (shared && s.total) {
            const int64_t ck = s.total * s.kv_heads * s.dim_k, cv = s.total * s.kv_heads * s.dim_v;
            shared_sum_kernel<T><<<sum_grid(ck), 256, 0, stm>>>(pk, (T *)dk, ck, s.heads / s.kv_heads, s.dim_k);
            shared_sum_kernel<T><<<sum_grid(cv), 256, 0, stm>>>(pv, (T *)dv, cv, s.heads / s.kv_heads, s.dim_v);
        }
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

extern "C" int dnatok_linear_attention_step(const dnatok_linear_shape *shape, const void *q, const void *k, const void *v,
                                            const float *log_decay, const float *state, void *y, float *new_state, void *stream)
{
    static const char *who = "dnatok_linear_attention_step";
    dnatok_linear_shape s;
    if (int rc = check_shape(who, shape, &dnatok_linear_shape::n_rows, &s)) return rc;
    shape = &s;
    if (s.n_rows == 0) return DNATOK_OK;
    LINEAR_REQUIRE(q && k && v && log_decay && y && new_state, "null buffer");
    DNATOK_REQUIRE(s.n_rows <= 65535, DNATOK_E_TOO_LARGE, "%s: at most 65535 rows", who);
    const dim3 grid((unsigned)s.heads, (unsigned)s.n_rows);
    const bool wide = s.dim_v % 4 == 0 && ((uintptr_t)state | (uintptr_t)new_state) % 16 == 0;
    with_type(s.dtype, [&](auto t) {
        using T = decltype(t);
        if (wide)
            linear_step_kernel<T, 4><<<grid, 256, 0, (hipStream_t)stream>>>(q_of(shape, q), k_of(shape, k), v_of(shape, v), log_decay,
                                                                            s.scale, state, (T *)y, new_state);
        else
            linear_step_kernel<T, 1><<<grid, 256, 0, (hipStream_t)stream>>>(q_of(shape, q), k_of(shape, k), v_of(shape, v), log_decay,
                                                                            s.scale, state, (T *)y, new_state);
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
