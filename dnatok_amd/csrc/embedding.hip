// Rows of an embedding for packed ids, y_t = scale W[id_t], and the weights' gradient, dW[v] = scale sum of dy_t over the tokens
// t of id v.  An id outside the table stands for no row: zeros, and no part of a gradient.
#include "lm_common.hpp"

#include <utility>

namespace dnatok {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Sixteen bytes of a row of `dim` elements from element `at` on, at any alignment; zeros behind the row's end.
template <typename T> struct Words {
    static constexpr int kCount = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(kCount)));
    typedef float floats __attribute__((ext_vector_type(kCount)));
};
template <typename T> __device__ __forceinline__ typename Words<T>::type load_words(const T *row, int64_t at, int64_t dim)
{
    typename Words<T>::type v{};
    if (at + Words<T>::kCount <= dim) {
        __builtin_memcpy(&v, row + at, 16);
    } else {
#pragma unroll
        for (int i = 0; i < Words<T>::kCount; ++i)
            if (at + i < dim) v[i] = row[at + i];
    }
    return v;
}
template <typename T> __device__ __forceinline__ void store_words(T *row, int64_t at, int64_t dim, typename Words<T>::type v)
{
    if (at + Words<T>::kCount <= dim) {
        __builtin_memcpy(row + at, &v, 16);
    } else {
#pragma unroll
        for (int i = 0; i < Words<T>::kCount; ++i)
            if (at + i < dim) row[at + i] = v[i];
    }
}

// Where a lane's sixteen bytes begin: the last ones of a row end with it, so that they overlap those in front of them and hold (and write)
// the same values there.  -1: none.  (Only rows of less than sixteen bytes are taken by elements.)
template <typename T> __device__ __forceinline__ int64_t word_at(int64_t word, int64_t dim)
{
    const int64_t at = word * Words<T>::kCount;
    if (at >= dim) return -1;
    return at + Words<T>::kCount > dim && dim >= Words<T>::kCount ? dim - Words<T>::kCount : at;
}
template <typename T> __device__ __forceinline__ int64_t words_at(int64_t dim)
{
    return word_at<T>((int64_t)blockIdx.y * 64 + (threadIdx.x & 63), dim);
}

// Rows that fill no more than half of a wave: 64 >> shift of them lie next to each other in it.  -1: wider ones.
static int narrow_shift(int64_t dim, int64_t size)
{
    const int64_t words = (dim * size + 15) / 16;
    if (words > 32) return -1;
    int shift = 0;
    while ((1 << shift) < words) ++shift;
    return shift;
}

// ---- rows for ids --------------------------------------------------------------------------------------

constexpr int kEmbedAhead = 8;                     // rows that a wave has under way

// A wave copies a run of tokens' rows, sixteen bytes to a lane, eight rows under way.  Bound by the writes: 524,288 rows of 512 bfloat16
// (537 MB; the table stays in the caches) 113 us, 4.75 TB/s, as much as a copy; 1,000,003 rows of 203 floats 167 us, 4.9 TB/s (147 in a training
// step, behind work that leaves fewer writes to finish).
template <typename T, typename ID>
__global__ __launch_bounds__(256) void embed_kernel(const ID *ids, int64_t n, int32_t run, const T *weight, int64_t w_stride,
                                                    int64_t vocab, int64_t dim, float scale, T *y)
{
    typedef Words<T> W;
    const int lane = threadIdx.x & 63;
    const int64_t first = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * run;
    const int64_t at = words_at<T>(dim);
    for (int64_t t0 = first; t0 < first + run && t0 < n; t0 += kEmbedAhead) {
        const int here = n - t0 < kEmbedAhead ? (int)(n - t0) : kEmbedAhead;
        int64_t mine = lane < here ? (int64_t)ids[t0 + lane] : -1;
        if (mine < 0 || mine >= vocab) mine = -1;
        const int32_t low = (int32_t)mine;         // (below 2^31, or -1)
        typename W::type v[kEmbedAhead];
#pragma unroll
        for (int i = 0; i < kEmbedAhead; ++i) {
            const int32_t id = __builtin_amdgcn_readlane(low, i);
            v[i] = typename W::type{};
            if (id >= 0 && at >= 0) v[i] = load_words(weight + id * w_stride, at, dim);
        }
#pragma unroll
        for (int i = 0; i < kEmbedAhead; ++i) {
            if (i >= here || at < 0) break;
            store_words(y + (t0 + i) * dim, at, dim,
                        __builtin_convertvector(__builtin_convertvector(v[i], typename W::floats) * scale, typename W::type));
        }
    }
}

// The same for narrow rows.  (1,000,000 rows of 16, 64, 128 and 256 bfloat16: 12, 25, 44 and 103 us, with a row to a wave 63, 63, 66 and
// 123; bytes written at the rate of a copy 7, 27, 54 and 108.)
template <typename T, typename ID>
__global__ __launch_bounds__(256) void embed_narrow_kernel(const ID *ids, int64_t n, int32_t run, int shift, const T *weight, int64_t w_stride,
                                                           int64_t vocab, int64_t dim, float scale, T *y)
{
    typedef Words<T> W;
    const int lane = threadIdx.x & 63, mine = lane >> shift, rows = 64 >> shift;
    const int64_t first = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * run, end = n - first < run ? n : first + run;
    const int64_t at = word_at<T>(lane & ((1 << shift) - 1), dim);
    for (int64_t t0 = first + mine; t0 < end; t0 += kEmbedAhead * rows) {
        int64_t id[kEmbedAhead];
        typename W::type v[kEmbedAhead];
#pragma unroll
        for (int i = 0; i < kEmbedAhead; ++i) id[i] = t0 + i * rows < end ? (int64_t)ids[t0 + i * rows] : -1;
#pragma unroll
        for (int i = 0; i < kEmbedAhead; ++i) {
            v[i] = typename W::type{};
            if (id[i] >= 0 && id[i] < vocab && at >= 0) v[i] = load_words(weight + id[i] * w_stride, at, dim);
        }
#pragma unroll
        for (int i = 0; i < kEmbedAhead; ++i)
            if (t0 + i * rows < end && at >= 0)
                store_words(y + (t0 + i * rows) * dim, at, dim,
                            __builtin_convertvector(__builtin_convertvector(v[i], typename W::floats) * scale, typename W::type));
    }
}

// ---- tokens sorted by id -----------------------------------------------------------------------------

// Keys are ids, those outside the table the number behind its last row.  A pass sorts by up to eight of their bits: a workgroup
// counts its tile's digits, a scan gives each tile its place for each digit, and a workgroup writes its tile there, the tokens of one
// digit in their order.  So tokens of one id stay in their order, and a sum over them is the same in every call.  Tiles of 1,024 tokens:
// a pass over 262,144 takes 5 + 3 + 7 us.  (Tiles of 8,192 leave CUs without work: 40,000 tokens and 32,000 ids 107 us for the whole
// gradient instead of 46, 262,144 159 instead of 95, 8,000,000 450 instead of 433; the same dy each time, partly in the cache behind L2.)
constexpr int kSortThreads = 256, kSortWaves = kSortThreads / 64, kDigits = 256;
constexpr int kSortPerLane = 4, kSortTile = kSortThreads * kSortPerLane;
constexpr int kSmallSort = 8192, kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64;

struct Token {
    uint32_t key, at;
};

template <typename ID> __device__ __forceinline__ uint32_t key_of(ID id, uint32_t vocab)
{
    return id >= 0 && (uint64_t)id < vocab ? (uint32_t)id : vocab;
}
// The lanes with this lane's digit.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool here)
{
    uint64_t same = __ballot(here);
    for (int b = 0; b < bits; ++b) {
        const uint64_t one = __ballot(digit >> b & 1);
        same &= digit >> b & 1 ? one : ~one;
    }
    return same;
}

template <typename ID>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const ID *ids, const Token *tokens, uint32_t n, uint32_t vocab,
                                                                  int shift, int bits, uint32_t *counts)
{
    __shared__ uint32_t count[kDigits];
    for (int i = threadIdx.x; i < kDigits; i += kSortThreads) count[i] = 0;
    __syncthreads();
    const uint32_t first = blockIdx.x * kSortTile, mask = (1u << bits) - 1;
    const int lane = threadIdx.x & 63;
    uint32_t key[kSortPerLane];
#pragma unroll
    for (int j = 0; j < kSortPerLane; ++j) {
        const uint32_t i = first + j * kSortThreads + threadIdx.x;
        key[j] = i < n ? (ids ? key_of(ids[i], vocab) : tokens[i].key) : 0;
    }
#pragma unroll
    for (int j = 0; j < kSortPerLane; ++j) {
        const bool here = first + j * kSortThreads + threadIdx.x < n;
        const uint32_t digit = key[j] >> shift & mask;
        const uint64_t same = same_digit(digit, bits, here);
        if (here && (same & ((1ull << lane) - 1)) == 0) atomicAdd(&count[digit], (uint32_t)__popcll(same));
    }
    __syncthreads();
    for (int i = threadIdx.x; i <= (int)mask; i += kSortThreads) counts[(size_t)i * gridDim.x + blockIdx.x] = count[i];
}

// A workgroup to a digit: its tiles' counts become what lies in front of them, and their sum is left in totals.
__global__ __launch_bounds__(256) void sort_scan_kernel(uint32_t *counts, uint32_t tiles, uint32_t *totals)
{
    __shared__ uint32_t part[4];
    uint32_t *mine = counts + (size_t)blockIdx.x * tiles;
    uint32_t before = 0;
    for (uint32_t t0 = 0; t0 < tiles; t0 += 256) {
        const uint32_t t = t0 + threadIdx.x, v = t < tiles ? mine[t] : 0;
        const uint32_t upto = wave_inclusive_sum_u32(v);
        if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = upto;
        __syncthreads();
        uint32_t front = before;
        for (unsigned w = 0; w < threadIdx.x >> 6; ++w) front += part[w];
        if (t < tiles) mine[t] = front + upto - v;
        before += part[0] + part[1] + part[2] + part[3];
        __syncthreads();
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

template <typename ID>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(const ID *ids, const Token *tokens, uint32_t n, uint32_t vocab,
                                                                  int shift, int bits, const uint32_t *counts, const uint32_t *totals,
                                                                  Token *out)
{
    __shared__ uint32_t place[kSortWaves][kDigits], part[4];
    constexpr int kPerLane = kSortPerLane;
    const uint32_t mask = (1u << bits) - 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < kSortWaves * kDigits; i += kSortThreads) place[0][i] = 0;
    __syncthreads();
    // a wave has neighbouring tokens, 64 at a time
    const uint32_t first = blockIdx.x * kSortTile + wave * (64 * kPerLane);
    uint32_t key[kPerLane], at[kPerLane];
    uint64_t same[kPerLane];
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) {
        const uint32_t i = first + j * 64 + lane;
        at[j] = i;
        key[j] = 0;
        if (i < n) {
            if (ids) {
                key[j] = key_of(ids[i], vocab);
            } else {
                const Token t = tokens[i];
                key[j] = t.key;
                at[j] = t.at;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) {
        const bool here = first + j * 64 + lane < n;
        const uint32_t digit = key[j] >> shift & mask;
        same[j] = same_digit(digit, bits, here);
        if (here && (same[j] & ((1ull << lane) - 1)) == 0) atomicAdd(&place[wave][digit], (uint32_t)__popcll(same[j]));
    }
    __syncthreads();
    {   // the digits' places: in front of all of them, of the tile, of the waves
        const uint32_t d = threadIdx.x, all = d <= mask ? totals[d] : 0;
        const uint32_t upto = wave_inclusive_sum_u32(all);
        if (lane == 63) part[wave] = upto;
        __syncthreads();
        uint32_t from = upto - all;
        for (int w = 0; w < wave; ++w) from += part[w];
        if (d <= mask) {
            from += counts[(size_t)d * gridDim.x + blockIdx.x];
            for (int w = 0; w < kSortWaves; ++w) {
                const uint32_t here = place[w][d];
                place[w][d] = from;
                from += here;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) {
        const bool here = first + j * 64 + lane < n;
        const uint32_t digit = key[j] >> shift & mask;
        const uint64_t before = same[j] & ((1ull << lane) - 1);
        const uint32_t from = here ? place[wave][digit] : 0;
        __builtin_amdgcn_wave_barrier();
        if (here) {
            out[from + __popcll(before)] = Token{key[j], at[j]};
            if (before == 0) place[wave][digit] = from + __popcll(same[j]);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// Up to kSmallSort tokens in one workgroup: the same passes in LDS, one launch instead of six.  (The whole gradient for 2,500 and 8,000
// tokens, 32,000 rows of 512 bfloat16: 30 and 35 us, with launches of their own 37 and 39.)
template <typename ID>
__global__ __launch_bounds__(kSmallThreads) void sort_small_kernel(const ID *ids, uint32_t n, uint32_t vocab, int passes, int bits,
                                                                   Token *out)
{
    __shared__ uint32_t place[kSmallWaves][kDigits], part[kSmallWaves];
    __shared__ Token token[kSmallSort];
    constexpr int kPerLane = kSmallSort / kSmallThreads;
    const uint32_t mask = (1u << bits) - 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t each = ((n + kSmallThreads - 1) / kSmallThreads) * 64, first = wave * each;
    for (uint32_t i = threadIdx.x; i < n; i += kSmallThreads) token[i] = Token{key_of(ids[i], vocab), i};
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * bits;
        for (int i = threadIdx.x; i < kSmallWaves * kDigits; i += kSmallThreads) place[0][i] = 0;
        __syncthreads();
        Token mine[kPerLane];
        uint64_t same[kPerLane];
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) {
            const uint32_t i = first + j * 64 + lane;
            const bool here = (uint32_t)j * 64 < each && i < n;
            mine[j] = here ? token[i] : Token{0, 0};
            const uint32_t digit = mine[j].key >> shift & mask;
            same[j] = same_digit(digit, bits, here);
            if (here && (same[j] & ((1ull << lane) - 1)) == 0) atomicAdd(&place[wave][digit], (uint32_t)__popcll(same[j]));
        }
        __syncthreads();
        uint32_t all = 0;
        if (threadIdx.x < kDigits)
            for (int w = 0; w < kSmallWaves; ++w) all += place[w][threadIdx.x];
        const uint32_t upto = wave_inclusive_sum_u32(all);
        if (lane == 63) part[wave] = upto;
        __syncthreads();
        if (threadIdx.x < kDigits) {
            uint32_t from = upto - all;
            for (int w = 0; w < wave; ++w) from += part[w];
            for (int w = 0; w < kSmallWaves; ++w) {
                const uint32_t here = place[w][threadIdx.x];
                place[w][threadIdx.x] = from;
                from += here;
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) {
            const bool here = (uint32_t)j * 64 < each && first + j * 64 + lane < n;
            const uint32_t digit = mine[j].key >> shift & mask;
            const uint64_t before = same[j] & ((1ull << lane) - 1);
            const uint32_t from = here ? place[wave][digit] : 0;
            __builtin_amdgcn_wave_barrier();
            if (here) {
                token[from + __popcll(before)] = mine[j];
                if (before == 0) place[wave][digit] = from + __popcll(same[j]);
            }
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
    }
    for (uint32_t i = threadIdx.x; i < n; i += kSmallThreads) out[i] = token[i];
}

// ---- sums over the tokens of an id -------------------------------------------------------------------

constexpr int kGradAhead = 8;                      // rows of dy that a wave has under way
constexpr int kZeroRows = 64;                      // rows of the gradient that a wave looks at for ids that do not occur

// (The pointers that are written through are arguments of their own: kept in here, the compiler at times no longer knew that they
// point to memory.)
struct GradArgs {
    const Token *tokens;
    uint32_t n, vocab, tiles;
    int32_t run;                                   // tokens of a tile, a power of two
    const void *dy;
    int64_t dy_stride, dim;
    float scale;
};

// The first token whose key is not below `key`.
__device__ __forceinline__ uint32_t first_of(const Token *tokens, uint32_t n, uint32_t key)
{
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (tokens[mid].key < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// The rows of ids that do not occur, for a wave's kZeroRows rows.
template <typename T> __device__ __forceinline__ void clear_absent(const GradArgs &a, uint32_t rows, T *grad)
{
    const int lane = threadIdx.x & 63;
    const int64_t at = words_at<T>(a.dim);
    const uint32_t row = rows * kZeroRows + lane;
    bool empty = row < a.vocab;
    if (empty) {
        const uint32_t i = first_of(a.tokens, a.n, row);
        empty = i == a.n || a.tokens[i].key != row;
    }
    uint64_t left = __ballot(empty);
    while (left) {
        const int i = __builtin_ctzll(left);
        left &= left - 1;
        if (at >= 0) store_words(grad + (int64_t)(row - lane + i) * a.dim, at, a.dim, typename Words<T>::type{});
    }
}

// A lane's part of a run's sum: a row of the gradient, or of `part` if the run goes on outside of the tile.
template <typename T> __device__ __forceinline__ void put_sum(const GradArgs &a, uint32_t key, bool goes_on, float *part, T *grad, int64_t at,
                                                              const typename Words<T>::floats &sum)
{
    typedef Words<T> W;
    if (key >= a.vocab || at < 0) return;
    if (!goes_on) {
        store_words(grad + (int64_t)key * a.dim, at, a.dim, __builtin_convertvector(sum * a.scale, typename W::type));
    } else if (at + W::kCount <= a.dim) {
        __builtin_memcpy(part + at, &sum, sizeof(sum));
    } else {
#pragma unroll
        for (int i = 0; i < W::kCount; ++i)
            if (at + i < a.dim) part[at + i] = sum[i];
    }
}

// A wave to a tile of the sorted tokens and 64 x 16 bytes of their rows: it adds up runs of one id.  A run inside the tile is a
// row of the gradient; one that goes on in front of the tile or behind it leaves its sum in parts [tiles, 2, dim].  Further waves clear the
// rows of ids that do not occur.  Eight rows of dy under way: 262,144 rows of 512 bfloat16 in the order of 32,000 ids 89 us (301 MB,
// 3.4 TB/s), 1,000,003 rows of 203 floats and 12 ids 227 us (812 MB, 3.6 TB/s).  (Sixteen rows under way: the whole gradient of 262,144 rows
// takes 134 us instead of 95.)
template <typename T> __global__ __launch_bounds__(256) void embed_grad_kernel(GradArgs a, float *parts, T *grad)
{
    typedef Words<T> W;
    const int lane = threadIdx.x & 63;
    const int64_t at = words_at<T>(a.dim);
    const uint32_t tile = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= (a.tiles + 3) / 4 * 4) {
        clear_absent(a, tile - (a.tiles + 3) / 4 * 4, grad);
        return;
    }
    if (tile >= a.tiles) return;
    const uint32_t begin = tile * a.run, end = a.n - begin < (uint32_t)a.run ? a.n : begin + a.run;
    const uint32_t front = begin ? a.tokens[begin - 1].key : ~0u, back = end < a.n ? a.tokens[end].key : ~0u;
    typename W::floats sum{};
    uint32_t key = a.tokens[begin].key;
    bool from_front = key == front;
    const auto finish = [&](bool goes_on) {
        put_sum<T>(a, key, from_front || goes_on, parts + ((int64_t)tile * 2 + !from_front) * a.dim, grad, at, sum);
    };
    for (uint32_t t0 = begin; t0 < end; t0 += 64) {
        const uint32_t mine_at = t0 + lane < end ? t0 + lane : end - 1;
        const Token mine = a.tokens[mine_at];
        for (int j0 = 0; j0 < 64 && t0 + j0 < end; j0 += kGradAhead) {
            typename W::type v[kGradAhead];
#pragma unroll
            for (int i = 0; i < kGradAhead; ++i) {
                const uint32_t row = __builtin_amdgcn_readlane(mine.at, j0 + i);
                v[i] = typename W::type{};
                if (at >= 0) v[i] = load_words((const T *)a.dy + (int64_t)row * a.dy_stride, at, a.dim);
            }
            const int here = end - t0 - j0 < (uint32_t)kGradAhead ? (int)(end - t0 - j0) : kGradAhead;
#pragma unroll
            for (int i = 0; i < kGradAhead; ++i) {
                if (i < here) {
                    const uint32_t next = __builtin_amdgcn_readlane(mine.key, j0 + i);
                    if (next != key) {
                        finish(false);
                        key = next;
                        from_front = false;
                        sum = typename W::floats{};
                    }
                    sum += __builtin_convertvector(v[i], typename W::floats);
                }
            }
        }
    }
    finish(key == back);
}

// The same for rows that fill no more than a quarter of a wave: 64 >> shift tiles to a wave, each with as many of its lanes.  (1,000,000 x 64
// bfloat16: 32 us, with a tile to a wave and twice the tiles 60; of two rows to a wave 1,000,000 x 192 takes 160 us instead of 157.)
template <typename T> __global__ __launch_bounds__(256) void embed_grad_narrow_kernel(GradArgs a, int shift, float *parts, T *grad)
{
    typedef Words<T> W;
    const int lane = threadIdx.x & 63, rows = 64 >> shift;
    const uint32_t blocks = (a.tiles + rows * 4 - 1) / (rows * 4);
    if (blockIdx.x >= blocks) {
        clear_absent(a, (blockIdx.x - blocks) * 4 + (threadIdx.x >> 6), grad);
        return;
    }
    const uint32_t tile = (blockIdx.x * 4 + (threadIdx.x >> 6)) * rows + (lane >> shift);
    if (tile >= a.tiles) return;
    const int64_t at = word_at<T>(lane & ((1 << shift) - 1), a.dim);
    const uint32_t begin = tile * a.run, end = a.n - begin < (uint32_t)a.run ? a.n : begin + a.run;
    const uint32_t front = begin ? a.tokens[begin - 1].key : ~0u, back = end < a.n ? a.tokens[end].key : ~0u;
    typename W::floats sum{};
    Token coming[kGradAhead];
#pragma unroll
    for (int i = 0; i < kGradAhead; ++i) coming[i] = a.tokens[begin + i < end ? begin + i : end - 1];
    uint32_t key = coming[0].key;
    bool from_front = key == front;
    const auto finish = [&](bool goes_on) {
        put_sum<T>(a, key, from_front || goes_on, parts + ((int64_t)tile * 2 + !from_front) * a.dim, grad, at, sum);
    };
    for (uint32_t t0 = begin; t0 < end; t0 += kGradAhead) {
        Token token[kGradAhead];
        typename W::type v[kGradAhead];
#pragma unroll
        for (int i = 0; i < kGradAhead; ++i) {
            token[i] = coming[i];
            v[i] = typename W::type{};
            if (at >= 0) v[i] = load_words((const T *)a.dy + (int64_t)token[i].at * a.dy_stride, at, a.dim);
        }
#pragma unroll
        for (int i = 0; i < kGradAhead; ++i) {
            const uint32_t t = t0 + kGradAhead + i;
            coming[i] = a.tokens[t < end ? t : end - 1];
        }
#pragma unroll
        for (int i = 0; i < kGradAhead; ++i) {
            if (t0 + i >= end) break;
            if (token[i].key != key) {
                finish(false);
                key = token[i].key;
                from_front = false;
                sum = typename W::floats{};
            }
            sum += __builtin_convertvector(v[i], typename W::floats);
        }
    }
    finish(key == back);
}

// Few tokens: a wave to a row of the gradient looks through all of their ids, and adds up what it finds.  One launch and no sort: 128
// tokens take 4.1, 4.1 and 9.8 us with 12, 4,096 and 32,000 rows of 512 bfloat16 (sorted 14.4, 22.4 and 25.4), and where all are
// one id, which one wave then adds up, 16.4, 16.9 and 23.2 (15.2, 25.2 and 27.8); 256 of one id take 31 (17 with 12 rows, 27 with 4,096).
constexpr int kFewTokens = 128;
template <typename T, typename ID>
__global__ __launch_bounds__(256) void embed_grad_few_kernel(const ID *ids, uint32_t n, const T *dy, int64_t dy_stride, int64_t vocab,
                                                             int64_t dim, float scale, T *grad)
{
    typedef Words<T> W;
    const int lane = threadIdx.x & 63;
    const int64_t at = words_at<T>(dim);
    for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < vocab; row += (int64_t)gridDim.x * 4) {
        typename W::floats sum{};
        for (uint32_t t0 = 0; t0 < n; t0 += 64) {
            uint64_t found = __ballot(t0 + lane < n && (int64_t)ids[t0 + lane < n ? t0 + lane : 0] == row);
            while (found) {
                typename W::type v[kGradAhead];
#pragma unroll
                for (int i = 0; i < kGradAhead; ++i) {
                    v[i] = typename W::type{};
                    if (found && at >= 0) v[i] = load_words(dy + (int64_t)(t0 + __builtin_ctzll(found)) * dy_stride, at, dim);
                    found &= found - 1;
                }
#pragma unroll
                for (int i = 0; i < kGradAhead; ++i) sum += __builtin_convertvector(v[i], typename W::floats);
            }
        }
        if (at >= 0) store_words(grad + row * dim, at, dim, __builtin_convertvector(sum * scale, typename W::type));
    }
}

// Runs that begin in one tile and end in another: their parts, added up in order.  A wave to a tile looks whether such a run begins there,
// and adds it up by itself if it ends less than sixteen tiles on; a longer one is added up by the workgroup's waves and then in
// their order.  (With a workgroup to each tile 7,800 tiles took 38 us, most of them to begin waves that leave at once.)
constexpr int kJoinWaves = 16, kJoinAhead = 8;
template <typename T> __global__ __launch_bounds__(kJoinWaves * 64) void embed_join_kernel(GradArgs a, const float *parts, T *grad)
{
    typedef Words<T> W;
    __shared__ typename W::floats part[kJoinWaves][64];
    __shared__ uint32_t lasts[kJoinWaves], keys[kJoinWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t at = words_at<T>(a.dim);
    const auto piece = [&](uint32_t t, uint32_t first, uint32_t last) {
        typename W::floats v{};
        if (t <= last && at >= 0) {
            const float *p = parts + ((int64_t)t * 2 + (t == first)) * a.dim;
            if (at + W::kCount <= a.dim) {
                __builtin_memcpy(&v, p + at, sizeof(v));
            } else {
#pragma unroll
                for (int i = 0; i < W::kCount; ++i)
                    if (at + i < a.dim) v[i] = p[at + i];
            }
        }
        return v;
    };
    const auto put = [&](uint32_t key, const typename W::floats &sum) {
        if (at >= 0) store_words(grad + (int64_t)key * a.dim, at, a.dim, __builtin_convertvector(sum * a.scale, typename W::type));
    };
    // the last tile of the run that ends this one, if it begins here and goes on: it begins there, behind the tile's begin or at it with
    // another id in front
    const auto find = [&](uint32_t tile, uint32_t *of) -> uint32_t {
        const uint32_t begin = tile * (uint32_t)a.run, end = begin + (uint32_t)a.run;
        if (end >= a.n) return 0;
        const uint32_t next = end + (uint32_t)a.run < a.n ? end + (uint32_t)a.run : a.n - 1;
        const uint32_t key = a.tokens[end].key, mine = a.tokens[end - 1].key, head = a.tokens[begin].key,
                       front = begin ? a.tokens[begin - 1].key : ~0u, after = a.tokens[next].key;
        if (key >= a.vocab || mine != key || (head == key && front == key)) return 0;
        *of = key;
        if (after != key) return tile + 1;
        uint32_t lo = next, hi = a.n;              // the last token of the id, 64 places at once (lo has it, hi does not)
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo - 1 + 63) / 64, place = lo + step * (lane + 1);
            const int n = __popcll(__ballot(place < hi && a.tokens[place < hi ? place : lo].key == key));
            lo += step * n;
            hi = hi - lo > step ? lo + step : hi;
        }
        return lo / (uint32_t)a.run;
    };
    const uint32_t own = blockIdx.x * kJoinWaves + wave;
    uint32_t key = 0, last = own < a.tiles ? find(own, &key) : 0;
    if (last && last - own < kJoinWaves) {
        typename W::floats sum{};
        for (uint32_t t = own; t <= last; t += 2) {
            const auto v = piece(t, own, last), u = piece(t + 1, own, last);
            sum += v;
            sum += u;
        }
        put(key, sum);
        last = 0;
    }
    if (lane == 0) {
        lasts[wave] = last;
        keys[wave] = key;
    }
    __syncthreads();
    for (int w = 0; w < kJoinWaves; ++w) {
        const uint32_t first = blockIdx.x * kJoinWaves + w;
        last = lasts[w];
        if (!last) continue;
        typename W::floats sum{};
        for (uint32_t t = first + wave; t <= last; t += kJoinWaves * kJoinAhead) {
            typename W::floats v[kJoinAhead];
#pragma unroll
            for (int i = 0; i < kJoinAhead; ++i) v[i] = piece(t + i * kJoinWaves, first, last);
#pragma unroll
            for (int i = 0; i < kJoinAhead; ++i) sum += v[i];
        }
        part[wave][lane] = sum;
        __syncthreads();
        if (wave == 0) {
            for (int i = 1; i < kJoinWaves; ++i) sum += part[i][lane];
            put(keys[w], sum);
        }
        __syncthreads();
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
    DNATOK_REQUIRE(n < (1ll << 31) && vocab < (1ll << 31) - 1 && dim <= (1ll << 22), DNATOK_E_TOO_LARGE,
                   "%s: at most 2^31 tokens and rows of 2^22 elements", who);
    return DNATOK_OK;
}

// Blocks of 64 x 16 bytes of a row.
static int64_t blocks_of(int64_t dim, int64_t size) { return (dim * size + 1023) / 1024; }

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
    EMBED_REQUIRE(__builtin_isfinite(scale), "the scale must be finite");
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        with_ids(id_bytes, [&](auto i) {
            using ID = decltype(i);
            // two rounds of rows to a wave, or one if that takes no more than 32,768 waves (524,288 rows of 512 bfloat16: 112.9 us with
            // two, 114.2 with one, 116.1 with four; 1,000,003 of 203 floats: 167 with two, 161 with one, 181 with four)
            const int shift = narrow_shift(dim, sizeof(T));
            if (shift >= 0) {
                const int64_t once = kEmbedAhead * (64 >> shift);
                int64_t run = n <= 32768 * once ? once : 2 * once;
                while (n / run > (1 << 22)) run *= 2;
                embed_narrow_kernel<T, ID><<<(unsigned)((n + run * 4 - 1) / (run * 4)), 256, 0, (hipStream_t)stream>>>(
                    (const ID *)ids, n, (int32_t)run, shift, (const T *)weight, weight_stride, vocab, dim, scale, (T *)y);
                return;
            }
            const int64_t blocks = blocks_of(dim, sizeof(T));
            int64_t run = n * blocks <= 32768 * kEmbedAhead ? kEmbedAhead : 2 * kEmbedAhead;
            while (n / run > (1 << 22)) run *= 2;  // (a grid ends at 2^32 threads)
            embed_kernel<T, ID><<<dim3((unsigned)((n + run * 4 - 1) / (run * 4)), (unsigned)blocks), 256, 0, (hipStream_t)stream>>>(
                (const ID *)ids, n, (int32_t)run, (const T *)weight, weight_stride, vocab, dim, scale, (T *)y);
        });
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}

// What the backward pass needs besides its arguments: tokens sorted by id (twice, where they go from one place to the other), counts of
// digits, and parts of sums.
struct GradPlan {
    uint32_t tiles, sort_tiles;
    int32_t run, passes, bits;
    size_t other, counts, totals, parts, bytes;    // offsets
};
static GradPlan plan_of(int64_t n, int64_t vocab, int64_t dim)
{
    GradPlan p{};
    int bits = 1;
    while ((vocab >> bits) != 0) ++bits;           // (keys go up to vocab itself)
    p.passes = (bits + 7) / 8;
    p.bits = (bits + p.passes - 1) / p.passes;
    p.sort_tiles = (uint32_t)((n + kSortTile - 1) / kSortTile);
    // about 2,048 waves of wide rows, of 16-bit elements, or 1,024 with several narrow ones: shorter tiles write more parts of sums, longer
    // ones leave CUs without work (the whole gradient, bfloat16, ids of falling frequency, the same dy each time, partly in the cache behind
    // L2: 262,144 x 512, 32,000 ids, 95 us, with half or twice the waves 111 and 97; 1,000,003 x 203, 12 ids, 149, 167 and 172;
    // 1,000,000 x 64, 4,096 ids, 86, with half 106; 8,000,000 x 32, 32,000 ids, 433, 545 and 438)
    const int64_t narrow = (1 << 19) / (dim < 32 ? 32 : dim), wide = (1 << 20) / (dim < 128 ? 128 : dim);
    p.run = 16;
    while (p.run < (1 << 20) && n / p.run > (narrow > wide ? narrow : wide)) p.run *= 2;
    p.tiles = (uint32_t)((n + p.run - 1) / p.run);
    const bool small = n <= kSmallSort;
    const auto place = [&](size_t bytes) {
        const size_t at = p.bytes;
        p.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    place((size_t)n * sizeof(Token));
    p.other = place(small ? 0 : (size_t)n * sizeof(Token));
    p.counts = place(small ? 0 : (size_t)p.sort_tiles * kDigits * 4);
    p.totals = place(small ? 0 : kDigits * 4);
    p.parts = place((size_t)p.tiles * 2 * dim * 4);
    return p;
}

extern "C" size_t dnatok_embedding_work_bytes(int64_t n, int64_t vocab, int64_t dim)
{
    return n > kFewTokens && vocab > 0 && dim > 0 ? plan_of(n, vocab, dim).bytes : 0;
}

template <typename ID>
static const Token *sort_tokens(const ID *ids, uint32_t n, uint32_t vocab, const GradPlan &p, char *work, hipStream_t s)
{
    Token *from = (Token *)work, *to = (Token *)(work + p.other);
    if (n <= kSmallSort) {
        sort_small_kernel<ID><<<1, kSmallThreads, 0, s>>>(ids, n, vocab, p.passes, p.bits, from);
        return from;
    }
    uint32_t *counts = (uint32_t *)(work + p.counts), *totals = (uint32_t *)(work + p.totals);
    for (int pass = 0; pass < p.passes; ++pass) {
        const ID *source = pass ? nullptr : ids;
        sort_count_kernel<ID><<<p.sort_tiles, kSortThreads, 0, s>>>(source, from, n, vocab, pass * p.bits, p.bits, counts);
        sort_scan_kernel<<<1u << p.bits, 256, 0, s>>>(counts, p.sort_tiles, totals);
        sort_place_kernel<ID><<<p.sort_tiles, kSortThreads, 0, s>>>(source, from, n, vocab, pass * p.bits, p.bits, counts, totals, to);
        std::swap(from, to);
    }
    return from;
}

extern "C" int dnatok_embedding_backward(const void *ids, int32_t id_bytes, int64_t n, const void *dy, int64_t dy_stride, int32_t dtype,
                                         int64_t vocab, int64_t dim, const float *scale_h, void *grad, void *work, size_t work_bytes,
                                         void *stream)
{
    static const char *who = "dnatok_embedding_backward";
    if (int rc = check_embedding(who, id_bytes, n, dy_stride, dtype, vocab, dim)) return rc;
    if (vocab == 0 || dim == 0) return DNATOK_OK;
    EMBED_REQUIRE((n == 0 || (ids && dy)) && grad && scale_h, "null buffer");
    EMBED_REQUIRE(work_bytes >= dnatok_embedding_work_bytes(n, vocab, dim) && (work || !work_bytes), "work space too small");
    EMBED_REQUIRE((uintptr_t)work % 16 == 0, "work space must be 16-byte aligned");
    const float scale = *scale_h;
    EMBED_REQUIRE(__builtin_isfinite(scale), "the scale must be finite");
    hipStream_t s = (hipStream_t)stream;
    if (n <= kFewTokens) {
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            with_ids(id_bytes, [&](auto i) {
                using ID = decltype(i);
                const unsigned rows = (unsigned)(vocab < 65536 * 4 ? (vocab + 3) / 4 : 65536);
                embed_grad_few_kernel<T, ID><<<dim3(rows, (unsigned)blocks_of(dim, sizeof(T))), 256, 0, s>>>(
                    (const ID *)ids, (uint32_t)n, (const T *)dy, dy_stride, vocab, dim, scale, (T *)grad);
            });
        });
        DNATOK_HIP_TRY(hipGetLastError());
        return DNATOK_OK;
    }
    const GradPlan p = plan_of(n, vocab, dim);
    const Token *tokens = nullptr;
    with_ids(id_bytes, [&](auto i) {
        using ID = decltype(i);
        tokens = sort_tokens((const ID *)ids, (uint32_t)n, (uint32_t)vocab, p, (char *)work, s);
    });
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        const GradArgs a{tokens, (uint32_t)n, (uint32_t)vocab, p.tiles, p.run, dy, dy_stride, dim, scale};
        float *parts = (float *)((char *)work + p.parts);
        const unsigned blocks = (unsigned)blocks_of(dim, sizeof(T)), zeros = (unsigned)((vocab + kZeroRows * 4 - 1) / (kZeroRows * 4));
        const int shift = narrow_shift(dim, sizeof(T));
        if (shift >= 0 && shift <= 4) {
            const unsigned each = 4 * (64 >> shift);
            embed_grad_narrow_kernel<T><<<(p.tiles + each - 1) / each + zeros, 256, 0, s>>>(a, shift, parts, (T *)grad);
        } else {
            embed_grad_kernel<T><<<dim3((p.tiles + 3) / 4 + zeros, blocks), 256, 0, s>>>(a, parts, (T *)grad);
        }
        if (p.tiles > 1)
            embed_join_kernel<T><<<dim3((p.tiles - 1 + kJoinWaves - 1) / kJoinWaves, blocks), kJoinWaves * 64, 0, s>>>(a, parts, (T *)grad);
    });
    DNATOK_HIP_TRY(hipGetLastError());
    return DNATOK_OK;
}
