// Keys and values appended to the paged int8 cache, keys (and queries) rotated on the way.
//
// A block of the cache (one page of one KV head) holds int8 values times one power of two 2^e. With
// the new tokens' largest magnitude a, e has to satisfy a <= 127 * 2^e: with a = f * 2^x, f in [1/2, 1),
// that is x - 7 for f <= 127/128 and x - 6 otherwise. A block that is continued keeps the larger of
// this and the exponent it has; when it grows, the integers held already are shifted right with
// rounding to nearest even. Rotation and quantisation are evaluated in double (two exact products and
// one sum): a value next to the border between two integers falls the right way.
#include "paged.hpp"

namespace rmlk {
namespace {

constexpr int kThreads = 256;
constexpr int kLowestExponent = -126;

template <typename T>
struct AppendArgs {
    PagedArgs c;
    const T *k, *v, *q;
    T *q_out;
    const float *cos, *sin;
    int64_t k_stride, v_stride, q_stride;
    int64_t positions;
    int32_t heads;
    int32_t pieces;      // upper bound of (sequence, page) pairs: the first blocks of the grid, per KV head
    int64_t q_units;     // rows * heads * D / 16 units of q
};

// The pages that sequence s writes to, at most fresh / page_size + 2, are numbered from
// first[s] / page_size + 2 s: no two sequences share a number, and the grid need not be a rectangle
// over the longest sequence.

__device__ __forceinline__ double block_max(double v, double *lds) {
    v = wave_max(v);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    double r = lds[0];
    for (int i = 1; i < kThreads / kWave; ++i) r = lds[i] > r ? lds[i] : r;
    __syncthreads();
    return r;
}

__device__ __forceinline__ int exponent_for(double a) {
    if (a == 0.0) return kLowestExponent;
    int x;
    const double f = frexp(a, &x);
    const int e = f <= 127.0 / 128.0 ? x - 7 : x - 6;
    return max(kLowestExponent, min(127, e));
}

__device__ __forceinline__ int8_t to_step(double x, int e) {
    const int n = static_cast<int>(rint(ldexp(x, -e)));
    return static_cast<int8_t>(min(127, max(-127, n)));
}

template <typename T, int D>
__device__ __forceinline__ double rotated(const AppendArgs<T> &g, const T *row, int64_t pos, int d) {
    const double x = to_float(row[d]);
    if (!g.cos) return x;
    const double other = d < D / 2 ? -to_float(row[d + D / 2]) : to_float(row[d - D / 2]);
    return x * static_cast<double>(g.cos[pos * D + d]) + other * static_cast<double>(g.sin[pos * D + d]);
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(AppendArgs<T> g) {
    __shared__ double lds[kThreads / kWave];
    const int tid = threadIdx.x;
    const int kv_blocks = g.pieces * g.c.kv_heads;
    if (!starts_ascend(g.c)) {
        if (blockIdx.x == 0 && tid == 0) raise_error(g.c);
        return;
    }
    if (static_cast<int>(blockIdx.x) >= kv_blocks) {
        // queries: one element per thread and trip
        const int64_t total = g.c.rows * g.heads * D;
        for (int64_t i = (static_cast<int64_t>(blockIdx.x) - kv_blocks) * kThreads + tid; i < total;
             i += static_cast<int64_t>(gridDim.x - kv_blocks) * kThreads) {
            const int d = static_cast<int>(i % (D / 2));
            if (i % D >= D / 2) continue;
            const int64_t rh = i / D;
            const int64_t row = rh / g.heads;
            const int h = static_cast<int>(rh % g.heads);
            Sequence q;
            if (!sequence_at(g.c, sequence_of_row(g.c, row), q) || q.length < q.fresh || row < q.row ||
                row >= q.row + q.fresh)
                continue;
            const int64_t pos = q.length - q.fresh + (row - q.row);
            if (g.cos && pos >= g.positions) continue;
            const T *src = g.q + row * g.q_stride + static_cast<int64_t>(h) * D;
            const double a = rotated<T, D>(g, src, pos, d), b = rotated<T, D>(g, src, pos, d + D / 2);
            T *dst = g.q_out + (row * g.heads + h) * D;
            dst[d] = static_cast<T>(a);
            dst[d + D / 2] = static_cast<T>(b);
        }
        return;
    }
    const int piece = blockIdx.x / g.c.kv_heads, head = blockIdx.x % g.c.kv_heads;
    const int s = sequence_of(g.c, piece, 1 << g.c.page_shift, 2);
    if (s < 0) return;
    const int index = piece - ((g.c.first[s] >> g.c.page_shift) + 2 * s);   // of the pages it writes to
    Sequence q;
    if (!sequence_at(g.c, s, q) || q.length < q.fresh) {
        if (index == 0 && head == 0 && tid == 0) raise_error(g.c);
        return;
    }
    const int size = 1 << g.c.page_shift;
    const int begin_pos = q.length - q.fresh;
    const int64_t page_at = static_cast<int64_t>(begin_pos >> g.c.page_shift) + index;   // in the table
    const int64_t page_pos = page_at << g.c.page_shift;
    if (q.fresh == 0 || page_pos >= q.length) return;
    const int slot0 = page_pos < begin_pos ? static_cast<int>(begin_pos - page_pos) : 0;
    int slot1 = min(static_cast<int64_t>(size), q.length - page_pos);
    const int32_t page = g.c.table[s * g.c.table_stride + page_at];
    if (page < 0 || page >= g.c.pages) {
        if (tid == 0) raise_error(g.c);
        return;
    }
    if (g.cos && page_pos + slot1 > g.positions) {
        if (tid == 0) raise_error(g.c);
        slot1 = static_cast<int>(max(static_cast<int64_t>(slot0), g.positions - page_pos));
        if (slot1 == slot0) return;
    }
    const int tokens = slot1 - slot0;
    const int64_t row0 = q.row + (page_pos + slot0 - begin_pos);
    const int64_t block = static_cast<int64_t>(page) * g.c.kv_heads + head;
    for (int which = 0; which < 2; ++which) {
        const T *src = which ? g.v + row0 * g.v_stride : g.k + row0 * g.k_stride;
        const int64_t stride = which ? g.v_stride : g.k_stride;
        src += static_cast<int64_t>(head) * D;
        int8_t *dst = (which ? g.c.v : g.c.k) + block * size * D;
        float *scale = (which ? g.c.v_scale : g.c.k_scale) + block;
        auto value = [&](int t, int d) {
            const T *row = src + t * stride;
            return which ? static_cast<double>(to_float(row[d])) : rotated<T, D>(g, row, page_pos + slot0 + t, d);
        };
        auto at = [&](int slot, int d) { return which ? d * size + slot : slot * D + d; };
        double top = 0.0;
        bool finite = true;
        for (int i = tid; i < tokens * D; i += kThreads) {
            const double x = value(i / D, i % D);
            finite = finite && fabs(x) <= 1.7976931348623157e308;
            top = fabs(x) > top ? fabs(x) : top;
        }
        finite = __syncthreads_and(finite);
        top = block_max(top, lds);
        const float held = *scale;
        const bool poisoned = !finite || (slot0 > 0 && held != held);
        int e = exponent_for(top);
        int e_held = e;
        if (slot0 > 0 && !poisoned) {
            // a power of two as the appends leave it; anything else counts by its exponent
            e_held = max(kLowestExponent, min(127, static_cast<int>((__float_as_uint(held) >> 23) & 255u) - 127));
            e = max(e, e_held);
        }
        if (e > e_held && slot0 > 0) {
            for (int i = tid; i < slot0 * D; i += kThreads) {
                int8_t &b = dst[at(i / D, i % D)];
                b = to_step(static_cast<double>(b), e - e_held);
            }
        }
        for (int i = tid; i < tokens * D; i += kThreads)
            dst[at(slot0 + i / D, i % D)] = poisoned ? 0 : to_step(value(i / D, i % D), e);
        __syncthreads();     // (the scale has been read by every wavefront)
        if (tid == 0) *scale = poisoned ? __uint_as_float(0x7fc00000u) : ldexpf(1.f, e);
    }
}

}  // namespace
}  // namespace rmlk

using namespace rmlk;

extern "C" {

int32_t rmlk_hip_paged_append(rmlk_stream_t stream, int32_t dtype, const rmlk_paged_cache *cache,
                              const rmlk_paged_batch *batch, const void *k, int64_t k_stride, const void *v,
                              int64_t v_stride, const float *cos, const float *sin, int64_t positions, int64_t heads,
                              const void *q, int64_t q_stride, void *q_out, int32_t *err_flag) {
    hipStream_t st = as_stream(stream);
    PagedArgs c{};
    if (const int32_t bad = paged_args(cache, batch, err_flag, &c); bad != RMLK_OK) return bad;
    if (!is_activation(dtype)) return RMLK_ERR_UNSUPPORTED;
    if ((cos == nullptr) != (sin == nullptr) || (q == nullptr) != (q_out == nullptr)) return RMLK_ERR_NULL_POINTER;
    if (positions < 0 || (q && heads < 1)) return RMLK_ERR_INVALID_ARGUMENT;
    if (q && heads % c.kv_heads != 0) return RMLK_ERR_SIZE_MISMATCH;
    if (q && heads > 0xffff) return RMLK_ERR_TOO_LARGE;
    if (c.seqs == 0 || c.rows == 0) return RMLK_OK;
    if (!k || !v) return RMLK_ERR_NULL_POINTER;
    if (const int32_t bad = paged_pointers(cache, batch); bad != RMLK_OK) return bad;
    const int d = cache->head_dim;
    const int64_t unit = dtype == RMLK_FLOAT ? 4 : 8;     // elements of 16 bytes
    if (k_stride < static_cast<int64_t>(c.kv_heads) * d || v_stride < static_cast<int64_t>(c.kv_heads) * d ||
        (q && q_stride < heads * d))
        return RMLK_ERR_SIZE_MISMATCH;
    if (k_stride % unit || v_stride % unit || (q && q_stride % unit) || !aligned16(k) || !aligned16(v) ||
        !aligned16(q) || !aligned16(q_out) || !aligned16(cos) || !aligned16(sin))
        return RMLK_ERR_UNSUPPORTED;
    const int64_t pieces = (c.rows >> c.page_shift) + 2 * c.seqs;
    if (pieces * c.kv_heads > (1 << 23)) return RMLK_ERR_TOO_LARGE;
    const int64_t q_elems = q ? c.rows * heads * d : 0;
    const int64_t q_blocks = (q_elems + 16 * kThreads - 1) / (16 * kThreads);
    return with_activation(dtype, [&](auto tag) {
        using T = decltype(tag);
        AppendArgs<T> g{};
        g.c = c;
        g.k = static_cast<const T *>(k);
        g.v = static_cast<const T *>(v);
        g.q = static_cast<const T *>(q);
        g.q_out = static_cast<T *>(q_out);
        g.cos = cos;
        g.sin = sin;
        g.k_stride = k_stride;
        g.v_stride = v_stride;
        g.q_stride = q_stride;
        g.positions = positions;
        g.heads = static_cast<int32_t>(heads);
        g.pieces = static_cast<int32_t>(pieces);
        const int64_t blocks = pieces * c.kv_heads + (q_blocks < (1 << 22) ? q_blocks : (1 << 22));
        if (d == 64) paged_append_kernel<T, 64><<<static_cast<uint32_t>(blocks), kThreads, 0, st>>>(g);
        else paged_append_kernel<T, 128><<<static_cast<uint32_t>(blocks), kThreads, 0, st>>>(g);
        return launch_status();
    });
}

}  // extern "C"
