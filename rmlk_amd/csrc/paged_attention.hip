// Attention over the paged int8 cache: out = Softmax(q . K^T * scale) . V per sequence, a query seeing the
// tokens up to its own position.
#include <cmath>

#include "paged.hpp"

namespace rmlk {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

template <typename T>
struct AttendArgs {
    PagedArgs c;
    const T *q;
    T *out;
    int64_t q_stride;
    int32_t heads;
    float scale;         // of the scores, with log2(e)
};

// A wavefront per (row, head): 64 keys at a time, a key per lane for the scores and a head dim (or two)
// per lane for the output.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void attend_rows_kernel(AttendArgs<T> g) {
    if (!starts_ascend(g.c)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) raise_error(g.c);
        return;
    }
    const int lane = threadIdx.x % kWave;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / kWave) + threadIdx.x / kWave;
    if (item >= g.c.rows * g.heads) return;
    const int64_t row = item / g.heads;
    const int head = static_cast<int>(item % g.heads), kv = head / (g.heads / g.c.kv_heads);
    Sequence s;
    const int seq = sequence_of_row(g.c, row);
    if (!sequence_at(g.c, seq, s)) {
        if (lane == 0) raise_error(g.c);
        return;
    }
    if (row < s.row || row >= s.row + s.fresh) return;
    const int limit = s.length - s.fresh + static_cast<int>(row - s.row) + 1;   // tokens it sees
    const int size = 1 << g.c.page_shift;
    const int32_t *table = g.c.table + seq * g.c.table_stride;
    const T *q = g.q + row * g.q_stride + static_cast<int64_t>(head) * D;
    float m = -INFINITY, sum = 0.f, acc[D / kWave] = {};
    for (int t0 = 0; t0 < limit; t0 += kWave) {
        const int t = t0 + lane;
        float x = -INFINITY, vs = 0.f;
        int64_t block = 0;
        if (t < limit) {
            const int32_t page = table[t >> g.c.page_shift];
            if (page < 0 || page >= g.c.pages) {
                raise_error(g.c);
            } else {
                block = static_cast<int64_t>(page) * g.c.kv_heads + kv;
                const int8_t *k = g.c.k + (block * size + (t & (size - 1))) * D;
                float dot = 0.f;
                for (int d = 0; d < D; ++d) dot = fmaf(to_float(q[d]), static_cast<float>(k[d]), dot);
                vs = g.c.v_scale[block];
                // (a scale that is NaN, of K or of V, makes the score NaN)
                x = dot * (g.c.k_scale[block] + 0.f * vs) * g.scale;
            }
        }
        const bool any_nan = __any(x != x);
        const float top = any_nan ? __uint_as_float(0x7fc00000u) : fmaxf(m, wave_max(x));
        if (top == -INFINITY) continue;
        const float alpha = exp2f(m - top), p = exp2f(x - top);
        m = top;
        sum = sum * alpha + wave_sum(p);
#pragma unroll
        for (int i = 0; i < D / kWave; ++i) acc[i] *= alpha;
        const int here = min(kWave, limit - t0);
        const float pv = vs == vs ? p * vs : 0.f;
        for (int j = 0; j < here; ++j) {
            const float w = __shfl(pv, j, kWave);
            const int64_t b = __shfl(static_cast<long long>(block), j, kWave);
            const int8_t *v = g.c.v + b * size * D + ((t0 + j) & (size - 1));
#pragma unroll
            for (int i = 0; i < D / kWave; ++i)
                acc[i] = fmaf(w, static_cast<float>(v[static_cast<int64_t>(i * kWave + lane) * size]), acc[i]);
        }
    }
    T *out = g.out + (row * g.heads + head) * D;
#pragma unroll
    for (int i = 0; i < D / kWave; ++i) out[i * kWave + lane] = static_cast<T>(m == -INFINITY ? 0.f : acc[i] / sum);
}

int32_t attend_checks(int32_t dtype, const rmlk_paged_cache *cache, const rmlk_paged_batch *batch, int64_t heads,
                      int32_t *err_flag, PagedArgs *c) {
    if (const int32_t bad = paged_args(cache, batch, err_flag, c); bad != RMLK_OK) return bad;
    if (!is_activation(dtype)) return RMLK_ERR_UNSUPPORTED;
    if (heads < 1) return RMLK_ERR_INVALID_ARGUMENT;
    if (heads % c->kv_heads != 0) return RMLK_ERR_SIZE_MISMATCH;
    if (heads > 0xffff) return RMLK_ERR_TOO_LARGE;
    return RMLK_OK;
}

}  // namespace
}  // namespace rmlk

using namespace rmlk;

extern "C" {

size_t rmlk_hip_paged_attention_workspace_size(int32_t dtype, const rmlk_paged_cache *cache,
                                               const rmlk_paged_batch *batch, int64_t heads) {
    PagedArgs c{};
    if (attend_checks(dtype, cache, batch, heads, nullptr, &c) != RMLK_OK) return 0;
    return 0;
}

int32_t rmlk_hip_paged_attention(rmlk_stream_t stream, int32_t dtype, const rmlk_paged_cache *cache,
                                 const rmlk_paged_batch *batch, int64_t heads, const void *q, int64_t q_stride,
                                 int32_t scale_is_mul, float scale, void *workspace, size_t workspace_bytes,
                                 void *out, int32_t *err_flag) {
    hipStream_t st = as_stream(stream);
    PagedArgs c{};
    if (const int32_t bad = attend_checks(dtype, cache, batch, heads, err_flag, &c); bad != RMLK_OK) return bad;
    if (c.seqs == 0 || c.rows == 0) return RMLK_OK;
    if (!q || !out) return RMLK_ERR_NULL_POINTER;
    if (const int32_t bad = paged_pointers(cache, batch); bad != RMLK_OK) return bad;
    const int d = cache->head_dim;
    const int64_t unit = dtype == RMLK_FLOAT ? 4 : 8;
    if (q_stride < heads * d) return RMLK_ERR_SIZE_MISMATCH;
    if (q_stride % unit || !aligned16(q) || !aligned16(out)) return RMLK_ERR_UNSUPPORTED;
    const int64_t blocks = (c.rows * heads + 3) / 4;
    if (blocks > (1 << 23)) return RMLK_ERR_TOO_LARGE;
    return with_activation(dtype, [&](auto tag) {
        using T = decltype(tag);
        AttendArgs<T> g{};
        g.c = c;
        g.q = static_cast<const T *>(q);
        g.out = static_cast<T *>(out);
        g.q_stride = q_stride;
        g.heads = static_cast<int32_t>(heads);
        g.scale = (scale_is_mul ? scale : 1.f / scale) * kLog2e;
        if (d == 64) attend_rows_kernel<T, 64><<<static_cast<uint32_t>(blocks), kThreads, 0, st>>>(g);
        else attend_rows_kernel<T, 128><<<static_cast<uint32_t>(blocks), kThreads, 0, st>>>(g);
        return launch_status();
    });
}

}  // extern "C"
