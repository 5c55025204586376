// Keys and values appended to the paged int8 cache, keys (and queries) rotated on the way.
//
// A block of the cache (one page of one KV head) holds int8 values times one power of two 2^e. With
// the new tokens' largest magnitude a, e has to satisfy a <= 127 * 2^e: with a = f * 2^x, f in [1/2, 1),
// that is x - 7 for f <= 127/128 and x - 6 otherwise. A block that is continued keeps the larger of
// this and the exponent it has; when it grows, the integers held already are shifted right with
// rounding to nearest even. Rotation and quantisation are evaluated in double, two exact products and their
// sum rounded to odd: such a sum lies on a border (between two integers, or 127 * 2^e, numbers of few bits) only if
// the real one does, and on the same side of it otherwise, so that every value falls the right way.
#include <cmath>

#include "paged.hpp"

namespace rmlk {
namespace {

constexpr int kLowestExponent = -126;
constexpr int kHeads = 2;      // heads of q that a thread rotates with one row of the tables

template <typename T>
struct AppendArgs {
    PagedArgs c;
    const T *k, *v, *q;
    T *q_out;
    const float *cos, *sin;
    int64_t k_stride, v_stride, q_stride;
    int64_t positions;
    int32_t heads;
    int32_t pieces;      // upper bound of the pages written to: the first blocks of the grid, per KV head
    int64_t q_units;     // units of q: D / 16 per row and kHeads heads
};

__device__ __forceinline__ int exponent_for(double a) {
    if (a == 0.0) return kLowestExponent;
    int x;
    const double f = frexp(a, &x);
    const int e = f <= 127.0 / 128.0 ? x - 7 : x - 6;
    return max(kLowestExponent, min(127, e));
}

// 2^e as a double, |e| < 1000
__device__ __forceinline__ double power(int e) {
    return __longlong_as_double(static_cast<long long>(e + 1023) << 52);
}
__device__ __forceinline__ uint32_t to_byte(double x, double inverse_step) {
    const int n = static_cast<int>(rint(x * inverse_step));
    return static_cast<uint32_t>(min(127, max(-127, n))) & 255u;
}
// (a float times a power of two is exact, or so small that it rounds to zero)
__device__ __forceinline__ uint32_t to_byte(float x, float inverse_step) {
    const int n = static_cast<int>(rintf(x * inverse_step));
    return static_cast<uint32_t>(min(127, max(-127, n))) & 255u;
}
__device__ __forceinline__ uint64_t to_bytes(const double (&x)[8], double inverse_step) {
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo |= to_byte(x[i], inverse_step) << (8 * i);
        hi |= to_byte(x[4 + i], inverse_step) << (8 * i);
    }
    return static_cast<uint64_t>(hi) << 32 | lo;
}

// cos and sin of eight dims d .. of the first half of a row and of the eight that rotate with them.
struct Turn {
    float c0[8], s0[8], c1[8], s1[8];
};
template <int D>
__device__ __forceinline__ void load_turn(Turn &t, const float *cos, const float *sin, int64_t pos, int d) {
    load_row(cos + pos * D + d, t.c0);
    load_row(sin + pos * D + d, t.s0);
    load_row(cos + pos * D + d + D / 2, t.c1);
    load_row(sin + pos * D + d + D / 2, t.s1);
}
// a + b rounded to 53 bits, towards the neighbour whose last bit is 1 where it is not exact (the error of the sum as in
// Knuth's two-sum; rounding to odd as Boldo and Melquiond describe it). Sums that are not finite stay as they are.
__device__ __forceinline__ double sum_to_odd(double a, double b) {
    const double s = a + b, from_b = s - a, err = (a - (s - from_b)) + (b - from_b);
    long long bits = __double_as_longlong(s);
    const bool inexact = err > 0.0 || err < 0.0;
    bits += inexact && !(bits & 1) ? ((err > 0.0) == (s > 0.0) ? 1 : -1) : 0;
    return __longlong_as_double(bits);
}
// Zero for numbers of up to 9 bits, as the borders are.
__device__ __forceinline__ uint32_t bits_behind_nine(double x) {
    return static_cast<uint32_t>(__double2hiint(x) & 0xfff) | static_cast<uint32_t>(__double2loint(x));
}
__device__ __forceinline__ void rotate_eight(const float (&a)[8], const float (&b)[8], const Turn &t, bool turn,
                                             double (&lo)[8], double (&hi)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double x = a[i], y = b[i];
        lo[i] = turn ? x * t.c0[i] + -y * t.s0[i] : x;
        hi[i] = turn ? y * t.c1[i] + x * t.s1[i] : y;
    }
}
// The same with sums to odd.
__device__ __forceinline__ void rotate_eight_to_odd(const float (&a)[8], const float (&b)[8], const Turn &t,
                                                    double (&lo)[8], double (&hi)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double x = a[i], y = b[i];
        lo[i] = sum_to_odd(x * t.c0[i], -y * t.s0[i]);
        hi[i] = sum_to_odd(y * t.c1[i], x * t.s1[i]);
    }
}

// (STREAMING: past the caches, whose lines would have to be written back when the kernel ends)
template <bool STREAMING, typename T>
__device__ __forceinline__ void store_eight(T *to, const double (&x)[8]) {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(x[i]);
#pragma unroll
    for (size_t u = 0; u < sizeof(T) / 2; ++u)
        store_unit<STREAMING>(to + u * (16 / sizeof(T)), reinterpret_cast<const u32x4 *>(v)[u]);
}

// The same for a 16-bit result, in float: the rounding error of one product is carried along, so that nothing is
// lost where the two cancel, and the result is off by 2^-23 of itself before it is rounded.
__device__ __forceinline__ float two_products(float x, float c, float y, float s) {
    const float p = y * s, rest = fmaf(y, s, -p);
    return fmaf(x, c, p) + (fabsf(p) < INFINITY ? rest : 0.f);
}
template <bool STREAMING, typename T>
__device__ __forceinline__ void store_rotated(T *to, int half, const float (&a)[8], const float (&b)[8], const Turn &t,
                                              bool turn) {
    if constexpr (sizeof(T) == 4) {
        double lo[8], hi[8];
        rotate_eight(a, b, t, turn, lo, hi);
        store_eight<STREAMING>(to, lo);
        store_eight<STREAMING>(to + half, hi);
    } else {
        T lo[8], hi[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo[i] = static_cast<T>(turn ? two_products(a[i], t.c0[i], -b[i], t.s0[i]) : a[i]);
            hi[i] = static_cast<T>(turn ? two_products(b[i], t.c1[i], a[i], t.s1[i]) : b[i]);
        }
        store_unit<STREAMING>(to, *reinterpret_cast<const u32x4 *>(lo));
        store_unit<STREAMING>(to + half, *reinterpret_cast<const u32x4 *>(hi));
    }
}

// Blocks 0 .. pieces * kv_heads - 1: a block takes one page of one sequence and KV head, K and V. Its threads
// load all new values of it at once (PK units of 8 + 8 rotating dims of K, 2 PK units of 8 dims of V each),
// agree on the two largest magnitudes and write: one trip over the values. V is turned in LDS when more
// than a few tokens come, so that the runs of new slots of a dim go out as whole words. The other blocks
// rotate q.
// Single tokens are a chain of trips to memory (the sequence, its page, values and scales): 64 of them, 8 KV heads
// of 64 dims, 5.1 us. Prompts are bound by the bytes and by that chain in about equal parts: 2275 tokens of 8
// sequences in bfloat16, 8 KV heads of 128 dims and 32 heads of q (53.6 MB) take 18.2 us, 13 us without q.
// Measured and dropped: K and V in blocks of their own (20.8 became 26 us), units of 4 + 4 dims (25 us), q by
// one or four heads per thread (1.1 us more; 2.2 us more with single tokens). Queries of 16-bit types turned in
// double took 22.5 us when float took 20.8, plain stores of them 20.8 where streaming ones take 18.1 (with the
// attention that reads them behind, 100 us either way; the queries of single tokens are stored as usual).
template <typename T, int D, int THREADS, int PK>
__global__ __launch_bounds__(THREADS, PK < 4 ? 3 : 2) void paged_append_kernel(AppendArgs<T> g) {
    constexpr int kUnitsK = D / 16, kUnitsV = D / 8;              // units of a token
    constexpr int kTokensK = THREADS / kUnitsK, kTokensV = THREADS / kUnitsV;   // tokens of one trip
    constexpr int kMostTokens = PK * kTokensK < 128 ? PK * kTokensK : 128, kPad = kMostTokens + 4;
    __shared__ double lds[2][THREADS / kWave];
    __shared__ __align__(16) uint8_t turned[D][kPad];
    const int tid = threadIdx.x, lane = tid % kWave;
    const int kv_blocks = g.pieces * g.c.kv_heads;
    if (static_cast<int>(blockIdx.x) >= kv_blocks) {
        if (!starts_ascend(g.c)) return;
        const int64_t first_unit = (static_cast<int64_t>(blockIdx.x) - kv_blocks) * THREADS;
        // a unit: eight + eight dims of kHeads heads of a row, which share their row of the tables
        const int groups = (g.heads + kHeads - 1) / kHeads;
        for (int64_t u = first_unit + tid; u < g.q_units; u += static_cast<int64_t>(gridDim.x - kv_blocks) * THREADS) {
            const int64_t rg = u / kUnitsK;
            const int d = static_cast<int>(u % kUnitsK) * 8;
            const int row = static_cast<int>(rg / groups), h0 = static_cast<int>(rg % groups) * kHeads;
            Sequence q;
            if (!sequence_of_row(g.c, row, q) || q.length < q.fresh) continue;
            const int64_t pos = q.length - q.fresh + (row - q.row);
            if (g.cos && pos >= g.positions) continue;
            const T *from = g.q + row * g.q_stride + d;
            T *to = g.q_out + static_cast<int64_t>(row) * g.heads * D + d;
            float x[kHeads][2][8];
#pragma unroll
            for (int i = 0; i < kHeads; ++i)
                if (h0 + i < g.heads) {
                    load_row(from + (h0 + i) * D, x[i][0]);
                    load_row(from + (h0 + i) * D + D / 2, x[i][1]);
                }
            Turn turn;
            if (g.cos) load_turn<D>(turn, g.cos, g.sin, pos, d);
#pragma unroll
            for (int i = 0; i < kHeads; ++i)
                if (h0 + i < g.heads)
                    store_rotated<(THREADS > kWave)>(to + (h0 + i) * D, D / 2, x[i][0], x[i][1], turn, g.cos != nullptr);
        }
        return;
    }
    const int head = blockIdx.x % g.c.kv_heads;
    Item item;
    // (a sequence's items: the pages it writes to)
    if (!find_item(g.c, blockIdx.x / g.c.kv_heads,
                   [&](const Sequence &q) {
                       const int last = (q.length - 1) >> g.c.page_shift, begin = (q.length - q.fresh) >> g.c.page_shift;
                       return q.length < q.fresh ? 1 : last - begin + 1;
                   },
                   item)) {
        if (blockIdx.x == 0 && tid == 0) raise_error(g.c);
        return;
    }
    if (item.s < 0) return;
    const Sequence q = item.q;
    const int s = item.s, index = item.index;
    if (!in_bounds(g.c, q) || q.length < q.fresh) {
        if (head == 0 && tid == 0) raise_error(g.c);
        return;
    }
    const int size = 1 << g.c.page_shift;
    const int begin_pos = q.length - q.fresh;
    const int64_t page_at = static_cast<int64_t>(begin_pos >> g.c.page_shift) + index;   // in the table
    const int64_t page_pos = page_at << g.c.page_shift;
    const int slot0 = page_pos < begin_pos ? static_cast<int>(begin_pos - page_pos) : 0;
    int slot1 = static_cast<int>(min(static_cast<int64_t>(size), q.length - page_pos));
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
    const int64_t row0 = q.row + (page_pos + slot0 - begin_pos), pos0 = page_pos + slot0;
    const int64_t block = static_cast<int64_t>(page) * g.c.kv_heads + head;
    int8_t *k_block = g.c.k + block * size * D, *v_block = g.c.v + block * size * D;
    const float k_held = g.c.k_scale[block], v_held = g.c.v_scale[block];

    double k_lo[PK][8], k_hi[PK][8];
    float v[2 * PK][8];
    const int unit_k = tid % kUnitsK * 8, unit_v = tid % kUnitsV * 8;
#pragma unroll
    for (int i = 0; i < 2 * PK; ++i) {
        const int t = i * kTokensV + tid / kUnitsV;
        if (t < tokens) load_row(g.v + (row0 + t) * g.v_stride + static_cast<int64_t>(head) * D + unit_v, v[i]);
    }
    double k_top = 0.0, odd = 0.0;
    bool on_border = false;
    uint32_t v_bits = 0;
#pragma unroll
    for (int i = 0; i < PK; ++i) {
        const int t = i * kTokensK + tid / kUnitsK;
        if (t < tokens) {
            const T *from = g.k + (row0 + t) * g.k_stride + static_cast<int64_t>(head) * D + unit_k;
            float x[2][8];
            load_row(from, x[0]);
            load_row(from + D / 2, x[1]);
            Turn turn;
            if (g.cos) load_turn<D>(turn, g.cos, g.sin, pos0 + t, unit_k);
            rotate_eight(x[0], x[1], turn, g.cos != nullptr, k_lo[i], k_hi[i]);
            uint32_t behind = ~0u, second = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                behind = min(behind, min(bits_behind_nine(k_lo[i][e]), bits_behind_nine(k_hi[i][e])));
                second |= __float_as_uint(turn.s0[e]) | __float_as_uint(turn.s1[e]);
            }
            on_border = on_border || (behind == 0 && second << 1 != 0);     // (without a second product all is exact)
        }
    }
    // A sum that rounding has not moved onto a border lies on the real one's side of all of them: to odd only where
    // one is on a border now (for every sum, 64 single tokens take 5.6 us, so 5.1).
    if (g.cos && __any(on_border)) {
#pragma unroll
        for (int i = 0; i < PK; ++i) {
            const int t = i * kTokensK + tid / kUnitsK;
            if (t < tokens) {
                const T *from = g.k + (row0 + t) * g.k_stride + static_cast<int64_t>(head) * D + unit_k;
                float x[2][8];
                load_row(from, x[0]);
                load_row(from + D / 2, x[1]);
                Turn turn;
                load_turn<D>(turn, g.cos, g.sin, pos0 + t, unit_k);
                rotate_eight_to_odd(x[0], x[1], turn, k_lo[i], k_hi[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < PK; ++i) {
        if (i * kTokensK + tid / kUnitsK < tokens) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                k_top = fmax(k_top, fmax(fabs(k_lo[i][e]), fabs(k_hi[i][e])));
                odd = fma(k_lo[i][e], 0.0, fma(k_hi[i][e], 0.0, odd));    // NaN: a value that is not finite
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2 * PK; ++i)
        if (i * kTokensV + tid / kUnitsV < tokens) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v_bits = max(v_bits, __float_as_uint(v[i][e]) & 0x7fffffffu);
        }
    if (odd != 0.0) k_top = INFINITY;
    k_top = wave_max(k_top);
    v_bits = wave_max(v_bits);
    double v_top = v_bits >= 0x7f800000u ? static_cast<double>(INFINITY) : static_cast<double>(__uint_as_float(v_bits));
    if constexpr (THREADS > kWave) {
        if (lane == 0) {
            lds[0][tid / kWave] = k_top;
            lds[1][tid / kWave] = v_top;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < THREADS / kWave; ++i) {
            k_top = fmax(k_top, lds[0][i]);
            v_top = fmax(v_top, lds[1][i]);
        }
    }
    // the step of a block: what its new values need, and what it has if it goes on
    auto step = [&](double top, float held, int &e_held, bool &marked) {
        marked = top == static_cast<double>(INFINITY) || (slot0 > 0 && held != held);
        int e = marked ? 0 : exponent_for(top);
        e_held = e;
        if (slot0 > 0 && !marked) {
            // (a power of two as the appends leave it; anything else counts by its exponent)
            e_held = max(kLowestExponent, min(127, static_cast<int>((__float_as_uint(held) >> 23) & 255u) - 127));
            e = max(e, e_held);
        }
        return e;
    };
    int k_was, v_was;
    bool k_marked, v_marked;
    const int k_e = step(k_top, k_held, k_was, k_marked), v_e = step(v_top, v_held, v_was, v_marked);
    // values held already, in the new step
    if (k_e > k_was) {
        uint32_t *words = reinterpret_cast<uint32_t *>(k_block);
        const double shrink = power(k_was - k_e);
        for (int i = tid; i < slot0 * D / 4; i += THREADS) {
            const uint32_t w = words[i];
            uint32_t n = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) n |= to_byte(static_cast<double>(static_cast<int8_t>(w >> (8 * e))), shrink) << (8 * e);
            words[i] = n;
        }
    }
    if (v_e > v_was) {
        const double shrink = power(v_was - v_e);
        for (int i = tid; i < slot0 * D; i += THREADS) {
            int8_t &b = v_block[i / slot0 * size + i % slot0];
            b = static_cast<int8_t>(to_byte(static_cast<double>(b), shrink));
        }
    }
    const double k_inv = k_marked ? 0.0 : power(-k_e);
    const float v_inv = v_marked ? 0.f : static_cast<float>(power(-v_e));
#pragma unroll
    for (int i = 0; i < PK; ++i) {
        const int t = i * kTokensK + tid / kUnitsK;
        if (t < tokens) {
            int8_t *to = k_block + (slot0 + t) * D + unit_k;
            *reinterpret_cast<uint64_t *>(to) = k_marked ? 0 : to_bytes(k_lo[i], k_inv);
            *reinterpret_cast<uint64_t *>(to + D / 2) = k_marked ? 0 : to_bytes(k_hi[i], k_inv);
        }
    }
    const bool turn = tokens > 4;
#pragma unroll
    for (int i = 0; i < 2 * PK; ++i) {
        const int t = i * kTokensV + tid / kUnitsV;
        if (t < tokens) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint8_t b = v_marked ? 0 : static_cast<uint8_t>(to_byte(v[i][e], v_inv));
                if (turn) turned[unit_v + e][t] = b;
                else v_block[(unit_v + e) * size + slot0 + t] = static_cast<int8_t>(b);
            }
        }
    }
    if (turn) {
        __syncthreads();
        // words of four slots; those at the ends that hold older slots byte by byte
        const int w0 = slot0 / 4, w1 = (slot1 + 3) / 4;
        for (int i = tid; i < D * (w1 - w0); i += THREADS) {
            const int d = i / (w1 - w0), w = w0 + i % (w1 - w0);
            int8_t *to = v_block + d * size + w * 4;
            if (w * 4 >= slot0 && w * 4 + 4 <= slot1) {
                uint32_t n = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) n |= static_cast<uint32_t>(turned[d][w * 4 + e - slot0]) << (8 * e);
                *reinterpret_cast<uint32_t *>(to) = n;
            } else {
                for (int e = 0; e < 4; ++e)
                    if (w * 4 + e >= slot0 && w * 4 + e < slot1) to[e] = static_cast<int8_t>(turned[d][w * 4 + e - slot0]);
            }
        }
    }
    if (tid == 0) {
        const float nan = __uint_as_float(0x7fc00000u);
        g.c.k_scale[block] = k_marked ? nan : static_cast<float>(power(k_e));
        g.c.v_scale[block] = v_marked ? nan : static_cast<float>(power(v_e));
    }
}

template <typename T, int D, int THREADS, int PK>
int32_t launch_append(hipStream_t st, AppendArgs<T> g) {
    const int64_t q_blocks = (g.q_units + THREADS - 1) / THREADS;
    const int64_t blocks = static_cast<int64_t>(g.pieces) * g.c.kv_heads + (q_blocks < (1 << 22) ? q_blocks : (1 << 22));
    paged_append_kernel<T, D, THREADS, PK><<<static_cast<uint32_t>(blocks), THREADS, 0, st>>>(g);
    return launch_status();
}

// A wavefront per block where no sequence brings more tokens than it takes in one trip; 256 threads and as many
// trips as a page needs otherwise.
template <typename T, int D>
int32_t launch_append_for(hipStream_t st, const AppendArgs<T> &g) {
    const int64_t page = static_cast<int64_t>(1) << g.c.page_shift;
    const int64_t units = (g.c.max_new < page ? g.c.max_new : page) * (D / 16);     // of one block's K at most
    if (units <= 64) return launch_append<T, D, 64, 1>(st, g);
    if (units <= 256) return launch_append<T, D, 256, 1>(st, g);
    if (units <= 512) return launch_append<T, D, 256, 2>(st, g);
    if constexpr (D == 128) return launch_append<T, D, 256, 4>(st, g);
    return RMLK_ERR_UNSUPPORTED;      // (128 tokens of 64 dims are 512 units)
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
    if (q && q == q_out && q_stride != heads * d) return RMLK_ERR_INVALID_ARGUMENT;   // (rows would move under their readers)
    const int64_t pieces = (c.rows >> c.page_shift) + 2 * c.seqs;
    if (pieces * c.kv_heads > (1 << 23)) return RMLK_ERR_TOO_LARGE;
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
        g.q_units = q ? c.rows * ((heads + kHeads - 1) / kHeads) * (d / 16) : 0;
        return d == 64 ? launch_append_for<T, 64>(st, g) : launch_append_for<T, 128>(st, g);
    });
}

}  // extern "C"
