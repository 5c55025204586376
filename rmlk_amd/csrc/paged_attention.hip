// Attention over the paged int8 cache: out = Softmax(q . K^T * scale) . V per sequence, a query seeing the
// tokens up to its own position; prompts, chunks of prompts and single tokens alike.
//
// The rows of one KV head (its rep query heads times the sequence's new tokens) form one matrix, cut into
// tiles of rows. Long caches are split over several blocks besides, whose normalised results a second
// kernel joins.
//
// Everything is computed transposed, so that a query stays in one lane column from its scores to its
// output: S^T = K . Q^T by v_mfma_f32_16x16x32_f16 leaves four keys of a query in a lane, and the keys
// of a tile are assigned to the rows of the four S^T blocks such that a lane's sixteen weights belong to
// sixteen CONSECUTIVE tokens (16 g .. 16 g + 15 for lane group g): they are the B operand of
// O^T += V^T . P^T as they are, and the A operand is sixteen consecutive bytes of a row of the transposed
// V block. No score or weight passes through LDS; K and V come from memory in 16-byte loads, one tile ahead.
//
// int8 -> half: a byte b with its sign bit flipped, u = b + 128, under the high byte 0x64 is the half
// 1024 + u; one packed add of -1152 gives b (K), one packed fma (1024 + u) * f - 1152 f gives b * f
// exactly (V, f the page's step relative to the largest one of the block's keys, 2^E, which scales the output
// at the end). So pages with different steps mix in one MFMA. K's step goes to the scores.
//
// That holds while the steps lie close together: a wavefront's rows share E, and a row's outputs would vanish
// beside the step of a page that it does not see, or sees with next to no weight. So the steps are looked over
// first. Where they spread over more than 2^kSpread, or one is no power of two, V is widened as it is and the steps
// go to the weights, each row's products of weight and step relative to the largest of its own (the wide loops).
// Within the range a page's tokens lose what lies below 2^(kSpread - 31) of the row's largest product, less than V's
// own rounding (2^-8) even where 2^14 of them do. (A prompt of 2048 tokens, 32 heads of 64 dims, floats: 51 us, with a
// tenth of the pages 2^20 apart 79 us; 64 single tokens behind 100 .. 16384 keys 90 and 94 us. Looked over in the loops
// instead, tile by tile, prompts of 64 dims took 4 % longer, and a cache of far steps a second pass.)
//
// A float query is the sum of two halves (hi + lo, 22 bits), scaled by a power of two so that its
// largest element lies in [2^13, 2^14); a float weight likewise, exponentials being taken relative to
// the maximum less 7 and allowed to grow to 2^15 before the reference point moves (rescaling is rare),
// so weights down to 2^-18 of the largest keep 22 bits. For 16-bit types one half each: q is exact, a
// weight is off by 2^-11 of itself at most, as the output is.
#include <cmath>

#include "paged.hpp"

namespace rmlk {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTileKeys = 64;
constexpr float kBase = 7.f;          // log2 of the weight of a key that scores the reference maximum
constexpr float kLeastFactor = 1.17549435e-38f;
constexpr float kMostWeight = 15.f;   // log2 of the largest weight before the reference point moves
constexpr int kSpread = 6;            // log2 of the largest ratio of V's steps that share a reference

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct AttendArgs {
    PagedArgs c;
    const T *q;
    T *out;
    float *part;         // partial outputs [splits][rows * heads][D], then (max, sum) [splits][rows * heads][2]
    int64_t q_stride;
    int32_t heads, rep;
    float scale;         // of the scores, with log2(e)
    int32_t splits, chunk;   // tokens per split, a multiple of the tile
    int32_t fold;        // the second half of the items in ascending order
};

// the four bytes of a word as halves 1024 + (b + 128)
__device__ __forceinline__ void biased_halves(uint32_t w, h2 &lo, h2 &hi) {
    const uint32_t x = w ^ 0x80808080u;
    lo = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u));
    hi = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u));
}
__device__ __forceinline__ h8 eight(h2 a, h2 b, h2 c, h2 d) {
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ h8 widen(uint32_t w0, uint32_t w1) {
    const h2 bias = {static_cast<_Float16>(-1152.f), static_cast<_Float16>(-1152.f)};
    h2 a, b, c, d;
    biased_halves(w0, a, b);
    biased_halves(w1, c, d);
    return eight(a + bias, b + bias, c + bias, d + bias);
}
__device__ __forceinline__ h8 widen_scaled(uint32_t w0, uint32_t w1, h2 f, h2 bias) {
    h2 a, b, c, d;
    biased_halves(w0, a, b);
    biased_halves(w1, c, d);
    return eight(__builtin_elementwise_fma(a, f, bias), __builtin_elementwise_fma(b, f, bias),
                 __builtin_elementwise_fma(c, f, bias), __builtin_elementwise_fma(d, f, bias));
}

__device__ __forceinline__ float across_groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float across_groups_sum(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}

// One tile of keys on its way from memory: raw bytes of K and V, the steps of the page of the lane
// group's tokens.
template <int D>
struct Tile {
    u32x4 k[4][D / 64];
    u32x4 v[D / 16];
    float k_scale, v_scale;
    bool bad;            // the page lies outside the cache
};

// Sixteen NT rows of a wavefront's lane columns: what they see and their queries as halves.
template <typename T, int D, int NT>
struct Rows {
    static constexpr int P = sizeof(T) == 4 ? 2 : 1;   // half pieces of a query value and of a weight
    static constexpr int KH = D / 32;
    int limit[NT];             // tokens the row sees
    float factor[NT];          // of a score but for K's step
    h8 q[P][NT][KH];

    // rows r0 .. of the `rows` of one KV head of a sequence
    __device__ __forceinline__ void load(const AttendArgs<T> &g, const Sequence &s, int kv, int r0, int rows) {
        const int lane = threadIdx.x % kWave, col = lane % 16, grp = lane / 16;
        const int past = s.length - s.fresh;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = r0 + n * 16 + col;
            const bool live = r < rows;
            limit[n] = live ? past + r / g.rep + 1 : 0x7fffffff;   // (a row that is not there: no mask, zeros)
            float x[D / 64][16];
            const T *src = g.q + (s.row + (live ? r / g.rep : 0)) * g.q_stride +
                           static_cast<int64_t>(kv * g.rep + (live ? r % g.rep : 0)) * D + grp * 16;
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                load_row(src + c * 64, x[c]);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (!live) x[c][i] = 0.f;
                    const uint32_t bits = __float_as_uint(x[c][i]) & 0x7fffffffu;
                    top = bits > top ? bits : top;
                }
            }
            uint32_t other = __shfl_xor(top, 16, kWave);
            top = other > top ? other : top;
            other = __shfl_xor(top, 32, kWave);
            top = other > top ? other : top;
            const int e = max(-113, static_cast<int>(top >> 23) - 127);
            // (the scale's sign goes to the query: factors are positive)
            const float up = copysignf(__uint_as_float(static_cast<uint32_t>(13 - e + 127) << 23), g.scale);
            factor[n] = __uint_as_float(static_cast<uint32_t>(e - 13 + 127) << 23) * fabsf(g.scale);
            if (top >= 0x7f800000u) factor[n] = __uint_as_float(0x7fc00000u);   // (an infinity or a NaN in the row)
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float v = x[c][h * 8 + j] * up;
                        const _Float16 hi = static_cast<_Float16>(v);
                        q[0][n][c * 2 + h][j] = hi;
                        if constexpr (P == 2) q[1][n][c * 2 + h][j] = static_cast<_Float16>(v - static_cast<float>(hi));
                    }
        }
    }
};

// The cache as one KV head of one sequence sees it. Addresses are a 32-bit page times a 32-bit pitch (at most
// 65535 heads of 16 KB) behind a base that is the same in all lanes: one wide multiply each.
template <int D>
struct View {
    const int8_t *k, *v;
    const float *k_scale, *v_scale;
    const int32_t *table;
    uint32_t pages, pitch, heads;
    int shift, size, last_page;
    template <typename T>
    __device__ __forceinline__ View(const AttendArgs<T> &g, const Sequence &s, int seq, int kv)
        : k(g.c.k), v(g.c.v), k_scale(g.c.k_scale + kv), v_scale(g.c.v_scale + kv),
          table(g.c.table + seq * g.c.table_stride), pages(static_cast<uint32_t>(g.c.pages)), heads(g.c.kv_heads),
          shift(g.c.page_shift), size(1 << g.c.page_shift), last_page((s.length > 0 ? s.length - 1 : 0) >> shift) {
        k += kv * size * D;
        v += kv * size * D;
        pitch = heads * static_cast<uint32_t>(size * D);
    }
    __device__ __forceinline__ int page_at(int token) const { return min(token >> shift, last_page); }
    __device__ __forceinline__ uint32_t page_of(int token) const {
        return static_cast<uint32_t>(table[static_cast<uint32_t>(page_at(token))]);
    }
    __device__ __forceinline__ bool has(uint32_t page) const { return page < pages; }
    __device__ __forceinline__ const int8_t *at(const int8_t *base, uint32_t page, uint32_t offset) const {
        return base + static_cast<uint64_t>(page) * pitch + offset;
    }
    __device__ __forceinline__ uint64_t scale_at(uint32_t page) const { return static_cast<uint64_t>(page) * heads; }
};

// What a wavefront has of its rows' softmax: outputs (times 2^-E), sums, reference points.
template <typename T, int D, int NT>
struct Softmax {
    static constexpr int P = Rows<T, D, NT>::P, DT = D / 16, KH = D / 32;
    f32x4 acc[DT][NT];
    float sum[NT], ref[NT];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            sum[n] = 0.f;
            ref[n] = -3.402823466e38f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d][n] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // S^T of a tile: k_frag(jj, h) gives K's operands.
    typedef f32x4 Scores[4][NT];
    template <typename KF>
    __device__ __forceinline__ void scores(const Rows<T, D, NT> &rows, KF &&k_frag, Scores &sc) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[j][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int q = 0; q < KH; ++q) {
                const h8 kf = k_frag(j, q);
#pragma unroll
                for (int p = P - 1; p >= 0; --p)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        sc[j][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, rows.q[p][n][q], sc[j][n], 0, 0, 0);
            }
        }
    }
    // Hides what a row does not see and moves the reference point where a score lies too far above it; c: the factors
    // of the scores. kc is K's step of the lane group's tokens, t0 the tile's first token, masked whether any row of
    // the wavefront does not see all of it, bad whether the lane group's tokens are hidden from everyone. A hidden
    // score becomes -inf before it is scaled: factors are kept positive, and where a row sees none of the lane
    // group's tokens its factor is replaced, so that a step that is no number reaches only the rows that see the
    // block.
    // WIDE: the outputs have a reference of their own.
    template <bool WIDE = false>
    __device__ __forceinline__ void refer(const Rows<T, D, NT> &rows, Scores &sc, float (&c)[NT], float kc, int t0,
                                          bool masked, bool bad) {
        const int key = t0 + threadIdx.x % kWave / 16 * 16;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            c[n] = rows.factor[n] * kc;
            c[n] = c[n] < kLeastFactor ? kLeastFactor : c[n];
        }
        if (masked) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                c[n] = rows.limit[n] <= key || bad ? kLeastFactor : c[n];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    sc[i / 4][n][i % 4] = key + i < rows.limit[n] && !bad ? sc[i / 4][n][i % 4] : -INFINITY;
            }
        }
        // (factors are positive: the largest score has the largest exponent; the reference point is finite, so that
        // the exponent of a hidden score stays -inf)
        float top[NT];
        bool beyond = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            top[n] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) top[n] = fmaxf(top[n], sc[i / 4][n][i % 4]);
            beyond = fmaf(top[n], c[n], -ref[n]) > kMostWeight || beyond;
        }
        if (__any(beyond)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float now = fmaxf(ref[n], across_groups_max(top[n] * c[n]) - kBase);
                const float alpha = now == ref[n] ? 1.f : __builtin_amdgcn_exp2f(ref[n] - now);
                ref[n] = now;
                sum[n] *= alpha;
                if constexpr (!WIDE) {
#pragma unroll
                    for (int d = 0; d < DT; ++d) acc[d][n] *= alpha;
                }
            }
        }
    }
    // The weights of half hh of a tile, as P^T operands.
    typedef h8 Weights[P][NT];
    __device__ __forceinline__ void weights(const Scores &sc, const float (&c)[NT], int hh, Weights &pf) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const f32x4 &four = sc[hh * 2 + i / 4][n];
                const f32x2 w = {__builtin_amdgcn_exp2f(fmaf(four[i % 4], c[n], -ref[n])),
                                 __builtin_amdgcn_exp2f(fmaf(four[i % 4 + 1], c[n], -ref[n]))};
                const h2 hi = __builtin_convertvector(w, h2);
                pf[0][n][i] = hi[0];
                pf[0][n][i + 1] = hi[1];
                if constexpr (P == 2) {
                    sum[n] += w[0];
                    sum[n] += w[1];
                    const f32x2 rest = {w[0] - static_cast<float>(hi[0]), w[1] - static_cast<float>(hi[1])};
                    const h2 lo = __builtin_convertvector(rest, h2);
                    pf[1][n][i] = lo[0];
                    pf[1][n][i + 1] = lo[1];
                } else {
                    // (the sum of the weights as they are multiplied: their rounding cancels in part)
                    sum[n] = __builtin_amdgcn_fdot2(hi, h2{static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)}, sum[n], false);
                }
            }
    }
    // O^T of half hh of a tile: v_frag(d, hh) gives V's operands.
    template <typename VF>
    __device__ __forceinline__ void outputs(VF &&v_frag, int hh, const Weights &pf) {
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const h8 va = v_frag(d, hh);
#pragma unroll
            for (int p = P - 1; p >= 0; --p)
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    acc[d][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pf[p][n], acc[d][n], 0, 0, 0);
        }
    }
    // What the outputs are relative to where steps lie far apart: 2^num of the products of weight and step, a row's
    // own, moved like ref and by the same bound. num is a whole number, so that a step's exponent adds to it exactly.
    typedef float Reference[NT];
    __device__ __forceinline__ void clear(Reference &num) {
        clear();
#pragma unroll
        for (int n = 0; n < NT; ++n) num[n] = ref[n];
    }
    // One tile from beginning to end, V as integers; step: the step of the lane group's tokens.
    template <typename KF, typename VF>
    __device__ __forceinline__ void wide_tile(const Rows<T, D, NT> &rows, KF &&k_frag, VF &&v_frag, float kc, float step,
                                              int t0, bool masked, bool bad, Reference &num) {
        Scores sc;
        float c[NT];
        scores(rows, k_frag, sc);
        refer<true>(rows, sc, c, kc, t0, masked, bad);
        int e = -200;
        float m = 0.f;
        if (step != 0.f && fabsf(step) <= 3.402823466e38f && !bad) m = frexpf(step, &e);
        const float exponent = static_cast<float>(e);
        float top[NT];
        bool beyond = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            top[n] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) top[n] = fmaxf(top[n], sc[i / 4][n][i % 4]);
            top[n] = fmaf(top[n], c[n], exponent);
            beyond = top[n] - num[n] > kMostWeight || beyond;
        }
        if (__any(beyond)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float now = fmaxf(num[n], rintf(across_groups_max(top[n]) - kBase));
                const float alpha = now == num[n] ? 1.f : __builtin_amdgcn_exp2f(num[n] - now);
                num[n] = now;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[d][n] *= alpha;
            }
        }
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            Weights pf;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float from = exponent - num[n];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float s = sc[hh * 2 + i / 4][n][i % 4];
                    sum[n] += __builtin_amdgcn_exp2f(fmaf(s, c[n], -ref[n]));
                    float w = __builtin_amdgcn_exp2f(fmaf(s, c[n], from)) * m;
                    // (the product as it is rounded to float: formed once more inside a multiplication that rounds to
                    // half, a tie falls the other way, and the rest below belongs to another half)
                    asm("" : "+v"(w));
                    const _Float16 hi = static_cast<_Float16>(w);
                    pf[0][n][i] = hi;
                    if constexpr (P == 2) pf[1][n][i] = static_cast<_Float16>(w - static_cast<float>(hi));
                }
            }
            outputs(v_frag, hh, pf);
        }
    }
    // The outputs relative to a power of two again, each row's own.
    __device__ __forceinline__ void close_range(const Reference &num, int (&unit)[NT]) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float whole = rintf(ref[n]), f = __builtin_amdgcn_exp2f(whole - ref[n]);
            unit[n] = static_cast<int>(fmaxf(-1000.f, fminf(1000.f, num[n] - whole)));
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d][n] *= f;
        }
    }
    // One tile from beginning to end.
    template <typename KF, typename VF>
    __device__ __forceinline__ void tile(const Rows<T, D, NT> &rows, KF &&k_frag, VF &&v_frag, float kc, int t0,
                                         bool masked, bool bad) {
        Scores sc;
        float c[NT];
        scores(rows, k_frag, sc);
        refer(rows, sc, c, kc, t0, masked, bad);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            Weights pf;
            weights(sc, c, hh, pf);
            outputs(v_frag, hh, pf);
        }
    }
};

// The steps of V of a block's keys. One that is no number does not count.
struct Steps {
    int most = 0, least = 0x7f000000, others = 0;      // as bits: floats order like them
    template <typename V>
    __device__ __forceinline__ float step_of(const V &view, uint32_t page) const {
        return view.v_scale[view.scale_at(view.has(page) ? page : 0)];
    }
    __device__ __forceinline__ void take(float step, bool counts) {
        counts = counts && fabsf(step) <= 3.402823466e38f;
        const int bits = __float_as_int(step);
        most = counts ? max(most, bits) : most;
        least = counts ? min(least, bits) : least;
        others |= counts ? bits & 0x7fffff : 0;
    }
    // pages `first` .. `last` of a sequence, every stride-th of them
    template <typename V>
    __device__ __forceinline__ void look(const V &view, int first, int last, int stride) {
#pragma unroll 4
        for (int i = first; i <= last; i += stride) {
            const uint32_t page = static_cast<uint32_t>(view.table[static_cast<uint32_t>(i)]);
            take(step_of(view, page), view.has(page));
        }
    }
    // the whole wavefront's
    __device__ __forceinline__ void join() {
#pragma unroll
        for (int d = kWave / 2; d > 0; d /= 2) {
            most = max(most, __shfl_xor(most, d, kWave));
            least = min(least, __shfl_xor(least, d, kWave));
        }
        most = __builtin_amdgcn_readfirstlane(most);
        least = __builtin_amdgcn_readfirstlane(least);
        others = __any(others != 0);
    }
    __device__ __forceinline__ int exponent() const { return (most >> 23) - 127; }
    __device__ __forceinline__ bool far() const { return (most >> 23) - (least >> 23) > kSpread || others != 0; }
};

template <typename T>
__device__ __forceinline__ void store_four(T *to, const f32x4 &o) {
    if constexpr (sizeof(T) == 4) {
        __builtin_nontemporal_store(o, reinterpret_cast<f32x4 *>(to));
    } else {
        T v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(o[e]);
        __builtin_nontemporal_store(*reinterpret_cast<u32x2 *>(v), reinterpret_cast<u32x2 *>(to));
    }
}

// Means of means are formed with weights that add up to less than one: values next to the largest float stay inside
// it. (A power of two: nothing is rounded.)
__device__ __forceinline__ int unit_of(float total) {
    int e;
    frexpf(total, &e);
    return total > 0.f && total < INFINITY ? e : 0;
}

// Where a row's outputs go: the result, or (more than one split) a part of it with its statistics.
template <typename T, int D>
struct Output {
    T *out;           // null: a part
    float *part;
    float2 *stats;
    bool nothing;     // another split's

    __device__ __forceinline__ Output(const AttendArgs<T> &g, const Sequence &s, int kv, int r, int split) {
        const int token = r / g.rep;
        const int64_t at = (s.row + token) * static_cast<int64_t>(g.heads) + kv * g.rep + r % g.rep;
        const bool whole = s.length - s.fresh + token + 1 <= g.chunk;     // (all it sees lies in the first split)
        const int64_t all_rows = g.c.rows * g.heads;
        nothing = whole && split > 0;
        out = whole ? g.out + at * D : nullptr;
        part = g.part + (split * all_rows + at) * D;
        stats = reinterpret_cast<float2 *>(g.part + g.splits * all_rows * D) + split * all_rows + at;
    }
    // four neighbouring outputs
    __device__ __forceinline__ void put(int d, const f32x4 &o, float ref, float total) const {
        if (nothing) return;
        if (out) {
            store_four(out + d, o);
        } else {
            *reinterpret_cast<f32x4 *>(part + d) = o;
            if (d == 0) *stats = float2{ref, total};
        }
    }
};

// The place of a block in the work: KV head, sequence, first row, split. False: nothing to do.
struct Place {
    int kv, seq, split, r0, rows, most, least, begin, end;
    Sequence s;
};
template <typename T>
__device__ __forceinline__ bool find_place(const AttendArgs<T> &g, int tile_rows, Place &p) {
    // Blocks of one KV head next to each other would meet on different XCDs (workgroups go round robin): the
    // head is the fastest index, so with eight of them an XCD reads one head's cache.
    p.kv = blockIdx.x % g.c.kv_heads;
    // A sequence's items: its row tiles for every split it reaches. Last items first: with a causal prompt they
    // see the most keys; in a launch that fits the chip at once (fold) the second half of them goes the other
    // way, so that the blocks that share a compute unit have the same work together.
    auto tiles = [&](const Sequence &q) { return (q.fresh * g.rep + tile_rows - 1) / tile_rows; };
    Item item;
    if (!find_item(g.c, blockIdx.x / g.c.kv_heads,
                   [&](const Sequence &q) { return tiles(q) * (q.length <= g.chunk ? 1 : (q.length + g.chunk - 1) / g.chunk); },
                   item,
                   [&](int total, int order) {
                       const int half = (total + 1) / 2;
                       return order >= total ? -1 : !g.fold || order < half ? total - 1 - order : order - half;
                   })) {
        if (blockIdx.x == 0 && threadIdx.x == 0) raise_error(g.c);
        return false;
    }
    if (item.s < 0) return false;
    p.s = item.q;
    p.seq = item.s;
    if (!in_bounds(g.c, p.s)) {
        if (threadIdx.x == 0) raise_error(g.c);
        return false;
    }
    const int row_tiles = tiles(p.s);
    p.split = item.index / row_tiles;
    p.rows = p.s.fresh * g.rep;
    p.r0 = (item.index - p.split * row_tiles) * tile_rows;
    const int past = p.s.length - p.s.fresh;           // position of the sequence's first row
    p.most = past + min(p.r0 + tile_rows - 1, p.rows - 1) / g.rep + 1;   // tokens the last row sees
    p.least = past + p.r0 / g.rep + 1;
    p.begin = p.split * g.chunk;
    if (p.split > 0 && p.begin >= p.most) return false;
    p.end = min(p.most, p.begin + g.chunk);
    return true;
}

// Few rows (16 * NT of them): the wavefronts of a block deal the tiles of keys out among themselves, everything
// in registers. Bound by the cache's bytes: 64 single tokens behind 100 .. 16384 keys (8 KV heads of 128 dims, 415
// MB) take 90 us with the join, 4.6 TB/s, where a large copy reaches 5.1. A single token behind 640 keys takes
// 7.5 us, a chain of trips to memory: the sequence, its pages, the two or three tiles that each of the four wavefronts
// of its eight blocks (one per KV head) takes one after the other, the wavefronts' meeting.
template <typename T, int D, int NT, int WAVES>
__global__ __launch_bounds__(WAVES *kWave, 2) void attend_few_kernel(AttendArgs<T> g) {
    constexpr int DT = D / 16, KC = D / 64, R = 16 * NT, kPad = D + 4;
    extern __shared__ __align__(16) float lds[];   // [WAVES][R][kPad], then (max, sum) [WAVES][R]
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int col = lane % 16, grp = lane / 16;
    Place p;
    if (!find_place(g, R, p)) return;
    Rows<T, D, NT> rows;
    rows.load(g, p.s, p.kv, p.r0, p.rows);
    Softmax<T, D, NT> soft;
    soft.clear();
    const View<D> view(g, p.s, p.seq, p.kv);
    int step_exp = 0;          // E
    // pages of the tokens whose K rows (by lane column) and whose V columns (by lane group) a lane loads
    auto pages_of = [&](int t0, uint32_t &pk, uint32_t &pv) {
        pk = view.page_of(t0 + (col / 4) * 16);
        pv = view.page_of(t0 + grp * 16);
    };
    auto fetch = [&](Tile<D> &t, int t0, uint32_t pk, uint32_t pv) {
        t.bad = !view.has(pv);
        if (t.bad) raise_error(g.c);
        pk = view.has(pk) ? pk : 0;
        pv = t.bad ? 0 : pv;
        const int mask = view.size - 1;
        const int8_t *k = view.at(view.k, pk, ((t0 + (col / 4) * 16 + col % 4) & mask) * D + grp * 16);
        const int8_t *v = view.at(view.v, pv, ((t0 + grp * 16) & mask) + col * view.size);
        t.k_scale = view.k_scale[view.scale_at(pv)];
        t.v_scale = view.v_scale[view.scale_at(pv)];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < KC; ++c) t.k[j][c] = *reinterpret_cast<const u32x4 *>(k + j * 4 * D + c * 64);
#pragma unroll
        for (int d = 0; d < DT; ++d) t.v[d] = *reinterpret_cast<const u32x4 *>(v + d * 16 * view.size);
    };
    auto compute = [&](const Tile<D> &t, int t0) {
        // V's steps relative to the largest; a step that is no number marks the scores instead
        const bool odd = !(fabsf(t.v_scale) <= 3.402823466e38f) || t.bad;
        const _Float16 f1 = static_cast<_Float16>(odd ? 0.f : ldexpf(t.v_scale, -step_exp));
        const _Float16 b1 = static_cast<_Float16>(-1152.f) * f1;
        const h2 vf = {f1, f1}, vbias = {b1, b1};
        const float kc = odd && !t.bad ? __uint_as_float(0x7fc00000u) : t.k_scale;
        soft.tile(
            rows,
            [&](int j, int q) {
                const u32x4 raw = t.k[j][q / 2];
                return q % 2 ? widen(raw[2], raw[3]) : widen(raw[0], raw[1]);
            },
            [&](int d, int hh) { return widen_scaled(t.v[d][2 * hh], t.v[d][2 * hh + 1], vf, vbias); }, kc, t0,
            t0 + kTileKeys > p.least || __any(t.bad), t.bad);
    };

    // tiles begin + 64 * (wave + i * WAVES): the next one is on its way while one is computed, the page
    // numbers of the one after that besides
    constexpr int kStride = kTileKeys * WAVES;
    int t0 = p.begin + wave * kTileKeys;
    int unit[NT] = {};         // of the outputs, a row's
    if (t0 < p.end) {
        // the steps' pages come beside the first tile's, the steps beside the tile
        constexpr int kAhead = 4;
        const int first = (p.begin >> view.shift) + lane, last = view.page_at((p.end - 1) | (kTileKeys - 1));
        uint32_t ahead[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            ahead[i] = static_cast<uint32_t>(view.table[static_cast<uint32_t>(min(first + i * kWave, last))]);
        Tile<D> one, two;
        uint32_t pk, pv;
        pages_of(t0, pk, pv);
        uint32_t next_pk = 0, next_pv = 0;
        if (t0 + kStride < p.end) pages_of(t0 + kStride, next_pk, next_pv);
        Steps steps;
        float step[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) step[i] = steps.step_of(view, ahead[i]);
        fetch(one, t0, pk, pv);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) steps.take(step[i], view.has(ahead[i]));
        steps.look(view, first + kAhead * kWave, last, kWave);
        steps.join();
        step_exp = steps.exponent();
#pragma unroll
        for (int n = 0; n < NT; ++n) unit[n] = step_exp;
        if (__builtin_expect(steps.far(), 0)) {
            typename Softmax<T, D, NT>::Reference num;
            soft.clear(num);
            for (; t0 < p.end; t0 += kStride) {
                Tile<D> t;
                uint32_t pk, pv;
                pages_of(t0, pk, pv);
                fetch(t, t0, pk, pv);
                const bool marked = !(fabsf(t.v_scale) <= 3.402823466e38f) && !t.bad;
                soft.wide_tile(
                    rows,
                    [&](int j, int q) {
                        const u32x4 raw = t.k[j][q / 2];
                        return q % 2 ? widen(raw[2], raw[3]) : widen(raw[0], raw[1]);
                    },
                    [&](int d, int hh) { return widen(t.v[d][2 * hh], t.v[d][2 * hh + 1]); },
                    marked ? __uint_as_float(0x7fc00000u) : t.k_scale, t.v_scale, t0,
                    t0 + kTileKeys > p.least || __any(t.bad), t.bad, num);
            }
            soft.close_range(num, unit);
        } else {
            while (true) {
                auto half_step = [&](Tile<D> &now, Tile<D> &next) {
                    const int t1 = t0 + kStride, t2 = t1 + kStride;
                    const bool more = t1 < p.end;
                    if (more) {
                        const uint32_t a = next_pk, b = next_pv;
                        if (t2 < p.end) pages_of(t2, next_pk, next_pv);
                        fetch(next, t1, a, b);
                    }
                    compute(now, t0);
                    t0 = t1;
                    return more;
                };
                if (!half_step(one, two)) break;
                if (!half_step(two, one)) break;
            }
        }
    }

    // a wavefront's own mean first (bounded by the largest |v|), then the mean of the means
    float2 *stats = reinterpret_cast<float2 *>(lds + WAVES * R * kPad);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const float total = across_groups_sum(soft.sum[n]);
        const float inv = total == 0.f ? 0.f : 1.f / total;
        if (grp == 0) stats[wave * R + n * 16 + col] = float2{soft.ref[n], total};
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            f32x4 o = soft.acc[d][n] * inv;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = ldexpf(o[i], unit[n]);
            *reinterpret_cast<f32x4 *>(lds + (wave * R + n * 16 + col) * kPad + d * 16 + grp * 4) = o;
        }
    }
    __syncthreads();
    for (int i = tid; i < R * (D / 4); i += WAVES * kWave) {
        const int row = i / (D / 4), d = i % (D / 4) * 4;
        if (p.r0 + row >= p.rows) break;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stats[w * R + row].x);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float total = 0.f, weight[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float2 st = stats[w * R + row];
            weight[w] = st.y == 0.f ? 0.f : st.y * __builtin_amdgcn_exp2f(st.x - top);
            total += weight[w];
        }
        const int unit = unit_of(total);
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
            o += *reinterpret_cast<const f32x4 *>(lds + (w * R + row) * kPad + d) * ldexpf(weight[w], -unit);
        o *= total == 0.f ? 0.f : 1.f / ldexpf(total, -unit);
        Output<T, D>(g, p.s, p.kv, p.r0 + row, p.split).put(d, o, top, total);
    }
}

// Many rows: four wavefronts of 16 * NT rows each walk the same tiles of keys. A wavefront fetches and widens a
// quarter of a tile and leaves it in LDS as the MFMA operands it is (64 lanes x 16 bytes each, read back as
// they were written: no bank conflicts); two buffers, one barrier per tile. What widening costs, and the
// trips to the caches, are shared by the block's rows. Neither pipe is full: a prompt of 8192 tokens has the vector
// pipes busy 63 % and the matrix pipes 42 % of the cycles, 2048 tokens of 64 dims in floats 45 and 25 %. Beside the 64
// MFMAs of a tile (D = 128, 16-bit types) a wavefront has some 270 vector instructions (32 exponentials and as many
// arguments and maxima, the widening, addresses), and only a part of them runs under MFMAs: with two wavefronts per
// SIMD, sixteen v_mfma_f32_16x16x32_f16 each take 541 cycles alone, 578, 595, 713 and 825 with one to four
// multiply-adds behind every one of them, 566 with an exponential. So the scores of the next tile are computed beside
// the weights of this one (a prompt of 8192 tokens, 32 heads of 128 dims: 627 us without when it took 585 so; now
// 576, 955 TFLOP/s of the causal half), the largest score is looked for before the factors are applied, and an address is
// one wide multiply. Measured and dropped: wavefront priorities (592 us), orders of MFMAs and vector instructions
// given to the compiler (no faster), branches around the last fetch (the registers they hold).
constexpr int kManyWaves = 4;
template <typename T, int D, int NT>
__global__ __launch_bounds__(kManyWaves *kWave, 2) void attend_many_kernel(AttendArgs<T> g) {
    constexpr int DT = D / 16, KC = D / 64, KH = D / 32, R = 16 * NT * kManyWaves, DW = DT / kManyWaves;
    extern __shared__ __align__(16) u32x4 frags[];   // K [2][4][KH][64 lanes], V [2][DT][2][64 lanes]
    const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int col = lane % 16, grp = lane / 16;
    Place p;
    if (!find_place(g, R, p)) return;
    const int my_r0 = p.r0 + wave * 16 * NT;
    Rows<T, D, NT> rows;
    rows.load(g, p.s, p.kv, my_r0, p.rows);
    Softmax<T, D, NT> soft;
    soft.clear();
    const int past = p.s.length - p.s.fresh;
    const int my_least = past + my_r0 / g.rep + 1;

    const View<D> view(g, p.s, p.seq, p.kv);
    // a quarter of a tile: the K rows of one S^T block, DW row blocks of V
    struct Raw {
        u32x4 k[KC], v[DW];
        float k_scale, v_scale;       // of V's tile
        bool bad;
    };
    auto k_page = [&](int t0) { return view.page_of(t0 + (col / 4) * 16); };
    auto v_page = [&](int t0) { return view.page_of(t0 + grp * 16); };
    auto fetch_k = [&](Raw &t, int t0, uint32_t page) {
        const int8_t *k = view.at(view.k, view.has(page) ? page : 0,
                                  ((t0 + (col / 4) * 16 + wave * 4 + col % 4) & (view.size - 1)) * D + grp * 16);
#pragma unroll
        for (int c = 0; c < KC; ++c) t.k[c] = *reinterpret_cast<const u32x4 *>(k + c * 64);
    };
    auto fetch_v = [&](Raw &t, int t0, uint32_t page) {
        t.bad = !view.has(page);
        if (t.bad) raise_error(g.c);
        page = t.bad ? 0 : page;
        const int8_t *v = view.at(view.v, page, ((t0 + grp * 16) & (view.size - 1)) + (wave * DW * 16 + col) * view.size);
        t.k_scale = view.k_scale[view.scale_at(page)];
        t.v_scale = view.v_scale[view.scale_at(page)];
#pragma unroll
        for (int d = 0; d < DW; ++d) t.v[d] = *reinterpret_cast<const u32x4 *>(v + d * 16 * view.size);
    };
    // what every wavefront knows of a tile whose V is in LDS
    struct Ready {
        float kc;
        bool bad;
    };
    Steps steps;
    constexpr int kKFrags = 4 * KH, kVFrags = 2 * DT;
    u32x4 *const k_lds = frags + lane, *const v_lds = frags + 2 * kKFrags * kWave + lane;
    auto widen_k = [&](const Raw &t, int buf) {
        u32x4 *to = k_lds + buf * kKFrags * kWave;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            to[(wave * KH + 2 * c) * kWave] = __builtin_bit_cast(u32x4, widen(t.k[c][0], t.k[c][1]));
            to[(wave * KH + 2 * c + 1) * kWave] = __builtin_bit_cast(u32x4, widen(t.k[c][2], t.k[c][3]));
        }
    };
    auto widen_v = [&](const Raw &t, int buf) {
        const bool odd = !(fabsf(t.v_scale) <= 3.402823466e38f) || t.bad;
        const _Float16 f1 = static_cast<_Float16>(odd ? 0.f : ldexpf(t.v_scale, -steps.exponent()));
        const _Float16 b1 = static_cast<_Float16>(-1152.f) * f1;
        const h2 vf = {f1, f1}, vbias = {b1, b1};
        u32x4 *to = v_lds + buf * kVFrags * kWave;
#pragma unroll
        for (int d = 0; d < DW; ++d)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
                to[((wave * DW + d) * 2 + hh) * kWave] =
                    __builtin_bit_cast(u32x4, widen_scaled(t.v[d][2 * hh], t.v[d][2 * hh + 1], vf, vbias));
        return Ready{odd && !t.bad ? __uint_as_float(0x7fc00000u) : t.k_scale, t.bad};
    };

    int unit[NT] = {};       // of the outputs, a row's
    if (p.begin < p.end) {
        // each wavefront looks over a quarter of the pages' steps
        int *const shares = reinterpret_cast<int *>(frags);
        steps.look(view, (p.begin >> view.shift) + tid, view.page_at((p.end - 1) | (kTileKeys - 1)), kManyWaves * kWave);
        steps.join();
        if (lane < 3) shares[wave * 3 + lane] = lane == 0 ? steps.most : lane == 1 ? steps.least : steps.others;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kManyWaves; ++w) {
            steps.most = max(steps.most, __builtin_amdgcn_readfirstlane(shares[w * 3]));
            steps.least = min(steps.least, __builtin_amdgcn_readfirstlane(shares[w * 3 + 1]));
            steps.others |= __builtin_amdgcn_readfirstlane(shares[w * 3 + 2]);
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n) unit[n] = steps.exponent();
    }
    if (__builtin_expect(p.begin < p.end && steps.far(), 0)) {
        // one tile after the other
        Raw raw;
        typename Softmax<T, D, NT>::Reference num;
        soft.clear(num);
        for (int t0 = p.begin; t0 < p.end; t0 += kTileKeys) {
            fetch_k(raw, t0, k_page(t0));
            fetch_v(raw, t0, v_page(t0));
            __syncthreads();      // everyone has read what the buffers hold
            widen_k(raw, 0);
#pragma unroll
            for (int d = 0; d < DW; ++d)
#pragma unroll
                for (int hh = 0; hh < 2; ++hh)
                    v_lds[((wave * DW + d) * 2 + hh) * kWave] =
                        __builtin_bit_cast(u32x4, widen(raw.v[d][2 * hh], raw.v[d][2 * hh + 1]));
            __syncthreads();
            const bool marked = !(fabsf(raw.v_scale) <= 3.402823466e38f) && !raw.bad;
            soft.wide_tile(
                rows, [&](int j, int q) { return __builtin_bit_cast(h8, k_lds[(j * KH + q) * kWave]); },
                [&](int d, int hh) { return __builtin_bit_cast(h8, v_lds[(d * 2 + hh) * kWave]); },
                marked ? __uint_as_float(0x7fc00000u) : raw.k_scale, raw.v_scale, t0,
                t0 + kTileKeys > my_least || __any(raw.bad), raw.bad, num);
        }
        soft.close_range(num, unit);
    } else if (p.begin < p.end) {
        // K is one tile ahead of V: a tile's scores are computed beside the weights of the tile before it, so that
        // the matrix cores and the other units have work at the same time. (Past the last tile the scores are of
        // what the buffer happens to hold, and are not used.)
        Raw raw;
        fetch_k(raw, p.begin, k_page(p.begin));
        fetch_v(raw, p.begin, v_page(p.begin));
        Ready ready = widen_v(raw, 0);
        widen_k(raw, 0);
        if (p.begin + kTileKeys < p.end) {
            fetch_k(raw, p.begin + kTileKeys, k_page(p.begin + kTileKeys));
            widen_k(raw, 1);
        }
        uint32_t pk = k_page(p.begin + 2 * kTileKeys), pv = v_page(p.begin + kTileKeys);
        int buf = 0;        // of this tile
        typename Softmax<T, D, NT>::Scores sc;
        auto score = [&](int from, typename Softmax<T, D, NT>::Scores &to) {
            const u32x4 *k = k_lds + from * kKFrags * kWave;
            soft.scores(rows, [&](int j, int q) { return __builtin_bit_cast(h8, k[(j * KH + q) * kWave]); }, to);
        };
        __syncthreads();
        score(0, sc);
        for (int t0 = p.begin; t0 < p.end; t0 += kTileKeys) {
            const int t1 = t0 + kTileKeys, t2 = t1 + kTileKeys;
            fetch_v(raw, t1, pv);
            fetch_k(raw, t2, pk);
            pk = k_page(t2 + kTileKeys);
            pv = v_page(t2);
            __syncthreads();      // V of this tile and K of the next are in LDS, the other buffers have been read by everyone
            // (a wavefront whose rows see nothing of the tile goes along: the branch around it cost more, in copies
            // of the accumulators where its two sides meet)
            float c[NT];
            soft.refer(rows, sc, c, ready.kc, t0, t1 > my_least || __any(ready.bad), ready.bad);
            const u32x4 *v = v_lds + buf * kVFrags * kWave;
            auto v_frag = [&](int d, int hh) { return __builtin_bit_cast(h8, v[(d * 2 + hh) * kWave]); };
            typename Softmax<T, D, NT>::Weights pf[2];
            typename Softmax<T, D, NT>::Scores next;
            if constexpr (Softmax<T, D, NT>::P * D < 256) {
                score(buf ^ 1, next);
                soft.weights(sc, c, 0, pf[0]);
                soft.weights(sc, c, 1, pf[1]);
                soft.outputs(v_frag, 0, pf[0]);
                soft.outputs(v_frag, 1, pf[1]);
            } else {
                soft.weights(sc, c, 0, pf[0]);
                soft.outputs(v_frag, 0, pf[0]);
                soft.weights(sc, c, 1, pf[1]);
                soft.outputs(v_frag, 1, pf[1]);
                score(buf ^ 1, next);
            }
            ready = widen_v(raw, buf ^ 1);
            widen_k(raw, buf);
            buf ^= 1;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int n = 0; n < NT; ++n) sc[j][n] = next[j][n];
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const float total = across_groups_sum(soft.sum[n]);
        const float inv = total == 0.f ? 0.f : 1.f / total;
        const int r = my_r0 + n * 16 + col;
        if (r >= p.rows) continue;
        const Output<T, D> out(g, p.s, p.kv, r, p.split);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            f32x4 o = soft.acc[d][n] * inv;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = ldexpf(o[i], unit[n]);
            out.put(d * 16 + grp * 4, o, soft.ref[n], total);
        }
    }
}

// The splits of the rows that see more than one, joined: D / 4 lanes per (row, head).
template <typename T, int D>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs<T> g) {
    constexpr int kLanes = D / 4, kRows = 256 / kLanes;
    const int64_t all_rows = g.c.rows * g.heads;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kLanes;
    const int64_t row = at / g.heads;
    const int d = threadIdx.x % kLanes * 4;
    Sequence s;
    if (!starts_ascend(g.c) || at >= all_rows || !sequence_of_row(g.c, row, s)) return;
    const int limit = s.length - s.fresh + static_cast<int>(row - s.row) + 1;
    if (limit <= g.chunk) return;
    const int parts = (limit + g.chunk - 1) / g.chunk;
    const float2 *stats = reinterpret_cast<const float2 *>(g.part + g.splits * all_rows * D) + at;
    const float *part = g.part + at * D + d;
    // groups of eight parts, their loads in flight together; the reference point moves between groups
    constexpr int kGroup = 8;
    float top = -INFINITY, total = 0.f;
    int unit = 0;        // of o
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < parts; i0 += kGroup) {
        float2 st[kGroup];
        f32x4 v[kGroup];
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
            const int64_t from = min(i0 + i, parts - 1) * all_rows;
            st[i] = stats[from];
            v[i] = *reinterpret_cast<const f32x4 *>(part + from * D);
            if (i0 + i >= parts) st[i].y = 0.f;
        }
        float now = top;
#pragma unroll
        for (int i = 0; i < kGroup; ++i) now = fmaxf(now, st[i].x);
        const float alpha = total == 0.f ? 0.f : __builtin_amdgcn_exp2f(top - now);
        top = now;
        total *= alpha;
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
            st[i].y = st[i].y == 0.f ? 0.f : st[i].y * __builtin_amdgcn_exp2f(st[i].x - top);
            total += st[i].y;
        }
        const int was = unit;
        unit = unit_of(total);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = ldexpf(o[j] * alpha, was - unit);
#pragma unroll
        for (int i = 0; i < kGroup; ++i) o += v[i] * ldexpf(st[i].y, -unit);
    }
    store_four(g.out + at * D + d, o * (total == 0.f ? 0.f : 1.f / ldexpf(total, -unit)));
}

// How a call is cut: rows per block, tiles of rows, splits of the keys.
struct Plan {
    bool many;
    int nt;
    int64_t pieces;
    int32_t splits, chunk;
    size_t workspace;
};
constexpr int kFewWaves = 4;

Plan plan_for(const PagedArgs &c, int32_t dtype, int head_dim, int64_t heads) {
    Plan p{};
    const int64_t rep = heads / c.kv_heads, rows = c.max_new * rep;
    p.many = rows > 32;
    p.nt = p.many ? 2 : rows <= 16 || head_dim == 128 ? 1 : 2;
    const int64_t tile = 16 * p.nt * (p.many ? kManyWaves : 1);
    // upper bound of the row tiles; exact where all sequences bring the same rows (a sequence that brings more than
    // the call allows, be that none, is a tile that reports it)
    const int64_t ragged = c.rows * rep / tile + c.seqs, even = c.seqs * (rows > 0 ? (rows + tile - 1) / tile : 1);
    p.pieces = ragged < even ? ragged : even;
    const int64_t step = kTileKeys * (p.many ? 1 : kFewWaves);
    const int64_t len = c.max_length > 0 ? c.max_length : 1;
    const int64_t blocks = p.pieces * c.kv_heads;
    // Splits of the keys. A part costs its rows a trip through memory, and the call a second kernel.
    // Many rows: as many as make two blocks per compute unit (they are resident together: 512 rows behind 8192
    // keys, 8 KV heads of 128 dims, take 94 us in 4 splits = 512 blocks, 104 us in 6, 105 in 8, 134 in 16; a
    // prompt of 2048 tokens in one piece 58 us, in two 71); in a ragged call, where most sequences do not reach
    // the bounds, four times that (six sequences of 1 .. 512 rows behind 512 .. 16384 keys: 132 us, 195 us without
    // the factor, 131 us with twice, 145 us with eight times); prompts with little before them are not thinned out
    // for being ragged.
    // Few rows: a block per compute unit, and pieces of 2048 keys beyond 4096, so that sequences of different
    // lengths even out (64 sequences of 100 .. 16384 keys: 91 us, in pieces of 4096 109 us, of 1024 97 us; 32
    // sequences of 4096 keys: 52 us in one piece, 57 us in two). Up to 1024 keys the second kernel costs more
    // than it saves.
    int64_t splits;
    if (p.many) {
        const bool uneven = c.rows < c.seqs * c.max_new && c.max_length > 2 * c.max_new;
        splits = (uneven ? 8 : 2) * kNumCU / blocks;
    } else {
        splits = len <= 1024 ? 1 : (kNumCU + blocks - 1) / blocks;
        if (len > 4096 && splits < (len + 2047) / 2048) splits = (len + 2047) / 2048;
    }
    if (splits < 1) splits = 1;
    const int64_t most = p.many ? (len + 511) / 512 : (len + step - 1) / step;
    splits = splits < most ? splits : most;
    splits = splits < 64 ? splits : 64;
    const int64_t chunk = ((len + splits - 1) / splits + step - 1) / step * step;
    p.chunk = static_cast<int32_t>(chunk);
    p.splits = static_cast<int32_t>((len + chunk - 1) / chunk);
    p.workspace = p.splits > 1 ? static_cast<size_t>(p.splits) * c.rows * heads * (head_dim + 2) * sizeof(float) : 0;
    return p;
}

template <typename T, int D, int NT>
int32_t launch_few(hipStream_t st, const AttendArgs<T> &g, int64_t blocks) {
    constexpr int lds = kFewWaves * 16 * NT * ((D + 4) * 4 + 8);
    attend_few_kernel<T, D, NT, kFewWaves><<<static_cast<uint32_t>(blocks), kFewWaves * kWave, lds, st>>>(g);
    return launch_status();
}

template <typename T, int D>
int32_t launch_many(hipStream_t st, const AttendArgs<T> &g, int64_t blocks) {
    constexpr int NT = 2;
    constexpr int lds = 2 * (4 * (D / 32) + 2 * (D / 16)) * kWave * 16;
    static_assert(lds <= 64 * 1024, "no more than a block has without asking");
    attend_many_kernel<T, D, NT><<<static_cast<uint32_t>(blocks), kManyWaves * kWave, lds, st>>>(g);
    return launch_status();
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
    if (attend_checks(dtype, cache, batch, heads, nullptr, &c) != RMLK_OK || c.seqs == 0 || c.rows == 0) return 0;
    return plan_for(c, dtype, cache->head_dim, heads).workspace;
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
    const Plan plan = plan_for(c, dtype, d, heads);
    const int64_t blocks = plan.pieces * c.kv_heads * plan.splits;
    const int64_t join_blocks = (c.rows * heads * (d / 4) + 255) / 256;
    if (blocks > (1 << 23) || join_blocks > (1 << 23) || c.rows * heads > 0x3fffffff) return RMLK_ERR_TOO_LARGE;
    if (plan.workspace > 0) {
        if (!workspace) return RMLK_ERR_NULL_POINTER;
        if (!aligned16(workspace)) return RMLK_ERR_UNSUPPORTED;
        if (workspace_bytes < plan.workspace) return RMLK_ERR_WORKSPACE;
    }
    return with_activation(dtype, [&](auto tag) {
        using T = decltype(tag);
        AttendArgs<T> g{};
        g.c = c;
        g.q = static_cast<const T *>(q);
        g.out = static_cast<T *>(out);
        g.part = static_cast<float *>(workspace);
        g.q_stride = q_stride;
        g.heads = static_cast<int32_t>(heads);
        g.rep = static_cast<int32_t>(heads / c.kv_heads);
        g.scale = (scale_is_mul ? scale : 1.f / scale) * kLog2e;
        g.splits = plan.splits;
        g.chunk = plan.chunk;
        g.fold = plan.many && blocks <= 3 * kNumCU;
        int32_t bad;
        if (plan.many) bad = d == 64 ? launch_many<T, 64>(st, g, blocks) : launch_many<T, 128>(st, g, blocks);
        else if (d == 64) bad = plan.nt == 1 ? launch_few<T, 64, 1>(st, g, blocks) : launch_few<T, 64, 2>(st, g, blocks);
        else bad = launch_few<T, 128, 1>(st, g, blocks);
        if (bad != RMLK_OK || plan.splits == 1) return bad;
        if (d == 64) attend_join_kernel<T, 64><<<static_cast<uint32_t>(join_blocks), 256, 0, st>>>(g);
        else attend_join_kernel<T, 128><<<static_cast<uint32_t>(join_blocks), 256, 0, st>>>(g);
        return launch_status();
    });
}

}  // extern "C"
