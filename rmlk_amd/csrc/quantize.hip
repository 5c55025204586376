// Rows of activations (or of weights) to int8 with one scale per row, plain or behind RMSNorm.
//
//   scale = float(max|y| / 127),   q = y / scale rounded to nearest even
//
// A value close to the border between two integers must fall the right way whatever the arithmetic
// does, or the result depends on the kernel: where y is a float, q0 = rint(y * (1 / scale)) is the
// right integer or its neighbour, and r = fma(-q0, scale, y) is exact (q0 has 7 bits, and r, at most
// about scale / 2, is a multiple of the smaller operand's last bit), so comparing |r| with scale / 2
// decides exactly. Behind the norm y is a real number that is evaluated in double.
#include "paged.hpp"

namespace rmlk {
namespace {

constexpr float kSmallest = 0x1p-100f;   // rows below it are stored as zeros: 127 / max|y| stays finite

template <int THREADS, typename T, typename Op>
__device__ __forceinline__ T block_reduce(T v, T *lds, Op op) {
    if constexpr (THREADS == kWave) return v;
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    T r = lds[0];
#pragma unroll
    for (int i = 1; i < THREADS / kWave; ++i) r = op(r, lds[i]);
    __syncthreads();
    return r;
}

// Eight values of a row from column c on, zeros behind its end. Rows start where their elements do: the memory takes
// 16-byte accesses at any address (4118 rows of 2941 bfloat16 14.1 us, element by element 15.9; 1729 rows of 9254
// floats with the norm 33 us, 131 us element by element and held in registers).
template <typename T>
__device__ __forceinline__ void load_eight(const T *row, int c, int cols, T (&out)[8]) {
    if (c + 8 <= cols) {
#pragma unroll
        for (size_t u = 0; u < sizeof(T) / 2; ++u)
            reinterpret_cast<u32x4 *>(out)[u] = load_unit(row + c + u * (16 / sizeof(T)));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = c + e < cols ? row[c + e] : static_cast<T>(0.f);
    }
}
template <typename T>
__device__ __forceinline__ void store_eight(T *row, int c, int cols, const T (&v)[8]) {
    if (c + 8 <= cols) {
#pragma unroll
        for (size_t u = 0; u < sizeof(T) / 2; ++u)
            store_unit(row + c + u * (16 / sizeof(T)), reinterpret_cast<const u32x4 *>(v)[u]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < cols) row[c + e] = v[e];
    }
}
__device__ __forceinline__ uint64_t pack_eight(const int (&n)[8]) {
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        lo |= static_cast<uint32_t>(n[e] & 255) << (8 * e);
        hi |= static_cast<uint32_t>(n[4 + e] & 255) << (8 * e);
    }
    return static_cast<uint64_t>(hi) << 32 | lo;
}

// A block per row, which it holds in registers: CH units of eight values per thread, one pass over memory.
// CH = 0: a row of any length, read twice (the second time from the caches). Bound by the memory: 4096 rows of 8192
// floats, 168 MB, take 34.2 us = 4.9 TB/s, where a large copy reaches 5.1. (Streaming stores of q: 31.9 us, but what
// reads q next then waits for the memory: with a product of q and its scales behind it 133 us against 112.)
template <typename T, int THREADS, int CH>
__global__ __launch_bounds__(THREADS) void quantize_rows_kernel(const T *__restrict__ xs, int64_t ldx, int64_t rows,
                                                                int32_t cols, int8_t *__restrict__ qs, int64_t ldq,
                                                                float *__restrict__ scale) {
    __shared__ uint32_t lds[THREADS / kWave];
    const int padded = (cols + 15) & ~15, tid = threadIdx.x;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *x = xs + row * ldx;
        int8_t *q = qs + row * ldq;
        T held[CH > 0 ? CH : 1][8];
        // magnitudes compare like their bits, NaN and infinity above everything finite
        uint32_t top = 0;
        auto magnitude = [&](const T (&v)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(to_float(v[e])) & 0x7fffffffu);
        };
        if constexpr (CH > 0) {
#pragma unroll
            for (int i = 0; i < CH; ++i) load_eight(x, (i * THREADS + tid) * 8, cols, held[i]);
#pragma unroll
            for (int i = 0; i < CH; ++i) magnitude(held[i]);
        } else {
            for (int c = tid * 8; c < cols; c += THREADS * 8) {
                load_eight(x, c, cols, held[0]);
                magnitude(held[0]);
            }
        }
        top = block_reduce<THREADS>(wave_max(top), lds, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
        const float amax = __uint_as_float(top);
        const bool zero = !(amax >= kSmallest) || top >= 0x7f800000u;
        const float s = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : zero ? 0.f : amax / 127.f;
        const float inv = zero ? 0.f : 1.f / s, half = 0.5f * s;
        auto quantize = [&](const T (&v)[8], int c) {
            int n[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = to_float(v[e]), q0 = rintf(y * inv), r = fmaf(-q0, s, y), a = fabsf(r);
                n[e] = static_cast<int>(q0);
                if (a > half || (a == half && (n[e] & 1))) n[e] += r > 0.f ? 1 : -1;
                n[e] = zero ? 0 : min(127, max(-127, n[e]));
            }
            *reinterpret_cast<uint64_t *>(q + c) = pack_eight(n);
        };
        if constexpr (CH > 0) {
#pragma unroll
            for (int i = 0; i < CH; ++i)
                if (const int c = (i * THREADS + tid) * 8; c < padded) quantize(held[i], c);
        } else {
            for (int c = tid * 8; c < padded; c += THREADS * 8) {
                load_eight(x, c, cols, held[0]);
                quantize(held[0], c);
            }
        }
        if (tid == 0) scale[row] = s;
    }
}

// The same behind RMSNorm: y = x * f * gamma with f = 1 / sqrt(mean(x^2) + eps). The products x * gamma are exact
// in double (48 bits); their largest magnitude times f is the row's, and
// y / scale = x * gamma * (f / scale). One row of 2048 floats with a sum takes 2.9 us: a launch, a trip to memory
// and three reductions over the block.
template <typename T, int THREADS, int CH>
__global__ __launch_bounds__(THREADS) void norm_quantize_kernel(const T *xs, const T *bs, const float *__restrict__ gamma,
                                                                float eps, int64_t rows, int32_t cols, T *sums,
                                                                int8_t *__restrict__ qs, int64_t ldq,
                                                                float *__restrict__ scale) {
    __shared__ double lds[THREADS / kWave], lds2[THREADS / kWave], lds3[THREADS / kWave];
    const int padded = (cols + 15) & ~15, tid = threadIdx.x;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *x = xs + row * cols, *b = bs ? bs + row * cols : nullptr;
        T *sum = bs ? sums + row * cols : nullptr;
        int8_t *q = qs + row * ldq;
        T held[CH > 0 ? CH : 1][8];
        float gm[CH > 0 ? CH : 1][8];
        double square = 0.0, top = 0.0, odd = 0.0;
        // forms the sum of a unit where there is one, adds up squares, finds the largest product with gamma
        auto measure = [&](int c, T (&v)[8], const T (&w)[8], const float (&gm)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (b) v[e] = static_cast<T>(to_float(v[e]) + to_float(w[e]));
                const double y = to_float(v[e]), p = y * static_cast<double>(gm[e]);
                square = fma(y, y, square);
                top = fmax(top, fabs(p));
                odd = fma(p, 0.0, odd);       // NaN with the first product that is not finite
            }
            if (b && c < cols) store_eight(sum, c, cols, v);
        };
        if constexpr (CH > 0) {
            T w[CH][8];
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int c = (i * THREADS + tid) * 8;
                load_eight(x, c, cols, held[i]);
                if (b) load_eight(b, c, cols, w[i]);
                load_eight(gamma, c, cols, gm[i]);
            }
#pragma unroll
            for (int i = 0; i < CH; ++i) measure((i * THREADS + tid) * 8, held[i], w[i], gm[i]);
        } else {
            for (int c = tid * 8; c < cols; c += THREADS * 8) {
                T w[8];
                load_eight(x, c, cols, held[0]);
                if (b) load_eight(b, c, cols, w);
                load_eight(gamma, c, cols, gm[0]);
                measure(c, held[0], w, gm[0]);
            }
        }
        auto add = [](double a, double c) { return a + c; };
        square = block_reduce<THREADS>(wave_sum(square), lds, add);
        odd = block_reduce<THREADS>(wave_sum(odd), lds2, add);
        top = block_reduce<THREADS>(wave_max(top), lds3, [](double a, double c) { return c > a ? c : a; });
        const double f = 1.0 / sqrt(square / cols + static_cast<double>(eps));
        const double amax = top * f;
        const float s_of = static_cast<float>(amax / 127.0);
        // (infinite squares, an infinite or NaN product, a scale beyond float)
        const bool bad = !(odd == 0.0) || !(square <= 1.7976931348623157e308) || !(s_of <= 3.402823466e38f);
        const bool zero = bad || amax < static_cast<double>(kSmallest);
        const float s = bad ? __uint_as_float(0x7fc00000u) : zero ? 0.f : s_of;
        const double to_step = zero ? 0.0 : f / static_cast<double>(s);
        auto quantize = [&](const T (&v)[8], const float (&gm)[8], int c) {
            int n[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double p = static_cast<double>(to_float(v[e])) * static_cast<double>(gm[e]);
                n[e] = zero ? 0 : min(127, max(-127, static_cast<int>(rint(p * to_step))));
            }
            *reinterpret_cast<uint64_t *>(q + c) = pack_eight(n);
        };
        if constexpr (CH > 0) {
#pragma unroll
            for (int i = 0; i < CH; ++i)
                if (const int c = (i * THREADS + tid) * 8; c < padded) quantize(held[i], gm[i], c);
        } else {
            for (int c = tid * 8; c < padded; c += THREADS * 8) {
                load_eight(b ? sum : x, c, cols, held[0]);      // (every thread reads back what it wrote itself)
                load_eight(gamma, c, cols, gm[0]);
                quantize(held[0], gm[0], c);
            }
        }
        if (tid == 0) scale[row] = s;
    }
}

// f(threads, units per thread) as constants: a wavefront for short rows, larger blocks for longer ones. Rows of up
// to 16384 values are held in registers, behind the norm, which has gamma and a second operand besides, of up to
// 4096: longer ones are read twice by 512 threads (4096 rows of 8192 floats with a sum: 95 us; held by 256 threads
// 120, by 1024 threads 102 us; read twice by 256 threads 100. One row: 5.2, 5.8, 4.9 and 6.0 us).
template <bool NORM, typename F>
int32_t with_row_shape(int32_t cols, F &&f) {
    using std::integral_constant;
    const int units = (cols + 15) / 16 * 2;
    if (units <= 64) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (units <= 256) return f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    if (units <= 512) return f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    if constexpr (NORM) {
        return f(integral_constant<int, 512>{}, integral_constant<int, 0>{});
    } else {
        if (units <= 1024) return f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
        if (units <= 2048) return f(integral_constant<int, 256>{}, integral_constant<int, 8>{});
        return f(integral_constant<int, 256>{}, integral_constant<int, 0>{});
    }
}
inline uint32_t row_blocks(int64_t rows) { return static_cast<uint32_t>(rows < (1 << 20) ? rows : (1 << 20)); }

int32_t row_checks(int32_t dtype, int64_t rows, int64_t cols, const void *q, int64_t ldq) {
    if (rows < 0 || cols < 0) return RMLK_ERR_INVALID_ARGUMENT;
    if (!is_activation(dtype)) return RMLK_ERR_UNSUPPORTED;
    if (ldq % 16 != 0 || !aligned16(q)) return RMLK_ERR_UNSUPPORTED;
    if (ldq < cols) return RMLK_ERR_SIZE_MISMATCH;
    if (rows > 0x7fffffff || cols > 0x3fffffff) return RMLK_ERR_TOO_LARGE;
    return RMLK_OK;
}

}  // namespace
}  // namespace rmlk

using namespace rmlk;

extern "C" {

int32_t rmlk_hip_quantize_rows(rmlk_stream_t stream, int32_t dtype, int64_t rows, int64_t cols, const void *x,
                               int64_t ldx, void *q, int64_t ldq, float *scale) {
    hipStream_t st = as_stream(stream);
    if (const int32_t bad = row_checks(dtype, rows, cols, q, ldq); bad != RMLK_OK) return bad;
    if (ldx < cols) return RMLK_ERR_SIZE_MISMATCH;
    if (rows == 0 || cols == 0) return RMLK_OK;
    if (!x || !q || !scale) return RMLK_ERR_NULL_POINTER;
    return with_activation(dtype, [&](auto tag) {
        using T = decltype(tag);
        return with_row_shape<false>(static_cast<int32_t>(cols), [&](auto threads, auto units) {
            constexpr int THREADS = decltype(threads)::value, CH = decltype(units)::value;
            quantize_rows_kernel<T, THREADS, CH>
                <<<row_blocks(rows), THREADS, 0, st>>>(static_cast<const T *>(x), ldx, rows, static_cast<int32_t>(cols),
                                                       static_cast<int8_t *>(q), ldq, scale);
            return launch_status();
        });
    });
}

int32_t rmlk_hip_rmsnorm_quantize_rows(rmlk_stream_t stream, int32_t dtype, int64_t rows, int64_t cols,
                                       const void *x, const void *b, const float *gamma, float eps, void *sum_out,
                                       void *q, int64_t ldq, float *scale) {
    hipStream_t st = as_stream(stream);
    if (const int32_t bad = row_checks(dtype, rows, cols, q, ldq); bad != RMLK_OK) return bad;
    if (rows == 0 || cols == 0) return RMLK_OK;
    if (!x || !gamma || !q || !scale || (b == nullptr) != (sum_out == nullptr)) return RMLK_ERR_NULL_POINTER;
    return with_activation(dtype, [&](auto tag) {
        using T = decltype(tag);
        return with_row_shape<true>(static_cast<int32_t>(cols), [&](auto threads, auto units) {
            constexpr int THREADS = decltype(threads)::value, CH = decltype(units)::value;
            norm_quantize_kernel<T, THREADS, CH><<<row_blocks(rows), THREADS, 0, st>>>(
                static_cast<const T *>(x), static_cast<const T *>(b), gamma, eps, rows, static_cast<int32_t>(cols),
                static_cast<T *>(sum_out), static_cast<int8_t *>(q), ldq, scale);
            return launch_status();
        });
    });
}

}  // extern "C"
