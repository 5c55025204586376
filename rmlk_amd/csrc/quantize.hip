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

constexpr int kThreads = 256;
constexpr float kSmallest = 0x1p-100f;   // rows below it are stored as zeros: 127 / max|y| stays finite

// block-wide sum / max of one value per thread (four wavefronts)
template <typename T, typename Op>
__device__ __forceinline__ T block_reduce(T v, T *lds, Op op) {
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    T r = lds[0];
#pragma unroll
    for (int i = 1; i < kThreads / kWave; ++i) r = op(r, lds[i]);
    __syncthreads();
    return r;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const T *__restrict__ x, int64_t ldx, int32_t cols,
                                                                 int8_t *__restrict__ q, int64_t ldq,
                                                                 float *__restrict__ scale) {
    __shared__ uint32_t lds[kThreads / kWave];
    const int64_t row = blockIdx.x;
    x += row * ldx;
    q += row * ldq;
    // magnitudes compare like their bits, NaN and infinity above everything finite
    uint32_t top = 0;
    for (int j = threadIdx.x; j < cols; j += kThreads) top = max(top, __float_as_uint(to_float(x[j])) & 0x7fffffffu);
    top = block_reduce(wave_max(top), lds, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    const float amax = __uint_as_float(top);
    const bool zero = !(amax >= kSmallest) || top >= 0x7f800000u;
    const float s = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : zero ? 0.f : amax / 127.f;
    const float inv = zero ? 0.f : 1.f / s, half = 0.5f * s;
    const int padded = (cols + 15) & ~15;
    for (int j = threadIdx.x; j < padded; j += kThreads) {
        int n = 0;
        if (j < cols && !zero) {
            const float v = to_float(x[j]);
            const float q0 = rintf(v * inv);
            const float r = fmaf(-q0, s, v);
            n = static_cast<int>(q0);
            const float a = fabsf(r);
            if (a > half || (a == half && (n & 1))) n += r > 0.f ? 1 : -1;
            n = min(127, max(-127, n));
        }
        q[j] = static_cast<int8_t>(n);
    }
    if (threadIdx.x == 0) scale[row] = s;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_quantize_kernel(const T *x, const T *b, const float *__restrict__ gamma,
                                                                 float eps, int32_t cols, T *sum_out,
                                                                 int8_t *__restrict__ q, int64_t ldq,
                                                                 float *__restrict__ scale) {
    __shared__ double lds_d[kThreads / kWave];
    __shared__ uint64_t lds_u[kThreads / kWave];
    const int64_t row = blockIdx.x;
    x += row * cols;
    q += row * ldq;
    if (b) {
        b += row * cols;
        sum_out += row * cols;
    }
    double square = 0.0;
    for (int j = threadIdx.x; j < cols; j += kThreads) {
        float v = to_float(x[j]);
        if (b) {
            const T t = static_cast<T>(v + to_float(b[j]));
            sum_out[j] = t;
            v = to_float(t);
        }
        square += static_cast<double>(v) * static_cast<double>(v);
    }
    square = block_reduce(wave_sum(square), lds_d, [](double a, double c) { return a + c; });
    const double factor = 1.0 / sqrt(square / cols + static_cast<double>(eps));
    const T *y = b ? sum_out : x;     // (every thread reads back what it wrote itself)
    uint64_t top = 0;
    for (int j = threadIdx.x; j < cols; j += kThreads) {
        const double v = to_float(y[j]) * factor * static_cast<double>(gamma[j]);
        const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v)) & 0x7fffffffffffffffull;
        top = u > top ? u : top;
    }
    top = block_reduce(wave_max(top), lds_u, [](uint64_t a, uint64_t c) { return a > c ? a : c; });
    const double amax = __longlong_as_double(static_cast<long long>(top));
    const float s_of = static_cast<float>(amax / 127.0);
    const bool bad = !(s_of <= 3.402823466e38f);   // NaN, infinite, or beyond what a scale can hold
    const bool zero = bad || amax < static_cast<double>(kSmallest);
    const float s = bad ? __uint_as_float(0x7fc00000u) : zero ? 0.f : s_of;
    const double inv = zero ? 0.0 : 1.0 / static_cast<double>(s);
    const int padded = (cols + 15) & ~15;
    for (int j = threadIdx.x; j < padded; j += kThreads) {
        int n = 0;
        if (j < cols && !zero)
            n = static_cast<int>(rint(to_float(y[j]) * factor * static_cast<double>(gamma[j]) * inv));
        q[j] = static_cast<int8_t>(min(127, max(-127, n)));
    }
    if (threadIdx.x == 0) scale[row] = s;
}

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
        quantize_rows_kernel<T><<<static_cast<uint32_t>(rows), kThreads, 0, st>>>(
            static_cast<const T *>(x), ldx, static_cast<int32_t>(cols), static_cast<int8_t *>(q), ldq, scale);
        return launch_status();
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
        norm_quantize_kernel<T><<<static_cast<uint32_t>(rows), kThreads, 0, st>>>(
            static_cast<const T *>(x), static_cast<const T *>(b), gamma, eps, static_cast<int32_t>(cols),
            static_cast<T *>(sum_out), static_cast<int8_t *>(q), ldq, scale);
        return launch_status();
    });
}

}  // extern "C"
