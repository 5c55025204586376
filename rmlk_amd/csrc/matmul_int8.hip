// c[m, n] = (a . wt^T) * a_scale[row] * w_scale[column] (+ residual), a and wt int8 (K-contiguous).
// The integer sums are exact in 32 bits (k < 2^17, |values| <= 128), whatever their order; the
// epilogue scales them in float and rounds once to the output type.
#include "paged.hpp"

namespace rmlk {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct Int8Args {
    const int8_t *a;
    const int8_t *w;
    const float *a_scale;
    const float *w_scale;
    const T *residual;
    T *c;
    int64_t lda, ldw, ldr, ldc;
    int32_t m, n, k;
};

template <typename T>
__device__ __forceinline__ void store_scaled(const Int8Args<T> &g, int row, int col, int32_t sum) {
    float v = static_cast<float>(sum) * g.a_scale[row] * g.w_scale[col];
    if (g.residual) v += to_float(g.residual[row * g.ldr + col]);
    g.c[row * g.ldc + col] = static_cast<T>(v);
}

// bytes k .. of a 16-byte unit cleared
__device__ __forceinline__ u32x4 clear_tail(u32x4 v, int valid) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = valid - 4 * i;
        v[i] = left >= 4 ? v[i] : left <= 0 ? 0u : v[i] & ((1u << (8 * left)) - 1u);
    }
    return v;
}

// A thread per output.
template <typename T>
__global__ __launch_bounds__(kThreads) void int8_outputs_kernel(Int8Args<T> g) {
    const int col = blockIdx.x * 64 + threadIdx.x % 64;
    const int row = blockIdx.y * 4 + threadIdx.x / 64;
    if (row >= g.m || col >= g.n) return;
    const int8_t *a = g.a + row * g.lda, *w = g.w + col * g.ldw;
    int32_t sum = 0;
    for (int k0 = 0; k0 < g.k; k0 += 16) {
        const u32x4 av = clear_tail(*reinterpret_cast<const u32x4 *>(a + k0), g.k - k0);
        const u32x4 wv = *reinterpret_cast<const u32x4 *>(w + k0);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_sdot4(av[i], wv[i], sum, false);
    }
    store_scaled(g, row, col, sum);
}

}  // namespace
}  // namespace rmlk

using namespace rmlk;

extern "C" {

size_t rmlk_hip_matmul_int8_workspace_size(int64_t, int64_t, int64_t) { return 0; }

int32_t rmlk_hip_matmul_int8(rmlk_stream_t stream, int32_t dtype, int64_t m, int64_t n, int64_t k, const void *a,
                             int64_t lda, const float *a_scale, const void *wt, int64_t ldw, const float *w_scale,
                             const void *residual, int64_t ldr, void *workspace, size_t workspace_bytes, void *c,
                             int64_t ldc) {
    hipStream_t st = as_stream(stream);
    if (m < 0 || n < 0 || k < 0 || (residual && ldr < 0)) return RMLK_ERR_INVALID_ARGUMENT;
    if (!is_activation(dtype)) return RMLK_ERR_UNSUPPORTED;
    if (m == 0 || n == 0) return RMLK_OK;
    if ((k > 0 && (!a || !wt)) || !a_scale || !w_scale || !c) return RMLK_ERR_NULL_POINTER;
    if (lda < k || ldw < k || ldc < n || (residual && ldr != 0 && ldr < n)) return RMLK_ERR_SIZE_MISMATCH;
    if (k >= 131072 || m > 0xffff * 4 || n > 0x3fffffff) return RMLK_ERR_TOO_LARGE;
    if (lda % 16 != 0 || ldw % 16 != 0 || !aligned16(a) || !aligned16(wt)) return RMLK_ERR_UNSUPPORTED;
    const size_t need = rmlk_hip_matmul_int8_workspace_size(m, n, k);
    if (need > 0) {
        if (!workspace) return RMLK_ERR_NULL_POINTER;
        if (workspace_bytes < need) return RMLK_ERR_WORKSPACE;
    }
    return with_activation(dtype, [&](auto tag) {
        using T = decltype(tag);
        Int8Args<T> g{};
        g.a = static_cast<const int8_t *>(a);
        g.w = static_cast<const int8_t *>(wt);
        g.a_scale = a_scale;
        g.w_scale = w_scale;
        g.residual = static_cast<const T *>(residual);
        g.c = static_cast<T *>(c);
        g.lda = lda;
        g.ldw = ldw;
        g.ldr = ldr;
        g.ldc = ldc;
        g.m = static_cast<int32_t>(m);
        g.n = static_cast<int32_t>(n);
        g.k = static_cast<int32_t>(k);
        int8_outputs_kernel<T><<<dim3(static_cast<uint32_t>((n + 63) / 64), static_cast<uint32_t>((m + 3) / 4)),
                                 kThreads, 0, st>>>(g);
        return launch_status();
    });
}

}  // extern "C"
