// What the kernels of the 8-bit serving path share: activation types and the paged int8 cache.
#pragma once

#include "common.hpp"

namespace rmlk {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Activation types: float, _Float16, __bf16. to_float is exact; the casts back round to nearest even.
typedef _Float16 half_t;
typedef __bf16 bf16_t;

template <typename T>
__device__ __forceinline__ float to_float(T x) {
    return static_cast<float>(x);
}

// N values of type T (N * sizeof(T) a multiple of 16 bytes) from a 16-byte aligned address, widened.
template <typename T, int N>
__device__ __forceinline__ void load_row(const T *p, float (&out)[N]) {
    static_assert(N * sizeof(T) % 16 == 0, "whole 16-byte units");
    T v[N];
#pragma unroll
    for (size_t i = 0; i < N * sizeof(T) / 16; ++i)
        reinterpret_cast<u32x4 *>(v)[i] = reinterpret_cast<const u32x4 *>(p)[i];
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = to_float(v[i]);
}

// 16 bytes at any element's address: the memory takes such accesses wherever they start.
typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
__device__ __forceinline__ u32x4 load_unit(const T *p) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const u32x4_at4 *>(p);
    else return *reinterpret_cast<const u32x4_at2 *>(p);
}
template <bool STREAMING = false, typename T>
__device__ __forceinline__ void store_unit(T *p, u32x4 v) {
    if constexpr (STREAMING && sizeof(T) == 4) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_at4 *>(p));
    else if constexpr (STREAMING) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_at2 *>(p));
    else if constexpr (sizeof(T) == 4) *reinterpret_cast<u32x4_at4 *>(p) = v;
    else *reinterpret_cast<u32x4_at2 *>(p) = v;
}

inline bool is_activation(int32_t dtype) {
    return dtype == RMLK_FLOAT || dtype == RMLK_FLOAT16 || dtype == RMLK_BFLOAT16;
}

// f(T{}) with the element type of an activation dtype.
template <typename F>
inline int32_t with_activation(int32_t dtype, F &&f) {
    switch (dtype) {
        case RMLK_FLOAT: return f(float{});
        case RMLK_FLOAT16: return f(half_t{});
        case RMLK_BFLOAT16: return f(bf16_t{});
        default: return RMLK_ERR_UNSUPPORTED;
    }
}

inline bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

struct PagedArgs {
    int8_t *k;
    int8_t *v;
    float *k_scale;
    float *v_scale;
    const int32_t *first;
    const int32_t *length;
    const int32_t *table;
    int64_t table_stride;
    int64_t rows;
    int64_t pages;
    int64_t max_new, max_length;
    int32_t seqs;
    int32_t kv_heads;
    int32_t page_shift;      // log2 of the page size
    int32_t *err;
};

// Argument checks of the two structs, and the kernel arguments they give.
inline int32_t paged_args(const rmlk_paged_cache *cache, const rmlk_paged_batch *batch, int32_t *err_flag,
                          PagedArgs *g) {
    if (!cache || !batch) return RMLK_ERR_NULL_POINTER;
    if (cache->pages < 0 || cache->kv_heads < 1 || batch->seqs < 0 || batch->rows < 0 || batch->max_new < 0 ||
        batch->max_length < 0 || batch->table_stride < 0)
        return RMLK_ERR_INVALID_ARGUMENT;
    const int32_t ps = cache->page_size;
    if ((ps != 16 && ps != 32 && ps != 64 && ps != 128) || (cache->head_dim != 64 && cache->head_dim != 128))
        return RMLK_ERR_UNSUPPORTED;
    // what the kernels count with 32 bits
    if (cache->pages > 0x7fffffff || batch->seqs > 0xffff || cache->kv_heads > 0xffff ||
        batch->rows > 0x3fffffff || batch->max_length > 0x3fffffff || batch->max_new > 0x3fffffff)
        return RMLK_ERR_TOO_LARGE;
    g->k = static_cast<int8_t *>(cache->k);
    g->v = static_cast<int8_t *>(cache->v);
    g->k_scale = cache->k_scale;
    g->v_scale = cache->v_scale;
    g->first = batch->first;
    g->length = batch->length;
    g->table = batch->page_table;
    g->table_stride = batch->table_stride;
    g->rows = batch->rows;
    g->pages = cache->pages;
    g->max_new = batch->max_new < batch->rows ? batch->max_new : batch->rows;
    const int64_t room = batch->table_stride > (0x3fffffff / ps) ? 0x3fffffff : batch->table_stride * ps;
    g->max_length = batch->max_length < room ? batch->max_length : room;
    g->seqs = static_cast<int32_t>(batch->seqs);
    g->kv_heads = cache->kv_heads;
    g->page_shift = ps == 16 ? 4 : ps == 32 ? 5 : ps == 64 ? 6 : 7;
    g->err = err_flag;
    return RMLK_OK;
}

// The pointers of a call that has something to do.
inline int32_t paged_pointers(const rmlk_paged_cache *cache, const rmlk_paged_batch *batch) {
    if (!batch->first || !batch->length) return RMLK_ERR_NULL_POINTER;
    if (batch->table_stride > 0 && !batch->page_table) return RMLK_ERR_NULL_POINTER;
    if ((!cache->k || !cache->v || !cache->k_scale || !cache->v_scale) && cache->pages > 0)
        return RMLK_ERR_NULL_POINTER;
    if (cache->pages == 0) return RMLK_ERR_INVALID_ARGUMENT;    // nowhere to read from, nowhere to write to
    if (!aligned16(cache->k) || !aligned16(cache->v)) return RMLK_ERR_UNSUPPORTED;
    return RMLK_OK;
}

// Rows, new tokens and length of a sequence, and whether they keep to the call's bounds.
struct Sequence {
    int32_t row;       // its first row
    int32_t fresh;     // its rows
    int32_t length;    // tokens it holds, these included
};
// (`first` ascends within the rows: locate has said so)
__device__ __forceinline__ bool in_bounds(const PagedArgs &g, const Sequence &q) {
    return q.fresh <= g.max_new && q.length >= 0 && q.length <= g.max_length;
}

// The work of a ragged call, cut into items: sequence s has count(its numbers) of them, numbered one after
// the other, so that the grid (an upper bound of their sum) has its idle blocks at the end only: idle
// blocks among the others leave compute units with less work than their neighbours. Every wavefront
// works the numbering out for itself in one trip over `first` and `length` (a few cache lines).
struct Item {
    int s;            // its sequence, -1: none (the number is behind the last item)
    int index;        // among the sequence's items
    Sequence q;
};
struct NoOrder {
    __device__ __forceinline__ int operator()(int, int item) const { return item; }
};

__device__ __forceinline__ int wave_prefix_sum(int v) {
#pragma unroll
    for (int step = 1; step < kWave; step *= 2) {
        const int from = __shfl_up(v, step, kWave);
        v += static_cast<int>(threadIdx.x % kWave) >= step ? from : 0;
    }
    return v;
}

// Item number order(total, item). False when `first` does not ascend within 0 .. rows; a sequence that leaves
// the call's bounds counts as one item (which reports it).
template <typename C, typename O = NoOrder>
__device__ __forceinline__ bool find_item(const PagedArgs &g, int item, C &&count, Item &found, O &&order = O{}) {
    const int lane = static_cast<int>(threadIdx.x % kWave);
    auto numbers = [&](int i, Sequence &q, bool &good) {
        q.row = g.first[i];
        q.fresh = g.first[i + 1] - q.row;
        q.length = g.length[i];
        good = good && q.row >= 0 && q.fresh >= 0 && q.row + static_cast<int64_t>(q.fresh) <= g.rows;
        return q.fresh == 0 ? 0 : in_bounds(g, q) ? count(q) : 1;
    };
    found.s = -1;
    bool good = true;
    if (g.seqs == 1) {
        const int n = numbers(0, found.q, good);
        if (!good) return false;
        item = order(n, item);
        if (item >= 0 && item < n) {
            found.s = 0;
            found.index = item;
        }
        return true;
    }
    int total = 0;
    if (g.seqs > kWave) {
        for (int base = 0; base < g.seqs; base += kWave) {
            Sequence q;
            int n = 0;
            if (base + lane < g.seqs) n = numbers(base + lane, q, good);
            total += __builtin_amdgcn_readlane(wave_prefix_sum(n), kWave - 1);
        }
        item = order(total, item);
    }
    int before = 0;
    for (int base = 0; base < g.seqs; base += kWave) {
        Sequence q{0, 0, 0};
        int n = 0;
        if (base + lane < g.seqs) n = numbers(base + lane, q, good);
        const int upto = before + wave_prefix_sum(n);
        const int last = __builtin_amdgcn_readlane(upto, kWave - 1);
        if (g.seqs <= kWave) item = order(last, item);
        const uint64_t here = __ballot(item >= upto - n && item < upto);
        if (here) {
            const int at = __ffsll(static_cast<unsigned long long>(here)) - 1;
            found.s = base + at;
            found.index = item - __builtin_amdgcn_readlane(upto - n, at);
            found.q.row = __builtin_amdgcn_readlane(q.row, at);
            found.q.fresh = __builtin_amdgcn_readlane(q.fresh, at);
            found.q.length = __builtin_amdgcn_readlane(q.length, at);
        }
        before = last;
    }
    return __all(good);
}

// first[0 .. seqs] ascends within 0 .. rows.
__device__ __forceinline__ bool starts_ascend(const PagedArgs &g) {
    bool good = true;
    for (int i = static_cast<int>(threadIdx.x % kWave); i < g.seqs; i += kWave) {
        const int32_t lo = g.first[i], hi = g.first[i + 1];
        good = good && lo >= 0 && lo <= hi && hi <= g.rows;
    }
    return __all(good);
}

// The sequence of a row by bisection, for work whose lanes differ in it (of sequences that share a start: the
// last, which is the one that has rows).
__device__ __forceinline__ bool sequence_of_row(const PagedArgs &g, int64_t row, Sequence &q) {
    int lo = 0, hi = g.seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (g.first[mid] <= row) lo = mid;
        else hi = mid;
    }
    q.row = g.first[lo];
    q.fresh = g.first[lo + 1] - q.row;
    q.length = g.length[lo];
    return in_bounds(g, q) && row >= q.row && row < q.row + q.fresh;
}

__device__ __forceinline__ void raise_error(const PagedArgs &g) {
    if (g.err) *g.err = 1;
}

}  // namespace rmlk
