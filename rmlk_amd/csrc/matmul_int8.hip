// c[m, n] = (a . wt^T) * a_scale[row] * w_scale[column] (+ residual), a and wt int8 (K-contiguous).
// The integer sums are exact in 32 bits (k < 2^17, |values| <= 128), whatever their order; the
// epilogue scales them in float and rounds once to the output type.
//
// Three kernels. With few rows the weights are what is read, once: a block takes 16 channels and all the
// rows, its wavefronts deal K out among themselves and meet in LDS (int8_few_rows_kernel), or, given
// channels enough, a block streams tiles of channels past rows that it keeps (int8_wide_kernel).
// Beyond, tiles of a and wt go through LDS (int8_tiles_kernel).
#include "paged.hpp"

namespace rmlk {
namespace {

typedef int32_t v4i __attribute__((ext_vector_type(4)));
typedef int32_t v16i __attribute__((ext_vector_type(16)));

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
    int32_t tiles_m, tiles_n;
    int32_t *sums;       // K split over blocks: the integer sums [splits][m][n rounded up to 8]
    int32_t k_per_split;
};

template <typename T>
__device__ __forceinline__ void store_scaled(const Int8Args<T> &g, int row, int col, int32_t sum, float sa, float sw) {
    float v = static_cast<float>(sum) * sa * sw;
    if (g.residual) v += to_float(g.residual[row * g.ldr + col]);
    g.c[row * g.ldc + col] = static_cast<T>(v);
}

// bytes `valid` .. of a 16-byte unit cleared (valid may be negative or beyond 16)
__device__ __forceinline__ u32x4 clear_tail(u32x4 v, int valid) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = valid - 4 * i;
        v[i] = left >= 4 ? v[i] : left <= 0 ? 0u : v[i] & ((1u << (8 * left)) - 1u);
    }
    return v;
}

// 16 channels x 16 * MT rows per block, v_mfma_i32_16x16x64_i8 with the channels as its rows: lane (l % 16,
// l / 16) holds 16 consecutive bytes of channel l % 16, and of row l % 16 of a, straight from memory. A
// wavefront takes every WAVES-th run of 256 bytes of K. Bytes of a behind k are cleared, so what the
// weights hold there does not matter; units behind k are read from the row's start instead. One row, 2048 channels,
// K = 2048 (4.2 MB): 3.7 us, a launch and two trips to memory.
template <typename T, int MT, int WAVES>
__global__ __launch_bounds__(WAVES *kWave) void int8_few_rows_kernel(Int8Args<T> g) {
    __shared__ int32_t parts[WAVES][MT][kWave][4];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int n0 = blockIdx.x * 16;
    const int8_t *w = g.w + static_cast<int64_t>(min(n0 + lane % 16, g.n - 1)) * g.ldw;
    const int8_t *a[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) a[t] = g.a + static_cast<int64_t>(min(t * 16 + lane % 16, g.m - 1)) * g.lda;
    v4i acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = v4i{0, 0, 0, 0};
    for (int k0 = wave * 256; k0 < g.k; k0 += WAVES * 256) {
        u32x4 wv[4], av[4][MT];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = k0 + j * 64 + lane / 16 * 16, from = at < g.k ? at : 0;
            wv[j] = *reinterpret_cast<const u32x4 *>(w + from);
#pragma unroll
            for (int t = 0; t < MT; ++t) av[j][t] = *reinterpret_cast<const u32x4 *>(a[t] + from);
        }
        if (k0 + 256 > g.k) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int t = 0; t < MT; ++t) av[j][t] = clear_tail(av[j][t], g.k - (k0 + j * 64 + lane / 16 * 16));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t)
                acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, wv[j]),
                                                               __builtin_bit_cast(v4i, av[j][t]), acc[t], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) *reinterpret_cast<v4i *>(parts[wave][t][lane]) = acc[t];
    __syncthreads();
    for (int i = tid; i < MT * 256; i += WAVES * kWave) {
        const int row = i / 16, col = i % 16;        // outputs of a row next to each other
        if (row >= g.m || n0 + col >= g.n) continue;
        // C layout: lane (row % 16) + 16 * (channel / 4), register channel % 4
        int32_t sum = 0;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) sum += parts[v][row / 16][row % 16 + col / 4 * 16][col % 4];
        store_scaled(g, row, n0 + col, sum, g.a_scale[row], g.w_scale[n0 + col]);
    }
}

// The same for many channels and more than a few rows: a block keeps its share of a in registers (KU units
// of 64 bytes of K per wavefront) and streams tile after tile of 16 channels past it, the loads of the
// next tile in flight while one is summed up; the sums meet in two LDS buffers in turn, one barrier per
// tile. The block's wavefronts read whole rows of weights together. Bound by the memory: 8 rows, 128256
// channels, K = 2048 take 50 us (5.3 TB/s), the kernel above, which reads a again for every tile, 55 us;
// with one row 45 and 41 us. Measured and dropped: tiles of 32 and 64 channels (51 and 56 us), runs of
// neighbouring tiles per block (55 us), a wavefront per tile with a in LDS (51 us).
constexpr int kWideWaves = 8;
template <typename T, int MT, int KU>
__global__ __launch_bounds__(kWideWaves *kWave) void int8_wide_kernel(Int8Args<T> g) {
    __shared__ int32_t parts[2][kWideWaves][MT][kWave][4];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int tiles = (g.n + 15) / 16;
    // wavefront w takes the units w, w + 8, ..: a tile's loads of one j cover 512 bytes of every row
    u32x4 av[KU][MT];
    int from[KU];
#pragma unroll
    for (int j = 0; j < KU; ++j) {
        const int at = (j * kWideWaves + wave) * 64 + lane / 16 * 16;
        from[j] = at < g.k ? at : 0;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int8_t *a = g.a + static_cast<int64_t>(min(t * 16 + lane % 16, g.m - 1)) * g.lda;
            av[j][t] = clear_tail(*reinterpret_cast<const u32x4 *>(a + from[j]), g.k - at);
        }
    }
    auto fetch = [&](u32x4 (&to)[KU], int tile) {
        const int8_t *w = g.w + static_cast<int64_t>(min(tile * 16 + lane % 16, g.n - 1)) * g.ldw;
#pragma unroll
        for (int j = 0; j < KU; ++j) to[j] = *reinterpret_cast<const u32x4 *>(w + from[j]);
    };
    u32x4 now[KU], next[KU];
    int tile = blockIdx.x;
    fetch(now, tile);
    auto one_tile = [&](u32x4 (&cur)[KU], u32x4 (&ahead)[KU], int buf) {
        const int after = tile + gridDim.x;
        if (after < tiles) fetch(ahead, after);
        v4i acc[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t] = v4i{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < KU; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t)
                acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, cur[j]),
                                                               __builtin_bit_cast(v4i, av[j][t]), acc[t], 0, 0, 0);
#pragma unroll
        for (int t = 0; t < MT; ++t) *reinterpret_cast<v4i *>(parts[buf][wave][t][lane]) = acc[t];
        // (a buffer is written again two tiles later, behind the barrier of the tile between)
        __syncthreads();
        for (int i = tid; i < MT * 256; i += kWideWaves * kWave) {
            const int row = i / 16, col = i % 16, n = tile * 16 + col;
            if (row >= g.m || n >= g.n) continue;
            int32_t sum = 0;
#pragma unroll
            for (int v = 0; v < kWideWaves; ++v) sum += parts[buf][v][row / 16][row % 16 + col / 4 * 16][col % 4];
            store_scaled(g, row, n, sum, g.a_scale[row], g.w_scale[n]);
        }
        tile = after;
        return after < tiles;
    };
    while (true) {
        if (!one_tile(now, next, 0)) break;
        if (!one_tile(next, now, 1)) break;
    }
}

// Block tile (32 TM WM) x (32 TN WN), WM x WN wavefronts of 32 TM x 32 TN, K steps of 128 bytes: whole
// cache lines (with steps of 64 bytes every line crossed from the L2 twice).
// LDS rows are 128 bytes (eight 16-byte units), unpadded - a direct load writes 64 lanes x 16 bytes as one
// contiguous KiB, eight rows - and unit u of row r lives at position u ^ ((r >> 1) & 7) of its row, so
// that the sixteen lanes a 128-bit fragment read serves together cover all banks once. The stage for K
// step s + STAGES - 1 is requested in the first quarter of step s into the one read in step s - 1 (loads
// complete in order: vmcnt tells when the next stage is there); one barrier per K step, in its last
// quarter, behind which the first fragments of the next step are read. LDS reads and direct loads are
// dealt out between the MFMAs. Rows behind m and n are read from the last row and not stored.
// 4096 x 8192 x 8192 in tiles of 256 x 256: 250 us, 2200 TOP/s, where the library's product reaches 2430 and the
// matrix pipes are busy half of the cycles (a higher share lowers the clock). 509 x 8192 x 2048 in 256 tiles of
// 128 x 128: 13.4 - 13.9 us; a K step takes 0.58 us, 32 KB per compute unit from the L2s (14.5 TB/s in all; whether
// that is the L2s' limit has not been shown), launch and first step 3.3 us, the stores 2 us. Measured and dropped there: 2 x 2
// wavefronts (17.8 us at the time of 17.3), 64 x 128 tiles, two blocks per compute unit (20.3 us), two stages (23.2).
// Rows of a and wt that start inside a cache line make every step's 128 bytes cross from the L2 as two lines:
// 635 x 26100 x 3550 takes 124 us with a pitch of 3552, 95 us with one of 3584.
template <typename T, int TM, int TN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(WM *WN *kWave) void int8_tiles_kernel(Int8Args<T> g) {
    constexpr int NW = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, BK = 128, CHUNKS = 4;
    constexpr int kAStage = BM * BK, kStage = (BM + BN) * BK;
    constexpr int A_LOADS = BM / 8 / NW, B_LOADS = BN / 8 / NW, kLoads = A_LOADS + B_LOADS;
    extern __shared__ __align__(16) unsigned char smem[];

    // Tiles in groups of GM x GN that an XCD works on at a time (workgroups go to the XCDs round robin),
    // so that its L2 fetches each row of a group once.
    const int total = g.tiles_m * g.tiles_n, per_xcd = (total + 7) / 8;
    const int t = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;
    if (static_cast<int>(blockIdx.x / 8) >= per_xcd || t >= total) return;
    constexpr int GM = 8;
    const int group = t / (GM * g.tiles_n), first_m = group * GM;
    const int gm = min(GM, g.tiles_m - first_m);
    const int in_group = t - group * GM * g.tiles_n;
    const int tile_m = first_m + in_group % gm, tile_n = in_group / gm;
    const int m0 = tile_m * BM, n0 = tile_n * BN;
    const int k_begin = blockIdx.y * g.k_per_split, k_here = min(g.k - k_begin, g.k_per_split);
    const int n_steps = k_here / BK;

    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int wm = wave / WN, wn = wave % WN;
    const int l32 = lane % 32, half = lane / 32;

    // lane l of piece q (eight rows) fills LDS unit l of the piece: row l / 8, position l % 8
    uint32_t a_voff[A_LOADS], b_voff[B_LOADS];
    auto piece_row = [&](int q) { return q * 8 + lane / 8; };
    auto piece_unit = [&](int q) { return (lane % 8) ^ ((piece_row(q) >> 1) & 7); };
#pragma unroll
    for (int j = 0; j < A_LOADS; ++j) {
        const int q = wave + NW * j;
        a_voff[j] = static_cast<uint32_t>(min(piece_row(q), g.m - 1 - m0) * g.lda + piece_unit(q) * 16);
    }
#pragma unroll
    for (int j = 0; j < B_LOADS; ++j) {
        const int q = wave + NW * j;
        b_voff[j] = static_cast<uint32_t>(min(piece_row(q), g.n - 1 - n0) * g.ldw + piece_unit(q) * 16);
    }
    const int8_t *a_ptr = g.a + static_cast<int64_t>(m0) * g.lda + k_begin;
    const int8_t *b_ptr = g.w + static_cast<int64_t>(n0) * g.ldw + k_begin;
    const uint32_t lds0 =
        __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem)) + wave * 1024u);

    auto direct_load = [&](uint32_t lds_addr, const int8_t *base, uint32_t voff) {
        // (one wait state between a scalar write of M0 and the LDS-bound load that reads it)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                     :
                     : "s"(lds_addr), "v"(voff), "s"(base)
                     : "memory", "m0");
    };
    auto load_op = [&](int buf, auto o_tag) {
        constexpr int o = decltype(o_tag)::value;
        const uint32_t base = lds0 + static_cast<uint32_t>(buf * kStage);
        if constexpr (o < A_LOADS) direct_load(base + o * NW * 1024, a_ptr, a_voff[o]);
        else direct_load(base + kAStage + (o - A_LOADS) * NW * 1024, b_ptr, b_voff[o - A_LOADS]);
    };
    auto load_stage = [&](int buf) {
        static_for<kLoads>([&](auto o_tag) { load_op(buf, o_tag); });
        a_ptr += BK;
        b_ptr += BK;
    };

    // LDS addresses of the fragments of every chunk, moved to the next stage at the end of a step
    uint32_t a_addr[CHUNKS], b_addr[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t off = l32 * BK + ((c * 2 + half) ^ ((l32 >> 1) & 7)) * 16;
        a_addr[c] = wm * TM * 32 * BK + off;
        b_addr[c] = kAStage + wn * TN * 32 * BK + off;
    }
    u32x4 af[2][TM], bf[2][TN];
    constexpr int kFragOps = TM + TN;
    auto frag_op = [&](int c, auto s_tag, auto o_tag) {
        constexpr int s = decltype(s_tag)::value, o = decltype(o_tag)::value;
        if constexpr (o < TN) bf[s][o] = *reinterpret_cast<const u32x4 *>(smem + b_addr[c] + o * 32 * BK);
        else af[s][o - TN] = *reinterpret_cast<const u32x4 *>(smem + a_addr[c] + (o - TN) * 32 * BK);
    };
    int stage = 0;
    auto next_stage = [&]() {
        const uint32_t move = stage + 1 == STAGES ? -(STAGES - 1) * kStage : kStage;
        stage = stage + 1 == STAGES ? 0 : stage + 1;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            a_addr[c] += move;
            b_addr[c] += move;
        }
    };

    v16i acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

    constexpr int NM = TM * TN;
    auto mfma_at = [&](auto s_tag, auto q_tag) {
        constexpr int s = decltype(s_tag)::value, q = decltype(q_tag)::value, i = q / TN, j = q % TN;
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(v4i, af[s][i]),
                                                          __builtin_bit_cast(v4i, bf[s][j]), acc[i][j], 0, 0, 0);
    };
    using Slot0 = std::integral_constant<int, 0>;
    using Slot1 = std::integral_constant<int, 1>;
    constexpr int kBarrierAt = NM / 4;
    auto k_step = [&](int fill, auto load_tag, auto more_tag) {
        constexpr bool LOAD = decltype(load_tag)::value, MORE = decltype(more_tag)::value;
        static_for<CHUNKS - 1>([&](auto c_tag) {
            constexpr int c = decltype(c_tag)::value;
            using Now = std::integral_constant<int, c % 2>;
            using Next = std::integral_constant<int, (c + 1) % 2>;
            static_for<NM>([&](auto q_tag) {
                constexpr int q = decltype(q_tag)::value;
                mfma_at(Now{}, q_tag);
                static_for<kFragOps>([&](auto o_tag) {
                    constexpr int o = decltype(o_tag)::value;
                    if constexpr (o * NM / kFragOps == q) frag_op(c + 1, Next{}, o_tag);
                });
                if constexpr (LOAD && c == 0)
                    static_for<kLoads>([&](auto o_tag) {
                        constexpr int o = decltype(o_tag)::value;
                        if constexpr (o * NM / kLoads == q) load_op(fill, o_tag);
                    });
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        if constexpr (LOAD) {
            a_ptr += BK;
            b_ptr += BK;
        }
        constexpr int room = NM - kBarrierAt - 1;
        static_for<NM>([&](auto q_tag) {
            constexpr int q = decltype(q_tag)::value;
            mfma_at(Slot1{}, q_tag);
            if constexpr (MORE && q == kBarrierAt) {
                // this wavefront has read all of this stage and its part of the next one has landed;
                // then the block meets
                if constexpr (LOAD)
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * kLoads) : "memory");
                else
                    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                asm volatile("s_barrier" ::: "memory");
                next_stage();
            }
            if constexpr (MORE) {
                static_for<kFragOps>([&](auto o_tag) {
                    constexpr int o = decltype(o_tag)::value;
                    constexpr int place = kBarrierAt + 1 + (kFragOps <= room ? o : o * room / kFragOps);
                    if constexpr ((place < NM ? place : NM - 1) == q)
                        frag_op(0, Slot0{}, o_tag);
                });
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    };

    if (n_steps > 0) {
        const int pre = n_steps < STAGES - 1 ? n_steps : STAGES - 1;
        for (int i = 0; i < pre; ++i) load_stage(i);
        if (pre == STAGES - 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * kLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        asm volatile("s_barrier" ::: "memory");
        static_for<kFragOps>([&](auto o_tag) { frag_op(0, Slot0{}, o_tag); });
        int fill = STAGES - 1, step = 0;
        for (; step + STAGES - 1 < n_steps; ++step) {
            k_step(fill, std::true_type{}, std::true_type{});
            fill = fill + 1 == STAGES ? 0 : fill + 1;
        }
        if constexpr (STAGES > 2)
            for (; step + 1 < n_steps; ++step) k_step(0, std::false_type{}, std::true_type{});
        k_step(0, std::false_type{}, std::false_type{});
    }
    if (k_here % BK != 0) {
        // the rest of K, through registers: what lies behind k is zero in a
        __syncthreads();
        const int left = k_here - n_steps * BK;
        const int64_t at = k_begin + static_cast<int64_t>(n_steps) * BK;
        const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < A_LOADS; ++j) {
            const int here = left - piece_unit(wave + NW * j) * 16;     // bytes from this lane's unit on
            u32x4 v = zero;
            if (here > 0)
                v = clear_tail(*reinterpret_cast<const u32x4 *>(g.a + static_cast<int64_t>(m0) * g.lda + at + a_voff[j]), here);
            *reinterpret_cast<u32x4 *>(smem + stage * kStage + (wave + NW * j) * 1024 + lane * 16) = v;
        }
#pragma unroll
        for (int j = 0; j < B_LOADS; ++j) {
            u32x4 v = zero;
            if (left > piece_unit(wave + NW * j) * 16)
                v = *reinterpret_cast<const u32x4 *>(g.w + static_cast<int64_t>(n0) * g.ldw + at + b_voff[j]);
            *reinterpret_cast<u32x4 *>(smem + stage * kStage + kAStage + (wave + NW * j) * 1024 + lane * 16) = v;
        }
        __syncthreads();
        static_for<CHUNKS>([&](auto c_tag) {
            constexpr int c = decltype(c_tag)::value;
            static_for<kFragOps>([&](auto o_tag) { frag_op(c, Slot0{}, o_tag); });
            static_for<NM>([&](auto q_tag) { mfma_at(Slot0{}, q_tag); });
        });
    }

    // The sums go through LDS, 32 rows of a wavefront's tile at a time, so that a lane has eight outputs of a row as
    // 16-byte units of c and the residual (an output per lane, 2 bytes each, took 150 us of a 417 us product of
    // 4096 x 8192 x 8192 with a residual). Units of neighbouring lanes are neighbours: a lane's two units of
    // floats lie half a tile apart (next to each other, every store touched twice the lines: 509 x 8192 x 2048 took
    // 17.3 us, then 16.0); units start at any element (2279 x 3228 x 120 halves 11.5 us, element by element where rows
    // are no whole units 22.3). In the tiles of 128 columns stores are streaming: the kernel leaves no lines to write back
    // when it ends (the same product 13.4 us; a layer of two products and the quantisation of their rows, 512 x 2048 x
    // 8192 floats, 49.7 us against 51.1). The large results of the largest tiles have been written back by then, and
    // are found closer by what reads them next (the same layer at 2048 rows: 113 us streamed, 107 us not), as are the
    // few rows of the smallest ones (32 rows: 30.8 and 30.4 us).
    constexpr bool kStreaming = BN == 128;
    constexpr int kUnit = 16 / sizeof(T);
    __syncthreads();
    constexpr int kCols = 32 * TN, kPad = kCols + 4, kLanesPerRow = kCols / 8, kRowsPerTrip = kWave / kLanesPerRow;
    constexpr int kTrips = 32 / kRowsPerTrip;
    int32_t *mine = reinterpret_cast<int32_t *>(smem) + wave * 32 * kPad;
    constexpr int kApart = sizeof(T) == 4 ? kCols / 2 : 4;       // from a lane's first four columns to its other four
    const int in_tile = lane % kLanesPerRow * (sizeof(T) == 4 ? 4 : 8), col = n0 + wn * kCols + in_tile;
    auto col_of = [&](int e) { return col + e / 4 * kApart + e % 4; };
    float sw[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sw[e] = g.w_scale[min(col_of(e), g.n - 1)];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        T res[kTrips][8];
        const int row0 = m0 + (wm * TM + i) * 32 + lane / kLanesPerRow;
        if (g.residual && !g.sums && col < g.n) {
#pragma unroll
            for (int q = 0; q < kTrips; ++q) {
                const int row = min(row0 + q * kRowsPerTrip, g.m - 1);
#pragma unroll
                for (size_t u = 0; u < sizeof(T) / 2; ++u)
                    if (const int at = col_of(4 * u); at + kUnit <= g.n)
                        reinterpret_cast<u32x4 *>(res[q])[u] = load_unit(g.residual + row * g.ldr + at);
            }
        }
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) mine[(8 * (r / 4) + 4 * half + r % 4) * kPad + j * 32 + l32] = acc[i][j][r];
        // (a wavefront reads back what it wrote itself: its LDS accesses stay in order)
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int q = 0; q < kTrips; ++q) {
            const int row = row0 + q * kRowsPerTrip;
            int32_t sum[8];
            const int32_t *from = mine + (lane / kLanesPerRow + q * kRowsPerTrip) * kPad + in_tile;
            *reinterpret_cast<u32x4 *>(sum) = *reinterpret_cast<const u32x4 *>(from);
            *reinterpret_cast<u32x4 *>(sum + 4) = *reinterpret_cast<const u32x4 *>(from + kApart);
            if (row >= g.m || col >= g.n) continue;
            if (g.sums) {
                int32_t *to = g.sums + (static_cast<int64_t>(blockIdx.y) * g.m + row) * ((g.n + 7) & ~7) + col;
                *reinterpret_cast<u32x4 *>(to) = *reinterpret_cast<u32x4 *>(sum);
                if (col + kApart < g.n) *reinterpret_cast<u32x4 *>(to + kApart) = *reinterpret_cast<u32x4 *>(sum + 4);
                continue;
            }
            const float sa = g.a_scale[row];
            T out[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float v = static_cast<float>(sum[e]) * sa * sw[e];
                if (g.residual) v += to_float(res[q][e]);
                out[e] = static_cast<T>(v);
            }
#pragma unroll
            for (size_t u = 0; u < sizeof(T) / 2; ++u) {
                const int at = col_of(4 * u);
                if (at + kUnit <= g.n) {
                    store_unit<kStreaming>(g.c + row * g.ldc + at, reinterpret_cast<u32x4 *>(out)[u]);
                } else {
#pragma unroll
                    for (int e = 0; e < kUnit; ++e)
                        if (at + e < g.n) store_scaled(g, row, at + e, sum[u * kUnit + e], sa, sw[u * kUnit + e]);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// The splits of K joined: eight outputs of a row per thread.
template <typename T>
__global__ __launch_bounds__(256) void int8_join_kernel(Int8Args<T> g, int32_t splits) {
    const int units = (g.n + 7) / 8;
    const int64_t slab = static_cast<int64_t>(g.m) * units * 8;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < static_cast<int64_t>(g.m) * units;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int row = static_cast<int>(i / units), col = static_cast<int>(i % units) * 8;
        v4i lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
        for (int s = 0; s < splits; ++s) {
            const v4i *from = reinterpret_cast<const v4i *>(g.sums + s * slab + i * 8);
            lo += from[0];
            hi += from[1];
        }
        const float sa = g.a_scale[row];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (col + e < g.n) store_scaled(g, row, col + e, e < 4 ? lo[e] : hi[e - 4], sa, g.w_scale[col + e]);
    }
}

template <typename T, int MT, int WAVES>
int32_t launch_few_rows(hipStream_t st, const Int8Args<T> &g) {
    const int64_t blocks = (static_cast<int64_t>(g.n) + 15) / 16;
    if (blocks * (WAVES * kWave) >= (static_cast<int64_t>(1) << 32)) return RMLK_ERR_TOO_LARGE;    // work items of a launch
    int8_few_rows_kernel<T, MT, WAVES><<<static_cast<uint32_t>(blocks), WAVES * kWave, 0, st>>>(g);
    return launch_status();
}

template <typename T, int MT, int KU>
int32_t launch_wide(hipStream_t st, const Int8Args<T> &g) {
    const int64_t tiles = (static_cast<int64_t>(g.n) + 15) / 16, resident = 2 * kNumCU;
    int8_wide_kernel<T, MT, KU>
        <<<static_cast<uint32_t>(tiles < resident ? tiles : resident), kWideWaves * kWave, 0, st>>>(g);
    return launch_status();
}

template <typename T, int TM, int TN, int WM, int WN, int STAGES>
int32_t launch_tiles(hipStream_t st, Int8Args<T> g, int32_t splits) {
    constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN, stages = STAGES * (BM + BN) * 128;
    constexpr int sums = WM * WN * 32 * (32 * TN + 4) * 4, lds = stages > sums ? stages : sums;
    static_assert(lds <= 160 * 1024, "LDS of a compute unit");
    g.tiles_m = (g.m + BM - 1) / BM;
    g.tiles_n = (g.n + BN - 1) / BN;
    const int64_t tiles = static_cast<int64_t>(g.tiles_m) * g.tiles_n;
    if (tiles > (1 << 21)) return RMLK_ERR_TOO_LARGE;
    auto kern = int8_tiles_kernel<T, TM, TN, WM, WN, STAGES>;
    static DynamicLdsGrant grant;
    if (const int32_t bad = grant.ensure(kern, lds); bad != RMLK_OK) return bad;
    kern<<<dim3(static_cast<uint32_t>((tiles + 7) / 8 * 8), static_cast<uint32_t>(splits)), WM * WN * kWave, lds, st>>>(g);
    return launch_status();
}

// Which kernel a size takes, and the splits of K.
enum Route { kFewRows, kWide, kTile64, kTile64x128, kTile128, kTile256 };
struct Plan {
    Route route;
    int32_t splits, k_per_split;
};
Plan plan_for(int64_t m, int64_t n, int64_t k) {
    auto tiles = [&](int bm, int bn) { return (m + bm - 1) / bm * ((n + bn - 1) / bn); };
    auto rounds = [&](int bm, int bn) { return (tiles(bm, bn) + kNumCU - 1) / kNumCU; };
    Plan p{kTile64, 1, static_cast<int32_t>(k)};
    // Each rule with both sides measured, in us, floats:
    //   few rows, else tiles of 64 x 64:  32 x 2048 x 4096 7.7, 10.0; 32 x 8192 x 2048 8.0, 7.0
    //   256 x 256, else 128 x 128, by the rounds of tiles (one of the large ones takes as long as 3.1 to 3.5 of the
    //   others):  2048 x 8192 x 2048 43, 49; 1792 rows 41, 46; 1536 rows 40, 38; 2304 rows 68, 59
    //   128 x 128, else 64 x 128:  352 x 8192 x 2048 11.4, 12.9; 256 rows 11.0, 10.0
    //   64 x 128, else 64 x 64:  100 x 16384 x 2048 13.2, 14.0; 128 x 8192 x 2048 9.5, 7.6
    if (m > 4 && m <= 32 && n >= 64 * kNumCU && k > 0 && k <= 4096) {
        p.route = kWide;
    } else if (m <= 16 || (m <= 32 && n * k <= (1 << 23))) {
        p.route = kFewRows;
    } else if (m > 128 && 10 * rounds(256, 256) <= 3 * rounds(128, 128)) {
        p.route = kTile256;
    } else if (m > 64 && tiles(128, 128) >= kNumCU * 11 / 16) {
        p.route = kTile128;
    } else if (tiles(64, 128) >= kNumCU) {
        p.route = kTile64x128;
    } else {
        // fewer tiles than compute units: a long K is split, at least 1024 bytes of it per block (the join is a
        // launch of 3 us; 128 x 2048 x 2048 takes 7 us in one piece, 11 us in four)
        int64_t s = kNumCU / tiles(64, 64);
        s = s < k / 1024 ? s : k / 1024;
        s = s < 8 ? s : 8;
        if (s > 1 && k >= 4096) {
            const int64_t per = ((k + s - 1) / s + 127) / 128 * 128;
            p.k_per_split = static_cast<int32_t>(per);
            p.splits = static_cast<int32_t>((k + per - 1) / per);
        }
    }
    return p;
}

template <typename T>
int32_t launch_int8(hipStream_t st, Int8Args<T> g, const Plan &p, void *workspace) {
    g.k_per_split = p.k_per_split;
    g.sums = p.splits > 1 ? static_cast<int32_t *>(workspace) : nullptr;
    switch (p.route) {
        case kFewRows:
            if (g.m > 16) return launch_few_rows<T, 2, 8>(st, g);
            return g.n >= 16 * 2 * kNumCU ? launch_few_rows<T, 1, 8>(st, g) : launch_few_rows<T, 1, 16>(st, g);
        case kWide:
            if (g.m > 16) return g.k <= 2048 ? launch_wide<T, 2, 4>(st, g) : launch_wide<T, 2, 8>(st, g);
            return g.k <= 2048 ? launch_wide<T, 1, 4>(st, g) : launch_wide<T, 1, 8>(st, g);
        case kTile256: return launch_tiles<T, 4, 2, 2, 4, 2>(st, g, 1);
        case kTile128: return launch_tiles<T, 1, 2, 4, 2, 4>(st, g, 1);
        case kTile64x128: return launch_tiles<T, 1, 2, 2, 2, 3>(st, g, 1);
        case kTile64: break;
    }
    if (const int32_t bad = launch_tiles<T, 1, 1, 2, 2, 4>(st, g, p.splits); bad != RMLK_OK || p.splits == 1) return bad;
    int8_join_kernel<T><<<grid_for(static_cast<int64_t>(g.m) * ((g.n + 7) / 8), 256), 256, 0, st>>>(g, p.splits);
    return launch_status();
}

}  // namespace
}  // namespace rmlk

using namespace rmlk;

extern "C" {

size_t rmlk_hip_matmul_int8_workspace_size(int64_t m, int64_t n, int64_t k) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    const Plan p = plan_for(m, n, k);
    return p.splits > 1 ? static_cast<size_t>(p.splits) * m * ((n + 7) / 8 * 8) * sizeof(int32_t) : 0;
}

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
    if (k >= 131072 || m > 0x3fffffff || n > 0x3fffffff || lda >= (1 << 23) || ldw >= (1 << 23)) return RMLK_ERR_TOO_LARGE;
    if (lda % 16 != 0 || ldw % 16 != 0 || !aligned16(a) || !aligned16(wt)) return RMLK_ERR_UNSUPPORTED;
    const size_t need = rmlk_hip_matmul_int8_workspace_size(m, n, k);
    if (need > 0) {
        if (!workspace) return RMLK_ERR_NULL_POINTER;
        if (!aligned16(workspace)) return RMLK_ERR_UNSUPPORTED;
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
        return launch_int8(st, g, plan_for(m, n, k), workspace);
    });
}

}  // extern "C"
