// Quantized matrix-matrix product for gfx950:
//     outs[m, s] = fp16( sum_k fp32(x[m, k]) * fp32(w16[k, s]) )
// where w16 is the fp16 matrix the reference's unpack step builds (two fp16
// roundings per weight in linear mode, one fused multiply-add in exponent mode).
//
// Two kernels.  matmul_kernel_pipe (further down) is the fast one, for any number of
// rows and outputs whose columns fill at least two thirds of whole tiles;
// matmul_kernel takes everything else.  Common to both: one
// workgroup owns a tile of outs; per K step the packed weights of the tile are
// read from HBM once, decoded and dequantised to fp16 ONCE by the workgroup and
// stored to LDS in MFMA operand layout: 16-byte chunks
// of 8 consecutive k for one column, chunk (kc, n) at kc*BN + n, which both the
// writes (lanes along n) and the MFMA operand reads (lanes along n) touch
// without bank conflicts.  The states tile is stored row-major with an XOR
// swizzle of the chunk index so that row-contiguous writes and column-of-rows
// operand reads are both conflict-free.  Accumulation is fp32 in the MFMA
// accumulators.
//
// matmul_kernel walks K in steps of 64 with the global loads of step k+1 issued
// before the MFMA phase of step k (register prefetch) and two barriers per step.
//
// Workgroups are renumbered so that the 8 XCDs (each with its own L2) take
// disjoint column ranges of the weight matrix.
#include "pipe.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace i4 {

constexpr int BK = 64;

// swizzle of the 16-byte chunk index inside a 128-byte row of the states tile
__device__ __forceinline__ int a_swz(int m) { return (m & 7) ^ ((m >> 3) & 1); }

// Raw packed data of one (32-row block, column) cell
template <int BITS, bool SPARSE>
struct Cell {
    uint32_t w[SPARSE ? 2 : BITS];
    uint32_t m;
};

template <int BITS, bool SPARSE>
__device__ __forceinline__ void load_cell(Cell<BITS, SPARSE>& c, const MatmulArgs& a, int blk, int col) {
    constexpr int ROWS = SPARSE ? 2 : BITS;
    const int64_t S = a.S;
    const uint32_t* p = a.matrix + (int64_t)blk * ROWS * S + col;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) c.w[r] = p[r * S];
    c.m = SPARSE ? a.mask[(int64_t)blk * S + col] : 0xFFFFFFFFu;
}

// General cell decode: 32 fp16 weights = 4 chunks of 8, bit-exact with the
// reference decode, any format and either quantisation mode.
template <int BITS, bool SPARSE>
__device__ __forceinline__ void dequant_cell_generic(const Cell<BITS, SPARSE>& c, h16 sc, h16 ze, h16x8 out[4]) {
    uint32_t codes[32];
    if constexpr (SPARSE) {
        uint64_t v = (uint64_t)c.w[0] | ((uint64_t)c.w[1] << 32);
#pragma unroll
        for (int t = 0; t < 32; ++t) {
            const bool k = (c.m >> t) & 1u;
            codes[t] = (uint32_t)v & 0xFu;
            v >>= k ? 4 : 0;
        }
    } else if constexpr (BITS == 3) {
        const uint64_t lo = (uint64_t)c.w[0] | ((uint64_t)c.w[1] << 32);
        const uint64_t hi = (uint64_t)c.w[1] | ((uint64_t)c.w[2] << 32);
#pragma unroll
        for (int t = 0; t < 32; ++t) {
            const int pos = 3 * t;
            codes[t] = pos + 3 <= 64 ? (uint32_t)(lo >> pos) & 7u : (uint32_t)(hi >> (pos - 32)) & 7u;
        }
    } else {
        constexpr int PER = 32 / BITS;
#pragma unroll
        for (int i = 0; i < BITS; ++i) {
            uint32_t v = c.w[i];
#pragma unroll
            for (int j = 0; j < PER; ++j) { codes[i * PER + j] = v & ((1u << BITS) - 1u); v >>= BITS; }
        }
    }
#pragma unroll
    for (int t = 0; t < 32; ++t) {
        h16 w = dequant_code<BITS>(codes[t], sc, ze);
        if (SPARSE && !((c.m >> t) & 1u)) w = (h16)0.0f;
        out[t >> 3][t & 7] = w;
    }
}

template <int BITS, bool SPARSE>
__device__ __forceinline__ void dequant_cell(const Cell<BITS, SPARSE>& c, h16 sc, h16 ze, h16x8 out[4]) {
    if constexpr (BITS == 4 && !SPARSE) {
        if (sc >= (h16)0.0f) {
            const LinearCoef co = {{sc, sc}, {ze, ze}};
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = dequant_chunk<4>(c.w[i], co);
            return;
        }
    }
    dequant_cell_generic<BITS, SPARSE>(c, sc, ze, out);
}

// T threads; thread t owns column t % BN of the weight tile and CPT of its
// (2 * BN / T) 32-row cells per K step.
template <int BITS, bool SPARSE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64, 2) void matmul_kernel(MatmulArgs a) {
    constexpr int WAVES_N = BN / WN, WAVES_M = BM / WM;
    constexpr int T = WAVES_M * WAVES_N * 64;
    constexpr int TM = WM / 32, TN = WN / 32;     // MFMA tiles per wave
    constexpr int A_CHUNKS = BM * 8 / T;          // 16-byte chunks of the states tile per thread
    constexpr int CPT = 2 * BN / T;               // weight cells per thread
    static_assert(BM * 8 % T == 0 && (T == BN || T == 2 * BN), "tile/thread mismatch");
    static_assert(CPT == 1 || CPT == 2, "one or two cells per thread");

    __shared__ __attribute__((aligned(16))) h16 As[BM * BK];
    __shared__ __attribute__((aligned(16))) h16 Bs[BK * BN];

    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int wm0 = (wave / WAVES_N) * WM, wn0 = (wave % WAVES_N) * WN;

    // XCD-aware renumbering: workgroup i runs on XCD i % 8; give each XCD a
    // contiguous range of column tiles and walk the row tiles fastest.
    int bid = blockIdx.x;
    const int total = a.tiles_m * a.tiles_n;
    {
        const int per_xcd = (total + 7) / 8;
        const int xcd = bid % 8, local = bid / 8;
        const int renum = xcd * per_xcd + local;
        if (total % 8 == 0) bid = renum;
    }
    const int tile_m = bid % a.tiles_m, tile_n = bid / a.tiles_m;
    const int m0 = tile_m * BM, s0 = tile_n * BN;
    const int64_t boff = blockIdx.z;
    const h16* x = a.x + boff * a.M * (int64_t)a.K;
    h16* outs = a.outs + boff * a.M * (int64_t)a.S;

    const int bn = t % BN, bhb0 = (t / BN) * CPT;
    const int bcol = min(s0 + bn, a.S - 1);

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    u32x4 areg[A_CHUNKS];
    Cell<BITS, SPARSE> cell[CPT];
    h16 sc, ze;

    auto load_tile = [&](int kt) {
#pragma unroll
        for (int i = 0; i < A_CHUNKS; ++i) {
            const int c = t + T * i, m = c >> 3, kc = c & 7;
            const int row = min(m0 + m, a.M - 1);
            areg[i] = *reinterpret_cast<const u32x4*>(x + (int64_t)row * a.K + kt * BK + kc * 8);
        }
#pragma unroll
        for (int q = 0; q < CPT; ++q) load_cell<BITS, SPARSE>(cell[q], a, kt * 2 + bhb0 + q, bcol);
        const int64_t gofs = (int64_t)(kt / a.group_units) * a.S + bcol;
        sc = a.scales[gofs];
        ze = a.zeros[gofs];
    };

    const int ktiles = a.K / BK;
    load_tile(0);
    for (int kt = 0; kt < ktiles; ++kt) {
        // registers -> LDS
#pragma unroll
        for (int i = 0; i < A_CHUNKS; ++i) {
            const int c = t + T * i, m = c >> 3, kc = c & 7;
            *reinterpret_cast<u32x4*>(&As[m * BK + ((kc ^ a_swz(m)) << 3)]) = areg[i];
        }
#pragma unroll
        for (int q = 0; q < CPT; ++q) {
            h16x8 w[4];
            dequant_cell<BITS, SPARSE>(cell[q], sc, ze, w);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<h16x8*>(&Bs[(((bhb0 + q) * 4 + e) * BN + bn) * 8]) = w[e];
        }
        __syncthreads();
        if (kt + 1 < ktiles) load_tile(kt + 1);

#pragma unroll
        for (int ks = 0; ks < BK / 16; ++ks) {
            const int kc = 2 * ks + (lane >> 5);
            h16x8 af[TM], bf[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int m = wm0 + i * 32 + (lane & 31);
                af[i] = *reinterpret_cast<const h16x8*>(&As[m * BK + ((kc ^ a_swz(m)) << 3)]);
            }
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int n = wn0 + j * 32 + (lane & 31);
                bf[j] = *reinterpret_cast<const h16x8*>(&Bs[(kc * BN + n) * 8]);
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[i], bf[j], acc[i][j], 0, 0, 0);
        }
        __syncthreads();
    }

    // epilogue: accumulator register r of lane l is row 8*(r/4) + 4*(l/32) + r%4,
    // column l%32 of its 32x32 tile
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int col = s0 + wn0 + j * 32 + (lane & 31);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = m0 + wm0 + i * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                if (row < a.M && col < a.S) outs[(int64_t)row * a.S + col] = (h16)acc[i][j][r];
            }
        }
}

template <int BITS, bool SPARSE, int NW, int TM, bool PING, bool SPLIT>
__global__ __launch_bounds__(NW * 128, NW == 2 ? 2 : 1) void matmul_kernel_pipe(MatmulArgs a) {
    constexpr int BM = TM * 32, BN = NW * 64;
    constexpr int A_ROWS = NW * 32;
    // (each stage of the states an array of its own: in one array every fragment read would wait for all loads in flight)
    constexpr int A_HALVES = (BM + A_ROWS - 1) / A_ROWS * A_ROWS * PK;
    __shared__ __attribute__((aligned(16))) h16 A0[A_HALVES], A1[A_HALVES], A2[A_HALVES], A3[A_HALVES], A4[A_HALVES], A5[A_HALVES];
    __shared__ __attribute__((aligned(16))) h16 Bs[P_STAGES * PK * BN];
    __shared__ __attribute__((aligned(16))) uint32_t Lut[SPARSE ? SPARSE_LUT_WORDS : 4];
    // (split-K: the workgroups of a tile are neighbours in the grid, so they run at about the same time;
    // the tiles before `split_from` are whole)
    const int total = a.tiles_m * a.tiles_n;
    int bid = blockIdx.x, split = 0, nsplit = 1, slot = 0;
    if constexpr (SPLIT) {
        const int v = (int)blockIdx.x - a.split_from;
        if (v >= 0) {
            bid = a.split_from + v / a.ksplit;
            split = v % a.ksplit;
            nsplit = a.ksplit;
            slot = (int)blockIdx.z * (total - a.split_from) + v / a.ksplit;       // counter and partial tiles
        }
    }
    int tile_m, tile_n;
    if (total % 8 == 0) {
        // XCD-aware numbering: workgroups are dealt round-robin to the 8 XCDs (each
        // with its own L2), so XCD x takes the contiguous range x * total / 8 ... of tiles
        const int per_xcd = total / 8, l = bid / 8;
        if (a.by_columns) {
            // ... walked one tile row at a time across the XCD's tile columns: the tiles in
            // flight on an XCD then share few rows of states, whose 64 bytes per row and K
            // step outweigh the packed weights' 16 bytes per column (measured: 1-5 % faster
            // than column by column)
            const int cols = per_xcd / a.tiles_m;
            tile_m = l / cols;
            tile_n = (bid % 8) * cols + l % cols;
        } else {
            bid = (bid % 8) * per_xcd + l;
            tile_m = bid % a.tiles_m, tile_n = bid / a.tiles_m;
        }
    } else {
        tile_m = bid % a.tiles_m, tile_n = bid / a.tiles_m;
    }
    const int64_t boff = blockIdx.z;
    h16* const As[A_STAGES] = {A0, A1, A2, A3, A4, A5};
    pipe_tile<BITS, SPARSE, TM, NW, PING, SPLIT>(a, tile_m * BM, tile_n * BN, a.x + boff * a.M * (int64_t)a.K,
                                          a.outs + boff * a.M * (int64_t)a.S, As, Bs, Lut, slot, split, nsplit);
}

template <int BITS, bool SPARSE, int NW, int TM = 8, bool PING = false>
static void launch_pipe(MatmulArgs a, int64_t B, hipStream_t st) {
    a.tiles_m = (a.M + TM * 32 - 1) / (TM * 32);
    a.tiles_n = (a.S + NW * 64 - 1) / (NW * 64);
    const int total = a.tiles_m * a.tiles_n;
    const dim3 grid(a.split_from + (total - a.split_from) * a.ksplit, 1, (unsigned)B), block(NW * 128);
    a.by_columns = a.tiles_n % 8 == 0;
    if (noting("matmul_kernel_pipe<bits=%d,%s,tile=%dx%d,%s> tiles=%d ksplit=%d split_from=%d workgroups=%u batch=%d", BITS,
               SPARSE ? "16:32" : "dense", TM * 32, NW * 64, PING ? "two-phase" : "plain", total, a.ksplit, a.split_from, grid.x, (int)B))
        return;
    if (a.ksplit > 1) hipLaunchKernelGGL((matmul_kernel_pipe<BITS, SPARSE, NW, TM, PING, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((matmul_kernel_pipe<BITS, SPARSE, NW, TM, PING, false>), grid, block, 0, st, a);
}

// The pipelined kernel takes any whole number of 64 columns; the last tile may be partly empty, up to half of the
// columns in all (128-column tiles: an eighth).  Before, such outputs went to the general tiles, which hide
// less of their loads and cannot split K (us, general / here: int4, K=9280, S=1600, 700 rows 135 / 54, S=14400, 1100 rows 422 /
// 351; int2 there 239 / 54 and 699 / 341; 16:32 280 / 73 and 846 / 385; int4, K=9280, S=9344 -- 256 x 128 tiles before --
// 1100 rows 280 / 214).
static bool tile_columns(int64_t S, int width, bool half) {
    return S % 64 == 0 && (S + width - 1) / width * width * 8 <= S * (half ? 12 : 9);
}

constexpr int64_t MM_SPLIT_MAX_TILES = 1024;             // counters: one int per tile in 4 KB
constexpr int64_t MM_SPLIT_MAX_BYTES = 192ll << 20;      // cap of the partial tiles

// ---- plan of the tiles.  Heights of 128 ... 256 rows in steps of 32, all 256 columns wide, one workgroup per CU, each K split
// `ksplit` ways or not, or only the tiles of a last, partly filled round (from `split_from` on): the candidate that a cost model
// finds cheapest, in us,
//     rounds of 256 workgroups, each  steps x step(height) x (1 + fill x share of the CUs^3) + fixed(height)      (*)
//     + (split: (way x ways + hand x share of the CUs) x height / 256)
// the last of several rounds with its share of the CUs raised towards 1 by `last`, full ones times `round`.  (*) is the power limit:
// a GPU filled to the last CU runs its K steps 40 % slower than an almost empty one.  Fitted per format to 870 ... 2050 timed
// launches (K = 1024 ... 28672, S = 1024 ... 28672, 257 ... 4096 rows); on these shapes its pick is 1.0 - 1.2 % off the best
// candidate on average, 9 - 16 % at worst.  Before, a tree of rules chose among 128, 192 and 256 rows and 256 x 128 tiles, of which
// the last are the best candidate on none of 210 shapes: above 512 rows this plan takes 10 % (int4), 15 % (int3), 14 % (int2) and
// 11 % (16:32) less time on average, at most 3 % more on a shape (us: int4, K=16128, S=3072, 1411 rows 217 / 151; K=9216, S=2304, 1151
// rows 98 / 70; int3, K=28096, S=2176, 880 rows 201 / 134; K=S=4096, 777 rows on S=11008 77 / 72).  Preferences on top of the model -- whole
// 256-row tiles, 16:32 split in 256 rows and never in 224 -- were made for single shapes and cost 2 % (90 random products of multiples
// of 256 rows; int4, K=20480, S=5120, 2048 rows 420 / 373) and 4 % (121 of 16:32; K=4096, S=8192, 896 rows 79.5 / 74.9).
struct TileCost { double step[5], fixed[5], fill, way, hand, round, last; };
static const TileCost tile_cost[4] = {                // int4, int3, int2, 16:32
    {{0.373, 0.434, 0.466, 0.521, 0.555}, {4.151, 4.233, 4.77, 4.391, 5.388}, 0.369, 2.82, 19.858, 1.065, 0.292},
    {{0.405, 0.462, 0.493, 0.536, 0.58}, {3.632, 4.086, 3.915, 4.283, 5.317}, 0.406, 2.965, 19.124, 1.027, 0.321},
    {{0.376, 0.423, 0.463, 0.515, 0.544}, {2.878, 3.789, 3.887, 3.45, 5.247}, 0.344, 2.974, 18.171, 1.042, 0.363},
    {{0.59, 0.659, 0.686, 0.759, 0.817}, {5.287, 5.577, 5.793, 5.759, 6.161}, 0.131, 3.381, 18.391, 1.061, 0.347}};
struct TilePlan { int tm; int ksplit; int64_t split_from, tiles; size_t part_bytes; double us; };
// `only`: this height alone (0: any); `scratch`: bytes for partial tiles, splits that need more are no candidates
static TilePlan plan_tiles(int bits, bool sparse, int64_t M, int64_t K, int64_t S, size_t scratch, int only) {
    TilePlan best{0, 1, 0, 0, 0, 1e30};
    const TileCost& c = tile_cost[sparse ? 3 : 4 - bits];
    const int64_t columns = (S + 255) / 256, steps = K / 32, forced = tuning(TUNE_MM_SPLIT), tail_knob = tuning(TUNE_MM_TAIL);
    const int64_t room = (int64_t)std::min<size_t>(scratch, MM_SPLIT_MAX_BYTES);
    for (int tm = 4; tm <= 8; ++tm) {
        if (only != 0 && tm != only) continue;
        const int64_t total = (M + 32 * tm - 1) / (32 * tm) * columns, tile_bytes = 32 * 256 * 4 * (int64_t)tm;
        const double share = tm / 8.0;
        auto one = [&](double n, double fill) { return n * c.step[tm - 4] * (1.0 + c.fill * fill * fill * fill) + c.fixed[tm - 4]; };
        auto take = [&](double us, int64_t ks, int64_t from) {
            if (us < best.us) best = TilePlan{tm, (int)ks, from, total, ks > 1 ? (size_t)((total - from) * ks * tile_bytes) : 0, us};
        };
        for (int64_t ks = 1; ks <= 8; ++ks) {
            if (ks > 1 && (steps / ks < 8 || total > MM_SPLIT_MAX_TILES || total * ks * tile_bytes > room || forced == 1)) break;
            const int64_t wgs = total * ks, rounds = (wgs + 255) / 256;
            const double n = (double)steps / ks, last = (wgs - (rounds - 1) * 256) / 256.0;
            double us = (rounds - 1) * c.round * one(n, 1.0) + one(n, rounds > 1 ? last + (1.0 - last) * c.last : last);
            if (ks > 1) us += (c.way * ks + c.hand * (rounds - 1 + last)) * share;
            take(forced >= 2 && ks == forced ? 0.0 : us, ks, 0);
        }
        // the tiles of the last round alone, over at most half of the GPU (two ways from 64 tiles on, where the second adds the first
        // one's partial tile to its registers and nothing else is read back) in shares of at least 32 steps (K=4096, S=8192, 2304 rows,
        // 32 tiles in the tail: eight ways 197 us, four ways 170)
        const int64_t tail = total % 256;
        if (tm != 8 || total <= 256 || tail == 0 || tail > 128 || tail_knob == 1 || (tail > 96 && K < 3072)) continue;
        const int64_t ks = std::min<int64_t>({std::max<int64_t>(2, 128 / tail), tail_knob >= 2 ? tail_knob : 8, steps / 32});
        if (ks < 2 || tail * ks * tile_bytes > room) continue;
        const double fill = tail * ks / 256.0;
        const double us = total / 256 * c.round * one(steps, 1.0) + one((double)steps / ks, fill + (1.0 - fill) * c.last) + (c.way * ks + c.hand * fill) * share;
        // (preferred within 5 %: the model has few of these to go by)
        take(us / 1.05, ks, total - tail);
    }
    best.us += 2.0;
    return best;
}

// ---- what earlier forms of the tile kernels split along K.  It decides still which workspaces the last chunk of a large batch is taken
// to have (last_chunk_as_others, a line of precision), and nothing else.  Shapes with at most 128 tiles of 256 x 256: 256 x 128 tiles
// (16:32: 256 x 256) with `ksplit` workgroups per tile, by a cost in K steps.
struct SplitPlan { int ksplit; int64_t tiles; int64_t tile_bytes; };
static SplitPlan plan_split(bool sparse, int64_t B, int64_t M, int64_t K, int64_t S) {
    const SplitPlan none{1, 0, 0};
    if (!tile_columns(S, sparse ? 256 : 128, sparse)) return none;
    const int64_t m_pad = (M + 255) / 256 * 256, tiles4 = m_pad / 256 * ((S + 255) / 256) * B;
    if (tiles4 > 128) return none;
    SplitPlan p{1, m_pad / 256 * ((S + (sparse ? 255 : 127)) / (sparse ? 256 : 128)) * B, sparse ? 256 * 256 * 4 : 256 * 128 * 4};
    if (p.tiles > MM_SPLIT_MAX_TILES) return none;
    const int64_t steps = K / 32, forced = tuning(TUNE_MM_SPLIT);
    auto cost = [&](int64_t ks) -> double {
        const int64_t wgs = p.tiles * ks, rounds = (wgs + 255) / 256;
        const double own = (double)(rounds * ((steps + ks - 1) / ks + 20));
        if (!sparse) return own + (ks > 1 ? 6.0 * ks : 0.0);
        const double fill = wgs >= 256 ? 1.0 : wgs / 256.0;
        return own * (1.0 + 0.39 * std::pow(fill, 3.2)) + (ks > 1 ? 5.0 * ks : 0.0);
    };
    int64_t best = 1;
    for (int64_t ks = 2; ks <= 8; ++ks) {
        if (steps / ks < 8 || p.tiles * ks * p.tile_bytes > MM_SPLIT_MAX_BYTES) break;
        if (forced == ks) { best = ks; break; }
        if (forced == 0 && cost(ks) < cost(best)) best = ks;
    }
    if (best < 2) return none;
    p.ksplit = (int)best;
    return p;
}

// and the tiles of a last round of 256 x 256 ones that fills at most half of the GPU
struct TailPlan { int ksplit; int64_t split_from, tiles; };
static TailPlan plan_tail(bool sparse, int64_t B, int64_t M, int64_t K, int64_t S) {
    const TailPlan none{1, 0, 0};
    if (B != 1 || !tile_columns(S, 256, sparse) || tuning(TUNE_MM_TAIL) == 1) return none;
    const int64_t total = (M + 255) / 256 * ((S + 255) / 256), tail = total % 256;
    if (total <= 256 || tail == 0 || tail > 128) return none;
    if (tail > 96 && K < 3072) return none;
    const int64_t cap = tuning(TUNE_MM_TAIL) >= 2 ? tuning(TUNE_MM_TAIL) : 8;
    const int64_t ks = std::min<int64_t>({std::max<int64_t>(2, 128 / tail), cap, K / 32 / 32});
    if (ks < 2 || tail * ks * (256 * 256 * 4) > MM_SPLIT_MAX_BYTES) return none;
    return TailPlan{(int)ks, total - tail, tail};
}

template <int BITS, bool SPARSE, int BM, int BN, int WM, int WN>
static void launch_tile(MatmulArgs a, int64_t B, hipStream_t st) {
    a.tiles_m = (a.M + BM - 1) / BM;
    a.tiles_n = (a.S + BN - 1) / BN;
    const dim3 grid(a.tiles_m * a.tiles_n, 1, (unsigned)B), block((BM / WM) * (BN / WN) * 64);
    if (noting("matmul_kernel<bits=%d,%s,tile=%dx%d> tiles=%u batch=%d", BITS, SPARSE ? "16:32" : "dense", BM, BN, grid.x, (int)B)) return;
    hipLaunchKernelGGL((matmul_kernel<BITS, SPARSE, BM, BN, WM, WN>), grid, block, 0, st, a);
}

// (the kernel addresses with 32-bit byte offsets into buffer resources: 256 rows of states,
// the whole packed matrix and the whole of scales / zeros have to stay below 2 GB each)
static bool pipe_shape(int bits, bool sparse, int64_t K, int64_t S, int64_t group_units) {
    const int64_t w_bytes = K / 32 * (sparse ? 2 : bits) * 4 * S, sz_bytes = (K / 64 + group_units - 1) / group_units * S * 2;
    return K <= (1 << 22) && S <= (1 << 27) && w_bytes < (1ll << 31) && sz_bytes < (1ll << 31);
}
// (a short K on a small dense grid: the pipelined kernel's prologue costs more than its faster steps return: 2048 rows,
// K=S=128 8.7 -> 5.3 us; 512 rows, K=512, S=1024 14.6 -> 10.7; from K = 1024 on there is nothing in it)
static bool takes_tiles(int bits, bool sparse, int64_t M, int64_t K, int64_t S, int64_t group_units) {
    return pipe_shape(bits, sparse, K, S, group_units) && tile_columns(S, 256, true) &&
           (sparse || K >= 1024 || (M + 255) / 256 * ((S + 255) / 256) > 128);
}

// ---- outputs of 128 columns, of which a tile of 256 would leave half empty: tiles of 128 x 128, two workgroups of four waves per CU, in the
// two phases as well.  On many rows the states' reads are the bound, 5.1 TB/s at 65536 rows.  K is split as many ways as fit 256 workgroups, in
// shares of 16 steps and more (int4, us: K=8192, 128 tiles 95 unsplit, two ways 69, three 73, four 75; 80 tiles three ways 38, four
// 44), or 512 where these are filled better (160 tiles, K=4096: one way 44, three 41; 96 tiles, K=16384: two ways 134, five 110) or the
// states are more than the 256 MB of the cache beside memory (110 tiles, K=28672: two ways 217, four 195).  Before, 256 x 128 tiles with
// the states through registers, whose decode spilled (int4, us, so / now: K=8192, 2048 rows 41.4 / 23.7, without room for a split 146 /
// 76, 65536 rows 249 / 211; K=4096, 600 rows 31.5 / 17.0; with 32x32x16 MFMAs and no spill 39.7, 126, 233, 30.4).
static bool takes_narrow_tiles(int bits, bool sparse, int64_t M, int64_t K, int64_t S, int64_t group_units) {
    const int64_t variant = tuning(TUNE_MM_VARIANT);
    return !sparse && M > 128 && pipe_shape(bits, sparse, K, S, group_units) && tile_columns(S, 128, false) &&
           (variant == 5 || (variant == 0 && K > 1024 && !tile_columns(S, 256, true)));
}
struct NarrowPlan { int ksplit; size_t part_bytes; };
static NarrowPlan plan_narrow(int64_t M, int64_t K, int64_t S, size_t scratch) {
    const int64_t tiles = (M + 127) / 128 * ((S + 127) / 128), steps = K / 32, forced = tuning(TUNE_MM_SPLIT), tile_bytes = 128 * 128 * 4;
    const int64_t room = (int64_t)std::min<size_t>(scratch, MM_SPLIT_MAX_BYTES);
    auto ways = [&](int64_t workgroups) { return std::max<int64_t>(1, std::min<int64_t>({8, workgroups / tiles, steps / 16})); };
    int64_t ks = forced >= 1 ? std::min(forced, steps / 8) : ways(256);
    if (forced < 1 && (ways(512) * 10 > ks * 22 || M * K * 2 > 256ll << 20)) ks = ways(512);
    if (tiles > MM_SPLIT_MAX_TILES) ks = 1;
    while (ks > 1 && tiles * ks * tile_bytes > room) --ks;
    return ks > 1 ? NarrowPlan{(int)ks, (size_t)(tiles * ks * tile_bytes)} : NarrowPlan{1, 0};
}

double tiles_us(int bits, bool sparse, int64_t M, int64_t K, int64_t S, int64_t group_units, size_t scratch) {
    return takes_tiles(bits, sparse, M, K, S, group_units) ? plan_tiles(bits, sparse, M, K, S, scratch, 0).us : 1e30;
}

// height of a forced variant's tiles, in 32 rows (0: none)
static int forced_height(int64_t variant) {
    static const int heights[12] = {0, 0, 0, 0, 0, 0, 8, 4, 6, 8, 5, 7};
    return variant >= 0 && variant < 12 ? heights[variant] : 0;
}

template <int BITS, bool SPARSE>
static void launch(MatmulArgs a, int64_t B, hipStream_t st, void* workspace, size_t workspace_bytes) {
    // variant 0 = automatic: the plan of the pipelined kernel's tiles; where that kernel does not take the shape its 128 x 128 tiles
    // or the general ones, 128 x 256, and 128 x 128 for narrow outputs or few rows
    const int variant = (int)tuning(TUNE_MM_VARIANT);
    const WorkspaceParts wsp = workspace_parts(workspace, workspace_bytes);
    // (a single row comes here where its matvec has a group longer than a launch covers: the size query asks nothing for it)
    const size_t scratch = wsp.counters != nullptr && B == 1 && (a.M > 1 || variant != 0) ? wsp.scratch_bytes : 0;
    a.counters = reinterpret_cast<int*>(wsp.counters);
    a.part = reinterpret_cast<float*>(wsp.scratch);
    const bool shape_ok = pipe_shape(BITS, SPARSE, a.K, a.S, a.group_units);
    const bool narrow = B == 1 && takes_narrow_tiles(BITS, SPARSE, a.M, a.K, a.S, a.group_units);
    const int only = forced_height(variant);
    const bool tiles = !narrow && (variant == 0 ? takes_tiles(BITS, SPARSE, a.M, a.K, a.S, a.group_units) : only != 0 && shape_ok && tile_columns(a.S, 256, true));
    if (narrow) {
        a.ksplit = plan_narrow(a.M, a.K, a.S, scratch).ksplit;
        if constexpr (!SPARSE) launch_pipe<BITS, false, 2, 4, true>(a, B, st);
    } else if (tiles) {
        const TilePlan p = plan_tiles(BITS, SPARSE, a.M, a.K, a.S, scratch, only);
        a.ksplit = p.ksplit;
        a.split_from = (int)p.split_from;
        // (variant 9 forces 256 x 256 without the two phases: 9 % slower, 16:32 4 %)
        if (variant == 9) launch_pipe<BITS, SPARSE, 4>(a, B, st);
        else if (p.tm == 4) launch_pipe<BITS, SPARSE, 4, 4, true>(a, B, st);
        else if (p.tm == 5) launch_pipe<BITS, SPARSE, 4, 5, true>(a, B, st);
        else if (p.tm == 6) launch_pipe<BITS, SPARSE, 4, 6, true>(a, B, st);
        else if (p.tm == 7) launch_pipe<BITS, SPARSE, 4, 7, true>(a, B, st);
        else launch_pipe<BITS, SPARSE, 4, 8, true>(a, B, st);
    } else if (variant == 3 || (variant != 1 && a.M > 512 && a.S >= 256 && !(!SPARSE && a.K <= 1024))) {
        launch_tile<BITS, SPARSE, 128, 256, 128, 64>(a, B, st);
    } else {
        launch_tile<BITS, SPARSE, 128, 128, 64, 64>(a, B, st);
    }
}

}  // namespace i4

using namespace i4;

extern "C" int int4mm_matmul(int bits, void* outs, const void* matrix, const void* multiplier,
                             const void* scales, const void* zeros, const void* sparse_mask,
                             const int4mm_shape* shape, void* workspace, size_t workspace_bytes,
                             void* stream) {
    int rc = validate_product(bits, outs, matrix, multiplier, scales, zeros, sparse_mask, shape, false);
    if (rc != INT4MM_OK) return rc;
    int64_t B = shape->batch, M = shape->seq_len;
    const int64_t K = shape->in_size, S = shape->out_size;
    if (B * M * S == 0) return INT4MM_OK;
    // Batches are contiguous ([B, M, K] states, [B, M, S] outputs) and every kernel's rows are independent: B
    // products of M rows are one product of B * M rows -- whole tiles instead of B padded ones (K=5120, S=20480: 32
    // batch elements of 20 rows 970 -> 152 us, 5 of 130 rows 258 -> 153).
    if (B > 1 && B * M <= ((int64_t)1 << 31) - 256) { M *= B; B = 1; }
    if (((M + 127) / 128) * ((S + 127) / 128) > 0x7FFFFFFF / 2) return INT4MM_ERR_SHAPE;
    const int64_t g = shape->group_size < 0 ? ONE_GROUP : shape->group_size;

    hipStream_t st = (hipStream_t)stream;
    // 2 .. 96 rows in all (batches are contiguous, so they flatten; on suitable shapes up to 512): the few-row
    // kernels, which read every packed word once for all rows -- unless a tile-kernel variant is forced
    if (B * M == 1 && !tuning(TUNE_NO_SKINNY) && !tuning(TUNE_MM_VARIANT) &&
        matvec_one_row(bits, (h16*)outs, (const uint32_t*)matrix, (const uint32_t*)sparse_mask, (const h16*)multiplier,
                       (const h16*)scales, (const h16*)zeros, K, S, g, st, workspace, workspace_bytes, &rc))
        return rc;
    if (B * M >= 2 && B * M <= 4 && !sparse_mask && !tuning(TUNE_NO_SKINNY) && !tuning(TUNE_MM_VARIANT) &&
        matvec_rows(bits, (h16*)outs, (const uint32_t*)matrix, (const h16*)multiplier, (const h16*)scales, (const h16*)zeros,
                    B * M, K, S, g, false, st, workspace, workspace_bytes))
        return check_launch("matmul");
    if (B * M >= 2 && B * M <= SK_WIDE_MAX_ROWS && !tuning(TUNE_NO_SKINNY) && !tuning(TUNE_MM_VARIANT) &&
        skinny_rows(bits, (h16*)outs, (const uint32_t*)matrix, (const h16*)multiplier, (const h16*)scales,
                    (const h16*)zeros, B * M, K, S, g, false, st, (const uint32_t*)sparse_mask, workspace, workspace_bytes, FOR_MATMUL))
        return check_launch("matmul");

    MatmulArgs a;
    a.outs = (h16*)outs;
    a.matrix = (const uint32_t*)matrix;
    a.mask = (const uint32_t*)sparse_mask;
    a.x = (const h16*)multiplier;
    a.scales = (const h16*)scales;
    a.zeros = (const h16*)zeros;
    a.M = (int)M;
    a.K = (int)K;
    a.S = (int)S;
    a.group_units = (int)(g / 64 > 0x7FFFFFF ? 0x7FFFFFF : g / 64);
    a.tiles_m = a.tiles_n = 0;
    a.by_columns = 0;
    a.ksplit = 1;
    a.split_from = 0;
    a.part = nullptr;
    a.counters = nullptr;

    if (sparse_mask) launch<4, true>(a, B, st, workspace, workspace_bytes);
    else if (bits == 4) launch<4, false>(a, B, st, workspace, workspace_bytes);
    else if (bits == 3) launch<3, false>(a, B, st, workspace, workspace_bytes);
    else launch<2, false>(a, B, st, workspace, workspace_bytes);
    return check_launch("matmul");
}

bool i4::last_chunk_as_others(bool sparse, int64_t B, int64_t n, int64_t K, int64_t S, int64_t group_units) {
    if (tuning(TUNE_NO_WIDE) >= 2) return true;
    const size_t others = rounded_room(sparse, SK_WIDE_MAX_ROWS, K, S, group_units, true), room = rounded_room(sparse, n, K, S, group_units, true);
    if (others == SIZE_MAX) return false;
    if (room <= others || room == SIZE_MAX) return true;                 // (never admitted: nothing to decide)
    const SplitPlan sp = plan_split(sparse, 1, B, K, S);
    const TailPlan tp = plan_tail(sparse, 1, B, K, S);
    size_t bytes = int4mm_workspace_bytes(S) + 2 * round_to_page(std::max(rounded_room(sparse, SK_WIDE_MAX_ROWS, K, S, 0, false),
                                                                          sp.ksplit > 1 ? (size_t)(sp.tiles * sp.ksplit * sp.tile_bytes) : 0));
    if (sp.ksplit == 1 && tp.ksplit > 1) bytes += 2 * round_to_page((size_t)(tp.tiles * tp.ksplit * (256 * 256 * 4)));
    return room <= bytes - ((bytes / 2) & ~size_t(4095));
}

// Workspace with which int4mm_matmul may split K for this shape: what the matvec needs, plus room for
// the partial tiles in the scratch half.  A smaller workspace is not an error: the product then runs unsplit.
extern "C" size_t int4mm_matmul_workspace_bytes(const int4mm_shape* shape, int sparse) {
    if (shape == nullptr) return 0;
    int64_t B = shape->batch, M = shape->seq_len;
    const int64_t K = shape->in_size, S = shape->out_size;
    size_t need = int4mm_workspace_bytes(S);
    // (below 128 columns two to four rows keep the launches that they have with the matvec's workspace)
    if (B <= 0 || M <= 0 || K < 64 || S < (B * M < 5 ? 128 : 64)) return need;
    if (B > 1 && B * M <= ((int64_t)1 << 31) - 256) { M *= B; B = 1; }           // (as int4mm_matmul does)
    // (a caller who asks with the sizes alone leaves matrix_rows or group_size 0)
    int bits = 0;
    for (const int b : {4, 3, 2})
        if (shape->matrix_rows * 32 == K * b) bits = b;
    const int64_t g = shape->group_size, group_units = g < 0 ? ONE_GROUP / 64 : g / 64;
    auto few = [&](int64_t rows, RowsCall call) { return skinny_workspace_bytes(bits, rows, K, S, sparse != 0, group_units, call); };
    size_t few_rows = B * M <= FEW_ROWS_MAX ? few(B * M, FOR_MATMUL) : 0;
    // (the matvec entry takes many batch elements of one row in chunks through the few-row kernels: as many as the kernel
    // for more rows takes, else even shares, which may be one fewer towards the end; its callers may ask with the flattened
    // shape too)
    if (B * M > FEW_ROWS_MAX && (shape->seq_len == 1 || B * M <= SK_WIDE_MAX_ROWS))
        for (const int64_t n : {std::min<int64_t>(B * M, SK_WIDE_MAX_ROWS), B * M > SK_WIDE_MAX_ROWS ? B * M % SK_WIDE_MAX_ROWS : 0}) {
            if (n < 2) continue;
            const bool as_others = B * M <= SK_WIDE_MAX_ROWS || n == SK_WIDE_MAX_ROWS || last_chunk_as_others(sparse != 0, B * M, n, K, S, group_units);
            if (as_others) few_rows = std::max(few_rows, few(n, FOR_MATVEC));
            for (const int64_t share : {exact_sums_at_once(n, S), exact_sums_at_once(B * M, S)})
                if ((n > FEW_ROWS_MAX || !as_others) && share >= 2)
                    few_rows = std::max({few_rows, few(share, EXACT_SUMS), few(std::max<int64_t>(2, share - 1), EXACT_SUMS)});
        }
    size_t part = few_rows;
    if (shape->seq_len == 1 && B * M > SK_WIDE_MAX_ROWS) {           // (chunks of the matvec entry: last_chunk_as_others)
        const SplitPlan sp = plan_split(sparse != 0, B, M, K, S);
        const TailPlan tp = plan_tail(sparse != 0, B, M, K, S);
        if (sp.ksplit > 1) part = std::max(part, (size_t)(sp.tiles * sp.ksplit * sp.tile_bytes));
        else if (tp.ksplit > 1) part = round_to_page(part) + (size_t)(tp.tiles * tp.ksplit * (256 * 256 * 4));
    }
    // (rows that the few-row kernels leave to the tiles are asked for as well: what a product is split into, and with it the order of its
    // sums, may not hang on what a workspace was made for)
    const int64_t variant = tuning(TUNE_MM_VARIANT);
    auto others_serve = [&](int b) {
        if (variant != 0 || tuning(TUNE_NO_SKINNY) || B != 1 || M > SK_WIDE_MAX_ROWS) return false;
        if (M <= FEW_ROWS_MAX) return M == 1 || few_rows_serve(b, sparse != 0, M, K, S, group_units);
        size_t bytes = 0;
        if (!wide_serves(b, sparse != 0, M, K, S, std::max<int64_t>(1, group_units), &bytes)) return false;
        part = std::max(part, bytes);
        return true;
    };
    for (const int b : {4, 3, 2}) {
        if (B != 1 || (sparse ? b != 4 : bits != 0 && b != bits) || others_serve(b)) continue;
        const int64_t gu = std::max<int64_t>(1, group_units);
        if (takes_narrow_tiles(b, sparse != 0, M, K, S, gu)) part = std::max(part, plan_narrow(M, K, S, SIZE_MAX).part_bytes);
        else if (variant != 0 || takes_tiles(b, sparse != 0, M, K, S, gu)) part = std::max(part, plan_tiles(b, sparse != 0, M, K, S, SIZE_MAX, forced_height(variant)).part_bytes);
    }
    return need + 2 * round_to_page(part);
}
