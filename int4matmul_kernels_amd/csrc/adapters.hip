// Low-rank adapters of many requests beside a shared projection:
//     outs[t, :] = fp16( base[t, :] + scales[a] * (x[t, :] down[a]^T) up[a] ),   a = ids[t / rows_per_id]
// with down [n, r, K] and up [n, r, S] in fp16; a row whose id is outside 0 ... n - 1 has no adapter and keeps its base.
//
// Two launches, or three.  shrink_kernel: h[t, :] = x[t, :] down[a]^T, a share of K per workgroup, fp32 partial sums to the workspace.
// expand_kernel: adds the shares up, scales, and adds h up[a] onto base.  Both take tiles of neighbouring rows and go through the
// DISTINCT adapters of a tile: one or two where rows come as prompts, up to all different where every row is a request's token.  Many rows
// with ids of their own are ordered by adapter first (plan_kernel, experts.hip), so that a tile has one: every tile through all of its
// adapters reads the factors as often as there are tiles.  What an adapter's weights hold reaches no row of another adapter (its
// products are formed for all rows of a tile and selected, not masked by a 0 that an infinity would turn into NaN).
//
// h is split into two halves of 11 bits each, after scaling its row by a power of two to 512 ... 1024, so that nothing overflows
// and 22 bits of it are multiplied: both products are on v_mfma_f32_16x16x32_f16, which are few beside the memory traffic.
//
// What bounds it: prompts, the traffic of base and outs (4096 rows, K=5120, S=20480, rank 16: 377 MB in 83 - 87 us, 4.4 TB/s, of which
// expand_kernel 72; a large copy does 4.9); requests with an adapter each, reading the factors (64 of rank 64: 164 MB in 48 us, expand_kernel
// 40 at 3.3 TB/s); small calls, two launches (one row 8 us; 777 rows of 24 adapters 16, the order 4 of them).  Rows of base and outs go through buffers whose
// lanes lie beyond where a row is not the workgroup's: with conditions around loads and stores instead 4096 rows took 98.
#include "experts.h"

#include <algorithm>
#include <cmath>

namespace i4 {

constexpr int AD_RSRC = 0x00020000;                   // raw buffer, 32-bit data format
constexpr uint32_t AD_BEYOND = 0x80000000u;           // ORed into a lane's offset: beyond the buffer, the load returns 0

struct AdapterArgs {
    h16* outs;
    const h16* base;
    const h16* x;
    const h16* down;
    const h16* up;
    const float* scales;
    const int* ids;
    float* part;                                      // [ksplit][rows][rank]
    int64_t rows;
    int rows_per_id;
    uint32_t id_magic;
    int adapters, rank, K, S;
    int ksplit, units_per_split;                      // units of 64 k
    // the distinct adapters of a tile are dealt to `deal` workgroups (a power of two) by the first row of each; deal_rows: every
    // deal-th bit from bit 0
    int deal;
    uint64_t deal_rows;
    int strips;                                       // expand: of 256 columns, per workgroup
    const int* offsets;                               // sorted: of each adapter's rows, and behind them those without one, in `order`
    const int* order;
};

// (rows < 2^22: check_adapters)
__device__ __forceinline__ int id_of(const AdapterArgs& a, int64_t row) { return magic_div((int)row, a.rows_per_id, a.id_magic); }

// A tile of up to 64 rows: neighbouring ones or, SORTED, up to `height` rows of one adapter.  Lane i holds row i's place among all rows
// and its id, -1 without one.  Rows of a tile are masks of 64 bits.
struct Tile {
    int row;                                          // (lanes without a row: some row of the tile)
    int id;
    int64_t first;                                    // where the tile's partial sums begin
    uint64_t there;                                   // rows that exist
    uint64_t with;                                    // rows that have an adapter
    uint64_t dealt;                                   // rows whose adapters are this workgroup's, where they are the first of theirs
};
template <bool SORTED>
__device__ __forceinline__ Tile tile_of(const AdapterArgs& a, int nth, int height, int lane, int deal) {
    Tile t = {};
    t.dealt = a.deal_rows << deal;
    if constexpr (SORTED) {
        Block b;
        if (find_block(a.offsets, a.adapters + 1, height, nth, lane, b) >= 0) return t;
        t.first = b.first;
        t.row = a.order[b.first + min(lane, b.count - 1)];
        const bool there = lane < b.count;
        t.id = there && b.expert < a.adapters ? b.expert : -1;
        t.there = __builtin_amdgcn_ballot_w64(there);
    } else {
        t.first = (int64_t)nth * height;
        const int64_t row = t.first + lane;
        const bool there = lane < height && row < a.rows;
        t.row = (int)min(row, a.rows - 1);
        const int v = there ? a.ids[id_of(a, row)] : -1;
        t.id = v >= 0 && v < a.adapters ? v : -1;
        t.there = __builtin_amdgcn_ballot_w64(there);
    }
    t.with = __builtin_amdgcn_ballot_w64(t.id >= 0);
    return t;
}
// rows of x, base or outs are addressed from the tile's first row or, sorted, from the first of all: a tile's row as a multiple of the
// row's bytes, and how many rows the buffer has
template <bool SORTED>
__device__ __forceinline__ int64_t buffer_row(const Tile& t) { return SORTED ? 0 : t.first; }
template <bool SORTED>
__device__ __forceinline__ int buffer_rows(const AdapterArgs& a, const Tile& t, int height) {
    return SORTED ? (int)a.rows : (int)min((int64_t)height, a.rows - t.first);
}
template <bool SORTED>
__device__ __forceinline__ uint32_t row_in_buffer(const Tile& t, int row) { return SORTED ? (uint32_t)__shfl(t.row, row) : (uint32_t)row; }
// calls f(adapter, its rows) for each of this workgroup's adapters
template <class F>
__device__ __forceinline__ void each_adapter(const Tile& t, F f) {
    uint64_t left = t.with & t.dealt;
    while (left) {
        const int row = __builtin_ctzll(left), adapter = __builtin_amdgcn_readlane(t.id, row);
        const uint64_t rows = __builtin_amdgcn_ballot_w64(t.id == adapter);
        left &= ~rows;
        if (__builtin_ctzll(rows) == row) f(adapter, rows);
    }
}

// 16 MT rows, 16 NT ranks, a share of K; the four waves share it out by units of 64 k
template <int MT, int NT, bool SORTED>
__global__ __launch_bounds__(256) void shrink_kernel(AdapterArgs a) {
    __shared__ __attribute__((aligned(16))) float red[4 * 16 * MT * 16 * NT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, q = lane >> 4;
    const int deal = blockIdx.z % a.deal, rank0 = blockIdx.z / a.deal * (16 * NT);
    const int units = a.K / 64, u0 = blockIdx.x * a.units_per_split, u1 = min(u0 + a.units_per_split, units);
    const uint32_t pitch = 2u * (uint32_t)a.K;
    const Tile tile = tile_of<SORTED>(a, blockIdx.y, 16 * MT, lane, deal);
    if (tile.with == 0) return;
    const int ranks_here = min(16 * NT, a.rank - rank0);
    const __amdgpu_buffer_rsrc_t x_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<h16*>(a.x) + buffer_row<SORTED>(tile) * a.K, 0, (int)(buffer_rows<SORTED>(a, tile, 16 * MT) * pitch), AD_RSRC);
    // lane group q takes k = 16 q ... 16 q + 15 of a unit in two steps: 128 bytes of a row per pair of steps
    const uint32_t at = (uint32_t)n * pitch + 32u * q;
    uint32_t x_at[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) x_at[m] = row_in_buffer<SORTED>(tile, 16 * m + n) * pitch + 32u * q;

    each_adapter(tile, [&](int cur, uint64_t rows) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t w_rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<h16*>(a.down) + ((int64_t)cur * a.rank + rank0) * a.K, 0, (int)(ranks_here * pitch), AD_RSRC);
        uint32_t xo[MT];                              // (only this adapter's rows are read)
#pragma unroll
        for (int m = 0; m < MT; ++m) xo[m] = x_at[m] | ((rows >> (16 * m + n)) & 1 ? 0u : AD_BEYOND);
        f32x4 acc[MT][NT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        // (two units a trip, the second one perhaps beyond the share: it reads as 0)
        for (int u = u0 + wave; u < u1; u += 8) {
            u32x4 xv[4][MT], wv[4][NT];
            const uint32_t beyond = u + 4 < u1 ? 0u : AD_BEYOND;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const uint32_t off = 128u * (u + (s >> 1) * 4) + 16u * (s & 1), past = s >> 1 ? beyond : 0u;
#pragma unroll
                for (int m = 0; m < MT; ++m) xv[s][m] = __builtin_amdgcn_raw_buffer_load_b128(x_rsrc, xo[m] | past, off, 0);
#pragma unroll
                for (int t = 0; t < NT; ++t) wv[s][t] = __builtin_amdgcn_raw_buffer_load_b128(w_rsrc, (at + 16u * t * pitch) | past, off, 0);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<h16x8>(xv[s][m]), bitcast<h16x8>(wv[s][t]), acc[m][t], 0, 0, 0);
        }
        // register r of tile (m, t) is row 16 m + 4 q + r, rank 16 t + n
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) red[((wave * 16 * MT) + 16 * m + 4 * q + r) * (16 * NT) + 16 * t + n] = acc[m][t][r];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MT * NT; ++i) {
            const int e = i * 256 + threadIdx.x, row = e / (16 * NT), rank = e % (16 * NT);
            const float sum = (red[e] + red[e + 256 * MT * NT]) + (red[e + 512 * MT * NT] + red[e + 768 * MT * NT]);
            if (((rows >> row) & 1) && rank < ranks_here)
                a.part[((int64_t)blockIdx.x * a.rows + tile.first + row) * a.rank + rank0 + rank] = sum;
        }
        __syncthreads();
    });
}

template <int CTRL>
__device__ __forceinline__ float dpp_fmax(float v) { return fmaxf(v, dpp_f32<CTRL>(v)); }

// 16 MT rows, `strips` times 256 columns: four waves of 64 columns, tile j of a wave takes columns 4 n + j.  LONG: more than 64
// ranks.  The first adapter's first PRE times 32 ranks and base are asked for a strip ahead.
template <int MT, bool LONG, int PRE, bool SORTED>
__global__ __launch_bounds__(256) void expand_kernel(AdapterArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, q = lane >> 4;
    const int deal = blockIdx.z;
    const int chunks = (a.rank + 31) / 32, pitch = chunks * 32 + 8;        // halves between the rows of h in LDS
    h16* const high = reinterpret_cast<h16*>(lds);
    h16* const low = high + 16 * MT * pitch;
    float* const unscale = reinterpret_cast<float*>(low + 16 * MT * pitch);
    const Tile tile = tile_of<SORTED>(a, blockIdx.y, 16 * MT, lane, deal);

    // ---- the rows that are written here: those of this workgroup's adapters and, in the first one, those without an adapter
    uint64_t mine = 0;
    int lead = -1;                                    // the first of these adapters
    each_adapter(tile, [&](int cur, uint64_t rows) __attribute__((always_inline)) {
        if (lead < 0) lead = cur;
        mine |= rows;
    });
    const uint64_t idle = deal == 0 && a.outs != a.base ? tile.there & ~tile.with : 0;
    if ((mine | idle) == 0) return;

    const int first_column = (blockIdx.x * a.strips * 4 + wave) * 64;
    const int end_column = min(a.S, (int)(blockIdx.x + 1) * a.strips * 256);
    const uint32_t row_bytes = 2u * (uint32_t)a.S;
    // rows of base and outs through buffers of the tile's rows: a row that is not to be read or written lies beyond
    const int tile_bytes = (int)((uint32_t)buffer_rows<SORTED>(a, tile, 16 * MT) * row_bytes);
    const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<h16*>(a.base) + buffer_row<SORTED>(tile) * a.S, 0, tile_bytes, AD_RSRC);
    const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(a.outs + buffer_row<SORTED>(tile) * a.S, 0, tile_bytes, AD_RSRC);
    uint32_t row_at[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) row_at[m][r] = row_in_buffer<SORTED>(tile, 16 * m + 4 * q + r) * row_bytes + 8u * n;
    auto offset = [&](int m, int r, uint64_t rows) __attribute__((always_inline)) {
        const int row = 16 * m + 4 * q + r;
        return row_at[m][r] | ((rows >> row) & 1 ? 0u : AD_BEYOND);
    };
    // ranks 32 ch + 8 q ... + 7 of columns 4 n ... 4 n + 3 of the strip at column c
    auto load_up = [&](u32x2 (&w)[8], int adapter, int c, int ch) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<h16*>(a.up) + (int64_t)adapter * a.rank * a.S + c, 0, (int)((a.rank - 1) * row_bytes + 128u), AD_RSRC);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __builtin_amdgcn_raw_buffer_load_b64(rsrc, (uint32_t)(32 * ch + 8 * q + i) * row_bytes + 8u * n, 0, 0);
    };
    u32x2 ahead[PRE][8], base[MT][4];
    uint32_t base_off[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) base_off[m][r] = offset(m, r, mine | idle);
    // (beyond the last strip: the last column's again, not used)
    auto ask_up = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int ch = 0; ch < PRE; ++ch) load_up(ahead[ch], max(lead, 0), min(c, a.S - 64), ch);       // (ranks that there are not read as 0)
    };
    auto ask_base = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) base[m][r] = __builtin_amdgcn_raw_buffer_load_b64(from, base_off[m][r], 2 * min(c, a.S - 64), 0);
    };
    ask_up(first_column);
    ask_base(first_column);

    // ---- h of these rows, 16, 32 or 64 lanes to a row
    {
        const int lanes = LONG || a.rank > 32 ? 64 : a.rank > 16 ? 32 : 16, per_wave = 64 / lanes;
        const int sub = lane & (lanes - 1);
#pragma unroll 1
        for (int row = wave * per_wave + lane / lanes; row < 16 * MT; row += 4 * per_wave) {
            const bool there = (mine >> row) & 1;
            if (__builtin_amdgcn_ballot_w64(there) == 0) continue;
            const int64_t at_row = tile.first + row;
            const int of = __shfl(tile.id, row);
            const float scale = there ? a.scales[of] : 0.f;
            float h[LONG ? 8 : 1], most = 0.f;
#pragma unroll
            for (int i = 0; i < (LONG ? 8 : 1); ++i) {
                const int rank = 64 * i + sub;
                float sum = 0.f;
                if (there && rank < a.rank) {
                    const float* const part = a.part + at_row * a.rank + rank;
                    const int64_t next = a.rows * a.rank;
                    int ks = 0;
                    for (; ks + 4 <= a.ksplit; ks += 4)
                        sum += (part[ks * next] + part[(ks + 1) * next]) + (part[(ks + 2) * next] + part[(ks + 3) * next]);
                    for (; ks < a.ksplit; ++ks) sum += part[ks * next];
                }
                h[i] = sum * scale;
                most = fmaxf(most, fabsf(h[i]));
            }
            most = dpp_fmax<0x140>(dpp_fmax<0x141>(dpp_fmax<0x4E>(dpp_fmax<0xB1>(most))));
            if (lanes >= 32) most = fmaxf(most, __shfl_xor(most, 16));
            if (lanes == 64) most = fmaxf(most, __shfl_xor(most, 32));
            // most = f 2^e, f in [0.5, 1): times 2^(10 - e)
            int e = 10;
            if (most > 0.f && most < INFINITY) e = max(__builtin_amdgcn_frexp_expf(most), -100);
            const float by = __builtin_ldexpf(1.f, 10 - e);
#pragma unroll
            for (int i = 0; i < (LONG ? 8 : 1); ++i) {
                const float v = h[i] * by;
                const h16 hi = (h16)v;
                // (an infinity or NaN is in the high part alone)
                const h16 lo = fabsf(v) < 65504.f ? (h16)(v - (float)hi) : (h16)0.f;
                for (int rank = 64 * i + sub; rank < min(chunks * 32, 64 * i + 64); rank += lanes) {
                    high[row * pitch + rank] = rank < 64 * i + lanes ? hi : (h16)0.f;
                    low[row * pitch + rank] = rank < 64 * i + lanes ? lo : (h16)0.f;
                }
            }
            if (sub == 0) unscale[row] = __builtin_ldexpf(1.f, e - 10);
        }
    }
    __syncthreads();

#pragma unroll 1
    for (int c = first_column; c < end_column; c += 256) {
        uint64_t left = tile.with & tile.dealt;
        while (left) {
            const int row = __builtin_ctzll(left), cur = __builtin_amdgcn_readlane(tile.id, row);
            const uint64_t rows = __builtin_amdgcn_ballot_w64(tile.id == cur);
            left &= ~rows;
            if (__builtin_ctzll(rows) != row) continue;
            f32x4 acc[MT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            auto multiply = [&](const u32x2 (&w)[8], int ch) __attribute__((always_inline)) {
                // turned so that a register holds two ranks of a column
                h16x8 b[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
                    u32x4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_perm(w[2 * i + 1][j >> 1], w[2 * i][j >> 1], sel);
                    b[j] = bitcast<h16x8>(v);
                }
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const int at = (16 * m + n) * pitch + 32 * ch + 8 * q;
                    const h16x8 hi = *reinterpret_cast<const h16x8*>(high + at), lo = *reinterpret_cast<const h16x8*>(low + at);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, b[j], acc[m][j], 0, 0, 0);
                        acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, b[j], acc[m][j], 0, 0, 0);
                    }
                }
            };
            int ch = 0;
            if (cur == lead) {
#pragma unroll
                for (int p = 0; p < PRE; ++p)
                    if (p < chunks) multiply(ahead[p], p);
                ch = PRE;
                if (c + 256 < end_column) ask_up(c + 256);
            }
            for (; ch < chunks; ++ch) {
                u32x2 w[8];
                load_up(w, cur, c, ch);
                multiply(w, ch);
            }
            // register r of tile (m, j) is row 16 m + 4 q + r: this adapter's are done
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const f32x4 by = *reinterpret_cast<const f32x4*>(unscale + 16 * m + 4 * q);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const h16x4 v = bitcast<h16x4>(base[m][r]);
                    h16x4 o;
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[j] = (h16)((float)v[j] + acc[m][j][r] * by[r]);
                    __builtin_amdgcn_raw_buffer_store_b64(bitcast<u32x2>(o), to, offset(m, r, rows), 2 * c, 0);
                }
            }
        }
        if (idle) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r) __builtin_amdgcn_raw_buffer_store_b64(base[m][r], to, offset(m, r, idle), 2 * c, 0);
        }
        if (c + 256 < end_column) ask_base(c + 256);
    }
}

// Rows ordered by adapter or not: ids per row, adapters, rank, K, S: 256, 16, 16, 5120, 5120 13.2 / 20.8; 256, 128, 16, 5120, 5120 23.1 / 23.8; 777,
// 24, 20, 2048, 1408 15.5 / 24.2; 777, 4, 16, 2048, 1408 13.5 / 12.6; 1500, 128, 16, 5120, 5120 26 / 125; 4096, 2, 16, 5120, 5120 43 / 45; 4096, 100,
// 64, 4096, 4096 84 / 473; where it does not gain, 128, 128, 16, 4096, 4096 16.7 / 13.0; one row 11.9 / 8.4.
// Only rows with an id each, up to 256 adapters and 65536 rows (the order reads all ids for every adapter) whose states and outputs are addressed with 31
// bits: beyond that a tile goes through all of its adapters, however many those are.
constexpr double SORTED_GAIN = 2.0;                   // tiles times their adapters over tiles of one adapter
struct AdapterPlan { int mt, nt, ksplit, units_per_split, deal_shrink, deal_expand, strips; bool sorted; int64_t tiles; };

// Measured, us a call, one side / the other: the adapters of a tile dealt to several workgroups or not, 777 rows of 24 adapters 23 / 226;
// until there are 256 / 512 / 1024 / 2048 / 4096 workgroups, the same rows 27 / 23 / 24 / 25 / 27 (not ordered), 64 requests with an adapter of rank 64
// each 56 / 48 / 52 / 48 / 47; shares of K of 8 units or of a thirtieth of it, the 777 rows 26 / 34; tiles of 16 or 32 rows for 4096 rows
// of prompts 97 / 86; workgroups that walk along the columns (1024 in all) or one for every 256 columns: the 64 requests 49 / 53, 4096
// rows of prompts 86 / 108.
static AdapterPlan plan_adapters(const int4mm_adapter_shape& sh) {
    AdapterPlan p;
    const int64_t T = sh.rows, units = sh.in_size / 64, n = sh.adapters;
    p.nt = sh.rank <= 16 ? 1 : sh.rank <= 32 ? 2 : 4;
    const int64_t rank_parts = (sh.rank + 16 * p.nt - 1) / (16 * p.nt);
    p.mt = T <= 1024 ? 1 : 2;
    p.tiles = (T + 16 * p.mt - 1) / (16 * p.mt);
    // sorted: what the tiles go through, the different adapters of 16 mt rows that ask for one each, against tiles of one adapter
    p.sorted = false;
    if (sh.rows_per_id == 1 && n <= 256 && T <= 65536 && T * std::max(sh.in_size, sh.out_size) * 2 < ((int64_t)1 << 31)) {
        const int64_t height = std::min<int64_t>(T, 16 * p.mt);
        const double different = n * (1.0 - std::pow(1.0 - 1.0 / n, (double)height));
        const int mt = T >= 24 * n ? 2 : 1;
        const int64_t tiles = std::min(T, n + 1 + T / (16 * mt));
        if (p.tiles * different > SORTED_GAIN * tiles) p.sorted = true, p.mt = mt, p.tiles = tiles;
    }
    // the most distinct adapters that a tile can hold, and the workgroups that its adapters are dealt to: until there are 512
    const int64_t distinct = p.sorted ? 1 : std::min<int64_t>({n, T, (16 * p.mt - 1) / std::min(sh.rows_per_id, T) + 2, 16 * p.mt});
    auto deal = [&](int64_t workgroups) {
        int d = 1;
        while (d < distinct && d < 16 && d * workgroups < 512) d *= 2;
        return d;
    };
    p.deal_shrink = deal(p.tiles * rank_parts);
    // (a share is at least the two units that a wave takes at once, and there are at most 16 to add up, fewer where the tiles are many:
    // every workgroup of expand_kernel adds them up.  Up to 1024 / 8192 workgroups, prompts of 256 rows, 16 adapters of rank 64, 8192 x 8192,
    // 74 / 94; 4096 rows of one of rank 128, 4096 x 11008, 134 / 152)
    const int64_t workgroups = p.tiles * rank_parts * p.deal_shrink;
    p.units_per_split = (int)std::max<int64_t>({8, (units + 15) / 16, (units * workgroups + 1023) / 1024});
    p.ksplit = (int)((units + p.units_per_split - 1) / p.units_per_split);
    const int64_t strips = (sh.out_size + 255) / 256;
    p.deal_expand = deal(p.tiles * strips);
    p.strips = (int)std::max<int64_t>(1, p.tiles * p.deal_expand * strips / 1024);
    return p;
}
struct AdapterParts { size_t offsets, order, part, total; };
static AdapterParts adapter_parts(const int4mm_adapter_shape& sh, const AdapterPlan& p) {
    auto round = [](size_t n) { return (n + 255) & ~size_t(255); };
    AdapterParts a;
    a.offsets = 0;
    a.order = p.sorted ? round(4 * (size_t)(sh.adapters + 2)) : 0;
    a.part = a.order + (p.sorted ? round(4 * (size_t)sh.rows) : 0);
    a.total = a.part + (size_t)p.ksplit * sh.rows * sh.rank * 4;
    return a;
}

static int check_adapters(const int4mm_adapter_shape* sh) {
    if (sh == nullptr) return INT4MM_ERR_NULL;
    const int64_t limit = (int64_t)1 << 31;
    if (sh->rows < 0 || sh->rows_per_id < 1 || sh->adapters < 1 || sh->rank < 1 || sh->rank > 512 || sh->in_size <= 0 ||
        sh->out_size <= 0 || sh->in_size % 64 != 0 || sh->out_size % 64 != 0)
        return INT4MM_ERR_SHAPE;
    if (sh->adapters >= limit || sh->rows > 16 * 65535 || sh->in_size * 2 * 64 >= limit || (sh->rank + 31) / 32 * 32 * sh->out_size * 2 >= limit)
        return INT4MM_ERR_SHAPE;
    return INT4MM_OK;
}

}  // namespace i4

using namespace i4;

extern "C" {

size_t int4mm_adapters_workspace_bytes(const int4mm_adapter_shape* sh) {
    if (check_adapters(sh) != INT4MM_OK || sh->rows == 0) return 0;
    return adapter_parts(*sh, plan_adapters(*sh)).total;
}

int int4mm_low_rank_add(void* outs, const void* base, const void* x, const void* down, const void* up, const void* scales,
                        const void* ids, const int4mm_adapter_shape* sh, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_adapters(sh)) return rc;
    if (sh->rows == 0) return INT4MM_OK;
    if (!outs || !base || !x || !down || !up || !scales || !ids) return INT4MM_ERR_NULL;
    const void* aligned[] = {outs, base, x, down, up, workspace};
    for (const void* ptr : aligned)
        if (reinterpret_cast<uintptr_t>(ptr) & 15) return INT4MM_ERR_ALIGN;
    if ((reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(ids)) & 3) return INT4MM_ERR_ALIGN;
    const AdapterPlan p = plan_adapters(*sh);
    const AdapterParts parts = adapter_parts(*sh, p);
    if (workspace == nullptr || workspace_bytes < parts.total) return INT4MM_ERR_WORKSPACE;
    AdapterArgs a;
    a.outs = static_cast<h16*>(outs);
    a.base = static_cast<const h16*>(base);
    a.x = static_cast<const h16*>(x);
    a.down = static_cast<const h16*>(down);
    a.up = static_cast<const h16*>(up);
    a.scales = static_cast<const float*>(scales);
    a.ids = static_cast<const int*>(ids);
    char* const ws = static_cast<char*>(workspace);
    int* const offsets = reinterpret_cast<int*>(ws + parts.offsets);
    int* const order = reinterpret_cast<int*>(ws + parts.order);
    a.offsets = offsets;
    a.order = order;
    a.part = reinterpret_cast<float*>(ws + parts.part);
    a.rows = sh->rows;
    a.rows_per_id = (int)std::min(sh->rows_per_id, sh->rows);
    a.id_magic = div_magic((uint32_t)a.rows_per_id);
    a.adapters = (int)sh->adapters;
    a.rank = (int)sh->rank;
    a.K = (int)sh->in_size;
    a.S = (int)sh->out_size;
    a.ksplit = p.ksplit;
    a.units_per_split = p.units_per_split;
    hipStream_t st = (hipStream_t)stream;
    if (p.sorted) {
        launch_rows_by_id(a.ids, offsets, order, (int)sh->rows, (int)sh->adapters + 1, st);
        if (const int rc = check_launch("low_rank_add")) return rc;
    }
    {
        a.deal = p.deal_shrink;
        a.deal_rows = ~0ull / ((1ull << a.deal) - 1);
        const dim3 grid(p.ksplit, (unsigned)p.tiles, (unsigned)(p.deal_shrink * ((sh->rank + 16 * p.nt - 1) / (16 * p.nt))));
#define SHRINK(MT, NT)                                                                                \
    if (p.sorted) hipLaunchKernelGGL((shrink_kernel<MT, NT, true>), grid, dim3(256), 0, st, a);       \
    else hipLaunchKernelGGL((shrink_kernel<MT, NT, false>), grid, dim3(256), 0, st, a)
        if (p.mt == 1) {
            if (p.nt == 1) { SHRINK(1, 1); } else if (p.nt == 2) { SHRINK(1, 2); } else { SHRINK(1, 4); }
        } else {
            if (p.nt == 1) { SHRINK(2, 1); } else if (p.nt == 2) { SHRINK(2, 2); } else { SHRINK(2, 4); }
        }
#undef SHRINK
        if (const int rc = check_launch("low_rank_add")) return rc;
    }
    a.deal = p.deal_expand;
    a.deal_rows = ~0ull / ((1ull << a.deal) - 1);
    a.strips = p.strips;
    const int height = 16 * p.mt;
    const dim3 grid((unsigned)((sh->out_size + 256 * p.strips - 1) / (256 * p.strips)), (unsigned)p.tiles, (unsigned)p.deal_expand);
    const size_t lds = (size_t)height * (((sh->rank + 31) / 32 * 32 + 8) * 4 + 4);
    auto expand = [&](void (*kernel)(AdapterArgs)) {
        // more than 64 KB of dynamic LDS (32 rows of more than 480 ranks) has to be requested
        if (lds > 64 * 1024) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        hipLaunchKernelGGL(kernel, grid, dim3(256), lds, st, a);
    };
#define EXPAND_AS(MT, SORTED)                                               \
    if (sh->rank <= 32) expand(expand_kernel<MT, false, 1, SORTED>);        \
    else if (sh->rank <= 64) expand(expand_kernel<MT, false, 2, SORTED>);   \
    else expand(expand_kernel<MT, true, 2, SORTED>)
#define EXPAND(MT) if (p.sorted) { EXPAND_AS(MT, true); } else { EXPAND_AS(MT, false); }
    if (p.mt == 1) { EXPAND(1) }
    else { EXPAND(2) }
#undef EXPAND
#undef EXPAND_AS
    return check_launch("low_rank_add");
}

}  // extern "C"
