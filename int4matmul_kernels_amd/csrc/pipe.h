// The step loop of the pipelined tile kernels, for one tile: matmul.hip launches it for a product with one matrix,
// experts_tiles.hip for the rows of each expert.
#pragma once

#include "decode.h"

#include <type_traits>

namespace i4 {

struct MatmulArgs {
    h16* outs;
    const uint32_t* matrix;
    const uint32_t* mask;
    const h16* x;
    const h16* scales;
    const h16* zeros;
    int M, K, S;
    int group_units;        // group size / 64
    int tiles_m, tiles_n;
    int by_columns;         // pipelined kernel: 1 = an XCD walks its range of tile columns row by row
    // split-K (pipelined kernel, grids that would leave most of the GPU idle): `ksplit` workgroups
    // share a tile, each walks 1 / ksplit of the K steps and stores its fp32 partial tile to
    // `part`; the one that arrives last (`counters`, one per tile) adds them up in split order
    int ksplit;
    float* part;
    int* counters;
    // tiles (in grid order) before `split_from` are not split: a grid whose last round would fill
    // at most half of the GPU splits only the tiles of that round
    int split_from;
};

// ---- the pipelined kernel: (TM * 32) x (NW * 64) tiles, 2 x NW waves of (TM * 16) x 64, K steps of 32.
//
// What bounds it is the power limit: at full load the clock falls to what the work of a K step allows, so energy per step counts,
// and beside it the step's length.  Hence
//  * v_mfma_f32_16x16x32_f16: a loop of nothing but MFMAs and their LDS reads, on all CUs and random data, does 1710 TFLOP/s where
//    32x32x16 ones do 1530 (a third less accumulator traffic per flop); at zeros, which cost no power, both do 2260;
//  * the states go from global memory straight to LDS, A_AHEAD steps ahead (six stages), which leaves the registers alone;
//  * decodes of 17 (int4, int2) and 24 (int3) instructions per chunk through the 8-bit float conversion and v_perm tables;
//  * scales and zeros are asked for once per pair of steps, int4's words of two columns in one load;
//  * the two halves of the workgroup run a step in opposite phases (PING): a SIMD holds a wave of each, one on the matrix
//    pipe, its decode in the shadow of its MFMAs, while the other does everything that touches the LDS or memory.  A wave's own
//    LDS stores between its MFMAs would hold these up (40 cycles each, on a step of 1024), and just before the barrier the
//    barrier; so what phase 1 stores at a step's start was decoded in the step before.  (1330 cycles a step with the
//    stores between the MFMAs, 1200 with those of the decode at its end, 1050 so, in a loop without global loads.)
// A tile of int4 or 16:32 that contains exponent-mode groups takes a second copy of the loop whose decode serves either mode;
// int2 and int3 have one decode for both.
//
// Measured, before (32x32x16 MFMAs, states through registers, magic-number decodes) / so, us: K=5120, S=20480, 2048 rows int4 398 /
// 346, int3 402 / 359, int2 394 / 337, 16:32 437 / 400, one group in 40 in exponent mode 464 / 369, int3 468 / 359; K=8192,
// S=28672, 4096 rows 1663 / 1430 (1.35 PFLOP/s); with the plan of the tiles below K=S=8192, 768 rows 146 / 107; K=20480, S=5120, 1024
// rows 265 / 206.
constexpr int PK = 32;            // K per step of the pipelined kernel

// Per-format constants of the pipelined kernel: packed rows per 32-row block and
// the number of packed words a thread loads per K step for its two chunks.
template <int BITS, bool SPARSE> struct PipeFmt;
template <> struct PipeFmt<4, false> { static constexpr int ROWS = 4, NWORDS = 2; };
template <> struct PipeFmt<3, false> { static constexpr int ROWS = 3, NWORDS = 2; };
template <> struct PipeFmt<2, false> { static constexpr int ROWS = 2, NWORDS = 1; };
template <> struct PipeFmt<4, true> { static constexpr int ROWS = 2, NWORDS = 2; };

constexpr int P_STAGES = 3, A_STAGES = 6;  // of the weights, of the states
constexpr int A_AHEAD = 5;                 // steps that the states are ahead
// immediate of s_waitcnt: at most so many vector memory and LDS operations outstanding
constexpr int wait_counts(int vm, int lgkm) { return (vm & 15) | 0x70 | lgkm << 8 | (vm >> 4) << 14; }

// Swizzle of the states stage: row m's 16-byte chunk c stands at c ^ pipe_swz(m).  A 16-byte LDS read is served in
// groups of lanes 0-3, 12-15, 20-27 and 4-11, 16-19, 28-31 (of each half wave); with lane = row + 16 chunk each group then
// touches all 64 banks once (247 bytes a cycle and CU; with (m >> 2) & 3, which suits 32 rows x 2 chunks, 127).
__device__ __forceinline__ int pipe_swz(int m) { return ((m >> 3) & 1) | (((m >> 1 ^ m >> 2) & 2)); }

// GATED (the first product of an expert): the tile's rows are those that `order` names; of a wave's 64 columns every four
// are two neighbouring ones of the gate and the same two of the other half of the matrix, so that a lane ends with pairs of
// both and stores h = silu(gate) * up; the tile is 128 columns of h, s0 counts both halves.
struct GatedRows {
    const int* order;              // of the tile's rows: pair = row top_k + slot
    int top_k, half;               // half: columns of the gate
    uint32_t bytes;                // of all rows
};
__device__ __forceinline__ float silu_times(float gate, float up) { return gate * __builtin_amdgcn_rcpf(1.f + __expf(-gate)) * up; }

// PING: the waves of the first half run phase 0, MFMAs first and then everything else; those of the second half phase 1,
// everything else first and the MFMAs last.  Without it all waves run phase 1.
// Out: what the results are stored as, h16 or float.
template <int BITS, bool SPARSE, int TM, int NW, bool PING, bool SPLIT, bool GATED = false, class Out = h16>
__device__ __forceinline__ void pipe_tile(const MatmulArgs& a, const int m0, const int s0, const h16* x,
                                          Out* outs, h16* const (&As)[A_STAGES], h16* Bs, uint32_t* lut, const int tile, const int split,
                                          const int nsplit, const GatedRows gated = {}) {
    constexpr int BM = TM * 32, BN = NW * 64, WM = TM * 16, WN = 64, TN = 4, T = 2 * NW * 64;
    constexpr int A_ROWS = T / 4;                                  // rows covered by one 16-byte load per thread
    constexpr int A_LOADS = (BM + A_ROWS - 1) / A_ROWS;            // such loads per thread and step (192 rows: the second half full)
    constexpr int B_STAGE = PK * BN;                               // halves per stage

    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm0 = (wave / NW) * WM, wn0 = (wave % NW) * WN;

    // states stage: row m at m * 64 bytes, 16-byte chunk c of the row at c ^ pipe_swz(m).  Thread t fills position t % 4 of rows
    // t / 4 + A_ROWS * i (rows >= M re-read row M - 1 and are dropped at the store), from global memory straight to LDS.
    const int a_row = t >> 2, a_chunk = (t & 3) ^ pipe_swz(a_row);            // (rows + A_ROWS: same swizzle)
    // every global address is a buffer resource (the tile's rows of states; the whole
    // of the packed matrix, mask, scales, zeros) plus a per-lane 32-bit byte offset that
    // never changes plus a workgroup-uniform 32-bit offset that moves with the K step:
    // buffer loads add the three themselves, no address arithmetic is left to the VALU
    // (the launcher admits only shapes whose tensors stay below 2 GB: pipe_shape)
    constexpr int RSRC_FLAGS = 0x00020000;               // raw buffer, 32-bit data format
    const __amdgpu_buffer_rsrc_t a_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<h16*>(GATED ? x : x + (int64_t)m0 * a.K), 0, GATED ? (int)gated.bytes : min(a.M - m0, BM) * a.K * 2, RSRC_FLAGS);
    uint32_t a_off[A_LOADS];
#pragma unroll
    for (int i = 0; i < A_LOADS; ++i) {
        int row = min(a_row + A_ROWS * i, min(a.M - m0, BM) - 1);
        if constexpr (GATED) row = gated.order[row] / gated.top_k;
        a_off[i] = (uint32_t)((row * a.K + a_chunk * 8) * 2);
    }
    auto dma_a = [&](int stage, uint32_t step_off) {
#pragma unroll
        for (int i = 0; i < A_LOADS; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(a_rsrc, (__attribute__((address_space(3))) void*)&As[stage][i * A_ROWS * PK + wave * 512], 16,
                                                     a_off[i], step_off, 0, 0);
    };

    // weights: a thread decodes two chunks of 8 rows of every K step.
    // int4: word `row` of two adjacent columns, one 8-byte load; the others: column bn, rows 16 bhb .. 16 bhb + 15 of the
    // step's 32-row block: int2 word bhb; int3 words bhb, bhb + 1 (bits 48 bhb .. 48 bhb + 47 of the block's 96-bit stream); 16:32
    // sparse: both words and the mask word of the block.
    // Column 4 n + j of a wave's 64 stands at position 16 j + (n ^ 4 (j / 2)) of its row of chunks: an MFMA tile takes every fourth
    // column, so that the four tiles leave a lane with four adjacent columns of a row, an 8-byte store.  The fragment reads, 256 bytes
    // a cycle, and the stores of either mapping, 128 bytes of eight lanes a cycle, touch every bank once (with n ^ 8 the stores of
    // int4 met twice on every second one: 16 conflict cycles per wave and step).
    // (a last tile that is not full: the columns beyond the last repeat the last 64 and are not written)
    using F = PipeFmt<BITS, SPARSE>;
    constexpr int NWORDS = F::NWORDS;
    constexpr bool PAIR = BITS == 4 && !SPARSE;
    constexpr int W_LOADS = PAIR ? 1 : NWORDS + (SPARSE ? 1 : 0);
    const int bn = PAIR ? t % (BN / 2) * 2 : t % BN, bhb = PAIR ? t / (BN / 2) : t / BN;
    const int of_wave = PAIR ? bn & 63 : 4 * ((bn & 15) ^ (bn >> 3 & 4)) + (bn >> 4 & 3);
    const int bcol = GATED ? min(s0 / 2 + (bn >> 6) * 32, gated.half - 32) + 2 * (of_wave >> 2) + (of_wave & 1) + (of_wave & 2 ? gated.half : 0)
                           : min(s0 + (bn & ~63), a.S - 64) + of_wave;
    int b_chunk[2];                                      // where the two chunks go (halves)
#pragma unroll
    for (int q = 0; q < 2; ++q)
        b_chunk[q] = 8 * (PAIR ? bhb * BN + (bn & ~63) + 16 * ((bn & 2) + q) + ((bn >> 2 & 15) ^ (bn << 1 & 4)) : (bhb * 2 + q) * BN + bn);
    struct Stage { uint32_t w[NWORDS]; uint32_t m; };
    // scale / zero travel as the aligned 32-bit word that holds the column's half
    // (sub-dword loads make the compiler wait for every outstanding load); `half_sel`
    // replicates the wanted half into both lanes of a packed register
    const uint32_t half_sel = (bcol & 1) ? 0x03020302u : 0x01000100u;
    uint32_t b_off[W_LOADS];
#pragma unroll
    for (int i = 0; i < (PAIR ? 1 : NWORDS); ++i)
        b_off[i] = (uint32_t)((((SPARSE ? 0 : bhb) + i) * a.S + bcol) * 4);
    const uint32_t m_off = (uint32_t)(bcol * 4);
    const uint32_t m_step = 4u * a.S;                    // bytes of one row of mask words
    const uint32_t sz_off = (uint32_t)((bcol & ~1) * 2);
    const uint32_t b_step = (uint32_t)(F::ROWS * 4) * a.S;   // bytes of packed weights per K step
    const uint32_t g_step = 2u * a.S;                    // bytes of one row of scales / zeros
    const int k_blocks = a.K / PK, n_groups = (k_blocks + a.group_units * 2 - 1) / (a.group_units * 2);
    const __amdgpu_buffer_rsrc_t w_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint32_t*>(a.matrix), 0, (int)(k_blocks * b_step), RSRC_FLAGS);
    const __amdgpu_buffer_rsrc_t m_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint32_t*>(SPARSE ? a.mask : a.matrix), 0, (int)(k_blocks * m_step), RSRC_FLAGS);
    const __amdgpu_buffer_rsrc_t sc_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<h16*>(a.scales), 0, (int)(n_groups * g_step), RSRC_FLAGS);
    const __amdgpu_buffer_rsrc_t ze_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<h16*>(a.zeros), 0, (int)(n_groups * g_step), RSRC_FLAGS);
    // cursor over K steps: byte offsets of the step's packed-weight rows, mask row and scale / zero row
    struct Cursor { uint32_t w, m, sz; int kt, left; };
    auto cursor_at = [&](int kt) {
        const int gu = a.group_units * 2, group = kt / gu;
        return Cursor{kt * b_step, SPARSE ? kt * m_step : 0u, group * g_step, kt, gu - kt % gu};
    };
    // scale and zero of the thread's column: of the pair of steps that is decoded, and as loaded for the next one (a group is
    // whole pairs of steps, and a workgroup starts with one)
    uint32_t next_s, next_z;
    auto load_b = [&](Stage& s, const Cursor& c, bool first_of_pair) {
        if constexpr (PAIR) {
            const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(w_rsrc, b_off[0], c.w, 0);
            s.w[0] = v.x;
            s.w[1] = v.y;
        } else {
#pragma unroll
            for (int i = 0; i < NWORDS; ++i) s.w[i] = __builtin_amdgcn_raw_buffer_load_b32(w_rsrc, b_off[i], c.w, 0);
        }
        if constexpr (SPARSE) s.m = __builtin_amdgcn_raw_buffer_load_b32(m_rsrc, m_off, c.m, 0);
        if (first_of_pair) {
            next_s = __builtin_amdgcn_raw_buffer_load_b32(sc_rsrc, sz_off, c.sz, 0);
            next_z = __builtin_amdgcn_raw_buffer_load_b32(ze_rsrc, sz_off, c.sz, 0);
        }
    };
    auto take_sz = [&](auto (&co)[PAIR ? 2 : 1]) {
#pragma unroll
        for (int q = 0; q < (PAIR ? 2 : 1); ++q) {
            const uint32_t sel = !PAIR ? half_sel : q ? 0x03020302u : 0x01000100u;
            co[q].set(as_h2(__builtin_amdgcn_perm(next_s, next_s, sel)), as_h2(__builtin_amdgcn_perm(next_z, next_z, sel)));
        }
    };
    // the 8 codes of the thread's chunk q (rows 16 bhb + 8 q .. + 7), LSB first
    const int i3_shift = 16 * bhb;
    auto chunk_bits = [&](const Stage& s, int q) -> uint32_t {
        if constexpr (BITS == 4) return s.w[q];
        else if constexpr (BITS == 2) return q ? s.w[0] >> 16 : s.w[0];
        else if (q == 0) return __builtin_amdgcn_alignbit(s.w[1], s.w[0], i3_shift);
        else return __builtin_amdgcn_alignbit(bhb ? 0u : s.w[1], bhb ? s.w[1] : s.w[0], i3_shift + 24);
    };
    // 16:32 sparse: mask bits of chunk q and its kept codes as consecutive nibbles: those from the skip-th on of the block's two
    // words, 4 bits each.  (Neither here nor above a shift of 64 bits by a register: where that is the last vector register that a
    // kernel has, this GPU shifts by something else now and then, and the compiler does not keep from it.  Behind 16 skipped codes
    // the chunk has none.)
    auto sparse_chunk = [&](const Stage& s, int q, uint32_t& v, uint32_t& m8) {
        const uint32_t m16 = (s.m >> (16 * bhb)) & 0xFFFFu;
        uint32_t skip = bhb ? __builtin_popcount(s.m & 0xFFFFu) : 0;
        if (q) skip += __builtin_popcount(m16 & 0xFFu);
        m8 = (m16 >> (8 * q)) & 0xFFu;
        v = __builtin_amdgcn_alignbit(skip < 8 ? s.w[1] : 0u, skip < 8 ? s.w[0] : s.w[1], 4 * skip);
    };
    auto decode = [&](const Stage& st, const auto (&co)[PAIR ? 2 : 1], h16x8 (&w)[2]) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const auto& c = co[PAIR ? q : 0];
            if constexpr (SPARSE) {
                uint32_t v, m8;
                sparse_chunk(st, q, v, m8);
                w[q] = dequant_chunk_sparse(v, m8, lut, c);
            } else {
                w[q] = dequant_chunk<BITS>(chunk_bits(st, q), c);
            }
        }
    };
    auto write_b = [&](const h16x8 (&w)[2], int stage) {
#pragma unroll
        for (int q = 0; q < 2; ++q) *reinterpret_cast<h16x8*>(&Bs[stage * B_STAGE + b_chunk[q]]) = w[q];
    };
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // fragment addresses (halves, inside a stage); a step's 32 k are four chunks, one per lane group of 16
    // (row offsets are multiples of 16: the same swizzle for all of a lane's rows)
    const int a_frag = (wm0 + (lane & 15)) * PK + (((lane >> 4) ^ pipe_swz(lane)) << 3);
    const int b_frag[2] = {((lane >> 4) * BN + wn0 + (lane & 15)) * 8, ((lane >> 4) * BN + wn0 + ((lane & 15) ^ 4)) * 8};
    auto load_frags = [&](int a_stage, int stage, h16x8 fa[TM], h16x8 fb[TN]) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
            fa[i] = *reinterpret_cast<const h16x8*>(&As[a_stage][a_frag + i * 16 * PK]);
#pragma unroll
        for (int j = 0; j < TN; ++j)
            fb[j] = *reinterpret_cast<const h16x8*>(&Bs[stage * B_STAGE + b_frag[j >> 1] + j * 128]);
    };
    auto mfma_step = [&](const h16x8 fa[TM], const h16x8 fb[TN]) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[i], fb[j], acc[i][j], 0, 0, 0);
    };

    // K steps kt0 .. last of the matrix belong to this workgroup (all of them unless SPLIT)
    const int ksteps = a.K / PK;
    // (whole pairs of steps; a share has at least four)
    const int kt0 = SPLIT ? ksteps / 2 * split / nsplit * 2 : 0;
    const int ktiles = (SPLIT ? ksteps / 2 * (split + 1) / nsplit * 2 : ksteps) - kt0;
    const int last = kt0 + ktiles - 1;

    // Cursors of the loads: weights run four K steps ahead of the MFMAs, states
    // A_AHEAD; both stop at the last step (the surplus loads re-read it, unused).
    Cursor cur = cursor_at(kt0);
    // (selects instead of branches: a branch here would split the scheduling
    // region of the step and invite the compiler to reuse the previous step's
    // scale / zero registers, which makes the step wait for its newest loads)
    // (plain integer arithmetic on purpose: conditions kept as booleans come out as
    // 64-bit lane-mask operations, several scalar instructions each)
    const int gu2 = a.group_units * 2;
    auto advance = [&]() {
        const int more = min(last - cur.kt, 1);                  // 1 until the last step is reached
        const int wrap = cur.left == 1 ? more : 0;
        cur.kt += more;
        cur.w += more * b_step;
        if constexpr (SPARSE) cur.m += more * m_step;
        cur.sz += wrap * g_step;
        cur.left += wrap * gu2 - more;
    };
    uint32_t a_cur = (uint32_t)kt0 * (PK * 2);
    int a_kt = kt0;
    auto advance_a = [&]() {
        const int more = min(last - a_kt, 1);
        a_kt += more;
        a_cur += more * (PK * 2);
    };
    Stage r[3];
    // the first steps' operands are requested before the look at the scales below, whose
    // round trip to memory they then share
    load_b(r[0], cur, true); advance();
    load_b(r[1], cur, false); advance();
#pragma unroll
    for (int i = 0; i < A_AHEAD; ++i) { dma_a(i, a_cur); advance_a(); }

    // Does any (group, column) of this tile use exponent quantisation (scale < 0
    // or NaN)?  One pass over the tile's scales (a few KB); the answer is
    // workgroup-uniform and selects between the pipelined loop, whose decode is
    // the linear one, and the one that also serves exponent groups.  (int2 and int3 have one decode for both.)
    bool tile_has_expo = false;
    if constexpr (BITS == 4) {
        int& any_expo = *reinterpret_cast<int*>(Bs);          // borrowed before the pipeline starts
        __syncthreads();
        if constexpr (SPARSE) {
            if (t < 256) sparse_lut_entry(lut, t);
        }
        if (t == 0) any_expo = 0;
        __syncthreads();
        {
            // the tile's scales are `groups` rows of BN / 2 aligned 32-bit words; the threads share them
            // out and fetch four words each per trip, all in flight together (one round trip to
            // memory instead of one per group)
            bool bad = false;
            const int groups = (ksteps + a.group_units * 2 - 1) / (a.group_units * 2);
            const int total = groups * (BN / 2);
            const uint32_t* tile_scales = reinterpret_cast<const uint32_t*>(a.scales + (GATED ? s0 / 2 : s0));
            const int64_t row_words = a.S / 2;
            const int last_word = GATED ? (gated.half - s0 / 2) / 2 - 1 : (a.S - s0) / 2 - 1;
            // (a gated tile's words are BN / 4 of the gate and as many of the other half)
            auto word = [&](int i) { return GATED ? min(i % (BN / 4), last_word) + (i & BN / 4 ? gated.half / 2 : 0) : min(i, last_word); };
            for (int i0 = t; i0 < total; i0 += 4 * T) {
                uint32_t v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i = min(i0 + k * T, total - 1);
                    v[k] = tile_scales[(int64_t)(i / (BN / 2)) * row_words + word(i % (BN / 2))];
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const h16x2 h = as_h2(v[k]);
                    bad |= !(h.x >= (h16)0.0f) | !(h.y >= (h16)0.0f);
                }
            }
            if (__builtin_amdgcn_ballot_w64(bad) != 0 && lane == 0) any_expo = 1;
        }
        __syncthreads();
        tile_has_expo = any_expo != 0;
        __syncthreads();
    }

    // Step kt, u = kt % 6, weights' stage b = kt % 3, states' stage u.  On entry states and decoded weights of
    // steps kt and kt + 1 are complete.  The step stores the decoded weights of step kt + 2 and asks for the packed ones of
    // kt + 4 and the states of kt + A_AHEAD.  Phase 0:
    // MFMAs, on fragments fetched in the step before, beside the decode of step kt + 2's weights; then stores, loads, the next
    // step's fragments.  Phase 1: the step's own fragments, stores of what the step before decoded, loads; then MFMAs
    // beside the decode of step kt + 3's weights.
    h16x8 fa[TM], fb[TN], dec[2];
    auto walk = [&](auto mode) {
        Coef<BITS, decltype(mode)::value> co[PAIR ? 2 : 1];
        auto body = [&](auto phase_tag, int u, Stage& r_new, const Stage& r_dec) {
            constexpr int phase = decltype(phase_tag)::value;
            const int b = u % P_STAGES, b1 = (u + 1) % P_STAGES, b2 = (u + 2) % P_STAGES;
            auto stores_and_loads = [&]() {
                write_b(dec, b2);
                __builtin_amdgcn_sched_barrier(0);
                dma_a((u + A_AHEAD) % A_STAGES, a_cur);
                load_b(r_new, cur, u % 2 == 0);
                advance_a();
                advance();
                __builtin_amdgcn_sched_barrier(0);
            };
            if constexpr (phase == 1) {
                load_frags(u, b, fa, fb);
                __builtin_amdgcn_sched_barrier(0);
                stores_and_loads();
            }
            if ((u + phase) % 2 == 0) take_sz(co);
            decode(r_dec, co, dec);
            mfma_step(fa, fb);
            // (the decode in the shadow of the MFMAs: one occupies the pipe for 16 cycles, and up to two other vector instructions per
            // MFMA go beside it.  Spread over the last two thirds, so that the packed words need not have arrived yet: 261 us where
            // three behind each of the first MFMAs take 288, 16 tiles at K = 16384; at full load 2 - 3 %)
            constexpr int MFMAS = TM * TN, LATE = MFMAS / 3, DECODE = (SPARSE ? 64 : BITS == 3 ? 52 : 40) + (decltype(mode)::value ? 26 : 0);
#pragma unroll
            for (int e = 0; e < MFMAS; ++e) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                const int n = e < LATE ? 0 : (e - LATE + 1) * DECODE / (MFMAS - LATE) - (e - LATE) * DECODE / (MFMAS - LATE);
                if (n == 1) __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
                else if (n == 2) __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
                else if (n == 3) __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
                else if (n == 4) __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
                else if (n > 4) __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (phase == 0) stores_and_loads();
            // the step's stores are complete (lgkmcnt(0)) and, of the loads, all but the last two steps'
            __builtin_amdgcn_s_waitcnt(wait_counts(2 * (A_LOADS + W_LOADS) + 2, 0));
            if constexpr (phase == 0) {
                load_frags((u + 1) % A_STAGES, b1, fa, fb);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        take_sz(co);
        decode(r[0], co, dec);
        write_b(dec, 0);
        decode(r[1], co, dec);
        write_b(dec, 1);
        __builtin_amdgcn_s_waitcnt(wait_counts(0, 15));         // steps 0 ... A_AHEAD - 1 of the states
        load_b(r[2], cur, true); advance();             // step 2
        load_b(r[0], cur, false); advance();            // step 3
        __syncthreads();
        // weight stages and registers rotate with period 3, the states' stages with 6: six steps per trip, unrolled so that
        // all of them are compile-time names
        auto run = [&](auto phase_tag) {
            constexpr int ahead = 2 + decltype(phase_tag)::value;
            for (int kt = 0; kt < ktiles; kt += 6) {
#pragma unroll
                for (int u = 0; u < 6; ++u) {
                    if (u > 0 && kt + u >= ktiles) break;
                    body(phase_tag, u, r[(u + 1) % 3], r[(u + ahead) % 3]);
                }
            }
        };
        if (PING && wave < NW) {
            load_frags(0, 0, fa, fb);
            if constexpr (PING) run(std::integral_constant<int, 0>{});
        } else {
            take_sz(co);
            decode(r[2], co, dec);
            run(std::integral_constant<int, 1>{});
        }
    };
    if (BITS == 4 && tile_has_expo) walk(std::bool_constant<BITS == 4>{});
    else walk(std::false_type{});
    // (no load to LDS is in flight any more when the LDS is used otherwise or given back)
    __builtin_amdgcn_s_waitcnt(wait_counts(0, 15));
    if (SPLIT && nsplit > 1) {
        // Every workgroup of the tile stores its partial accumulators (16 bytes per lane and
        // store: register group g of thread t at (g * T + t) * 16 -- whole cache lines per wave)
        // and then counts itself in; whoever finds all the others counted adds the partials up
        // in split order (its own included, from memory: the sum has one order whoever is
        // last) and writes the tile.  Stores and loads go straight through to memory
        // (system-scope cache policy), the counter is a device-scope atomic: no cache-wide
        // fence, no waiting.  (Two workgroups per tile: the last one adds the other's partial to
        // its own registers -- a sum of two terms has one value in either order.)
        constexpr int SLOT_BYTES = BM * BN * 4, THROUGH = 17;      // sc0 | sc1
        char* const slots = reinterpret_cast<char*>(a.part) + (int64_t)tile * nsplit * SLOT_BYTES;
        const __amdgpu_buffer_rsrc_t mine = __builtin_amdgcn_make_buffer_rsrc(
            slots + (int64_t)split * SLOT_BYTES, 0, SLOT_BYTES, RSRC_FLAGS);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                __builtin_amdgcn_raw_buffer_store_b128(bitcast<u32x4>(acc[i][j]), mine, ((i * TN + j) * T + t) * 16, 0, THROUGH);
        __builtin_amdgcn_s_waitcnt(0);                 // every store of this thread has been acknowledged
        int* const flag = reinterpret_cast<int*>(Bs);
        __syncthreads();
        if (t == 0) *flag = __hip_atomic_fetch_add(a.counters + tile, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (*flag != nsplit - 1) return;
        if (t == 0) __hip_atomic_store(a.counters + tile, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // clean for the next call
        if (nsplit > 2) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        for (int sp = nsplit > 2 ? 0 : 1 - split; sp < (nsplit > 2 ? nsplit : 2 - split); ++sp) {
            const __amdgpu_buffer_rsrc_t theirs = __builtin_amdgcn_make_buffer_rsrc(
                slots + (int64_t)sp * SLOT_BYTES, 0, SLOT_BYTES, RSRC_FLAGS);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    acc[i][j] += bitcast<f32x4>(__builtin_amdgcn_raw_buffer_load_b128(theirs, ((i * TN + j) * T + t) * 16, 0, THROUGH));
        }
    }
    if constexpr (GATED) {
        const int c = s0 / 2 + wn0 / 2;
        if (c >= gated.half) return;
        h16* const out = outs + (int64_t)(wm0 + 4 * (lane >> 4)) * gated.half + c + 2 * (lane & 15);
        const int left = a.M - (wm0 + 4 * (lane >> 4));
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (16 * i + r < left)
                    *reinterpret_cast<h16x2*>(out + (int64_t)(16 * i + r) * gated.half) =
                        h16x2{(h16)silu_times(acc[i][0][r], acc[i][2][r]), (h16)silu_times(acc[i][1][r], acc[i][3][r])};
        return;
    }
    if (s0 + wn0 >= a.S) return;                       // (a wave's 64 columns are inside or outside as one)
    // register r of tile (i, j) is row 16 i + 4 (lane / 16) + r, column 4 (lane % 16) + j of the wave's
    typedef Out Out4 __attribute__((ext_vector_type(4)));
    Out* const out = outs + (int64_t)(m0 + wm0 + 4 * (lane >> 4)) * a.S + s0 + wn0 + 4 * (lane & 15);
    const int rows = a.M - (m0 + wm0 + 4 * (lane >> 4));
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (16 * i + r < rows)
                *reinterpret_cast<Out4*>(out + (int64_t)(16 * i + r) * a.S) =
                    Out4{(Out)acc[i][0][r], (Out)acc[i][1][r], (Out)acc[i][2][r], (Out)acc[i][3][r]};
}

}  // namespace i4
