// The experts' gated feed-forward on packed weights: of tokens x [T, K] with the experts ids [T, k] and their weights [T, k]
//     h[t, j, :] = silu(x[t] up_e[:, :F]) * (x[t] up_e[:, F:]),   outs[t, :] = fp16( sum_j weights[t, j] * (h[t, j] down_e) ),
// e = ids[t, j]; a pair whose id is outside 0 ... E - 1 has no expert and adds nothing.  Sums are fp32; h is rounded to fp16 (it is
// an operand of the matrix instructions), and so is the result.
//
//   plan_kernel     pairs in the order of their experts, stable: where each expert's begin, the pairs, each pair's place (up to 256
//                   pairs: order_few, at the head of the first product)
//   rows_kernel     a product of the pairs of one expert, up to 32 at a time, with a strip of 64 columns (many pairs an expert:
//                   experts_tiles.hip)
//   combine_kernel  the weighted sum of a token's k results, fp32
//
// rows_kernel is bound by reading the packed weights and by the instructions that decode them.  The waves of a workgroup share K out,
// so nothing is shared through LDS in the loop: a lane loads 16 bytes of packed words, four neighbouring columns of the packed row
// that holds its 8 k, and each word is after its decode the operand of one v_mfma_f32_16x16x32_f16 whose columns are every fourth
// of the strip.  What is multiplied is what the codes stand for, exact in fp16; scale and zero are applied once per group to the sums
// (sum x w = s (sum x q - z sum x), the sum of x from a product with ones), which takes 7 instructions a word where rounded weights
// take 17 and is nearer to the exact product.  The partial sums of the waves meet in LDS.
//
// Measured (64 tokens, two of eight experts of 4096 x 11008, int4, us a call on one GPU): weights rounded, addresses computed, one lane
// for 16 bytes of every row of states 198; exact codes, buffer loads, two units in flight in the order that the waits go by 178; states
// read row by row and turned in LDS 172; states straight to LDS, blocks of up to 16 pairs with one row tile 155 - 166.  With all
// weights from cache 129 before the last step, without the fold of the groups' sums 107: not the bytes, the
// issue of the fold and the decode and the ends of the workgroups.  Three units in flight are slower (192: registers), so are strips that are
// neighbours on an XCD (193), and non-temporal loads where the weights fit the last-level cache (37 / 42, 16 experts of 2048 x 1408,
// 16 pairs each).
// Both heights share a kernel, whose registers are those of the two row tiles.  Compiled with one row tile alone, blocks of 16 pairs, it takes int4 43,
// int3 54 - 60, int2 51, 16:32 66 - 72 where this takes 53, 68, 58 - 63, 84 (64 experts of 2048 x 1024, 2 pairs each), at means of 8 to 16 the two cross, and
// at 32 it loses a fifth (8 experts of 4096 x 11008, int4 259 / 210): a kernel of its own for small means is left to do.
#include "experts.h"

#include <algorithm>
#include <cmath>

namespace i4 {

template <int BITS, bool SPARSE> struct RowsFmt;       // packed rows of a 32-row block, 16-byte loads of a lane per block
template <> struct RowsFmt<4, false> { static constexpr int ROWS = 4, LOADS = 1; };
template <> struct RowsFmt<3, false> { static constexpr int ROWS = 3, LOADS = 2; };
template <> struct RowsFmt<2, false> { static constexpr int ROWS = 2, LOADS = 1; };
template <> struct RowsFmt<4, true> { static constexpr int ROWS = 2, LOADS = 3; };

// ---- pairs in the order of their experts: workgroup e finds how many pairs belong to lower experts, and places its own.  Each
// of the 16 waves takes a share of the pairs, twice: counting, then placing; no atomics, the order is that of the pairs.
// A wave reads 256 pairs at a time, four neighbours a lane, and keeps the first 2048 of its share in registers: one trip to memory.
// REST: an id outside belongs to the last expert, and no places are asked for.
struct __attribute__((packed, aligned(4))) FourIds { int v[4]; };
template <bool REST>
__global__ __launch_bounds__(1024) void plan_kernel(const int* ids, int* offsets, int* order, int* place, int pairs, int experts) {
    constexpr int DEPTH = 8;
    __shared__ int of_wave[16], lower_of_wave[16];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), e = blockIdx.x;
    const int share = ((pairs + 15) / 16 + 255) & ~255, from = min(wave * share, pairs), to = min(from + share, pairs);
    int kept[DEPTH][4];
    auto load = [&](int (&v)[4], int at) __attribute__((always_inline)) {
        const int p = at + 4 * lane;
        if (p + 4 <= to) {
            const FourIds f = *reinterpret_cast<const FourIds*>(ids + p);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = f.v[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = p + j < to ? ids[p + j] : -1;
        }
        if constexpr (REST) {
            // (below 0: not a pair)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = p + j >= to ? -1 : (uint32_t)v[j] < (uint32_t)experts ? v[j] : experts - 1;
        }
    };
    int mine = 0, below = 0;
    auto count = [&](const int (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mine += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[j] == e));
            below += __builtin_popcountll(__builtin_amdgcn_ballot_w64((uint32_t)v[j] < (uint32_t)e));
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (from + 256 * d < to) load(kept[d], from + 256 * d);
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (from + 256 * d < to) count(kept[d]);
    for (int i = from + 256 * DEPTH; i < to; i += 256) {
        int v[4];
        load(v, i);
        count(v);
    }
    if (lane == 0) {
        of_wave[wave] = mine;
        lower_of_wave[wave] = below;
    }
    __syncthreads();
    int lower = 0, at = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        lower += lower_of_wave[w];
        at += w < wave ? of_wave[w] : 0;
        all += of_wave[w];
    }
    at += lower;
    if (t == 0) {
        offsets[e] = lower;
        if (e == experts - 1) offsets[experts] = lower + all;
    }
    const uint64_t before = (1ull << lane) - 1;
    auto put = [&](const int (&v)[4], int i) __attribute__((always_inline)) {
        uint64_t in[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) in[j] = __builtin_amdgcn_ballot_w64(v[j] == e);
        int where = at;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            where += __builtin_popcountll(in[j] & before);
            at += __builtin_popcountll(in[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int p = i + 4 * lane + j;
            if (v[j] == e) {
                order[where] = p;
                if constexpr (!REST) place[p] = where;
                ++where;
            } else if (!REST && e == 0 && p < to && (uint32_t)v[j] >= (uint32_t)experts) {
                place[p] = -1;
            }
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (from + 256 * d < to) put(kept[d], from + 256 * d);
    for (int i = from + 256 * DEPTH; i < to; i += 256) {
        int v[4];
        load(v, i);
        put(v, i);
    }
}

void launch_rows_by_id(const int* ids, int* offsets, int* order, int rows, int buckets, hipStream_t st) {
    hipLaunchKernelGGL(plan_kernel<true>, dim3(buckets), dim3(1024), 0, st, ids, offsets, order, (int*)nullptr, rows, buckets);
}

// The operand of a lane, 8 k of one column, from the words that it has loaded of a 32-row block: `lo` its packed word (int3: and the
// next, 16:32: and the block's second and its mask)
template <int BITS, bool SPARSE, class C>
__device__ __forceinline__ h16x8 operand_of(uint32_t lo, uint32_t hi, uint32_t mask, int q, const uint32_t* lut, const C& co) {
    if constexpr (SPARSE) {
        const uint32_t skip = __builtin_popcount(mask & ((1u << (8 * q)) - 1u));
        // the codes from the skip-th on.  (Not a shift of 64 bits: with its amount in the last vector register that a
        // kernel has, this GPU shifts by something else now and then, and the compiler does not keep from it.)
        return dequant_chunk_sparse(__builtin_amdgcn_alignbit(skip < 8 ? hi : 0u, skip < 8 ? lo : hi, 4 * skip), (mask >> (8 * q)) & 0xFFu, lut, co);
    } else if constexpr (BITS == 4) {
        return dequant_chunk<4>(lo, co);
    } else if constexpr (BITS == 2) {
        return dequant_chunk<2>(lo >> (16 * (q & 1)), co);
    } else {
        // bits 24 q ... 24 q + 23 of the 96
        return dequant_chunk<3>(__builtin_amdgcn_alignbit(q == 3 ? 0u : hi, q == 3 ? hi : lo, (32 - 8 * q) & 31), co);
    }
}
// a lane's first packed row of a 32-row block; int3 and 16:32 load the next one too
template <int BITS, bool SPARSE>
__device__ __forceinline__ uint32_t packed_row(int q) { return BITS == 4 && !SPARSE ? q : BITS == 2 ? q >> 1 : BITS == 3 ? (q > 0 ? q - 1 : 0) : 0; }
template <int BITS, bool SPARSE>
__device__ __forceinline__ uint32_t packed_row2(int q) { return SPARSE ? 1u : min(packed_row<BITS, SPARSE>(q) + 1u, 2u); }

// (A, B) of sum x w = A sum x value + B sum x.  (16:32 and a NaN scale: A is that NaN, since `value` may come from the linear decode, which
// has not met the scale; see any_negative)
template <bool SPARSE>
__device__ __forceinline__ void fold_factors(uint32_t s2, uint32_t z2, int odd, float& A, float& B) {
    const float s = (float)as_h2(s2)[odd], z = (float)as_h2(z2)[odd];
    const bool linear = s >= 0.f;
    A = linear ? s : SPARSE ? (s < 0.f ? 1.f : s) : -s;
    B = linear ? -s * z : z;
}
// a scale with its sign set anywhere in the wave: the decode that serves either mode
__device__ __forceinline__ bool any_negative(uint32_t a, uint32_t b) { return __builtin_amdgcn_ballot_w64(((a | b) & 0x80008000u) != 0) != 0; }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);        // raw, 32-bit data format
}
__device__ __forceinline__ void fill_lut(uint32_t* lut, int t, int threads) {
    for (int e = t; e < 256; e += threads) sparse_lut_entry(lut, e);
    __syncthreads();
}

// ---- a product of up to 32 pairs of one expert with 64 columns, 16 MT of them in a tile's rows.  UP: 32 columns of the gate and the same 32 of the other
// half; the source row of a pair is its token's, the result h.  Else: 64 columns, source and result by place.
constexpr int ROWS_HEIGHT = 32, ROWS_WAVES = 4;
// Few pairs: every workgroup of the first product orders them by itself, from LDS, and finds its block's; the first one writes the order
// down for the kernels behind.  A launch less: us a call, 16 experts of 2048 x 1408, int4, ordered by plan_kernel / so: 32 pairs 27.9 / 25.9, 180 pairs
// 30.9 / 29.4, 512 pairs 42.7 / 44.8.
constexpr int FEW_PAIRS = 256, FEW_EXPERTS = 256;
struct FewPairs { int ids[FEW_PAIRS], count[FEW_EXPERTS], before[FEW_EXPERTS], order[ROWS_HEIGHT]; };
struct NoPairs { int order[1]; };
__device__ __forceinline__ bool order_few(const ExpertsArgs& a, int want, FewPairs& f, Block& b) {
    constexpr int T = 64 * ROWS_WAVES;
    static_assert(FEW_EXPERTS <= T);
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    if (t < FEW_EXPERTS) f.count[t] = 0;
    for (int p = t; p < FEW_PAIRS; p += T) {
        const int v = p < a.few_pairs ? a.ids[p] : -1;
        f.ids[p] = (uint32_t)v < (uint32_t)a.experts ? v : -1;
    }
    __syncthreads();
    for (int p = t; p < a.few_pairs; p += T)
        if (f.ids[p] >= 0) atomicAdd(&f.count[f.ids[p]], 1);
    __syncthreads();
    // blocks and pairs of the experts up to each, in the halves of a word
    int blocks = 0, pairs = 0, skip = 0;
    bool found = false;
    for (int e0 = 0; e0 < a.experts; e0 += 64) {
        const int e = e0 + lane, c = e < a.experts ? f.count[e] : 0, own = (c + ROWS_HEIGHT - 1) / ROWS_HEIGHT << 16 | c;
        int upto = own;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(upto, d);
            upto += lane >= d ? o : 0;
        }
        if (blockIdx.x == 0 && wave == 0 && e < a.experts) {
            f.before[e] = pairs + ((upto - own) & 0xFFFF);
            const_cast<int*>(a.offsets)[e] = f.before[e];
        }
        const uint64_t beyond = __builtin_amdgcn_ballot_w64(blocks + (upto >> 16) > want);
        if (!found && beyond) {
            const int l = __builtin_ctzll(beyond);
            const int mine = __builtin_amdgcn_readlane(own, l), lower = __builtin_amdgcn_readlane(upto, l) - mine;
            skip = (want - blocks - (lower >> 16)) * ROWS_HEIGHT;
            b.expert = e0 + l;
            b.first = pairs + (lower & 0xFFFF) + skip;
            b.count = min(ROWS_HEIGHT, (mine & 0xFFFF) - skip);
            found = true;
        }
        const int all = __builtin_amdgcn_readlane(upto, 63);
        blocks += all >> 16;
        pairs += all & 0xFFFF;
    }
    if (blockIdx.x == 0) {
        if (t == 0) const_cast<int*>(a.offsets)[a.experts] = pairs;
        __syncthreads();
        for (int p = t; p < a.few_pairs; p += T) {
            const int v = f.ids[p];
            int where = -1;
            if (v >= 0) {
                where = f.before[v];
                for (int o = 0; o < p; ++o) where += f.ids[o] == v;
                const_cast<int*>(a.order)[where] = p;
            }
            a.place[p] = where;
        }
    }
    if (!found) return false;
    if (wave == 0) {
        int seen = 0;
        for (int i = 0; i < a.few_pairs; i += 64) {
            const bool mine = f.ids[i + lane] == b.expert;
            const uint64_t in = __builtin_amdgcn_ballot_w64(mine);
            const int at = seen + __builtin_popcountll(in & ((1ull << lane) - 1)) - skip;
            if (mine && at >= 0 && at < ROWS_HEIGHT) f.order[at] = i + lane;
            seen += __builtin_popcountll(in);
        }
    }
    __syncthreads();
    return true;
}

template <int BITS, bool SPARSE, int MT, bool UP>
__device__ __forceinline__ void rows_tile(const ExpertsArgs& a, const Block& block, char* const (&Xs)[2], uint32_t* lut, const int* few) {
    using F = RowsFmt<BITS, SPARSE>;
    constexpr int HEIGHT = 16 * MT, WAVES = ROWS_WAVES, DEPTH = 2;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int n = lane & 15, q = lane >> 4;
    const int expert = block.expert, first = block.first, count = block.count;
    const int strip = blockIdx.x % a.strips;
    if constexpr (SPARSE) fill_lut(lut, t, 64 * WAVES);
    const int half = a.S / 2;
    // lane n's four columns of the strip
    const int col = UP ? (n < 8 ? 0 : half - 32) + 32 * strip + 4 * n : 64 * strip + 4 * n;
    // every load is a buffer, an offset of the lane that does not change and a uniform one that moves with k
    const int units = a.K / 64, groups = (units + a.group_units - 1) / a.group_units;
    const uint32_t row_bytes = 4u * (uint32_t)a.S;
    const __amdgpu_buffer_rsrc_t w_rsrc = buffer_of(a.matrix + expert * a.matrix_stride, 2 * units * F::ROWS * row_bytes);
    const __amdgpu_buffer_rsrc_t m_rsrc = buffer_of(SPARSE ? a.mask + expert * a.mask_stride : a.matrix, 2 * units * row_bytes);
    const __amdgpu_buffer_rsrc_t s_rsrc = buffer_of(a.scales + expert * a.scale_stride, groups * (row_bytes / 2));
    const __amdgpu_buffer_rsrc_t z_rsrc = buffer_of(a.zeros + expert * a.scale_stride, groups * (row_bytes / 2));
    const __amdgpu_buffer_rsrc_t x_rsrc = UP ? buffer_of(a.x, a.x_bytes) : buffer_of(a.x + (int64_t)first * a.K, 2u * (uint32_t)count * a.K);
    // states: eight lanes read the 128 bytes of a row (one lane for 16 bytes of every row, as the operands want them, are 64 accesses of
    // the L1 a load, four times as many), straight to LDS of the wave's own: chunk c of row r stands at c ^ (r % 8)
    uint32_t x_off[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
        const int at = min(8 * i + (lane >> 3), count - 1);             // (rows beyond the last repeat it and are not written)
        const int row = !UP ? at : (a.few_pairs ? few[at] : a.order[first + at]) / a.top_k;
        x_off[i] = 2u * ((uint32_t)row * a.K + 8 * ((lane & 7) ^ (lane >> 3)));
    }
    const uint32_t w_off = 4u * col + packed_row<BITS, SPARSE>(q) * row_bytes, w_off2 = 4u * col + packed_row2<BITS, SPARSE>(q) * row_bytes;

    struct Unit {                                     // 64 k
        u32x4 w[2][F::LOADS];
        u32x2 s, z;
    };
    constexpr int UNIT_LOADS = 2 * MT + 2 * F::LOADS + 2;
    auto load = [&](Unit& u, char* stage, int unit) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < 2 * MT; ++c)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(x_rsrc, (__attribute__((address_space(3))) void*)(stage + wave * (HEIGHT * 128) + c * 1024), 16,
                                                     x_off[c], 128u * unit, 0, 0);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint32_t blk = (uint32_t)(2 * unit + b) * row_bytes;
            u.w[b][0] = __builtin_amdgcn_raw_buffer_load_b128(w_rsrc, w_off, blk * F::ROWS, 0);
            if constexpr (F::LOADS > 1) u.w[b][1] = __builtin_amdgcn_raw_buffer_load_b128(w_rsrc, w_off2, blk * F::ROWS, 0);
            if constexpr (SPARSE) u.w[b][2] = __builtin_amdgcn_raw_buffer_load_b128(m_rsrc, 4u * col, blk, 0);
        }
        const uint32_t g = (uint32_t)magic_div(unit, a.group_units, a.group_magic) * (row_bytes / 2);
        u.s = __builtin_amdgcn_raw_buffer_load_b64(s_rsrc, 2u * col, g, 0);
        u.z = __builtin_amdgcn_raw_buffer_load_b64(z_rsrc, 2u * col, g, 0);
    };

    f32x4 acc[MT][4], acc_x[MT], sum[MT][4];
    auto clear = [&](auto& v) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    auto clear_group = [&]() __attribute__((always_inline)) {
        clear(acc);
#pragma unroll
        for (int m = 0; m < MT; ++m) acc_x[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    clear_group();
    clear(sum);
    const h16x8 ones = bitcast<h16x8>(u32x4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u});
    auto multiply = [&](auto mode, const Unit& u, const char* stage) __attribute__((always_inline)) {
        h16x8 x[2][MT];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int m = 0; m < MT; ++m)
                x[b][m] = bitcast<h16x8>(*reinterpret_cast<const u32x4*>(stage + (wave * HEIGHT + 16 * m + n) * 128 + (((4 * b + q) ^ n) & 7) * 16));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            Values<BITS, SPARSE, decltype(mode)::value> co;
            const uint32_t sel = (j & 1) ? 0x03020302u : 0x01000100u;
            co.set(as_h2(__builtin_amdgcn_perm(u.s[j >> 1], u.s[j >> 1], sel)), as_h2(__builtin_amdgcn_perm(u.z[j >> 1], u.z[j >> 1], sel)));
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const h16x8 w = operand_of<BITS, SPARSE>(u.w[b][0][j], F::LOADS > 1 ? u.w[b][F::LOADS > 1][j] : 0u, F::LOADS > 2 ? u.w[b][F::LOADS - 1][j] : 0u, q, lut, co);
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[b][m], w, acc[m][j], 0, 0, 0);
            }
        }
        if constexpr (!SPARSE) {
            // (every column of this product is the rows' sums: a lane has those of the rows that it has results of)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int m = 0; m < MT; ++m) acc_x[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[b][m], ones, acc_x[m], 0, 0, 0);
        }
    };
    // the end of a group, or of the wave's part of one
    auto fold = [&](const Unit& u) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float A, B;
            fold_factors<SPARSE>(u.s[j >> 1], u.z[j >> 1], j & 1, A, B);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if constexpr (!SPARSE) sum[m][j][r] = fmaf(B, acc_x[m][r], sum[m][j][r]);
                    sum[m][j][r] = fmaf(A, acc[m][j][r], sum[m][j][r]);
                }
        }
        clear_group();
    };
    const int u0 = units * wave / WAVES, u1 = units * (wave + 1) / WAVES;
    // DEPTH units in flight; what would be beyond the last is the last again, from the L1 (a load under a condition would make
    // the compiler wait for more than it needs)
    if (u0 < u1) {
        int left = a.group_units - (u0 - magic_div(u0, a.group_units, a.group_magic) * a.group_units);
        Unit ring[DEPTH];
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            load(ring[d], Xs[d], min(u0 + d, u1 - 1));
            __builtin_amdgcn_sched_barrier(0);        // (in this order, which the waits in the loop go by)
        }
#pragma unroll 1
        for (int i = u0; i < u1; i += DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const Unit& now = ring[d];
                // all loads but those of the younger units have arrived
                __builtin_amdgcn_s_waitcnt(wait_counts((DEPTH - 1) * UNIT_LOADS, 15));
                __builtin_amdgcn_sched_barrier(0);
                if (i + d < u1) {
                    if (any_negative(now.s[0], now.s[1])) multiply(std::true_type{}, now, Xs[d]);
                    else multiply(std::false_type{}, now, Xs[d]);
                    if (--left == 0 || i + d == u1 - 1) {
                        fold(now);
                        left = a.group_units;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                load(ring[d], Xs[d], min(i + d + DEPTH, u1 - 1));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    // (no load to LDS is in flight any more)
    __builtin_amdgcn_s_waitcnt(wait_counts(0, 15));
    __syncthreads();
    // register r of tile (m, j): row 16 m + 4 q + r, column 4 n + j of the strip
    float* const red[2] = {reinterpret_cast<float*>(Xs[0]), reinterpret_cast<float*>(Xs[1])};
    float* const to = (wave < WAVES / 2 ? red[0] : red[1]) + wave % (WAVES / 2) * (HEIGHT * 64);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            *reinterpret_cast<f32x4*>(to + (16 * m + 4 * q + r) * 64 + 4 * n) = f32x4{sum[m][0][r], sum[m][1][r], sum[m][2][r], sum[m][3][r]};
    __syncthreads();
    auto total = [&](int row, int c) __attribute__((always_inline)) {
        f32x4 s = *reinterpret_cast<const f32x4*>(red[0] + row * 64 + c);
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += *reinterpret_cast<const f32x4*>(red[w / (WAVES / 2)] + (w % (WAVES / 2) * HEIGHT + row) * 64 + c);
        return s;
    };
    constexpr int QUADS = UP ? 8 : 16;                // quadruples of results in a row
    for (int i = t; i < HEIGHT * QUADS; i += 64 * WAVES) {
        const int row = i / QUADS, c = i % QUADS * 4;
        if (row >= count) break;
        if constexpr (UP) {
            const f32x4 gate = total(row, c), up = total(row, c + 32);
            h16x4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = (h16)silu_times(gate[j], up[j]);
            *reinterpret_cast<h16x4*>(a.h + (int64_t)(first + row) * half + 32 * strip + c) = o;
        } else {
            *reinterpret_cast<f32x4*>(a.part + (int64_t)(first + row) * a.S + 64 * strip + c) = total(row, c);
        }
    }
}

template <int BITS, bool SPARSE, bool UP>
__global__ __launch_bounds__(64 * ROWS_WAVES, 2) void rows_kernel(ExpertsArgs a) {
    constexpr int STAGE = ROWS_WAVES * ROWS_HEIGHT * 128;
    // the states of the two units in flight (arrays of their own, so that the compiler sees which loads a read has to wait for); behind
    // the loop the waves' partial sums
    __shared__ __attribute__((aligned(16))) char X0[STAGE], X1[STAGE];
    __shared__ __attribute__((aligned(16))) uint32_t lut[SPARSE ? SPARSE_LUT_WORDS : 4];
    char* const Xs[2] = {X0, X1};
    __shared__ std::conditional_t<UP, FewPairs, NoPairs> few;
    Block block;
    bool here = false, ordered = false;
    if constexpr (UP)
        if (a.few_pairs) {
            ordered = true;
            here = order_few(a, blockIdx.x / a.strips, few, block);
        }
    if (!ordered) here = find_block(a.offsets, a.experts, ROWS_HEIGHT, blockIdx.x / a.strips, threadIdx.x & 63, block) < 0;
    if (!here) return;
    if (block.count <= 16) rows_tile<BITS, SPARSE, 1, UP>(a, block, Xs, lut, few.order);
    else rows_tile<BITS, SPARSE, 2, UP>(a, block, Xs, lut, few.order);
}

// ---- few pairs, hardly two of them of the same expert: no order, a workgroup takes a pair and 64 columns, two launches in all.
// What bounds them at that size is latency and the issue of instructions.  The second product's workgroups of a token and a strip
// store their weighted sums write-through and count themselves in, and the last to arrive adds them up in the order of the slots: a
// sum of one order, whoever is last.  Measured, one token, eight of 64 experts of 2048 x 1024, a call: 14.5 us; with sixteen waves
// 15.8; with all pairs of a token in one workgroup, as one long K, which leaves three quarters of the CUs idle, 18.4; through
// plan_kernel, rows_kernel and combine_kernel 19.5.
template <int BITS, bool SPARSE, bool UP>
__global__ __launch_bounds__(512) void token_kernel(ExpertsArgs a) {
    using F = RowsFmt<BITS, SPARSE>;
    constexpr int WAVES = 8, DEPTH = 2, THROUGH = 17;        // THROUGH: sc0 | sc1, straight to memory
    __shared__ __attribute__((aligned(16))) float red[WAVES * 64];
    __shared__ __attribute__((aligned(16))) uint32_t lut[SPARSE ? SPARSE_LUT_WORDS : 4];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int n = lane & 15, q = lane >> 4, strip = blockIdx.x % a.strips, pair = blockIdx.x / a.strips;
    const int token = pair / a.top_k, half = a.S / 2;
    const int id = a.ids[pair];
    const bool valid = (uint32_t)id < (uint32_t)a.experts;
    if constexpr (UP) {
        // the second product's counters, one for each of its strips of the token
        if (strip == 0 && pair == token * a.top_k)
            for (int c = t; c < a.K / 64; c += 64 * WAVES) a.arrivals[token * (a.K / 64) + c] = 0;
        if (!valid) return;
    }
    const int col = UP ? (n < 8 ? 0 : half - 32) + 32 * strip + 4 * n : 64 * strip + 4 * n;
    const int units = a.K / 64, groups = (units + a.group_units - 1) / a.group_units;
    const uint32_t row_bytes = 4u * (uint32_t)a.S;
    const int64_t e = valid ? id : 0;
    const __amdgpu_buffer_rsrc_t w_rsrc = buffer_of(a.matrix + e * a.matrix_stride, 2 * units * F::ROWS * row_bytes);
    const __amdgpu_buffer_rsrc_t m_rsrc = buffer_of(SPARSE ? a.mask + e * a.mask_stride : a.matrix, 2 * units * row_bytes);
    const __amdgpu_buffer_rsrc_t s_rsrc = buffer_of(a.scales + e * a.scale_stride, groups * (row_bytes / 2));
    const __amdgpu_buffer_rsrc_t z_rsrc = buffer_of(a.zeros + e * a.scale_stride, groups * (row_bytes / 2));
    const __amdgpu_buffer_rsrc_t x_rsrc = buffer_of(a.x + (int64_t)(UP ? token : pair) * a.K, 2u * (uint32_t)a.K);
    const uint32_t w_off = 4u * col + packed_row<BITS, SPARSE>(q) * row_bytes, w_off2 = 4u * col + packed_row2<BITS, SPARSE>(q) * row_bytes;
    struct Unit {
        u32x4 w[2][F::LOADS];
        u32x4 x[2];
        u32x2 s, z;
    };
    auto load = [&](Unit& u, int unit) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint32_t blk = (uint32_t)(2 * unit + b) * row_bytes;
            u.w[b][0] = __builtin_amdgcn_raw_buffer_load_b128(w_rsrc, w_off, blk * F::ROWS, 0);
            if constexpr (F::LOADS > 1) u.w[b][1] = __builtin_amdgcn_raw_buffer_load_b128(w_rsrc, w_off2, blk * F::ROWS, 0);
            if constexpr (SPARSE) u.w[b][2] = __builtin_amdgcn_raw_buffer_load_b128(m_rsrc, 4u * col, blk, 0);
            // (all rows of the operand are the one row)
            u.x[b] = __builtin_amdgcn_raw_buffer_load_b128(x_rsrc, 16u * q, 128u * unit + 64u * b, 0);
        }
        const uint32_t g = (uint32_t)magic_div(unit, a.group_units, a.group_magic) * (row_bytes / 2);
        u.s = __builtin_amdgcn_raw_buffer_load_b64(s_rsrc, 2u * col, g, 0);
        u.z = __builtin_amdgcn_raw_buffer_load_b64(z_rsrc, 2u * col, g, 0);
    };
    f32x4 acc[4], acc_x;
    float sum[4];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        acc_x = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    clear();
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = 0.f;
    const h16x8 ones = bitcast<h16x8>(u32x4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u});
    auto multiply = [&](auto mode, const Unit& u) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            Values<BITS, SPARSE, decltype(mode)::value> co;
            const uint32_t sel = (j & 1) ? 0x03020302u : 0x01000100u;
            co.set(as_h2(__builtin_amdgcn_perm(u.s[j >> 1], u.s[j >> 1], sel)), as_h2(__builtin_amdgcn_perm(u.z[j >> 1], u.z[j >> 1], sel)));
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const h16x8 w = operand_of<BITS, SPARSE>(u.w[b][0][j], F::LOADS > 1 ? u.w[b][F::LOADS > 1][j] : 0u, F::LOADS > 2 ? u.w[b][F::LOADS - 1][j] : 0u, q, lut, co);
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<h16x8>(u.x[b]), w, acc[j], 0, 0, 0);
            }
        }
        if constexpr (!SPARSE) {
#pragma unroll
            for (int b = 0; b < 2; ++b) acc_x = __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<h16x8>(u.x[b]), ones, acc_x, 0, 0, 0);
        }
    };
    const int u0 = units * wave / WAVES, u1 = valid ? units * (wave + 1) / WAVES : u0;
    Unit ring[DEPTH];
    if (u0 < u1) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            load(ring[d], min(u0 + d, u1 - 1));
            __builtin_amdgcn_sched_barrier(0);        // (in this order, which the waits in the loop go by)
        }
    }
    if constexpr (SPARSE) fill_lut(lut, t, 64 * WAVES);
    if (u0 < u1) {
        int left = a.group_units - (u0 - magic_div(u0, a.group_units, a.group_magic) * a.group_units);
#pragma unroll 1
        for (int i = u0; i < u1; i += DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const Unit& now = ring[d];
                if (i + d < u1) {
                    if (any_negative(now.s[0], now.s[1])) multiply(std::true_type{}, now);
                    else multiply(std::false_type{}, now);
                    if (--left == 0 || i + d == u1 - 1) {         // the end of a group or of the wave's part
                        left = a.group_units;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float A, B;
                            fold_factors<SPARSE>(now.s[j >> 1], now.z[j >> 1], j & 1, A, B);
                            if constexpr (!SPARSE) sum[j] = fmaf(B, acc_x[0], sum[j]);
                            sum[j] = fmaf(A, acc[j][0], sum[j]);
                        }
                        clear();
                    }
                }
                load(ring[d], min(i + d + DEPTH, u1 - 1));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    if (q == 0) *reinterpret_cast<f32x4*>(red + wave * 64 + 4 * n) = f32x4{sum[0], sum[1], sum[2], sum[3]};
    __syncthreads();
    auto total = [&](int c) __attribute__((always_inline)) {
        float s = red[c];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += red[w * 64 + c];
        return s;
    };
    if constexpr (UP) {
        if (t < 32) a.h[(int64_t)pair * half + 32 * strip + t] = (h16)silu_times(total(t), total(t + 32));
    } else {
        if (wave != 0) return;
        const int slot = pair - token * a.top_k;
        const __amdgpu_buffer_rsrc_t parts = buffer_of(a.part + ((int64_t)token * a.strips + strip) * a.top_k * 64, a.top_k * 256);
        const float v = valid ? a.weights[pair] * total(t) : 0.f;
        __builtin_amdgcn_raw_buffer_store_b32(bitcast<uint32_t>(v), parts, 256u * slot + 4u * t, 0, THROUGH);
        __builtin_amdgcn_s_waitcnt(0);                // every store of the wave has been acknowledged
        int arrived = 0;
        if (t == 0) arrived = __hip_atomic_fetch_add(a.arrivals + token * a.strips + strip, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (__builtin_amdgcn_readfirstlane(arrived) != a.top_k - 1) return;
        float s = 0.f;
        for (int j = 0; j < a.top_k; ++j) s += bitcast<float>(__builtin_amdgcn_raw_buffer_load_b32(parts, 256u * j + 4u * t, 0, THROUGH));
        a.outs[(int64_t)token * a.S + 64 * strip + t] = (h16)s;
    }
}

// outs[t, :] = sum over j of weights[t, j] part[place[t, j], :]; a thread takes four columns
__global__ __launch_bounds__(256) void combine_kernel(h16* outs, const float* part, const float* weights, const int* place, int top_k, int S, int parts) {
    constexpr int N = 4;
    const int64_t t = blockIdx.x / parts;
    const int c = ((int)(blockIdx.x % parts) * 256 + threadIdx.x) * N;
    if (c >= S) return;
    f32x4 sum = {};
#pragma unroll 4
    for (int j = 0; j < top_k; ++j) {
        const int p = place[t * top_k + j];
        if (p < 0) continue;
        const float w = weights[t * top_k + j];
        const f32x4 v = *reinterpret_cast<const f32x4*>(part + (int64_t)p * S + c);
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] += w * v[i];
    }
    h16x4 o;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = (h16)sum[i];
    *reinterpret_cast<h16x4*>(outs + t * S + c) = o;
}

// ---- which kernels, by the pairs of an expert if all are asked alike (the host does not know how they are shared out).
//
// A pair by itself: one token, or so few pairs that hardly two of them share an expert.
//
// Blocks of rows_kernel up to a mean of 48, then tiles.  us a call, blocks / tiles:
//   16 experts of 2048 x 1408, mean 32    int4 45 / 56     int3 46 / 58     int2 44 / 52     16:32 58 / 78
//                                   48         51 / 54          60 / 59          57 / 53           73 / 77
//                                   64         61 / 56          71 / 62          67 / 55           85 / 80
//   8 experts of 4096 x 11008,      40         256 / 317        293 / 340        267 / 294         349 / 420
//                                   48         276 / 319        309 / 340        280 / 295         364 / 420
//                                   64         335 / 323        381 / 346        341 / 302         446 / 433
//
// The height of the tiles, for each product: a tile of up to 64 / 96 / 128 / 192 / 256 rows takes 8 us and, on a full grid, 0.43 / 0.47 / 0.53 / 0.69 /
// 0.86 a K step; the tiles are those of experts that are asked unevenly, with a deviation of half the mean beside that of independent choices.
constexpr int BLOCKS_UP_TO = 48;
struct ExpertsPlan { bool single, tiles; int up, down; };          // up, down: heights of the tiles
static double tiles_us(double mean, int experts, int height, int64_t strips, int64_t steps) {
    // (the middles of eight equal parts of the normal distribution)
    const double parts[] = {-1.534, -0.887, -0.489, -0.157, 0.157, 0.489, 0.887, 1.534}, step[] = {0.43, 0.43, 0.47, 0.53, 0.69, 0.69, 0.86, 0.86};
    const double deviation = std::sqrt(mean + 0.25 * mean * mean);
    double us = 0, tiles = 0, longest = 0;
    for (double z : parts) {
        const int rows = std::max(1, (int)(mean + deviation * z)), full = rows / height, rest = rows % height;
        const double whole = 8.0 + steps * step[height / 32 - 1], last = rest ? 8.0 + steps * step[(rest - 1) / 32] : 0.0;
        us += full * whole + last;
        tiles += full + (rest > 0);
        longest = std::max(longest, full ? whole : last);
    }
    const double each = us / tiles, rounds = tiles / 8 * experts * strips / 256.0;
    // (near one round it may as well be two)
    return rounds <= 1 ? longest + std::max(0.0, rounds - 0.9) * 3 * each : rounds * each + 0.7 * longest;
}
static ExpertsPlan plan_experts(const int4mm_experts_shape& sh) {
    const int64_t pairs = sh.tokens * sh.top_k, K = sh.in_size, F = sh.width;
    const double mean = (double)pairs / sh.experts;
    ExpertsPlan p{pairs <= 64 && (sh.tokens == 1 || 2 * pairs <= sh.experts), mean > BLOCKS_UP_TO, 128, 128};
    if (p.single || !p.tiles) return p;
    // (`row`: of the second product, whose tiles address their rows with 31 bits; 64 rows of any width that check_experts admits)
    auto height = [&](int64_t strips, int64_t steps, int64_t row) {
        int best = 64;
        for (int h : {96, 128, 192, 256})
            if (2 * h * row < (int64_t)1 << 31 && tiles_us(mean, (int)sh.experts, h, strips, steps) < tiles_us(mean, (int)sh.experts, best, strips, steps)) best = h;
        return best;
    };
    p.up = height((F + 127) / 128, K / 32, 0);
    p.down = height((K + 255) / 256, F / 32, F);
    return p;
}

template <bool UP>
static void rows_product(int bits, ExpertsArgs a, int64_t pairs, hipStream_t st) {
    a.strips = a.S / 64;
    const dim3 grid((unsigned)(std::min<int64_t>(pairs, a.experts + pairs / ROWS_HEIGHT) * a.strips)), block(64 * ROWS_WAVES);
    if (a.mask) hipLaunchKernelGGL((rows_kernel<4, true, UP>), grid, block, 0, st, a);
    else if (bits == 4) hipLaunchKernelGGL((rows_kernel<4, false, UP>), grid, block, 0, st, a);
    else if (bits == 3) hipLaunchKernelGGL((rows_kernel<3, false, UP>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((rows_kernel<2, false, UP>), grid, block, 0, st, a);
}

template <bool UP>
static void token_product(int bits, ExpertsArgs a, int64_t pairs, hipStream_t st) {
    a.strips = a.S / 64;
    const dim3 grid((unsigned)(pairs * a.strips)), block(512);
    if (a.mask) hipLaunchKernelGGL((token_kernel<4, true, UP>), grid, block, 0, st, a);
    else if (bits == 4) hipLaunchKernelGGL((token_kernel<4, false, UP>), grid, block, 0, st, a);
    else if (bits == 3) hipLaunchKernelGGL((token_kernel<3, false, UP>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((token_kernel<2, false, UP>), grid, block, 0, st, a);
}

// work-items of the largest grid that a call of so few tokens launches
static int64_t work_items(const int4mm_experts_shape& sh) {
    const ExpertsPlan plan = plan_experts(sh);
    const int64_t pairs = sh.tokens * sh.top_k, E = sh.experts, K = sh.in_size, F = sh.width;
    if (plan.single) return pairs * (std::max(K, 2 * F) / 64) * 512;
    if (!plan.tiles) return std::min(pairs, E + pairs / ROWS_HEIGHT) * (std::max(K, 2 * F) / 64) * (64 * ROWS_WAVES);
    auto tiles = [&](int height, int64_t S) { return (std::min(pairs, E + pairs / height) * ((S + 255) / 256) + 7) * 512; };
    return std::max(tiles(plan.up, 2 * F), tiles(plan.down, K));
}

// Tokens that go through the launches at once, in even shares: their states are addressed with 31 bits, of many pairs (a quarter
// of a million fill the GPU many times over) not all need a workspace at the same time, and a grid has fewer than 2^32 work-items.
constexpr int64_t PAIRS_AT_ONCE = (int64_t)1 << 18, GRID_ITEMS = ((int64_t)1 << 32) - 4096;
static int64_t tokens_at_once(const int4mm_experts_shape& sh) {
    int64_t most = std::max<int64_t>(1, std::min((((int64_t)1 << 31) - 1) / (2 * sh.in_size), PAIRS_AT_ONCE / sh.top_k));
    // (the most that any number of pairs takes: blocks up to their mean, the lowest tiles, 64 pairs by themselves; a pair never takes
    // more than 512 work-items a strip)
    const int64_t E = sh.experts, strips = std::max(sh.in_size, 2 * sh.width) / 64;
    if ((E + std::min(PAIRS_AT_ONCE, BLOCKS_UP_TO * E) / ROWS_HEIGHT) * strips * (64 * ROWS_WAVES) > GRID_ITEMS ||
        (E + PAIRS_AT_ONCE / 64) * ((strips + 3) / 4) * 512 > GRID_ITEMS || 64 * strips * 512 > GRID_ITEMS)
        most = std::min(most, std::max<int64_t>(1, GRID_ITEMS / (strips * 512) / sh.top_k));
    const int64_t shares = (sh.tokens + most - 1) / most;
    return shares <= 1 ? sh.tokens : (sh.tokens + shares - 1) / shares;
}

static int check_experts(int bits, const int4mm_experts_shape* sh, bool sparse) {
    if (sh == nullptr) return INT4MM_ERR_NULL;
    if (bits != 4 && bits != 3 && bits != 2) return INT4MM_ERR_BITS;
    if (sparse && bits != 4) return INT4MM_ERR_SPARSE_BITS;
    const int64_t limit = (int64_t)1 << 31, K = sh->in_size, F = sh->width, g = sh->group_size;
    if (sh->tokens < 0 || sh->top_k < 1 || sh->experts < 1 || sh->experts > 4096 || K <= 0 || F <= 0 || K % 64 != 0 || F % 64 != 0) return INT4MM_ERR_SHAPE;
    if (g == 0 || (g > 0 && g % 64 != 0)) return INT4MM_ERR_GROUP;
    const int64_t up_groups = g < 0 ? 1 : (K + g - 1) / g, down_groups = g < 0 ? 1 : (F + g - 1) / g;
    if (sh->up_groups != up_groups || sh->down_groups != down_groups) return INT4MM_ERR_SHAPE;
    // (a matrix, and 64 rows, are addressed with 31 bits)
    if (K >= limit / 128 || F >= limit / 128 || K * F >= limit) return INT4MM_ERR_SHAPE;
    if (sh->top_k > 1024 || sh->tokens >= limit) return INT4MM_ERR_SHAPE;
    // (where even a token's grid is too large)
    if (tokens_at_once(*sh) == 1) {
        int4mm_experts_shape one = *sh;
        one.tokens = 1;
        if (work_items(one) > GRID_ITEMS) return INT4MM_ERR_SHAPE;
    }
    return INT4MM_OK;
}

struct ExpertsParts { size_t offsets, order, place, arrivals, h, part, total; };
static ExpertsParts experts_parts(const int4mm_experts_shape& sh) {
    const int64_t tokens = tokens_at_once(sh);
    const size_t pairs = (size_t)(tokens * sh.top_k);
    auto round = [](size_t n) { return (n + 255) & ~size_t(255); };
    ExpertsParts p;
    p.offsets = 0;
    p.order = p.offsets + round(4 * (size_t)(sh.experts + 1));
    p.place = p.order + round(4 * pairs);
    p.arrivals = p.place + round(4 * pairs);              // (pairs by themselves: up to 64 tokens, also as the last share of many)
    p.h = p.arrivals + round(4 * (size_t)(std::min<int64_t>(tokens, 64) * (sh.in_size / 64)));
    p.part = p.h + round(2 * pairs * (size_t)sh.width);
    p.total = p.part + round(4 * pairs * (size_t)sh.in_size);
    return p;
}

static int experts_share(int bits, bool sparse, h16* outs, const h16* x, const float* weights, const int* ids, const void* up_matrix,
                         const void* up_scales, const void* up_zeros, const void* up_mask, const void* down_matrix, const void* down_scales,
                         const void* down_zeros, const void* down_mask, const int4mm_experts_shape* sh, const ExpertsParts& parts, char* ws,
                         hipStream_t st) {
    const int64_t pairs = sh->tokens * sh->top_k, K = sh->in_size, F = sh->width;
    const int E = (int)sh->experts;
    int* const place = reinterpret_cast<int*>(ws + parts.place);
    ExpertsArgs a;
    a.offsets = reinterpret_cast<int*>(ws + parts.offsets);
    a.order = reinterpret_cast<int*>(ws + parts.order);
    a.h = reinterpret_cast<h16*>(ws + parts.h);
    a.part = reinterpret_cast<float*>(ws + parts.part);
    a.arrivals = reinterpret_cast<int*>(ws + parts.arrivals);
    a.experts = E;
    a.top_k = (int)sh->top_k;
    a.group_units = (int)(sh->group_size < 0 ? std::max(K, F) / 64 : std::min(sh->group_size, std::max(K, F) + 63) / 64);
    a.group_magic = div_magic((uint32_t)a.group_units);
    a.ids = ids;
    a.weights = weights;
    a.outs = outs;
    const ExpertsPlan plan = plan_experts(*sh);
    a.place = place;
    a.few_pairs = !plan.single && !plan.tiles && pairs <= FEW_PAIRS && E <= FEW_EXPERTS ? (int)pairs : 0;
    if (!plan.single && !a.few_pairs)
        hipLaunchKernelGGL(plan_kernel<false>, dim3(E), dim3(1024), 0, st, a.ids, const_cast<int*>(a.offsets), const_cast<int*>(a.order), place, (int)pairs, E);
    if (const int rc = check_launch("experts_forward")) return rc;
    auto rows_of = [&](int64_t k) { return sparse ? k / 16 : k * bits / 32; };
    a.x = x;
    a.matrix = static_cast<const uint32_t*>(up_matrix);
    a.mask = static_cast<const uint32_t*>(up_mask);
    a.scales = static_cast<const h16*>(up_scales);
    a.zeros = static_cast<const h16*>(up_zeros);
    a.K = (int)K;
    a.S = (int)(2 * F);
    a.matrix_stride = rows_of(K) * 2 * F;
    a.mask_stride = K / 32 * 2 * F;
    a.scale_stride = sh->up_groups * 2 * F;
    a.x_bytes = (uint32_t)(sh->tokens * K * 2);
    if (plan.single) token_product<true>(bits, a, pairs, st);
    else if (plan.tiles) launch_experts_tiles(bits, a, plan.up, pairs, true, st);
    else rows_product<true>(bits, a, pairs, st);
    if (const int rc = check_launch("experts_forward")) return rc;
    a.x = a.h;
    a.matrix = static_cast<const uint32_t*>(down_matrix);
    a.mask = static_cast<const uint32_t*>(down_mask);
    a.scales = static_cast<const h16*>(down_scales);
    a.zeros = static_cast<const h16*>(down_zeros);
    a.K = (int)F;
    a.S = (int)K;
    a.matrix_stride = rows_of(F) * K;
    a.mask_stride = F / 32 * K;
    a.scale_stride = sh->down_groups * K;
    if (plan.single) {
        token_product<false>(bits, a, pairs, st);
        return check_launch("experts_forward");
    }
    if (plan.tiles) launch_experts_tiles(bits, a, plan.down, pairs, false, st);
    else rows_product<false>(bits, a, pairs, st);
    if (const int rc = check_launch("experts_forward")) return rc;
    const int columns = (int)((K + 1023) / 1024);
    hipLaunchKernelGGL(combine_kernel, dim3((unsigned)(sh->tokens * columns)), dim3(256), 0, st, a.outs, a.part, a.weights, place, a.top_k, (int)K, columns);
    return check_launch("experts_forward");
}

}  // namespace i4

using namespace i4;

extern "C" {

size_t int4mm_experts_workspace_bytes(const int4mm_experts_shape* sh) {
    if (check_experts(4, sh, false) != INT4MM_OK || sh->tokens == 0) return 0;
    return experts_parts(*sh).total;
}

int int4mm_experts_forward(int bits, void* outs, const void* x, const void* weights, const void* ids, const void* up_matrix,
                           const void* up_scales, const void* up_zeros, const void* up_mask, const void* down_matrix,
                           const void* down_scales, const void* down_zeros, const void* down_mask, const int4mm_experts_shape* sh,
                           void* workspace, size_t workspace_bytes, void* stream) {
    const bool sparse = up_mask != nullptr || down_mask != nullptr;
    if (const int rc = check_experts(bits, sh, sparse)) return rc;
    if (sh->tokens == 0) return INT4MM_OK;
    if (!outs || !x || !weights || !ids || !up_matrix || !up_scales || !up_zeros || !down_matrix || !down_scales || !down_zeros ||
        (sparse && (!up_mask || !down_mask)))
        return INT4MM_ERR_NULL;
    const void* aligned[] = {outs, x, up_matrix, up_scales, up_zeros, up_mask, down_matrix, down_scales, down_zeros, down_mask, workspace};
    for (const void* ptr : aligned)
        if (reinterpret_cast<uintptr_t>(ptr) & 15) return INT4MM_ERR_ALIGN;
    if ((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(ids)) & 3) return INT4MM_ERR_ALIGN;
    const ExpertsParts parts = experts_parts(*sh);
    if (workspace == nullptr || workspace_bytes < parts.total) return INT4MM_ERR_WORKSPACE;
    const int64_t share = tokens_at_once(*sh), K = sh->in_size, k = sh->top_k;
    for (int64_t t = 0; t < sh->tokens; t += share) {
        int4mm_experts_shape part = *sh;
        part.tokens = std::min(share, sh->tokens - t);
        if (const int rc = experts_share(bits, sparse, static_cast<h16*>(outs) + t * K, static_cast<const h16*>(x) + t * K,
                                         static_cast<const float*>(weights) + t * k, static_cast<const int*>(ids) + t * k, up_matrix, up_scales,
                                         up_zeros, up_mask, down_matrix, down_scales, down_zeros, down_mask, &part, parts,
                                         static_cast<char*>(workspace), (hipStream_t)stream))
            return rc;
    }
    return INT4MM_OK;
}

}  // extern "C"
