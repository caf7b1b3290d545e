// The experts' products where an expert has many rows: the pipelined tile kernel's step loop (pipe.h) over tiles of up to 64 ... 256 of
// an expert's pairs and 256 columns.  The first product gathers its rows (a pair's token) on their way to LDS and ends with the
// activation, so that neither a gathered copy of x nor the gate's and the other half's results pass through memory; the second one
// takes the pairs as they lie.
//
// Weights are rounded to fp16 as int4mm_dequantize's are: sums of exact codes would need a group's sums beside the running ones, twice 128 of
// the 256 registers that a lane has.  A pair's result is stored in fp32, as those of rows_kernel are: its weight, which may be what brings it into
// fp16's range, comes after it.  (In fp16 calls took 2 - 12 % less, 16:32 experts gaining most, and a result beyond 65504 was lost.)
//
// What bounds it: large batches the beginnings and ends of tiles, 8 us beside 55 and 27 in the steps, and then the power limit (4096 tokens, eight of 64 experts
// of 2048 x 1024, int4: 336 and 214 us for 275 and 137 GFLOP, matrix pipe busy 49 and 35 %); few rows the chain of a step, 0.44 us whatever the height.  One
// height for all of a launch's blocks instead: 510 us a call where blocks of their own took 466.
#include "experts.h"

#include <algorithm>

namespace i4 {

template <int BITS, bool SPARSE, int TM, bool GATED>
__device__ __forceinline__ void tile_of_height(const ExpertsArgs& a, const MatmulArgs& m, int first, int s0, h16* const (&As)[A_STAGES], h16* Bs, uint32_t* lut) {
    if constexpr (GATED)
        pipe_tile<BITS, SPARSE, TM, 4, true, false, true>(m, 0, s0, a.x, a.h + (int64_t)first * (a.S / 2), As, Bs, lut, 0, 0, 1,
                                                          GatedRows{a.order + first, a.top_k, a.S / 2, a.x_bytes});
    else
        pipe_tile<BITS, SPARSE, TM, 4, true, false, false, float>(m, 0, s0, a.x + (int64_t)first * a.K, a.part + (int64_t)first * a.S, As, Bs, lut, 0, 0, 1);
}

// A block of fewer rows than the launch's height takes the lowest tile that holds it, so that what is computed beyond an expert's last
// row is less than 64 rows of it.
template <int BITS, bool SPARSE, bool GATED>
__global__ __launch_bounds__(512, 1) void experts_tile_kernel(ExpertsArgs a) {
    constexpr int BN = 256, A_HALVES = 256 * PK;
    __shared__ __attribute__((aligned(16))) h16 A0[A_HALVES], A1[A_HALVES], A2[A_HALVES], A3[A_HALVES], A4[A_HALVES], A5[A_HALVES];
    __shared__ __attribute__((aligned(16))) h16 Bs[P_STAGES * PK * BN];
    __shared__ __attribute__((aligned(16))) uint32_t Lut[SPARSE ? SPARSE_LUT_WORDS : 4];
    const int lane = threadIdx.x & 63;
    // workgroups go round the 8 XCDs: each takes a range of the tiles, an expert's side by side
    Block b;
    const int blocks = find_block(a.offsets, a.experts, a.height, INT32_MAX, lane, b);
    const int total = blocks * a.strips, per_xcd = (total + 7) / 8;
    const int local = blockIdx.x / 8, tile = blockIdx.x % 8 * per_xcd + local;
    if (local >= per_xcd || tile >= total) return;
    find_block(a.offsets, a.experts, a.height, tile / a.strips, lane, b);

    MatmulArgs m = {};
    m.M = b.count;
    m.K = a.K;
    m.S = a.S;
    m.group_units = a.group_units;
    m.matrix = a.matrix + b.expert * a.matrix_stride;
    m.mask = SPARSE ? a.mask + b.expert * a.mask_stride : nullptr;
    m.scales = a.scales + b.expert * a.scale_stride;
    m.zeros = a.zeros + b.expert * a.scale_stride;
    h16* const As[A_STAGES] = {A0, A1, A2, A3, A4, A5};
    const int s0 = tile % a.strips * BN;
    if (b.count <= 64) tile_of_height<BITS, SPARSE, 2, GATED>(a, m, b.first, s0, As, Bs, Lut);
    else if (b.count <= 96) tile_of_height<BITS, SPARSE, 3, GATED>(a, m, b.first, s0, As, Bs, Lut);
    else if (b.count <= 128) tile_of_height<BITS, SPARSE, 4, GATED>(a, m, b.first, s0, As, Bs, Lut);
    else if (b.count <= 192) tile_of_height<BITS, SPARSE, 6, GATED>(a, m, b.first, s0, As, Bs, Lut);
    else tile_of_height<BITS, SPARSE, 8, GATED>(a, m, b.first, s0, As, Bs, Lut);
}

void launch_experts_tiles(int bits, ExpertsArgs a, int height, int64_t pairs, bool gated, hipStream_t st) {
    a.strips = (a.S + 255) / 256;
    a.height = height;
    const int64_t blocks = std::min<int64_t>(pairs, a.experts + pairs / height);
    const dim3 grid((unsigned)((blocks * a.strips + 7) / 8 * 8));
#define LAUNCH(BITS, SPARSE)                                                                                          \
    if (gated) hipLaunchKernelGGL((experts_tile_kernel<BITS, SPARSE, true>), grid, dim3(512), 0, st, a);              \
    else hipLaunchKernelGGL((experts_tile_kernel<BITS, SPARSE, false>), grid, dim3(512), 0, st, a)
    if (a.mask) { LAUNCH(4, true); }
    else if (bits == 4) { LAUNCH(4, false); }
    else if (bits == 3) { LAUNCH(3, false); }
    else { LAUNCH(2, false); }
#undef LAUNCH
}

}  // namespace i4
