// The experts' products where an expert has many rows: the pipelined tile kernel's step loop (pipe.h) over tiles of up to 32 TM of
// an expert's pairs and 256 columns.  The first product gathers its rows (a pair's token) on their way to LDS and ends with the
// activation, so that neither a gathered copy of x nor the gate's and the other half's results pass through memory; the second one
// takes the pairs as they lie.
#include "experts.h"

#include <algorithm>

namespace i4 {

template <int BITS, bool SPARSE, int TM, bool GATED>
__global__ __launch_bounds__(512, 1) void experts_tile_kernel(ExpertsArgs a) {
    constexpr int NW = 4, BM = TM * 32, BN = NW * 64, A_ROWS = NW * 32;
    constexpr int A_HALVES = (BM + A_ROWS - 1) / A_ROWS * A_ROWS * PK;
    __shared__ __attribute__((aligned(16))) h16 A0[A_HALVES], A1[A_HALVES], A2[A_HALVES], A3[A_HALVES], A4[A_HALVES], A5[A_HALVES];
    __shared__ __attribute__((aligned(16))) h16 Bs[P_STAGES * PK * BN];
    __shared__ __attribute__((aligned(16))) uint32_t Lut[SPARSE ? SPARSE_LUT_WORDS : 4];
    const int lane = threadIdx.x & 63;
    // workgroups go round the 8 XCDs: each takes a range of the tiles, an expert's side by side
    Block b;
    const int blocks = find_block(a.offsets, a.experts, BM, INT32_MAX, lane, b);
    const int total = blocks * a.strips, per_xcd = (total + 7) / 8;
    const int local = blockIdx.x / 8, tile = blockIdx.x % 8 * per_xcd + local;
    if (local >= per_xcd || tile >= total) return;
    find_block(a.offsets, a.experts, BM, tile / a.strips, lane, b);

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
    if constexpr (GATED)
        pipe_tile<BITS, SPARSE, TM, NW, true, false, true>(m, 0, s0, a.x, a.h + (int64_t)b.first * (a.S / 2), As, Bs, Lut, 0, 0, 1,
                                                           GatedRows{a.order + b.first, a.top_k, a.S / 2, a.x_bytes});
    else
        pipe_tile<BITS, SPARSE, TM, NW, true, false>(m, 0, s0, a.x + (int64_t)b.first * a.K, a.h + (int64_t)b.first * a.S, As, Bs, Lut, 0, 0, 1);
}

template <int BITS, bool SPARSE, bool GATED>
static void launch_height(ExpertsArgs a, int tm, int64_t pairs, hipStream_t st) {
    a.strips = (a.S + 255) / 256;
    const int64_t blocks = std::min<int64_t>(pairs, a.experts + pairs / (32 * tm));
    const dim3 grid((unsigned)((blocks * a.strips + 7) / 8 * 8));
    if (tm == 2) hipLaunchKernelGGL((experts_tile_kernel<BITS, SPARSE, 2, GATED>), grid, dim3(512), 0, st, a);
    else if (tm == 3) hipLaunchKernelGGL((experts_tile_kernel<BITS, SPARSE, 3, GATED>), grid, dim3(512), 0, st, a);
    else if (tm == 6) hipLaunchKernelGGL((experts_tile_kernel<BITS, SPARSE, 6, GATED>), grid, dim3(512), 0, st, a);
    else if (tm == 4) hipLaunchKernelGGL((experts_tile_kernel<BITS, SPARSE, 4, GATED>), grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((experts_tile_kernel<BITS, SPARSE, 8, GATED>), grid, dim3(512), 0, st, a);
}

void launch_experts_tiles(int bits, const ExpertsArgs& a, int tm, int64_t pairs, bool gated, hipStream_t st) {
#define FORMAT(BITS, SPARSE) (gated ? launch_height<BITS, SPARSE, true>(a, tm, pairs, st) : launch_height<BITS, SPARSE, false>(a, tm, pairs, st))
    if (a.mask) FORMAT(4, true);
    else if (bits == 4) FORMAT(4, false);
    else if (bits == 3) FORMAT(3, false);
    else FORMAT(2, false);
#undef FORMAT
}

}  // namespace i4
