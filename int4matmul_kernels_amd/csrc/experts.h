// What the experts' kernels share: their arguments, and which expert's pairs (or adapter's rows) a block of a grid takes.
#pragma once

#include "pipe.h"

namespace i4 {

struct ExpertsArgs {
    const h16* x;                  // source rows
    const uint32_t* matrix;
    const uint32_t* mask;
    const h16* scales;
    const h16* zeros;
    const int* offsets;            // [E + 1]: an expert's pairs among the ordered ones
    const int* order;              // [P]: pair of each place
    h16* h;                        // up: [P, F] by place
    float* part;                   // down: [P, S] by place
    const int* ids;
    const float* weights;
    h16* outs;
    int* place;                    // [P]: place of each pair, -1 without an expert
    int few_pairs;                 // rows_kernel, up: the pairs, where it orders them itself, else 0
    int* arrivals;                 // pairs by themselves: [tokens, strips] workgroups that have stored their sums
    int64_t matrix_stride, mask_stride, scale_stride;   // elements from an expert to the next
    int experts, top_k, K, S;      // S: columns of the matrix (up: 2 F)
    int group_units, strips;       // strips: of columns
    int height;                    // of the tiles
    uint32_t group_magic;
    uint32_t x_bytes;              // up: of all source rows
};

// Blocks of up to `height` pairs of one expert, in the order of the experts.  `expert`, `first` and `count` of block `want`;
// returns the number of blocks if there are no more than `want` of them, else -1.
struct Block { int expert, first, count; };
__device__ __forceinline__ int find_block(const int* offsets, int experts, int height, int want, int lane, Block& b) {
    int before = 0;
    for (int e0 = 0; e0 < experts; e0 += 64) {
        const int e = e0 + lane;
        const int from = offsets[min(e, experts)], to = offsets[min(e + 1, experts)];
        const int blocks = (to - from + height - 1) / height;
        int upto = blocks;                            // of this lane's and the lower lanes' experts
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(upto, d);
            upto += lane >= d ? o : 0;
        }
        const uint64_t beyond = __builtin_amdgcn_ballot_w64(before + upto > want);
        if (beyond) {
            const int l = __builtin_ctzll(beyond);
            const int nth = want - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(blocks, l));
            const int lo = __builtin_amdgcn_readlane(from, l), hi = __builtin_amdgcn_readlane(to, l);
            b.expert = e0 + l;
            b.first = lo + nth * height;
            b.count = min(height, hi - b.first);
            return -1;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return before;
}

// experts.hip: rows in the order of their ids, stable, an id outside 0 ... buckets - 2 in the last bucket; offsets [buckets + 1]
void launch_rows_by_id(const int* ids, int* offsets, int* order, int rows, int buckets, hipStream_t st);

// experts_tiles.hip: both products in tiles of up to `height` (64, 96, 128, 192 or 256) rows and 256 columns
void launch_experts_tiles(int bits, ExpertsArgs a, int height, int64_t pairs, bool gated, hipStream_t st);

}  // namespace i4
