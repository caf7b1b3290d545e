// Low-rank adapters of many requests beside a shared projection:
//     outs[t, :] = fp16( base[t, :] + scales[a] * (x[t, :] down[a]^T) up[a] ),   a = ids[t / rows_per_id]
// with down [n, r, K] and up [n, r, S] in fp16; a row whose id is outside 0 ... n - 1 has no adapter and keeps its base.
//
// Two launches.  shrink_kernel: h[t, :] = x[t, :] down[a]^T, a share of K per workgroup, fp32 partial sums to the workspace.
// expand_kernel: adds the shares up, scales, and adds h up[a] onto base.  Both take tiles of neighbouring rows and go through the
// DISTINCT adapters of a tile: one or two where rows come as prompts, up to all different where every row is a request's token.
// No sorting by adapter is needed, and what an adapter's weights hold reaches no row of another adapter (its products are
// formed for all rows of a tile and selected, not masked by a 0 that an infinity would turn into NaN).
//
// h is split into two halves of 11 bits each, after scaling its row by a power of two to 512 ... 1024, so that nothing overflows
// and 22 bits of it are multiplied: both products are on v_mfma_f32_16x16x32_f16, which are few beside the memory traffic.
#include "common.h"

#include <algorithm>
#include <climits>

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
    int deal;                                         // workgroup z takes every deal-th of a tile's distinct adapters
    int columns;                                      // expand: columns per workgroup
};

template <int CTRL>
__device__ __forceinline__ int dpp_min(int v) {
    return min(v, __builtin_amdgcn_update_dpp(INT_MAX, v, CTRL, 0xF, 0xF, false));
}
// the smallest of the values in a row of 16 lanes, the same in all rows
__device__ __forceinline__ int row_min(int v) {
    v = dpp_min<0xB1>(v);
    v = dpp_min<0x4E>(v);
    v = dpp_min<0x141>(v);
    v = dpp_min<0x140>(v);
    return __builtin_amdgcn_readfirstlane(v);
}

// (rows < 2^22: check_adapters)
__device__ __forceinline__ int id_of(const AdapterArgs& a, int64_t row) { return magic_div((int)row, a.rows_per_id, a.id_magic); }

// ids of the tile's rows: lane l holds those of rows l % 16 + 16 m; -1: no adapter
template <int MT>
__device__ __forceinline__ void tile_ids(int (&id)[MT], const AdapterArgs& a, int64_t row0, int lane) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int64_t row = row0 + 16 * m + (lane & 15);
        int v = row < a.rows ? a.ids[id_of(a, row)] : -1;
        id[m] = v >= 0 && v < a.adapters ? v : -1;
    }
}
// the smallest id above `last` in the tile (INT_MAX: none)
template <int MT>
__device__ __forceinline__ int next_id(const int (&id)[MT], int last) {
    int v = INT_MAX;
#pragma unroll
    for (int m = 0; m < MT; ++m) v = min(v, id[m] > last ? id[m] : INT_MAX);
    return row_min(v);
}

// 16 MT rows, 16 NT ranks from rank0 = 16 NT blockIdx.z', a share of K; the four waves share it out by units of 64 k
template <int MT, int NT>
__global__ __launch_bounds__(256) void shrink_kernel(AdapterArgs a) {
    __shared__ __attribute__((aligned(16))) float red[4 * 16 * MT * 16 * NT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, q = lane >> 4;
    const int64_t row0 = (int64_t)blockIdx.y * (16 * MT);
    const int deal = blockIdx.z % a.deal, rank0 = blockIdx.z / a.deal * (16 * NT);
    const int units = a.K / 64, u0 = blockIdx.x * a.units_per_split, u1 = min(u0 + a.units_per_split, units);
    const uint32_t pitch = 2u * (uint32_t)a.K;
    int id[MT];
    tile_ids<MT>(id, a, row0, lane);
    const int rows_here = (int)min((int64_t)(16 * MT), a.rows - row0), ranks_here = min(16 * NT, a.rank - rank0);
    const __amdgpu_buffer_rsrc_t x_rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<h16*>(a.x) + row0 * a.K, 0, (int)(rows_here * pitch), AD_RSRC);
    // lane group q takes k = 16 q ... 16 q + 15 of a unit in two steps: 128 bytes of a row per step pair
    const uint32_t at = (uint32_t)n * pitch + 32u * q;

    int last = -1;
    for (int index = 0;; ++index) {
        const int cur = next_id<MT>(id, last);
        if (cur == INT_MAX) break;
        last = cur;
        if (index % a.deal != deal) continue;
        const __amdgpu_buffer_rsrc_t w_rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<h16*>(a.down) + ((int64_t)cur * a.rank + rank0) * a.K, 0, (int)(ranks_here * pitch), AD_RSRC);
        uint32_t xo[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) xo[m] = (at + 16u * m * pitch) | (id[m] == cur ? 0u : AD_BEYOND);
        f32x4 acc[MT][NT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
        for (int u = u0 + wave; u < u1; u += 4) {
            u32x4 xv[2][MT], wv[2][NT];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int m = 0; m < MT; ++m) xv[s][m] = __builtin_amdgcn_raw_buffer_load_b128(x_rsrc, xo[m], 128u * u + 16u * s, 0);
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    wv[s][t] = __builtin_amdgcn_raw_buffer_load_b128(w_rsrc, at + 16u * t * pitch, 128u * u + 16u * s, 0);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s)
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
            const int64_t at_row = row0 + row;
            if (at_row < a.rows && rank < ranks_here && a.ids[id_of(a, at_row)] == cur)
                a.part[((int64_t)blockIdx.x * a.rows + at_row) * a.rank + rank0 + rank] = sum;
        }
        __syncthreads();
    }
}

// 16 MT rows, `columns` columns: four waves of 64 columns at a time
template <int MT>
__global__ __launch_bounds__(256) void expand_kernel(AdapterArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, q = lane >> 4;
    const int64_t row0 = (int64_t)blockIdx.y * (16 * MT);
    const int deal = blockIdx.z;
    const int chunks = (a.rank + 31) / 32, pitch = chunks * 32 + 8;        // halves between the rows of h in LDS
    h16* const high = reinterpret_cast<h16*>(lds);
    h16* const low = high + 16 * MT * pitch;
    float* const unscale = reinterpret_cast<float*>(low + 16 * MT * pitch);
    int id[MT];
    tile_ids<MT>(id, a, row0, lane);

    // ---- h of the tile's rows: a wave takes a row at a time
    for (int row = wave; row < 16 * MT; row += 4) {
        const int64_t at_row = row0 + row;
        const int of = at_row < a.rows ? a.ids[id_of(a, at_row)] : -1;
        const bool there = of >= 0 && of < a.adapters;
        const float scale = there ? a.scales[of] : 0.f;
        float most = 0.f;
        float h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            h[i] = 0.f;
            if (64 * i < a.rank) {
                const int rank = 64 * i + lane;
                if (there && rank < a.rank) {
                    float sum = 0.f;
                    for (int ks = 0; ks < a.ksplit; ++ks) sum += a.part[((int64_t)ks * a.rows + at_row) * a.rank + rank];
                    h[i] = sum * scale;
                }
                most = fmaxf(most, fabsf(h[i]));
            }
        }
#pragma unroll
        for (int d = 1; d < WAVE; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
        // most = f 2^e, f in [0.5, 1): times 2^(10 - e)
        int e = 10;
        if (most > 0.f && most < INFINITY) e = __builtin_amdgcn_frexp_expf(most);
        e = max(e, -100);
        const float by = __builtin_ldexpf(1.f, 10 - e);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int rank = 64 * i + lane;
            if (64 * i < a.rank && rank < chunks * 32) {
                const float v = h[i] * by;
                const h16 hi = (h16)v;
                // (an infinity or NaN is in the high part alone)
                const float rest = fabsf(v) < 65504.f ? v - (float)hi : 0.f;
                high[row * pitch + rank] = hi;
                low[row * pitch + rank] = (h16)rest;
            }
        }
        if (lane == 0) unscale[row] = __builtin_ldexpf(1.f, e - 10);
    }
    __syncthreads();

    const uint32_t row_bytes = 2u * (uint32_t)a.S;
    const int c_end = min((int)(blockIdx.x + 1) * a.columns, a.S);
    for (int c = blockIdx.x * a.columns + 64 * wave; c < c_end; c += 256) {
        // tile j takes columns 4 n + j of the wave's 64
        f32x4 sum[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        uint32_t mine = 0;                            // bit 4 m + r: row 16 m + 4 q + r is written here
        int last = -1;
        for (int index = 0;; ++index) {
            const int cur = next_id<MT>(id, last);
            if (cur == INT_MAX) break;
            last = cur;
            if (index % a.deal != deal) continue;
            const __amdgpu_buffer_rsrc_t w_rsrc = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<h16*>(a.up) + (int64_t)cur * a.rank * a.S + c, 0, (int)((a.rank - 1) * row_bytes + 128u), AD_RSRC);
            f32x4 acc[MT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int ch = 0; ch < chunks; ++ch) {
                // ranks 32 ch + 8 q ... + 7 of columns 4 n ... 4 n + 3, turned so that a register holds two ranks of a column
                u32x2 w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    w[i] = __builtin_amdgcn_raw_buffer_load_b64(w_rsrc, (uint32_t)(32 * ch + 8 * q + i) * row_bytes + 8u * n, 0, 0);
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
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool of_cur = __shfl(id[m], 4 * q + r) == cur;
                    mine |= of_cur ? 1u << (4 * m + r) : 0u;
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[m][j][r] = of_cur ? acc[m][j][r] : sum[m][j][r];
                }
        }
        // rows without an adapter are the first workgroup's
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool idle = __shfl(id[m], 4 * q + r) < 0;
                const int row = 16 * m + 4 * q + r;
                if (row0 + row < a.rows && (idle ? deal == 0 : (mine >> (4 * m + r)) & 1)) {
                    const int64_t at = (row0 + row) * a.S + c + 4 * n;
                    const h16x4 v = *reinterpret_cast<const h16x4*>(a.base + at);
                    const float by = unscale[row];
                    h16x4 o;
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[j] = idle ? v[j] : (h16)((float)v[j] + sum[m][j][r] * by);
                    *reinterpret_cast<h16x4*>(a.outs + at) = o;
                }
            }
    }
}

struct AdapterPlan { int shrink_mt, nt, ksplit, units_per_split, expand_mt, columns, deal_shrink, deal_expand; };

static AdapterPlan plan_adapters(const int4mm_adapter_shape& sh) {
    AdapterPlan p;
    const int64_t T = sh.rows, units = sh.in_size / 64;
    p.nt = sh.rank <= 16 ? 1 : sh.rank <= 32 ? 2 : 4;
    p.shrink_mt = T <= 256 ? 1 : 2;
    p.expand_mt = T <= 256 ? 1 : 4;
    const bool many = T <= 256;
    p.deal_shrink = many ? (int)std::min<int64_t>(16, std::min<int64_t>(T, sh.adapters)) : 1;
    p.deal_expand = p.deal_shrink;
    const int64_t tiles = (T + 16 * p.shrink_mt - 1) / (16 * p.shrink_mt) * ((sh.rank + 16 * p.nt - 1) / (16 * p.nt));
    const int64_t want = std::max<int64_t>(1, 1024 / (many ? T : tiles));
    p.units_per_split = (int)std::max<int64_t>(8, (units + want - 1) / want);
    p.ksplit = (int)((units + p.units_per_split - 1) / p.units_per_split);
    p.columns = 256 * (T <= 256 ? 1 : 4);
    return p;
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
    return (size_t)plan_adapters(*sh).ksplit * sh->rows * sh->rank * 4;
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
    if (workspace == nullptr || workspace_bytes < int4mm_adapters_workspace_bytes(sh)) return INT4MM_ERR_WORKSPACE;
    const AdapterPlan p = plan_adapters(*sh);
    AdapterArgs a;
    a.outs = static_cast<h16*>(outs);
    a.base = static_cast<const h16*>(base);
    a.x = static_cast<const h16*>(x);
    a.down = static_cast<const h16*>(down);
    a.up = static_cast<const h16*>(up);
    a.scales = static_cast<const float*>(scales);
    a.ids = static_cast<const int*>(ids);
    a.part = static_cast<float*>(workspace);
    a.rows = sh->rows;
    a.rows_per_id = (int)std::min(sh->rows_per_id, sh->rows);
    a.id_magic = div_magic((uint32_t)a.rows_per_id);
    a.adapters = (int)sh->adapters;
    a.rank = (int)sh->rank;
    a.K = (int)sh->in_size;
    a.S = (int)sh->out_size;
    a.ksplit = p.ksplit;
    a.units_per_split = p.units_per_split;
    a.columns = p.columns;
    hipStream_t st = (hipStream_t)stream;
    {
        a.deal = p.deal_shrink;
        const dim3 grid(p.ksplit, (unsigned)((sh->rows + 16 * p.shrink_mt - 1) / (16 * p.shrink_mt)),
                        (unsigned)(p.deal_shrink * ((sh->rank + 16 * p.nt - 1) / (16 * p.nt))));
#define SHRINK(MT, NT) hipLaunchKernelGGL((shrink_kernel<MT, NT>), grid, dim3(256), 0, st, a)
        if (p.shrink_mt == 1) {
            if (p.nt == 1) SHRINK(1, 1); else if (p.nt == 2) SHRINK(1, 2); else SHRINK(1, 4);
        } else {
            if (p.nt == 1) SHRINK(2, 1); else if (p.nt == 2) SHRINK(2, 2); else SHRINK(2, 4);
        }
#undef SHRINK
        if (const int rc = check_launch("low_rank_add")) return rc;
    }
    a.deal = p.deal_expand;
    const int height = 16 * p.expand_mt;
    const dim3 grid((unsigned)((sh->out_size + p.columns - 1) / p.columns), (unsigned)((sh->rows + height - 1) / height), (unsigned)p.deal_expand);
    const size_t lds = (size_t)height * (((sh->rank + 31) / 32 * 32 + 8) * 4 + 4);
    if (p.expand_mt == 1) hipLaunchKernelGGL((expand_kernel<1>), grid, dim3(256), lds, st, a);
    else hipLaunchKernelGGL((expand_kernel<4>), grid, dim3(256), lds, st, a);
    return check_launch("low_rank_add");
}

}  // extern "C"
