// Routing to experts: of every token's row of logits the k experts it goes to, and their weights.
//
//   p_e   = exp(l_e - max l) / sum over e of the same, or 1 / (1 + exp(-l_e));   a logit of -inf or NaN: the expert is out
//   key_e = l_e without a bias (the order of p, and logits that tie, tie exactly), p_e + b_e with one (NaN, -inf: out)
//   groups of E / G experts: score = the group's best key or the sum of its two best p (+ b); the best groups stay
//   the k best keys of what stays, ties to the lowest index; weight = p, over the sum of the k if asked for, times `scale`
//
// p, keys, scores and sums are held in 64 bits: which expert comes last can hang on a difference that 32 bits lose, and the
// weights are rounded once, at the end.  A wave takes a token; lane i holds experts i EPL ... i EPL + EPL - 1, so that of lanes
// with equal keys the lowest is the lowest index.  A choice is a maximum over the wave (four DPP steps, then scalar), a ballot
// and a lane read; keys are unsigned integers in the numbers' order, 0 for an expert that is out.
#include "common.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace i4 {

struct RouteArgs {
    float* weights;
    int* ids;
    const float* bias;
    int64_t tokens;
    double scale;
    int experts, top_k, groups, topk_groups, group_size, lanes_per_group;
    uint32_t group_magic;
    int softmax, top2, renormalize;
};

__device__ __forceinline__ uint32_t ordered(float f) {
    const uint32_t u = bitcast<uint32_t>(f + 0.0f);               // (-0 ties with 0)
    return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ uint64_t ordered(double f) {
    const uint64_t u = bitcast<uint64_t>(f + 0.0);
    return u ^ ((u >> 63) ? ~0ull : 1ull << 63);
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = dpp_max<0xB1>(v);     // quad_perm [1,0,3,2]
    v = dpp_max<0x4E>(v);     // quad_perm [2,3,0,1]
    v = dpp_max<0x141>(v);    // row_half_mirror
    v = dpp_max<0x140>(v);    // row_mirror
    const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
    const uint32_t c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
    return max(max(a, b), max(c, d));
}
// the lanes that hold the wave's largest key; 0 if that is 0
__device__ __forceinline__ uint64_t holders_of_max(uint32_t key) {
    const uint32_t m = wave_max(key);
    return m ? __builtin_amdgcn_ballot_w64(key == m) : 0;
}
__device__ __forceinline__ uint64_t holders_of_max(uint64_t key) {
    const uint32_t hi = (uint32_t)(key >> 32), lo = (uint32_t)key, m = wave_max(hi);
    if (m == 0) return 0;                                          // (an ordered number other than "out" has a high word)
    const uint64_t in = __builtin_amdgcn_ballot_w64(hi == m);
    if ((in & (in - 1)) == 0) return in;
    const uint32_t l = wave_max(hi == m ? lo : 0u);
    return __builtin_amdgcn_ballot_w64(hi == m && lo == l);
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) v += __shfl_xor(v, d);
    return v;
}

template <int EPL, bool BIAS, typename L>
__global__ __launch_bounds__(256) void route_kernel(const L* logits, RouteArgs a) {
    extern __shared__ double shown_all[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int64_t wanted = (int64_t)blockIdx.x * waves + wave, token = wanted < a.tokens ? wanted : a.tokens - 1;
    const L* const row = logits + token * a.experts;
    const int first = lane * EPL;

    float l[EPL];
    uint32_t top_key = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        l[i] = first + i < a.experts ? (float)row[first + i] : -INFINITY;
        if (!(l[i] > -INFINITY)) l[i] = -INFINITY;                // (NaN: out)
        top_key = max(top_key, ordered(l[i]));
    }
    // the largest logit, from its key
    const uint32_t top_bits = wave_max(top_key);
    const double top = (double)bitcast<float>(top_bits ^ ((top_bits >> 31) ? 0x80000000u : 0xFFFFFFFFu));
    // (at +inf the largest logits share p, by the limit)
    auto above_top = [&](double x) { return x == top ? 1.0 : exp(x - top); };

    double p[EPL], total = 1.0;
    const bool grouped = a.groups > 1;
    if (a.softmax) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            p[i] = l[i] > -INFINITY ? above_top((double)l[i]) : 0.0;
            sum += p[i];
        }
        total = wave_sum(sum);
        if (BIAS || (grouped && a.top2)) {
#pragma unroll
            for (int i = 0; i < EPL; ++i) p[i] /= total;
        }
    } else if (BIAS || (grouped && a.top2)) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) p[i] = 1.0 / (1.0 + exp(-(double)l[i]));
    }

    using Key = std::conditional_t<BIAS, uint64_t, uint32_t>;
    Key key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        if constexpr (BIAS) {
            const double v = p[i] + (first + i < a.experts ? (double)a.bias[first + i] : 0.0);
            key[i] = l[i] > -INFINITY && v > -INFINITY ? ordered(v) : 0;
            p[i] = v;
        } else {
            key[i] = l[i] > -INFINITY ? ordered(l[i]) : 0;
        }
    }

    if (grouped) {
        // scores: the lanes of a group read its members, keep their two best and merge them
        double* const shown = shown_all + wave * a.experts;
#pragma unroll
        for (int i = 0; i < EPL; ++i)
            if (first + i < a.experts) shown[first + i] = key[i] == 0 ? -INFINITY : BIAS || a.top2 ? p[i] : (double)l[i];
        __syncthreads();
        const int lpg = a.lanes_per_group, g = lane / lpg, sub = lane % lpg;
        double best = -INFINITY, second = -INFINITY;
        if (g < a.groups) {
            for (int m = sub; m < a.group_size; m += lpg) {
                const double v = shown[g * a.group_size + m];
                second = fmax(second, fmin(best, v));
                best = fmax(best, v);
            }
        }
        for (int d = 1; d < lpg; d *= 2) {
            const double ob = __shfl_xor(best, d), os = __shfl_xor(second, d);
            second = fmax(fmax(second, os), fmin(best, ob));
            best = fmax(best, ob);
        }
        const double score = a.top2 && second > -INFINITY ? best + second : best;
        uint64_t score_key = sub == 0 && g < a.groups && best > -INFINITY ? ordered(score) : 0;
        uint64_t kept = 0;                                         // a bit per group
        for (int j = 0; j < a.topk_groups; ++j) {
            const uint64_t in = holders_of_max(score_key);
            if (in == 0) break;
            const int winner = __builtin_ctzll(in);
            kept |= 1ull << (winner / lpg);
            if (lane == winner) score_key = 0;
        }
#pragma unroll
        for (int i = 0; i < EPL; ++i)
            if (!((kept >> (magic_div(first + i, a.group_size, a.group_magic) & 63)) & 1)) key[i] = 0;
    }

    int mine = -1;
    for (int j = 0; j < a.top_k; ++j) {
        Key best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < EPL; ++i) {
            const bool more = key[i] > best;
            best = more ? key[i] : best;
            at = more ? i : at;
        }
        const uint64_t in = holders_of_max(best);
        if (in == 0) break;
        const int winner = __builtin_ctzll(in);
        const int which = __builtin_amdgcn_readlane(at, winner);
        if (lane == j) mine = winner * EPL + which;
#pragma unroll
        for (int i = 0; i < EPL; ++i)
            if (lane == winner && i == which) key[i] = 0;
    }

    double w = 0.0;
    if (mine >= 0) {
        const double x = (double)(float)row[mine];
        w = a.softmax ? above_top(x) / total : 1.0 / (1.0 + exp(-x));
    }
    if (a.renormalize) {
        const double sum = wave_sum(w);
        if (sum > 0.0) w /= sum;
    }
    if (wanted < a.tokens && lane < a.top_k) {
        a.weights[token * a.top_k + lane] = (float)(w * a.scale);
        a.ids[token * a.top_k + lane] = mine;
    }
}

constexpr int64_t ROUTE_AT_ONCE = (int64_t)1 << 25;      // tokens of a launch: a grid has fewer than 2^32 work-items, 64 for a token

template <bool BIAS, typename L>
static int launch_route(const L* logits, RouteArgs a, hipStream_t st) {
    for (int64_t left = a.tokens; left > 0; left -= ROUTE_AT_ONCE) {
        a.tokens = std::min(left, ROUTE_AT_ONCE);
        // one wave a workgroup where that still leaves CUs without one, else four
        const int waves = a.tokens <= 512 ? 1 : 4;
        const dim3 grid((unsigned)((a.tokens + waves - 1) / waves)), block(64 * waves);
        const size_t lds = a.groups > 1 ? (size_t)waves * a.experts * sizeof(double) : 0;
        const int epl = (a.experts + 63) / 64;
        if (epl <= 1) hipLaunchKernelGGL((route_kernel<1, BIAS, L>), grid, block, lds, st, logits, a);
        else if (epl <= 2) hipLaunchKernelGGL((route_kernel<2, BIAS, L>), grid, block, lds, st, logits, a);
        else if (epl <= 4) hipLaunchKernelGGL((route_kernel<4, BIAS, L>), grid, block, lds, st, logits, a);
        else if (epl <= 8) hipLaunchKernelGGL((route_kernel<8, BIAS, L>), grid, block, lds, st, logits, a);
        else hipLaunchKernelGGL((route_kernel<16, BIAS, L>), grid, block, lds, st, logits, a);
        if (const int rc = check_launch("route_experts")) return rc;
        logits += a.tokens * a.experts;
        a.weights += a.tokens * a.top_k;
        a.ids += a.tokens * a.top_k;
    }
    return INT4MM_OK;
}

}  // namespace i4

using namespace i4;

extern "C" int int4mm_route_experts(void* weights, void* ids, const void* logits, const void* bias, const int4mm_route_shape* sh,
                                    void* stream) {
    if (sh == nullptr) return INT4MM_ERR_NULL;
    if (sh->tokens < 0 || sh->tokens > ((int64_t)1 << 31) - 4 || sh->experts < 1 || sh->experts > 1024) return INT4MM_ERR_SHAPE;
    if (sh->groups < 1 || sh->groups > 64 || sh->experts % sh->groups != 0 || sh->topk_groups < 1 || sh->topk_groups > sh->groups)
        return INT4MM_ERR_SHAPE;
    if (sh->top_k < 1 || sh->top_k > 64 || sh->top_k > sh->experts / sh->groups * sh->topk_groups) return INT4MM_ERR_SHAPE;
    if ((sh->scoring != 0 && sh->scoring != 1) || (sh->group_score != 0 && sh->group_score != 1) ||
        (sh->logits_bytes != 2 && sh->logits_bytes != 4) || !std::isfinite(sh->scale))
        return INT4MM_ERR_SHAPE;
    if (sh->tokens == 0) return INT4MM_OK;
    if (!weights || !ids || !logits) return INT4MM_ERR_NULL;
    const uintptr_t mis = (reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(bias)) & 3;
    if (mis != 0 || (reinterpret_cast<uintptr_t>(logits) & (sh->logits_bytes - 1)) != 0) return INT4MM_ERR_ALIGN;

    RouteArgs a;
    a.weights = static_cast<float*>(weights);
    a.ids = static_cast<int*>(ids);
    a.bias = static_cast<const float*>(bias);
    a.tokens = sh->tokens;
    a.scale = sh->scale;
    a.experts = (int)sh->experts;
    a.top_k = (int)sh->top_k;
    a.groups = (int)sh->groups;
    a.topk_groups = (int)sh->topk_groups;
    a.group_size = (int)(sh->experts / sh->groups);
    a.lanes_per_group = 1;
    while (2 * a.lanes_per_group * a.groups <= 64) a.lanes_per_group *= 2;
    a.group_magic = div_magic((uint32_t)a.group_size);
    a.softmax = sh->scoring == 0;
    a.top2 = sh->group_score;
    a.renormalize = sh->renormalize != 0;
    hipStream_t st = (hipStream_t)stream;
    if (sh->logits_bytes == 2) {
        const h16* l = static_cast<const h16*>(logits);
        return bias ? launch_route<true>(l, a, st) : launch_route<false>(l, a, st);
    }
    const float* l = static_cast<const float*>(logits);
    return bias ? launch_route<true>(l, a, st) : launch_route<false>(l, a, st);
}
