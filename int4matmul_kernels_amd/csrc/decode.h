// Decodes of packed codes to fp16 weights that the tile kernels and the experts' kernels share: chunks of 8 consecutive
// k of one column, in natural k order, bit-exact with the formats' definition.
#pragma once

#include "common.h"

#include <type_traits>

namespace i4 {

// ---- decodes of a chunk, 8 consecutive k of one column, bit-exact and in natural k order
// The coefficients of a column's group: {s, s}, {z, z} or what the decode makes of them.
// Linear mode: the reference's own two roundings, fp16(q - z), fp16(. * s).
struct LinearCoef {
    static constexpr bool EITHER = false;
    h16x2 s, z;
    __device__ __forceinline__ void set(h16x2 s2, h16x2 z2) { s = s2; z = z2; }
    __device__ __forceinline__ uint32_t weight(h16x2 q) const { return as_u32((q - z) * s); }
};
// Either mode, chosen per thread (a thread decodes whole columns, and the mode belongs to a (group, column)), without a branch:
//     A = P + N (one rounding),  w = fma(A, B, C) (one rounding)
// linear:   P = q, N = -z, B = s, C = -0:  fp16(q - z), then fp16(. * s) -- adding -0 changes nothing
// exponent: P = +-2^e, N = -0, B = -s, C = z:  the reference's single-rounded fma (matmul.cuh:127-136)
struct TwoModeCoef {
    static constexpr bool EITHER = true;
    uint32_t m;                                  // all ones in exponent mode (bit picks: a selection came out as a branch)
    h16x2 N, B, C;
    float scale;                                 // of the 8-bit floats: 2^9 for q, 1 for +-2^e
    __device__ __forceinline__ uint32_t pick(uint32_t e, uint32_t l) const { return (e & m) | (l & ~m); }
    __device__ __forceinline__ void set(h16x2 s2, h16x2 z2) {
        m = s2.x >= (h16)0.0f ? 0u : 0xFFFFFFFFu;
        N = as_h2(pick(0x80008000u, as_u32(z2) ^ 0x80008000u));
        B = as_h2(as_u32(s2) ^ (m & 0x80008000u));
        C = as_h2(pick(as_u32(z2), 0x80008000u));
        scale = bitcast<float>(pick(0x3F800000u, 0x44000000u));
    }
    __device__ __forceinline__ uint32_t weight(h16x2 P) const { return as_u32(__builtin_elementwise_fma(P + N, B, C)); }
    // four codes as bytes -> the 8-bit floats of q 2^-9 or +-2^e
    __device__ __forceinline__ uint32_t powers(uint32_t b) const {
        return pick(((b & 0x08080808u) << 4) | (((b & 0x07070707u) << 3) + 0x38383838u), b);
    }
};
// int2: the group's four weights, in either mode, are a v_perm table
struct Int2Coef {
    uint32_t T0, T1;
    __device__ __forceinline__ void set(h16x2 s2, h16x2 z2) {
        TwoModeCoef c;
        c.set(s2, z2);
        T0 = c.weight(as_h2(c.pick(0x40003C00u, 0x3C000000u)));
        T1 = c.weight(as_h2(c.pick(0xC000BC00u, 0x42004000u)));
    }
};
// int3: the eight values' upper bytes are one (their lower ones are 0)
struct Int3Coef : TwoModeCoef {
    uint32_t T0, T1;
    __device__ __forceinline__ void set(h16x2 s2, h16x2 z2) {
        TwoModeCoef::set(s2, z2);
        T0 = pick(0x4844403Cu, 0x42403C00u);
        T1 = pick(0xC8C4C0BCu, 0x47464544u);
    }
};
template <int BITS, bool TWO_MODES>
using Coef = std::conditional_t<BITS == 2, Int2Coef, std::conditional_t<BITS == 3, Int3Coef, std::conditional_t<TWO_MODES, TwoModeCoef, LinearCoef>>>;

// What the codes stand for alone, exact in fp16: q or, in a column in exponent mode, +-2^e.  Scale and zero are left to the sums:
//     sum x w = A sum x value + B sum x,   (A, B) = (s, -s z), in exponent mode (-s, z)
template <int BITS>
struct CodeValues {
    static constexpr bool EITHER = false;
    static constexpr uint32_t T0 = BITS == 2 ? 0x3C000000u : 0x42403C00u, T1 = BITS == 2 ? 0x42004000u : 0x47464544u;
    __device__ __forceinline__ void set(h16x2, h16x2) {}
    __device__ __forceinline__ uint32_t weight(h16x2 value) const { return as_u32(value); }
};
template <int BITS>
struct EitherValues : TwoModeCoef {
    uint32_t T0, T1;
    __device__ __forceinline__ void set(h16x2 s2, h16x2 z2) {
        TwoModeCoef::set(s2, z2);
        T0 = BITS == 2 ? pick(0x40003C00u, 0x3C000000u) : pick(0x4844403Cu, 0x42403C00u);
        T1 = BITS == 2 ? pick(0xC000BC00u, 0x42004000u) : pick(0xC8C4C0BCu, 0x47464544u);
    }
    __device__ __forceinline__ uint32_t weight(h16x2 value) const { return as_u32(value); }
};
// 16:32: a dropped row must not meet the zero either, so that is subtracted here, the one rounding; a column in exponent mode is
// complete
//     sum x w = A sum x value,   A = s, in exponent mode 1
struct KeptValues {
    static constexpr bool EITHER = false;
    h16x2 z;
    __device__ __forceinline__ void set(h16x2, h16x2 z2) { z = z2; }
    __device__ __forceinline__ uint32_t weight(h16x2 q) const { return as_u32(q - z); }
};
struct EitherKeptValues : TwoModeCoef {
    __device__ __forceinline__ void set(h16x2 s2, h16x2 z2) {
        TwoModeCoef::set(s2, z2);
        B = as_h2(pick(as_u32(B), 0x3C003C00u));
    }
};
template <int BITS, bool SPARSE, bool EITHER>
using Values = std::conditional_t<SPARSE, std::conditional_t<EITHER, EitherKeptValues, KeptValues>,
                                  std::conditional_t<EITHER, EitherValues<BITS>, CodeValues<BITS>>>;

// four codes of a word as bytes -> eight weights: a byte q < 16 is the 8-bit float q 2^-9
template <class C>
__device__ __forceinline__ h16x8 weights_of_bytes(uint32_t b03, uint32_t b47, const C& c) {
    float scale = 512.f;
    if constexpr (C::EITHER) {
        b03 = c.powers(b03);
        b47 = c.powers(b47);
        scale = c.scale;
    }
    return bitcast<h16x8>(u32x4{c.weight(from_fp8<false>(b03, scale)), c.weight(from_fp8<true>(b03, scale)),
                                c.weight(from_fp8<false>(b47, scale)), c.weight(from_fp8<true>(b47, scale))});
}

// `bits`: the chunk's codes, LSB first, BITS bits apart (bits above 8 * BITS are ignored).  17 (int4), 17 (int2) and 24 (int3)
// instructions; with magic numbers and their removal 20, 24 and 24, and twice as many for either mode
template <int BITS, class C>
__device__ __forceinline__ h16x8 dequant_chunk(uint32_t bits, const C& c) {
    if constexpr (BITS == 4) {
        const uint32_t even = bits & 0x0F0F0F0Fu, odd = (bits >> 4) & 0x0F0F0F0Fu;
        return weights_of_bytes(__builtin_amdgcn_perm(odd, even, 0x05010400u), __builtin_amdgcn_perm(odd, even, 0x07030602u), c);
    } else if constexpr (BITS == 2) {
        const uint32_t v = (bits & 0xFFFFu) | (bits << 14);               // code 2 j at bit 4 j, code 2 j + 1 at 16 + 4 j
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            r[j] = __builtin_amdgcn_perm(c.T1, c.T0, __umul24((v >> (4 * j)) & 0x00030003u, 0x0202u) + 0x01000100u);
        return bitcast<h16x8>(r);
    } else {
        const uint32_t u = bits & 0xFFFFFFu;
        const uint32_t v = (u & 0xFFFFu) | ((u << 13) & 0xFFFF0000u);      // codes 0, 2, 4 at bits 0, 6, 12, codes 1, 3, 5 at 16, 22, 28
        const uint32_t y = u >> 10;                                       // code 6 at bit 8, code 7 at 11
        const uint32_t sel[4] = {v << 8, v << 2, v >> 4, (y << 13) | y};
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = c.weight(as_h2(__builtin_amdgcn_perm(c.T1, c.T0, (sel[j] & 0x07000700u) | 0x000C000Cu)));
        return bitcast<h16x8>(r);
    }
}

// 16:32 sparse int4.  `v` holds the (up to 8) kept codes of one 8-row chunk as
// consecutive nibbles, `m8` the chunk's mask bits.  A 256-entry table in LDS
// (per mask byte four words of per-half keep masks and, in a table of their own so that lanes
// with different bytes meet on fewer banks, two v_perm selectors) spreads the kept codes to their rows: the even / odd nibbles are
// separated into bytes, v_perm picks for every row the byte of its rank.  Dropped rows
// are cleared at the end, so they are exactly zero.
constexpr int SPARSE_LUT_WORDS = 256 * 6, SPARSE_LUT_SELECTORS = 256 * 4;

__device__ __forceinline__ void sparse_lut_entry(uint32_t* lut, uint32_t e) {
    uint32_t sel[2] = {0, 0}, hm[4] = {0, 0, 0, 0};
    uint32_t rank = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool kept = (e >> i) & 1u;
        const uint32_t byte = kept ? ((rank & 1u) ? 4u + (rank >> 1) : (rank >> 1)) : 0x0Cu;
        sel[i >> 2] |= byte << (8 * (i & 3));
        if (kept) { hm[i >> 1] |= 0xFFFFu << (16 * (i & 1)); ++rank; }
    }
    *reinterpret_cast<u32x4*>(lut + e * 4) = u32x4{hm[0], hm[1], hm[2], hm[3]};
    *reinterpret_cast<u32x2*>(lut + SPARSE_LUT_SELECTORS + e * 2) = u32x2{sel[0], sel[1]};
}

template <class C>
__device__ __forceinline__ h16x8 dequant_chunk_sparse(uint32_t v, uint32_t m8, const uint32_t* lut, const C& c) {
    const u32x4 keep = *reinterpret_cast<const u32x4*>(lut + m8 * 4);
    const u32x2 sel = *reinterpret_cast<const u32x2*>(lut + SPARSE_LUT_SELECTORS + m8 * 2);
    const uint32_t even = v & 0x0F0F0F0Fu, odd = (v >> 4) & 0x0F0F0F0Fu;
    const u32x4 r = bitcast<u32x4>(weights_of_bytes(__builtin_amdgcn_perm(odd, even, sel.x), __builtin_amdgcn_perm(odd, even, sel.y), c));
    return bitcast<h16x8>(r & keep);             // (dropped rows -> +0)
}

}  // namespace i4
