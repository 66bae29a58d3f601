// Lane-group reductions, the f32 exponential and the steps on 32-bit selection
// keys that the routing kernels share (topk_softmax.hip, route.hip).
#pragma once

#include "cm_common.hpp"

namespace cm {

// Lane-group exchange step M (1, 2, 4, 8, 16, 32): a and b are the values of
// a lane pair that straddles the two halves of an aligned group of 2M lanes
// (quad xor 1 / 2 by DPP quad_perm, mirror inside 8 / 16 lanes by DPP
// row_half_mirror / row_mirror, the row swaps of v_permlane16 / 32_swap);
// both lanes of a pair get the same (a, b). All VALU, no LDS round trip.
// A symmetric combine of (a, b) over the steps M < LPR leaves every lane of
// an LPR-lane group with the reduction of the whole group.
template <int M>
__device__ __forceinline__ void lane_pair(uint32_t v, uint32_t& a, uint32_t& b) {
    if constexpr (M == 16 || M == 32) {
        const auto r = M == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false)
                               : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        a = r[0];
        b = r[1];
    } else {
        constexpr int ctrl = M == 1 ? 0xB1 : (M == 2 ? 0x4E : (M == 4 ? 0x141 : 0x140));
        a = v;
        b = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, ctrl, 0xF, 0xF, false);
    }
}

template <int M>
__device__ __forceinline__ float max_step(float v) {
    uint32_t a, b;
    lane_pair<M>(__float_as_uint(v), a, b);
    return fmaxf(__uint_as_float(a), __uint_as_float(b));
}
template <int M>
__device__ __forceinline__ double sum_step(double v) {
    const uint64_t u = __double_as_longlong(v);
    uint32_t al, bl, ah, bh;
    lane_pair<M>((uint32_t)u, al, bl);
    lane_pair<M>((uint32_t)(u >> 32), ah, bh);
    // a + b in the same order on both lanes of the pair: identical sums
    return __longlong_as_double(((uint64_t)ah << 32) | al) + __longlong_as_double(((uint64_t)bh << 32) | bl);
}

template <int LPR>
__device__ __forceinline__ float group_max(float v) {
    if constexpr (LPR >= 2) v = max_step<1>(v);
    if constexpr (LPR >= 4) v = max_step<2>(v);
    if constexpr (LPR >= 8) v = max_step<4>(v);
    if constexpr (LPR >= 16) v = max_step<8>(v);
    if constexpr (LPR >= 32) v = max_step<16>(v);
    if constexpr (LPR >= 64) v = max_step<32>(v);
    return v;
}

template <int LPR>
__device__ __forceinline__ double group_sum(double v) {
    if constexpr (LPR >= 2) v = sum_step<1>(v);
    if constexpr (LPR >= 4) v = sum_step<2>(v);
    if constexpr (LPR >= 8) v = sum_step<4>(v);
    if constexpr (LPR >= 16) v = sum_step<8>(v);
    if constexpr (LPR >= 32) v = sum_step<16>(v);
    if constexpr (LPR >= 64) v = sum_step<32>(v);
    return v;
}

// (value, expert) pairs ordered by value, then the lower expert: a total
// order, so the pairwise pick is symmetric and the group agrees on the top.
template <int M>
__device__ __forceinline__ void argmax_step(float& v, int& i) {
    uint32_t va, vb, ia, ib;
    lane_pair<M>(__float_as_uint(v), va, vb);
    lane_pair<M>((uint32_t)i, ia, ib);
    const float fa = __uint_as_float(va), fb = __uint_as_float(vb);
    const bool take_b = (fb > fa) | ((fb == fa) & ((int)ib < (int)ia));
    v = take_b ? fb : fa;
    i = take_b ? (int)ib : (int)ia;
}

template <int LPR>
__device__ __forceinline__ void group_argmax(float& v, int& i) {
    if constexpr (LPR >= 2) argmax_step<1>(v, i);
    if constexpr (LPR >= 4) argmax_step<2>(v, i);
    if constexpr (LPR >= 8) argmax_step<4>(v, i);
    if constexpr (LPR >= 16) argmax_step<8>(v, i);
    if constexpr (LPR >= 32) argmax_step<16>(v, i);
    if constexpr (LPR >= 64) argmax_step<32>(v, i);
}

// e^d in f32 arithmetic for an f32 d <= 0, within 1 ulp of the correctly
// rounded value wherever that is a normal number (d >= -87.33; checked on the
// GPU against exp_f32_f64 for every f32 d in that range: 96.7 % equal, the
// rest 1 ulp apart). t = d log2(e) is carried as th + tl: th = f32(d L) with
// L = f32(log2 e), tl = the product's rounding error (an exact fma) plus
// d (log2 e - L); then 2^t = 2^th (1 + tl ln 2) to first order, |tl| being
// below 2^-16. 2^th is the hardware v_exp_f32. Below the normal range the
// result is approximate (possibly 0); below -104 it is +0, as above.
__device__ __forceinline__ float exp_f32_fast(float d) {
#pragma clang fp contract(off)
    constexpr float L = 1.44269504088896341f;        // log2(e) rounded to f32
    constexpr float Llo = 1.9259629911783648e-08f;   // log2(e) - L
    constexpr float LN2 = 0.693147180559945309f;
    const float th = d * L;
    const float tl = __builtin_fmaf(d, Llo, __builtin_fmaf(d, L, -th));
    const float y = __builtin_amdgcn_exp2f(th);
    return d < -104.0f ? 0.0f : __builtin_fmaf(y, tl * LN2, y);
}

// The lanes of `mask` (a wave-wide lane mask) take b, the others keep a.
__device__ __forceinline__ uint32_t key_take32(uint32_t a, uint32_t b, uint64_t mask) {
    uint32_t r;
    asm("v_cndmask_b32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(mask));
    return r;
}
// max(v, v of the partner lane) in one DPP-modified v_max_u32 for the
// steps inside a row of 16 lanes (the s_nop covers the wait states between a
// VALU write of v and its DPP read, which the compiler does not track across
// inline asm).
template <int M>
__device__ __forceinline__ uint32_t key32_max_step(uint32_t v) {
    if constexpr (M == 1 || M == 2 || M == 4 || M == 8) {
        uint32_t r;
        if constexpr (M == 1)
            asm volatile("s_nop 1\n\tv_max_u32_dpp %0, %1, %1 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf"
                         : "=v"(r) : "v"(v));
        else if constexpr (M == 2)
            asm volatile("s_nop 1\n\tv_max_u32_dpp %0, %1, %1 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf"
                         : "=v"(r) : "v"(v));
        else if constexpr (M == 4)
            asm volatile("s_nop 1\n\tv_max_u32_dpp %0, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xf"
                         : "=v"(r) : "v"(v));
        else
            asm volatile("s_nop 1\n\tv_max_u32_dpp %0, %1, %1 row_mirror row_mask:0xf bank_mask:0xf"
                         : "=v"(r) : "v"(v));
        return r;
    } else {
        uint32_t a, b;
        lane_pair<M>(v, a, b);
        return a > b ? a : b;
    }
}
template <int LPR>
__device__ __forceinline__ uint32_t group_key32_max(uint32_t v) {
    if constexpr (LPR >= 2) v = key32_max_step<1>(v);
    if constexpr (LPR >= 4) v = key32_max_step<2>(v);
    if constexpr (LPR >= 8) v = key32_max_step<4>(v);
    if constexpr (LPR >= 16) v = key32_max_step<8>(v);
    if constexpr (LPR >= 32) v = key32_max_step<16>(v);
    if constexpr (LPR >= 64) v = key32_max_step<32>(v);
    return v;
}

}  // namespace cm
