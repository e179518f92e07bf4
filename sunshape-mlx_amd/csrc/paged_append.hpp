// The paged 4-bit cache's quantiser, as the appends use it (paged.hip,
// paged_rotate.hip).
#pragma once

#include "paged_common.hpp"

namespace ss {

// Largest and smallest of a group's values over the lanes that hold it (4, 8
// or 16 neighbours, 8 values each).  The lane moves stay within 16 lanes.
template <int LANES, typename F>
__device__ __forceinline__ int group_reduce(int v, F op) {
    v = op(v, dpp_mov_i<0xB1>(v));                  // quad_perm [1,0,3,2]
    v = op(v, dpp_mov_i<0x4E>(v));                  // quad_perm [2,3,0,1]
    if (LANES >= 8) v = op(v, dpp_mov_i<0x141>(v));   // row_half_mirror
    if (LANES >= 16) v = op(v, dpp_mov_i<0x140>(v));  // row_mirror
    return v;
}

// Quantises the 8 values x of this lane within its group of LANES lanes:
// returns their codes as a word, (scale, zero) as `meta`.
// zero = min, scale = round16((max - min) / 15), code = the nearest of
// 0 .. 15 to (x - zero) / scale, ties to even.  x - zero is one rounding;
// the quotient is never rounded: rcp guesses its integer part c, at most one
// off and then next to an integer, and the exact remainder r = d - c scale (an
// fma) adds one if r > scale/2, or r = scale/2 and c is odd.  Positive floats
// compare as integers, so that both are one test: bits(r) + (c odd) >
// bits(scale/2).
template <int LANES, bool BF>
__device__ __forceinline__ uint32_t quantize8(const float (&x)[8], uint32_t &meta) {
    float most = x[0], least = x[0];
    bool nan = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        most = fmaxf(most, x[e]);
        least = fminf(least, x[e]);
        nan |= x[e] != x[e];
    }
    // (a NaN's key is above every number's: the range is NaN then)
    int hi = nan ? INT32_MAX : ord_key(most), lo = ord_key(least);
    hi = group_reduce<LANES>(hi, [](int a, int b) { return max(a, b); });
    lo = group_reduce<LANES>(lo, [](int a, int b) { return min(a, b); });
    const float zero = ord_float(lo);
    const float range = __fdiv_rn(__fsub_rn(ord_float(hi), zero), 15.f);
    const uint32_t sb = to_bits16<BF>(range);
    const float scale = from_bits16<BF>(sb);
    if (!(scale < INFINITY)) {  // a value, or the range, is not finite
        meta = kNan16<BF> | (kNan16<BF> << 16);
        return 0;
    }
    meta = sb | (to_bits16<BF>(zero) << 16);
    if (!(scale > 0.f)) return 0;
    // (a bfloat16 scale below 2^-100 has no normal reciprocal: both sides times 2^64)
    const float up = BF && scale < 0x1p-100f ? 0x1p64f : 1.f;
    const float sc = scale * up, inv = __builtin_amdgcn_rcpf(sc);
    const int half = __float_as_int(0.5f * sc);
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float d = __fsub_rn(x[e], zero);
        if (BF) d *= up;
        const float f = floorf(d * inv);
        uint32_t c = (uint32_t)f;
        c += __float_as_int(fmaf(-f, sc, d)) + (int)(c & 1) > half;
        word |= min(c, 15u) << nibble_bit(e);
    }
    return word;
}

// Stores the value words of a wave's 8 tokens of one head, whose codes lie in
// `tile` token by token (lane e < 8 holds the slot of token e, -1: not stored).
// A word holds the 8 tokens of an aligned block of slots: where the wave's
// tokens are one whole block it stores the words; otherwise it clears and sets
// their bits with two atomics per block (bits of other tokens, which other
// waves may be writing, are kept; no order changes the result as long as no
// slot is given twice).
template <int D>
__device__ __forceinline__ void store_value_words(const PagedStore &st, const uint32_t (&tile)[8][D / 8 + 1], int h,
                                                  int lane, int my_slot) {
    wave_lds_sync();
    const int s0 = __builtin_amdgcn_readfirstlane(my_slot);
    const bool whole = s0 >= 0 && (s0 & 7) == 0 && __all(lane >= 8 || my_slot == s0 + lane);
    constexpr int DPL = D / 64;  // dims a lane
    uint32_t code[DPL][8];       // of its dims, token by token
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t u = tile[e][lane * DPL / 8];
#pragma unroll
        for (int k = 0; k < DPL; ++k) code[k][e] = (u >> nibble_bit((lane * DPL + k) & 7)) & 15u;
    }
    if (whole) {
        const int64_t row = (int64_t)(s0 >> st.log_page) * st.heads + h;
        const int blk = (s0 & ((1 << st.log_page) - 1)) >> 3;
        uint32_t *dst = st.v_codes + (((row << st.log_page) >> 3) + blk) * D + lane * DPL;
#pragma unroll
        for (int k = 0; k < DPL; ++k) {
            uint32_t u = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) u |= code[k][e] << nibble_bit(e);
            dst[k] = u;
        }
        return;
    }
    // block by block: tokens whose slots share it go together
    uint64_t left = __ballot(lane < 8 && my_slot >= 0);
    while (left) {
        const int first = __ffsll((unsigned long long)left) - 1;
        const int sb = __shfl(my_slot, first) >> 3;
        const uint64_t same = __ballot(lane < 8 && my_slot >= 0 && (my_slot >> 3) == sb) & left;
        left &= ~same;
        const int64_t slot8 = (int64_t)sb << 3;
        const int64_t row = (slot8 >> st.log_page) * st.heads + h;
        const int blk = ((int)slot8 & ((1 << st.log_page) - 1)) >> 3;
        uint32_t *dst = st.v_codes + (((row << st.log_page) >> 3) + blk) * D + lane * DPL;
        uint32_t keep = ~0u, set[DPL];
#pragma unroll
        for (int k = 0; k < DPL; ++k) set[k] = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (!((same >> e) & 1)) continue;
            const int bit = nibble_bit(__shfl(my_slot, e) & 7);
            keep &= ~(15u << bit);
#pragma unroll
            for (int k = 0; k < DPL; ++k) set[k] |= code[k][e] << bit;
        }
#pragma unroll
        for (int k = 0; k < DPL; ++k) {
            atomicAnd(dst + k, keep);
            atomicOr(dst + k, set[k]);
        }
    }
}

}  // namespace ss
