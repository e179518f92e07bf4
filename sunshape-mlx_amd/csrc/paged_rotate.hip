// The rotated append of the paged 4-bit cache: per-head norms of queries and
// keys, their rotation by position, and the append of keys and values.
//
//   y = (x r) w,  r = 1 / sqrt(mean x^2 + eps)            (with a norm)
//   (a, b) -> (a cos - b sin, b cos + a sin)              (pairs of dims)
//
// Every operation is rounded to float32 by itself (r and its mean in 64 bits
// and once to float32), so that the keys' 16-bit roundings, and with them the
// codes, are the same wherever this is computed: a fused multiply-add would
// move one code in some 10^5.
#include "paged_append.hpp"

namespace ss {

struct RotatedAppend {
    PagedStore st;
    const void *q, *k, *v;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
    const int32_t *slots, *positions;
    const float *table;  // [n_pos][rdim/2][2]: cos, sin
    const void *q_weight, *k_weight;
    void *out;           // queries, [n_tok][hq][D]
    double eps;
    int64_t n_tok, n_pos;
    int hq, rdim, neighbours, in_dtype, out_dtype, w_dtype, vec, zero_rest;
    int run;             // query heads of a wave
    uint32_t kv_items, q_items;
};

// Of one token: what a lane's 8 dims and their partners are multiplied by.
struct Turn {
    float c[8], s[8];
};

__device__ __forceinline__ float turned(float x, float c, float p, float s) {
#pragma clang fp contract(off)
    const float a = x * c, b = p * s;
    return a + b;
}

// The lane's place in the rotation: its dims 8w .. 8w+7, those of its partners,
// and whether they turn at all.
struct Place {
    int w, partner;
    bool turns, second;
    __device__ Place(int w_, int rdim, int neighbours) : w(w_) {
        turns = w * 8 < rdim;
        second = !neighbours && turns && w * 16 >= rdim;
        partner = neighbours || !turns ? w : second ? w - rdim / 16 : w + rdim / 16;
    }
};

// 8 pairs (or, neighbours, 4) of the table's row of `pos`; NaN past its end.
__device__ __forceinline__ void load_turn(const RotatedAppend &a, const Place &pl, int pos, Turn &t) {
    if (!pl.turns) {
#pragma unroll
        for (int e = 0; e < 8; ++e) t.c[e] = 1.f, t.s[e] = 0.f;
        return;
    }
    const bool there = (uint32_t)pos < (uint64_t)a.n_pos;
    const float *row = a.table + (int64_t)(there ? pos : 0) * a.rdim;
    if (a.neighbours) {
        const float4 *p = reinterpret_cast<const float4 *>(row + pl.w * 8);
        const float4 u[2] = {p[0], p[1]};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float c = i & 1 ? u[i / 2].z : u[i / 2].x, s = i & 1 ? u[i / 2].w : u[i / 2].y;
            t.c[2 * i] = t.c[2 * i + 1] = c;
            t.s[2 * i] = -s, t.s[2 * i + 1] = s;
        }
    } else {
        const float4 *p = reinterpret_cast<const float4 *>(row + (pl.second ? pl.partner : pl.w) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 u = p[i];
            t.c[2 * i] = u.x, t.c[2 * i + 1] = u.z;
            t.s[2 * i] = pl.second ? u.y : -u.y, t.s[2 * i + 1] = pl.second ? u.w : -u.w;
        }
    }
    if (!there)
#pragma unroll
        for (int e = 0; e < 8; ++e) t.c[e] = NAN;
}

// A double from another lane of the row.
template <int CTRL>
__device__ __forceinline__ double dpp_double(double v) {
    const int64_t b = __builtin_bit_cast(int64_t, v);
    const uint32_t lo = (uint32_t)dpp_mov_i<CTRL>((int)b), hi = (uint32_t)dpp_mov_i<CTRL>((int)(b >> 32));
    return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}

// 1 / sqrt(mean x^2 + eps) of the row that LANES neighbours hold.
template <int LANES>
__device__ __forceinline__ float row_norm(const float (&x)[8], double eps) {
    double s = 0.;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fma((double)x[e], (double)x[e], s);
    s += dpp_double<0xB1>(s);                   // quad_perm [1,0,3,2]
    s += dpp_double<0x4E>(s);                   // quad_perm [2,3,0,1]
    s += dpp_double<0x141>(s);                  // row_half_mirror
    if (LANES == 16) s += dpp_double<0x140>(s);  // row_mirror
    s = s * (1. / (8 * LANES)) + eps;
    // (two steps of Newton's: 2^-26 -> 2^-52 and better)
    double r = __builtin_amdgcn_rsq(s);
    if (s > 0. && s < (double)INFINITY) {
#pragma unroll
        for (int i = 0; i < 2; ++i) r = fma(0.5 * r, fma(-(s * r), r, 1.), r);
    }
    return (float)r;
}

// A row's 8 values x of this lane (xp: its partners' in halves), rotated.
template <int LANES>
__device__ __forceinline__ void rotate8(const RotatedAppend &a, const Place &pl, const Turn &t, bool norm,
                                        const float (&w)[8], const float (&wp)[8], float (&x)[8], float (&xp)[8]) {
    if (norm) {
        const float r = row_norm<LANES>(x, a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e], xp[e] = xp[e] * r * wp[e];
    }
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float p = pl.turns ? (a.neighbours ? x[e ^ 1] : xp[e]) : 0.f;
        y[e] = turned(x[e], t.c[e], p, t.s[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = y[e];
}

// Waves take 8 consecutive tokens of one KV head, or of a run of query heads.
template <int D, int GROUP, bool BF>
__global__ void __launch_bounds__(256) append_rotated_kernel(const RotatedAppend a) {
    constexpr int LPR = D / 8;     // lanes a row
    constexpr int RPP = 64 / LPR;  // rows a pass
    constexpr int PASSES = 8 / RPP;
    constexpr int G = D / GROUP;
    __shared__ uint32_t tile[4][8][LPR + 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t item = blockIdx.x * 4 + wave;
    if (item >= a.kv_items + a.q_items) return;  // whole waves leave; no barrier follows
    const bool kv = item < a.kv_items;
    if (!kv) item -= a.kv_items;
    const uint32_t heads = kv ? (uint32_t)a.st.heads : (uint32_t)(a.hq + a.run - 1) / (uint32_t)a.run;
    const uint32_t win = item / heads;
    const int h = (int)(item - win * heads);
    const int64_t t0 = (int64_t)win * 8;
    const Place pl(lane % LPR, a.rdim, a.neighbours);
    const void *weight = kv ? a.k_weight : a.q_weight;
    const bool norm = weight != nullptr;
    float w[8], wp[8];
    if (norm) {
        load8_f32(weight, a.w_dtype, 0, pl.w * 8, w);
        load8_f32(weight, a.w_dtype, 0, pl.partner * 8, wp);
    }
    // lane e < 8 holds the position and the slot of token t0 + e
    int my_pos = -1, my_slot = -1;
    if (lane < 8 && t0 + lane < a.n_tok) {
        my_pos = a.positions[t0 + lane];
        my_slot = a.slots[t0 + lane];
        if (my_pos < 0 || (uint32_t)my_slot >= (uint32_t)(a.st.n_pages << a.st.log_page)) my_slot = -1;
    }
    int pos_of[PASSES];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) pos_of[p] = __shfl(my_pos, p * RPP + lane / LPR);
    if (!kv) {
        const int h1 = min(a.hq, (h + 1) * a.run);
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int e = p * RPP + lane / LPR, pos = pos_of[p];
            const int64_t t = t0 + e;
            if (t >= a.n_tok || (pos < 0 && !a.zero_rest)) continue;
            Turn turn;
            if (pos >= 0) load_turn(a, pl, pos, turn);
            for (int head = h * a.run; head < h1; ++head) {
                float x[8], xp[8];
                if (pos >= 0) {
                    const int64_t from = t * a.q_st + head * a.q_sh;
                    load8_f32(a.q, a.in_dtype, a.vec, from + pl.w * 8, x);
                    load8_f32(a.q, a.in_dtype, a.vec, from + pl.partner * 8, xp);
                    rotate8<LPR>(a, pl, turn, norm, w, wp, x, xp);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = 0.f;
                }
                uint32_t u[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    u[i] = a.out_dtype == SS_BF16 ? pack16<true>(x[2 * i], x[2 * i + 1])
                                                  : pack16<false>(x[2 * i], x[2 * i + 1]);
                *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + (t * a.hq + head) * D + pl.w * 8) =
                    make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
        return;
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int e = p * RPP + lane / LPR, slot = __shfl(my_slot, e), pos = pos_of[p];
        const int64_t t = min(t0 + e, a.n_tok - 1);
        const int64_t row = (int64_t)(slot >> a.st.log_page) * a.st.heads + h;
        const int off = slot & ((1 << a.st.log_page) - 1), g = pl.w * 8 / GROUP;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            float x[8];
            if (side == 0) {
                float xp[8];
                Turn turn;
                load_turn(a, pl, max(pos, 0), turn);
                load8_f32(a.k, a.in_dtype, a.vec, t * a.k_st + h * a.k_sh + pl.w * 8, x);
                load8_f32(a.k, a.in_dtype, a.vec, t * a.k_st + h * a.k_sh + pl.partner * 8, xp);
                rotate8<LPR>(a, pl, turn, norm, w, wp, x, xp);
            } else {
                load8_f32(a.v, a.in_dtype, a.vec, t * a.v_st + h * a.v_sh + pl.w * 8, x);
            }
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const uint32_t u = pack16<BF>(x[i], x[i + 1]);
                x[i] = from_bits16<BF>(u & 0xffffu), x[i + 1] = from_bits16<BF>(u >> 16);
            }
            uint32_t meta;
            const uint32_t word = quantize8<GROUP / 8, BF>(x, meta);
            if (side) tile[wave][e][pl.w] = word;
            if (slot >= 0) {
                if (!side) a.st.k_codes[((row << a.st.log_page) + off) * LPR + pl.w] = word;
                if (pl.w % (GROUP / 8) == 0)
                    (side ? a.st.v_meta : a.st.k_meta)[((row * G + g) << a.st.log_page) + off] = meta;
            }
        }
    }
    store_value_words<D>(a.st, tile[wave], h, lane, my_slot);
}

}  // namespace ss

using namespace ss;

extern "C" int ss_append_rotated_paged(const ss_paged_store *store, const void *queries, const void *keys,
                                       const void *values, int in_dtype, int64_t n_tokens, int n_q_heads,
                                       int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh, int64_t v_st,
                                       int64_t v_sh, const int32_t *slots, const int32_t *positions,
                                       const ss_rotation *rotation, void *out, int zero_rest, void *stream) {
    RotatedAppend a{};
    int log_page;
    if (int rc = check_paged_store(store, &a.st, &log_page)) return rc;
    SS_REQUIRE(valid_dtype(in_dtype), "bad query/key/value dtype");
    SS_REQUIRE(rotation && rotation->table, "null rotation");
    const ss_rotation &ro = *rotation;
    SS_UNSUPPORTED(ro.rotary_dim >= 16 && ro.rotary_dim <= store->head_dim && ro.rotary_dim % 16 == 0,
                   "rotary_dim %d (a multiple of 16 up to head_dim)", ro.rotary_dim);
    SS_REQUIRE(ro.n_positions >= 1 && ((uintptr_t)ro.table & 15) == 0,
               "the rotary table must be 16-byte aligned and hold a position");
    SS_REQUIRE((!ro.q_weight && !ro.k_weight) || valid_dtype(ro.weight_dtype), "bad weight dtype");
    SS_REQUIRE(ro.eps >= 0., "eps must not be negative");
    SS_REQUIRE(n_q_heads >= 1 && n_tokens >= 0, "bad sizes");
    if (n_tokens == 0) return SS_OK;
    SS_REQUIRE(queries && keys && values && slots && positions && out, "null pointer argument");
    SS_REQUIRE(((uintptr_t)out & 15) == 0, "out must be 16-byte aligned");
    SS_UNSUPPORTED(n_tokens <= INT32_MAX, "too many tokens for one launch");
    const int64_t windows = (n_tokens + 7) / 8;
    a.run = 1;
    const int64_t kv_items = windows * a.st.heads, q_items = windows * ((n_q_heads + a.run - 1) / a.run);
    SS_UNSUPPORTED((kv_items + q_items + 3) / 4 <= kMostGroups, "%lld tokens of %d and %d heads: too many for one launch",
                   (long long)n_tokens, n_q_heads, a.st.heads);
    a.q = queries, a.k = keys, a.v = values;
    a.q_st = q_st, a.q_sh = q_sh, a.k_st = k_st, a.k_sh = k_sh, a.v_st = v_st, a.v_sh = v_sh;
    a.slots = slots, a.positions = positions, a.table = static_cast<const float *>(ro.table);
    a.q_weight = ro.q_weight, a.k_weight = ro.k_weight, a.w_dtype = ro.weight_dtype, a.eps = ro.eps;
    a.out = out, a.n_tok = n_tokens, a.n_pos = ro.n_positions, a.hq = n_q_heads;
    a.rdim = ro.rotary_dim, a.neighbours = ro.neighbours, a.in_dtype = in_dtype, a.zero_rest = zero_rest;
    a.out_dtype = in_dtype == SS_F32 ? store->dtype : in_dtype;
    a.kv_items = (uint32_t)kv_items, a.q_items = (uint32_t)q_items;
    // 16-byte loads where every row starts on 16 bytes
    const int per = in_dtype == SS_F32 ? 4 : 8;
    a.vec = (((uintptr_t)queries | (uintptr_t)keys | (uintptr_t)values) & 15) == 0 && q_st % per == 0 &&
            q_sh % per == 0 && k_st % per == 0 && k_sh % per == 0 && v_st % per == 0 && v_sh % per == 0;
    const dim3 grid((unsigned)((kv_items + q_items + 3) / 4));
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a); };
    const bool bf = store->dtype == SS_BF16;
    const int key = store->head_dim * 1000 + store->group_size;
    if (key == 128032) bf ? launch(append_rotated_kernel<128, 32, true>) : launch(append_rotated_kernel<128, 32, false>);
    else if (key == 128064) bf ? launch(append_rotated_kernel<128, 64, true>) : launch(append_rotated_kernel<128, 64, false>);
    else if (key == 128128) bf ? launch(append_rotated_kernel<128, 128, true>) : launch(append_rotated_kernel<128, 128, false>);
    else if (key == 64032) bf ? launch(append_rotated_kernel<64, 32, true>) : launch(append_rotated_kernel<64, 32, false>);
    else bf ? launch(append_rotated_kernel<64, 64, true>) : launch(append_rotated_kernel<64, 64, false>);
    SS_LAUNCH_CHECK("append_rotated_kernel launch");
    return SS_OK;
}
