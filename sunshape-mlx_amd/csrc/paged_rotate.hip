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
//
// A prompt of 8192 tokens, 32 query and 8 KV heads of 128 dims, with norms, takes
// 48 us (181 MB, 3.8 TB/s; 36 us at the rate of a large copy): vector issue (70 %
// of the cycles: a key's element costs some 30 operations, a value's 20, most of
// them the quantising, a query's 10) beside HBM.  256 tokens take 7.9 us, one
// 4.4: the chain from a position over the table's row to the codes.
#include "paged_append.hpp"

namespace ss {

// Query heads of a wave (1: 58 us, 2: 48 us, 4: 53 us for the prompt above).
constexpr int kMostRun = 2;
// Workgroups in a row of one kind, queries or keys and values, and such stripes
// that the two share in proportion: one kind after the other takes 62 us where
// stripes of 8 take 52, of 2 to 32 about as much (in an earlier form).
constexpr int kStripe = 8;
constexpr int kMix = 16;

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
    int hq, rdim, neighbours, in_dtype, out_dtype, w_dtype, vec, w_vec, zero_rest;
    int run, kv_share;   // query heads of a wave; of kMix stripes those of keys
    uint32_t kv_items, q_items;
};

// a c + b s, each operation rounded.
__device__ __forceinline__ float turned(float a, float c, float b, float s) {
#pragma clang fp contract(off)
    const float x = a * c, y = b * s;
    return x + y;
}

// 8 cosines and sines of the table's row of `pos` from pair `first` on, NaN past
// its end; 1 and 0 if the lane's dims do not turn.
__device__ __forceinline__ void load_turn(const RotatedAppend &a, bool turns, int pos, int first, float (&c)[8],
                                          float (&s)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = 1.f, s[e] = 0.f;
    if (!turns) return;
    const bool there = pos < a.n_pos;
    const float4 *p = reinterpret_cast<const float4 *>(a.table + (int64_t)(there ? pos : 0) * a.rdim + first * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 u = p[i];
        c[2 * i] = there ? u.x : NAN, c[2 * i + 1] = there ? u.z : NAN;
        s[2 * i] = u.y, s[2 * i + 1] = u.w;
    }
}

// 4 of them, twice each; the sines for (a, b) and (b, a), the first negative.
__device__ __forceinline__ void load_turn_twice(const RotatedAppend &a, bool turns, int pos, int first, float (&c)[8],
                                                float (&s)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = 1.f, s[e] = 0.f;
    if (!turns) return;
    const bool there = pos < a.n_pos;
    const float4 *p = reinterpret_cast<const float4 *>(a.table + (int64_t)(there ? pos : 0) * a.rdim + first * 2);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float4 u = p[i];
        c[4 * i] = c[4 * i + 1] = there ? u.x : NAN, c[4 * i + 2] = c[4 * i + 3] = there ? u.z : NAN;
        s[4 * i] = -u.y, s[4 * i + 1] = u.y, s[4 * i + 2] = -u.w, s[4 * i + 3] = u.w;
    }
}

// A double from another lane of the row.
template <int CTRL>
__device__ __forceinline__ double dpp_double(double v) {
    const int64_t b = __builtin_bit_cast(int64_t, v);
    const uint32_t lo = (uint32_t)dpp_mov_i<CTRL>((int)b), hi = (uint32_t)dpp_mov_i<CTRL>((int)(b >> 32));
    return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}

// s plus the squares of x, in 64 bits (of 16-bit values exact).
__device__ __forceinline__ double add_squares(const float (&x)[8], double s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fma((double)x[e], (double)x[e], s);
    return s;
}

// 1 / sqrt(mean + eps) of D values whose squares sum up to s over LANES lanes.
template <int D, int LANES>
__device__ __forceinline__ float row_norm(double s, double eps) {
    s += dpp_double<0xB1>(s);                     // quad_perm [1,0,3,2]
    s += dpp_double<0x4E>(s);                     // quad_perm [2,3,0,1]
    if (LANES >= 8) s += dpp_double<0x141>(s);    // row_half_mirror
    if (LANES >= 16) s += dpp_double<0x140>(s);   // row_mirror
    s = s * (1. / D) + eps;
    // (two steps of Newton's: 2^-26 -> 2^-52 and better)
    double r = __builtin_amdgcn_rsq(s);
    if (s > 0. && s < (double)INFINITY) {
#pragma unroll
        for (int i = 0; i < 2; ++i) r = fma(0.5 * r, fma(-(s * r), r, 1.), r);
    }
    return (float)r;
}

__device__ __forceinline__ void unpack_half(const uint4 &u, bool bf, float (&x)[8]) {
    if (bf)
        unpack16<__hip_bfloat16>(u, x);
    else
        unpack16<__half>(u, x);
}

// Queries: a lane holds 16 dims of a row, two chunks of 8 that turn together, so
// that a row is D/16 lanes; a wave takes 64 of them: as many tokens, and a run of
// heads one after the other, for which the table's row and the weights are
// loaded once.
template <int D>
__device__ __forceinline__ void rotate_queries(const RotatedAppend &a, uint32_t item, int lane) {
    constexpr int LANES = D / 16;
    const uint32_t runs = (uint32_t)(a.hq + a.run - 1) / (uint32_t)a.run;
    const uint32_t win = item / runs;
    const int h0 = (int)(item - win * runs) * a.run, h1 = min(a.hq, h0 + a.run);
    const int64_t t = (int64_t)win * (64 / LANES) + lane / LANES;
    if (t >= a.n_tok) return;  // (rows are whole groups of lanes)
    const int l = lane % LANES;
    const bool halves = !a.neighbours, turns = l * 16 < a.rdim, bf = a.in_dtype == SS_BF16;
    // first dims of the lane's chunks
    const int da = halves && turns ? l * 8 : l * 16, db = halves && turns ? l * 8 + a.rdim / 2 : l * 16 + 8;
    const int64_t from = t * a.q_st;
    const bool quick = a.vec && a.in_dtype != SS_F32;
    auto load = [&](int head, int d) {
        return *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + from + head * a.q_sh + d);
    };
    uint4 ra[kMostRun], rb[kMostRun];  // (all of the run on their way before the first is looked at)
    if (quick)
#pragma unroll
        for (int i = 0; i < kMostRun; ++i) {
            const int head = min(h0 + i, h1 - 1);
            ra[i] = load(head, da), rb[i] = load(head, db);
        }
    const int pos = a.positions[t];
    if (pos < 0 && !a.zero_rest) return;
    const bool norm = a.q_weight != nullptr;
    float wa[8], wb[8], c[8], s[8];
    if (norm) {
        load8_f32(a.q_weight, a.w_dtype, a.w_vec, da, wa);
        load8_f32(a.q_weight, a.w_dtype, a.w_vec, db, wb);
    }
    load_turn(a, turns && pos >= 0, pos, l * 8, c, s);
    uint16_t *to = static_cast<uint16_t *>(a.out) + (t * a.hq + h0) * D;
#pragma unroll
    for (int i = 0; i < kMostRun; ++i, to += D) {
        const int head = h0 + i;
        if (head >= h1) break;
        float x[8], y[8];
        if (quick) {
            unpack_half(ra[i], bf, x), unpack_half(rb[i], bf, y);
        } else {
            load8_f32(a.q, a.in_dtype, a.vec, from + head * a.q_sh + da, x);
            load8_f32(a.q, a.in_dtype, a.vec, from + head * a.q_sh + db, y);
        }
        if (norm) {
            const float r = row_norm<D, LANES>(add_squares(y, add_squares(x, 0.)), a.eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = x[e] * r * wa[e], y[e] = y[e] * r * wb[e];
        }
        if (turns) {
            if (halves) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float u = turned(x[e], c[e], -y[e], s[e]);
                    y[e] = turned(y[e], c[e], x[e], s[e]), x[e] = u;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    float u = turned(x[i], c[i / 2], -x[i + 1], s[i / 2]);
                    x[i + 1] = turned(x[i + 1], c[i / 2], x[i], s[i / 2]), x[i] = u;
                    u = turned(y[i], c[4 + i / 2], -y[i + 1], s[4 + i / 2]);
                    y[i + 1] = turned(y[i + 1], c[4 + i / 2], y[i], s[4 + i / 2]), y[i] = u;
                }
            }
        }
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = a.out_dtype == SS_BF16 ? pack16<true>(x[2 * i], x[2 * i + 1]) : pack16<false>(x[2 * i], x[2 * i + 1]);
            u[4 + i] = a.out_dtype == SS_BF16 ? pack16<true>(y[2 * i], y[2 * i + 1]) : pack16<false>(y[2 * i], y[2 * i + 1]);
        }
        if (pos < 0)
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = 0;
        *reinterpret_cast<uint4 *>(to + da) = make_uint4(u[0], u[1], u[2], u[3]);
        *reinterpret_cast<uint4 *>(to + db) = make_uint4(u[4], u[5], u[6], u[7]);
    }
}

// x of the lane that is half a row (of LPR lanes) away.
template <int LPR>
__device__ __forceinline__ float across_row(float x) {
    const int v = __float_as_int(x);
    if (LPR == 16) return __int_as_float(dpp_mov_i<0x128>(v));           // row_ror:8
    return __int_as_float(dpp_mov_i<0x1B>(dpp_mov_i<0x141>(v)));         // row_half_mirror, quad_perm [3,2,1,0]
}

// Waves take 8 consecutive tokens' keys or values of one KV head, a chunk of 8
// dims a lane as the append does (the other halves of its pairs come from
// another lane), or 64 lanes of query rows.
template <int D, int GROUP, bool BF>
__global__ void __launch_bounds__(256) append_rotated_kernel(const RotatedAppend a) {
    constexpr int LPR = D / 8;     // lanes a row
    constexpr int RPP = 64 / LPR;  // rows a pass
    constexpr int PASSES = 8 / RPP;
    constexpr int G = D / GROUP;
    __shared__ uint32_t tile[4][8][LPR + 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // of kMix stripes kv_share are of keys, spread evenly, the others of queries
    // (whole waves leave; no barrier follows)
    const uint32_t stripe = blockIdx.x / kStripe, mix = stripe / kMix, in_mix = stripe % kMix;
    const uint32_t keys = in_mix * a.kv_share / kMix;  // of the stripes before this one
    const bool kv = (in_mix + 1) * a.kv_share / kMix > keys;
    const uint32_t mine = kv ? mix * a.kv_share + keys : mix * (kMix - a.kv_share) + in_mix - keys;
    const uint32_t item = (mine * kStripe + blockIdx.x % kStripe) * 4 + wave;
    if (!kv) {
        if (item < a.q_items) rotate_queries<D>(a, item, lane);
        return;
    }
    if (item >= a.kv_items) return;
    const bool values = item & 1;
    const uint32_t win = (item >> 1) / (uint32_t)a.st.heads;
    const int h = (int)((item >> 1) - win * (uint32_t)a.st.heads);
    const int64_t t0 = (int64_t)win * 8;
    const int w = lane % LPR;  // the lane's chunk
    // lane e < 8 holds the position and the slot of token t0 + e
    int my_pos = -1, my_slot = -1;
    if (lane < 8 && t0 + lane < a.n_tok) {
        my_pos = a.positions[t0 + lane];
        my_slot = a.slots[t0 + lane];
        if (my_pos < 0 || (uint32_t)my_slot >= (uint32_t)(a.st.n_pages << a.st.log_page)) my_slot = -1;
    }
    int slot_of[PASSES], pos_of[PASSES];
    float x[PASSES][8];
    const void *const from = values ? a.v : a.k;
    const int64_t stride = values ? a.v_st : a.k_st, first = (int64_t)h * (values ? a.v_sh : a.k_sh) + w * 8;
    auto row_of = [&](int p) { return min(t0 + p * RPP + lane / LPR, a.n_tok - 1) * stride + first; };
    auto look_up = [&] {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            slot_of[p] = __shfl(my_slot, p * RPP + lane / LPR);
            pos_of[p] = max(__shfl(my_pos, p * RPP + lane / LPR), 0);
        }
    };
    if (a.vec && a.in_dtype != SS_F32) {
        uint4 raw[PASSES];  // (all before the first is looked at)
#pragma unroll
        for (int p = 0; p < PASSES; ++p)
            raw[p] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(from) + row_of(p));
        look_up();
#pragma unroll
        for (int p = 0; p < PASSES; ++p) unpack_half(raw[p], a.in_dtype == SS_BF16, x[p]);
    } else {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) load8_f32(from, a.in_dtype, a.vec, row_of(p), x[p]);
        look_up();
    }
    if (!values) {
        // the chunk of the lane's pairs' other halves, and whether it turns at all
        const bool halves = !a.neighbours, turns = w * 8 < a.rdim, second = halves && w * 16 >= a.rdim;
        const int partner = halves && turns ? (second ? w - a.rdim / 16 : w + a.rdim / 16) : w;
        // (neighbours: 4 pairs from 4w on, twice each)
        float c[PASSES][8], s[PASSES][8];
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            if (halves) {
                load_turn(a, turns, pos_of[p], (second ? partner : w) * 8, c[p], s[p]);
#pragma unroll
                for (int i = 0; i < 8; ++i) s[p][i] = second ? s[p][i] : -s[p][i];
            } else {
                load_turn_twice(a, turns, pos_of[p], w * 4, c[p], s[p]);
            }
        }
        if (a.k_weight) {
            float wk[8];
            load8_f32(a.k_weight, a.w_dtype, a.w_vec, w * 8, wk);
#pragma unroll
            for (int p = 0; p < PASSES; ++p) {
                const float r = row_norm<D, LPR>(add_squares(x[p], 0.), a.eps);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[p][i] = x[p][i] * r * wk[i];
            }
        }
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            float(&k)[8] = x[p];
            float other[8];  // of the pairs
            if (!halves) {
#pragma unroll
                for (int i = 0; i < 8; ++i) other[i] = k[i ^ 1];
            } else if (a.rdim == D) {
#pragma unroll
                for (int i = 0; i < 8; ++i) other[i] = across_row<LPR>(k[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) other[i] = __shfl(k[i], (lane & ~(LPR - 1)) | partner);
            }
            if (turns)
#pragma unroll
                for (int i = 0; i < 8; ++i) k[i] = turned(k[i], c[p][i], other[i], s[p][i]);
        }
    }
    uint32_t *const to_meta = values ? a.st.v_meta : a.st.k_meta;
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int e = p * RPP + lane / LPR, slot = slot_of[p];
        const int64_t row = (int64_t)(slot >> a.st.log_page) * a.st.heads + h;
        const int off = slot & ((1 << a.st.log_page) - 1), g = w * 8 / GROUP;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const uint32_t u = pack16<BF>(x[p][i], x[p][i + 1]);
            x[p][i] = from_bits16<BF>(u & 0xffffu), x[p][i + 1] = from_bits16<BF>(u >> 16);
        }
        uint32_t meta;
        const uint32_t word = quantize8<GROUP / 8, BF>(x[p], meta);
        if (values) tile[wave][e][w] = word;
        if (slot >= 0) {
            if (!values) a.st.k_codes[((row << a.st.log_page) + off) * LPR + w] = word;
            if (w % (GROUP / 8) == 0) to_meta[((row * G + g) << a.st.log_page) + off] = meta;
        }
    }
    if (values) store_value_words<D>(a.st, tile[wave], h, lane, my_slot);
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
    SS_UNSUPPORTED(n_tokens <= INT32_MAX, "too many tokens for one launch");
    // as many heads a wave of queries as leave two waves for every SIMD
    const int per_wave = 1024 / store->head_dim;  // tokens
    const int64_t q_windows = (n_tokens + per_wave - 1) / per_wave;
    a.run = (int)max((int64_t)1, min((int64_t)min(kMostRun, n_q_heads), q_windows * n_q_heads / (8 * device_cu_count())));
    const int64_t kv_items = (n_tokens + 7) / 8 * 2 * a.st.heads, q_items = q_windows * ((n_q_heads + a.run - 1) / a.run);
    a.kv_share = (int)max((int64_t)1, min((int64_t)kMix - 1, (kv_items * kMix + (kv_items + q_items) / 2) / (kv_items + q_items)));
    auto mixes_of = [](int64_t items, int share) { return (items + 4 * kStripe * share - 1) / (4 * kStripe * share); };
    const int64_t groups = max(mixes_of(kv_items, a.kv_share), mixes_of(q_items, kMix - a.kv_share)) * kMix * kStripe;
    SS_UNSUPPORTED(groups <= kMostGroups, "%lld tokens of %d and %d heads: too many for one launch",
                   (long long)n_tokens, n_q_heads, a.st.heads);
    SS_REQUIRE(queries && keys && values && slots && positions && out, "null pointer argument");
    SS_REQUIRE(((uintptr_t)out & 15) == 0, "out must be 16-byte aligned");
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
    a.w_vec = (((uintptr_t)ro.q_weight | (uintptr_t)ro.k_weight) & 15) == 0;
    const dim3 grid((unsigned)groups);
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
