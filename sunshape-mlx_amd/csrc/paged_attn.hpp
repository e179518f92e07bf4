// What the kernels of attention over the paged cache share (paged_attn.hip:
// the few query rows of decode steps, paged_prompt.hip: the many of prompts).
//
//   S[r][t] = sum_g s_tg (q_rg . c_tg) + z_tg sum(q_rg)
//   O[r][d] = sum_t p_rt (s'_tg c'_td + z'_tg),   g = d's group
//
// with c the keys' codes, s and z their scales and zeros (primed: the
// values').  A code enters the fp16 matrix products as 1 + c/64: put into the
// middle of the mantissa of a 1 it needs no conversion, 7 operations for 8
// codes, and sum(x c) = 64 (sum(x (1 + c/64)) - sum(x)), where the sum of the
// other operand starts the accumulator, joins the zero's part or is taken off
// at the end.  (5 operations would make it the fp16 subnormal c * 2^-24; but
// the matrix cores align products by their operands' exponent fields, so that
// subnormals lost up to 10 bits: sums of 64 were off by 1.1e-5 of their terms,
// against 1.2e-7.)
#pragma once

#include "paged_common.hpp"

namespace ss {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float2_t __attribute__((ext_vector_type(2)));

// How far, in log2, a score may pass the running maximum before the maximum
// moves: probabilities stay below 2^4, so p * scale stays within fp16 with
// scales normalised to 2^10.
constexpr float kLag = 4.f;
// Scores are kept less a reference of their row, which is 0 until the maximum
// passes this many log2 units and moves to the maximum then: the maximum times
// the factor is off by 2^-24 of itself, which scores of 2^28 would turn into
// infinite probabilities.
constexpr float kFar = 4096.f;
__device__ __forceinline__ bool is_far(float top, float factor) {
    return fabsf(top * factor) > kFar && top > -INFINITY;
}

// What a kernel is built for: causal or no mask alone; rows that see an interval
// of their own and requests that continue others; and scores that are capped
// or get a bias too (in a kernel of its own, as its scores take operations more).
enum { kPlain = 0, kRanges = 1, kScores = 2 };

struct PagedAttn {
    PagedStore st;
    const void *q;
    int64_t q_st, q_sh;
    void *out;
    const int32_t *table, *lengths, *starts;
    int64_t width, n_tokens;
    int n_req, hq, rep, q_dtype, causal, zero_rest, vec;
    float scale;
    int most_rows;      // requests with more query rows a KV head are the prompt kernel's
    int target;         // of the prompt kernel: workgroups that its parts fill
    int4 *cut;          // columns to be joined (each kernel's merge says what it lists)
    float *acc;         // [workgroups][2][rows of a workgroup][D]
    float *ml;          // [workgroups][2][rows of a workgroup][2]
    // kRanges:
    // of the prompt kernel: workgroups that may leave parts; up to how many columns
    // the longer ones are halved
    int slots, halved;
    const int32_t *open;     // tokens of its beginning that all rows of a request see, or null
    int window;              // tokens up to its own that a row sees; INT32_MAX: all
    // A pass over shared tokens: row i of request r is that of token rows[starts[r]
    // + i].x, at .y behind the r's tokens; its sums go to `part`, for the pass over
    // the own tokens of a request that continues parents[r] >= 0.
    const int2 *rows_of;
    const int32_t *parents;
    float *part;             // [n_tokens][hq][D], then [n_tokens][hq][2] (maximum, sum)
    // kScores:
    float cap;               // of the scores; 0: none
    const float *slopes;     // [hq], or null
};

// Tables do not change while the kernel runs: through the constant address
// space their uniform reads are scalar loads, which do not queue behind the
// stream of codes.
__device__ __forceinline__ int table_read(const int32_t *p, int64_t i) {
    return reinterpret_cast<const __attribute__((address_space(4))) int32_t *>(reinterpret_cast<uintptr_t>(p))[i];
}

// Eight 16-bit query elements from p (16-byte aligned if vec).
__device__ __forceinline__ uint4 load_query8(const uint16_t *p, int vec) {
    if (vec) return *reinterpret_cast<const uint4 *>(p);
    return make_uint4(p[0] | ((uint32_t)p[1] << 16), p[2] | ((uint32_t)p[3] << 16),
                      p[4] | ((uint32_t)p[5] << 16), p[6] | ((uint32_t)p[7] << 16));
}

// A request, from the tables on the device: its new tokens' first row, their
// number (n_all, of which n rows exist), its length, its query rows a KV head.
struct Request {
    int t0, n, n_all, len, rows;
    int open;  // (kRanges) tokens that all rows see
};

template <int MODE = kPlain>
__device__ __forceinline__ Request request(const PagedAttn &a, int r) {
    Request q;
    q.t0 = table_read(a.starts, r);
    q.n_all = table_read(a.starts, r + 1) - q.t0;
    q.n = q.t0 < 0 ? 0 : (int)max((int64_t)0, min((int64_t)q.n_all, a.n_tokens - q.t0));
    q.len = (int)max((int64_t)0, min((int64_t)table_read(a.lengths, r), a.width << a.st.log_page));
    q.rows = q.n * a.rep;
    q.open = 0;
    if (MODE != kPlain && a.open) q.open = max(0, min(table_read(a.open, r), q.len));
    return q;
}

// The tokens [first_seen, last_seen) that the request's new token i sees; both
// grow with i.
template <int MODE>
__device__ __forceinline__ int last_seen(const PagedAttn &a, const Request &q, int i) {
    if (!a.causal) return q.len;
    const int own = max(0, min(q.len, q.len - q.n_all + i + 1));
    return MODE == kPlain ? own : max(own, q.open);
}
template <int MODE>
__device__ __forceinline__ int first_seen(const PagedAttn &a, const Request &q, int i) {
    if (MODE == kPlain) return 0;
    return max(0, min(q.len, max(0, q.len - q.n_all + i + 1)) - a.window);
}

// The token whose query is row i of the request, and its position among the
// request's tokens.
template <int MODE>
__device__ __forceinline__ int2 token_at(const PagedAttn &a, const Request &q, int i) {
    if (MODE != kPlain && a.rows_of) {
        const int2 t = a.rows_of[q.t0 + i];
        return make_int2(max(0, min(t.x, (int)a.n_tokens - 1)), q.len + t.y);
    }
    return make_int2(q.t0 + i, q.len - q.n_all + i);
}

// Whether request r ends before it begins.  Starts that descend name no rows at
// all: requests that overlap might be more than 32 bits count.
__device__ __forceinline__ bool descends(const PagedAttn &a, int r) {
    return table_read(a.starts, r + 1) < table_read(a.starts, r);
}

// Elements i .. i+3 of the output (i a multiple of 4), of q's 16-bit type.
__device__ __forceinline__ void store_out4(const PagedAttn &a, int64_t i, float x0, float x1, float x2, float x3) {
    const half2_t h0 = __builtin_convertvector(float2_t{x0, x1}, half2_t);
    const half2_t h1 = __builtin_convertvector(float2_t{x2, x3}, half2_t);
    const uint32_t b0 = to_bits16<true>(x0) | (to_bits16<true>(x1) << 16);
    const uint32_t b1 = to_bits16<true>(x2) | (to_bits16<true>(x3) << 16);
    const bool f16 = a.q_dtype == SS_F16;
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + i) =
        make_uint2(f16 ? __builtin_bit_cast(uint32_t, h0) : b0, f16 ? __builtin_bit_cast(uint32_t, h1) : b1);
}

// Row (token t, query head `head`) is done: of its dims c .. c+3 the sums of
// values x, of probabilities l, both times 2^(kPart - m).  Every sum that leaves a
// kernel, or joins another's, is so: bfloat16's largest values stay finite (up to
// 2^20 tokens), and values down to 2^-102 keep their bits.
constexpr int kPart = -24;
template <int MODE, int D>
__device__ __forceinline__ void finish_row(const PagedAttn &a, int r, int64_t t, int head, int c, float m, float l,
                                           float x0, float x1, float x2, float x3) {
    const int64_t at = t * a.hq + head;
    if constexpr (MODE != kPlain) {
        float *const ml = a.part + a.n_tokens * a.hq * D + at * 2;
        float4 *const part = reinterpret_cast<float4 *>(a.part + at * D + c);
        if (a.rows_of || (a.part && table_read(a.parents, r) >= 0)) {
            if (a.rows_of) {
                *part = make_float4(x0, x1, x2, x3);
                if (c == 0) *reinterpret_cast<float2 *>(ml) = make_float2(m, l);
                return;
            }
            const float2 e = *reinterpret_cast<const float2 *>(ml);
            const float4 v = *part;
            const float top = fmaxf(m, e.x);
            const float f = m == top ? 1.f : fast_exp2(m - top), g = e.x == top ? 1.f : fast_exp2(e.x - top);
            l = f * l + g * e.y;
            x0 = f * x0 + g * v.x, x1 = f * x1 + g * v.y, x2 = f * x2 + g * v.z, x3 = f * x3 + g * v.w;
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    store_out4(a, at * D + c, x0 * inv, x1 * inv, x2 * inv, x3 * inv);
}

// A row's products x with tokens 16 (i / 8) + i % 8 become scores in log2 units,
// capped and biased, less the row's reference `ref`.  slope: the head's, in
// log2 units a token; far: how many tokens the row is behind token 0; by: what a
// row's products are multiplied with, and the cap in log2 units.
// A cap's tanh(u) is u times a polynomial of u^2 (of the least largest error below
// |u| = 5/8: 2^-23 of it; 9 operations each), above that 1 - 2 / (1 + exp(2 u)), off
// by 2^-22 (12 operations' time), which is computed where one of the wave's scores is
// that large, hidden ones among them, and taken for those that are.  So a score is
// off by 2^-21 of itself, and its bits are its own, whatever other rows' scores or the
// tokens are that no row sees.  (A prompt of 4093 tokens capped at 50, which few scores
// come near, 303 us; at 15 330, at 3 383.  One form for all of a wave's scores: 299 to
// 302, but small scores were off by 2^-22 of the cap beside a large one.)
// (A bias meets the reference first: both may be large, what is left of them is
// rounded once.)
struct ScoreScale {
    float gain, cap;
    // (The gain is a normal number, whatever the cap: more would make products of 0
    // NaN; for less the cap is lowered to what products below 2^125 do not reach.)
    __device__ ScoreScale(const PagedAttn &a, float factor) : gain(factor), cap(a.cap * kLog2e) {
        if (cap > 0.f) {
            cap = fminf(cap, factor * 0x1p126f);
            gain = fminf(factor / cap, 0x1.fffffep127f);
        }
    }
};
template <int N, bool BIAS, typename X>
__device__ __forceinline__ void apply_rule(const PagedAttn &a, float slope, const ScoreScale &by, float ref, float far, X &x) {
    auto rest = [&](int i) __attribute__((always_inline)) {
        return BIAS ? fmaf(-slope, fabsf(far - (float)(16 * (i / 8) + i % 8)), -ref) : -ref;
    };
    if (a.cap > 0.f) {
        const float cap = by.cap;
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] *= by.gain, most = fmaxf(most, fabsf(x[i]));
        auto small = [&](float u, int i) __attribute__((always_inline)) {
            const float v = u * u;
            float p = fmaf(v, 0.0150509445f, -0.0518218674f);
            p = fmaf(v, p, 0.133045261f);
            p = fmaf(v, p, -0.333319543f);
            p = fmaf(v, p, 0.999999893f);
            return fmaf(u * p, cap, rest(i));
        };
        if (__any(most > 0.625f)) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float u = x[i], e = __builtin_amdgcn_rcpf(1.f + fast_exp2(u * (2.f * kLog2e)));
                x[i] = fabsf(u) <= 0.625f ? small(u, i) : fmaf(-2.f * cap, e, cap + rest(i));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = small(x[i], i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = fmaf(x[i], by.gain, rest(i));
    }
}
template <int N, typename X>
__device__ __forceinline__ void apply_scores(const PagedAttn &a, float slope, const ScoreScale &by, float ref,
                                             float far, X &x) {
    if (a.slopes)
        apply_rule<N, true>(a, slope, by, ref, far, x);
    else
        apply_rule<N, false>(a, slope, by, ref, far, x);
}

// How a query row whose largest magnitude is `top` enters the products: times
// `down`, a power of two that brings it into fp16's range (16-bit queries stay
// exact) with the scale's sign; a sum of products times `factor` is then a
// score in log2 units (codes enter as c/64).  factor is at least 2^-124, or
// masked scores of -inf and the lag of 4 / factor would not be: rows that are
// smaller stay smaller in fp16.  A scale of 0 or NaN is in `down`.
struct QueryScale {
    float down, factor;
    __device__ QueryScale(float top, float scale) {
        const float f = fabsf(scale) * kLog2e * 64.f;
        const int e = (int)((__float_as_uint(f) >> 23) & 0xffu) - 127;  // f >= 2^e
        const int shift = max(row_exp_shift(top), min(-124 - e, 126));
        down = exp2i(-shift) * (scale < 0.f ? -1.f : scale > 0.f ? 1.f : scale);
        factor = fmaxf(f * exp2i(shift), 0x1p-124f);
    }
};

__device__ __forceinline__ int uniform_div(int a, int b) {
    return __builtin_amdgcn_readfirstlane((int)((uint32_t)a / (uint32_t)b));
}

// Where part i of `parts` begins in a column of n units: i n / parts rounded
// down, without the product, which reaches 2^32 (512 parts of 2^23 units).
__device__ __forceinline__ int part_begin(int i, int n, int parts) {
    const int each = uniform_div(n, parts);
    return i * each + uniform_div(i * (n - each * parts), parts);
}

// s_waitcnt vmcnt(N), the other counters unconstrained.
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

template <typename T>
using lds_ptr = __attribute__((address_space(3))) T *;

template <typename T>
__device__ __forceinline__ lds_ptr<T> as_lds(void *p) {
    return reinterpret_cast<lds_ptr<T>>(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)));
}

// A word's eight codes c as the four registers of an operand, 1 + c/64 each.
// (The constants in registers that the compiler does not see through: as
// literals they would take an and, an or where one instruction does both.)
struct CodeBits {
    uint32_t bits = 0x00f000f0u, one = 0x3c003c00u;
    __device__ CodeBits() { asm volatile("" : "+s"(bits), "+v"(one)); }
};
__device__ __forceinline__ half8_t codes_operand(uint32_t w, const CodeBits &k) {
    union {
        uint32_t u[4];
        half8_t h;
    } x;
    x.u[0] = ((w << 4) & k.bits) | k.one;
    x.u[1] = (w & k.bits) | k.one;
    x.u[2] = ((w >> 4) & k.bits) | k.one;
    x.u[3] = ((w >> 8) & k.bits) | k.one;
    return x.h;
}

template <int N>
__device__ __forceinline__ void read_words(const char *p, uint32_t (&w)[N]) {
    if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        w[0] = u.x, w[1] = u.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 u = reinterpret_cast<const uint4 *>(p)[i];
            w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
    }
}

// Halves of a (scale, zero) pair.
template <bool BF>
__device__ __forceinline__ float low16(uint32_t u) {
    if (BF) return __uint_as_float(u << 16);
    return (float)__builtin_bit_cast(half2_t, u)[0];
}
template <bool BF>
__device__ __forceinline__ float high16(uint32_t u) {
    if (BF) return __uint_as_float(u & 0xffff0000u);
    return (float)__builtin_bit_cast(half2_t, u)[1];
}

template <int N>
__device__ __forceinline__ float column_max(const float (&x)[N]) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
    return m;
}

constexpr int kPromptTile = 256;  // query rows of a workgroup of the prompt kernel

// The requests with more than most_rows query rows a KV head (paged_prompt.hip),
// with `workspace` of paged_prompt_bytes for n_tokens * rep rows in all (with
// less no column is cut; `uneven`: of calls with options, whose rows see what
// is before them).
size_t paged_prompt_bytes(const ss_paged_store *s, int64_t n_requests, int64_t rows, int most_rows, bool uneven);
int launch_paged_prompt(PagedAttn a, const ss_paged_store *s, int mode, int64_t n_groups, void *workspace, size_t workspace_bytes,
                        hipStream_t st);

}  // namespace ss
