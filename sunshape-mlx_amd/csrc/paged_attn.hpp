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
};

__device__ __forceinline__ Request request(const PagedAttn &a, int r) {
    Request q;
    q.t0 = table_read(a.starts, r);
    q.n_all = table_read(a.starts, r + 1) - q.t0;
    q.n = q.t0 < 0 ? 0 : (int)max((int64_t)0, min((int64_t)q.n_all, a.n_tokens - q.t0));
    q.len = (int)max((int64_t)0, min((int64_t)table_read(a.lengths, r), a.width << a.st.log_page));
    q.rows = q.n * a.rep;
    return q;
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

// Inclusive sum over the lanes before (lane moves, no LDS).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 -> rows 1, 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 -> rows 2, 3
    return v;
}

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
// less no column is cut).
size_t paged_prompt_bytes(const ss_paged_store *s, int64_t n_requests, int64_t rows, int most_rows);
int launch_paged_prompt(PagedAttn a, const ss_paged_store *s, void *workspace, size_t workspace_bytes,
                        hipStream_t st);

}  // namespace ss
