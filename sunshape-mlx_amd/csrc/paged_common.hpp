// The paged 4-bit cache's layout and 16-bit floats (paged.hip, paged_attn.hip).
#pragma once

#include "ss_common.hpp"

namespace ss {

struct PagedStore {
    uint32_t *k_codes;  // [n_pages][heads][P][D/8]
    uint32_t *v_codes;  // [n_pages][heads][P/8][D]
    uint32_t *k_meta;   // [n_pages][heads][G][P] (scale low, zero high)
    uint32_t *v_meta;
    int n_pages, heads, log_page;
};

// Workgroups of 256 threads in a launch: the runtime counts its threads in 32 bits.
constexpr int64_t kMostGroups = UINT32_MAX / 256;

// Checks a caller's store; its shape in *out.
int check_paged_store(const ss_paged_store *s, PagedStore *out, int *log_page);

// Bit of element j of a word of eight codes.
__host__ __device__ constexpr int nibble_bit(int j) { return 4 * (j >> 1) + 16 * (j & 1); }

template <bool BF>
constexpr uint32_t kNan16 = BF ? 0x7fc0u : 0x7e00u;

template <bool BF>
__device__ __forceinline__ float from_bits16(uint32_t u) {
    if (BF) return __uint_as_float(u << 16);
    return __half2float(__ushort_as_half((unsigned short)u));
}

// Nearest 16-bit float, ties to even.
template <bool BF>
__device__ __forceinline__ uint32_t to_bits16(float x) {
    if (BF) return __bfloat16_as_ushort(__float2bfloat16(x));
    return __half_as_ushort(__float2half(x));
}

// Two nearest 16-bit floats (one instruction), `a` in the low half.
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    if (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), b2));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), h2));
}

}  // namespace ss
