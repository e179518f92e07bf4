// Attention over a paged cache of 4-bit keys and values: the few query rows
// of decode steps and speculative verification (paged_prompt.hip takes the
// many rows of prompts).
//
//   S[r][t] = sum_g s_tg (q_rg . c_tg) + z_tg sum(q_rg)
//   O[r][d] = sum_t (p_rt s'_tg) c'_td + sum_t p_rt z'_tg,   g = d's group
//
// with c the keys' codes, s and z their scales and zeros (primed: the
// values').  Codes enter the matrix cores as they are: a 4-bit code in the
// low bits of a 16-bit half is the fp16 subnormal c * 2^-24, one place
// further left c * 2^-20, and v_mfma_f32_16x16x32_f16 takes subnormals
// exactly, so two masks and half a shift turn eight codes into the four
// registers of an operand and no code is ever converted.  The factor 16
// between the places is taken from the other operand (queries, respectively
// probabilities, of odd pairs times 2^-4); 2^24 goes into the factors that
// the sums are multiplied by in any case.
//
// Scales stay out of the operands: the 16 columns of both products are
// (row r, group g), a query entering column (r, g) with the dims of group g
// alone.  Keys are the A operand (16 tokens), so a lane holds, of one column,
// 4 tokens of each key tile; two key tiles whose token order is chosen so
// make exactly the lane's 8 tokens of the second product's B operand: the
// probabilities never leave the lane's registers.
#include <type_traits>

#include "paged_common.hpp"

namespace ss {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float2_t __attribute__((ext_vector_type(2)));

constexpr int kTile = 32;          // tokens a wave takes at a time
constexpr int kWaves = 4;          // waves of a workgroup
constexpr int kUnit = kTile * kWaves;
constexpr int kMaxSplits = 64;
constexpr int kStages = 4;         // tiles of a wave in LDS, one computed while the others arrive
constexpr int kNt = 2;             // cache policy of the stream: non-temporal
// How far, in log2, a score may pass the running maximum before the maximum
// moves: probabilities stay below 2^4, so p * scale stays within fp16 with
// scales normalised to 2^10.
constexpr float kLag = 4.f;

struct PagedAttn {
    PagedStore st;
    const void *q;
    int64_t q_st, q_sh;
    void *out;
    const int32_t *table, *lengths, *starts;
    int64_t width, n_tokens;
    int n_req, hq, rep, q_dtype, causal, zero_rest, vec;
    float scale;
    int splits, chunk;  // grid's splits; tokens of a split (a multiple of kUnit)
    int row_cap;        // rows a KV head that the workspace holds
    float *acc;         // [n_req][heads][row_cap][splits][D]
    float *ml;          // [n_req][heads][row_cap][splits][2]
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

// A request's rows, length and splits, from the tables on the device.
struct Request {
    int t0, n, n_all, len, rows, splits, chunk;
};

__device__ __forceinline__ Request request(const PagedAttn &a, int r) {
    Request q;
    q.t0 = table_read(a.starts, r);
    q.n_all = table_read(a.starts, r + 1) - q.t0;
    q.n = q.t0 < 0 ? 0 : (int)max((int64_t)0, min((int64_t)q.n_all, a.n_tokens - q.t0));
    q.len = (int)max((int64_t)0, min((int64_t)table_read(a.lengths, r), a.width << a.st.log_page));
    q.rows = q.n * a.rep;
    // more tokens than the launch was sized for: longer splits; more rows than
    // the workspace holds: one split, which writes the rows itself
    const int need = (q.len + a.splits - 1) / a.splits;
    q.chunk = max(a.chunk, (need + kUnit - 1) / kUnit * kUnit);
    q.splits = max(1, (q.len + q.chunk - 1) / q.chunk);
    if (q.rows > a.row_cap) {
        q.splits = 1;
        q.chunk = INT32_MAX;
    }
    return q;
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

// 32 tokens of one KV head as they lie in LDS: key rows, value blocks, the
// keys' and the values' (scale, zero) pairs [G][32].  16-byte pieces move
// within their row or block so that the reads below touch every bank once:
// piece c of key row t sits at place c ^ (t / 8) % (pieces a row), piece c of
// a value block at c ^ (c / 16) % 2.
template <int D, int G>
struct TileLds {
    static constexpr int kCodes = 16 * D;       // bytes of the keys' codes, and of the values'
    static constexpr int kMeta = G * kTile * 4; // bytes of the keys' pairs, and of the values'
    static constexpr int kBytes = 2 * (kCodes + kMeta);
    static constexpr int kKP = D / 32;          // 16-byte pieces of a key row
    static constexpr int kVP = D / 4;           // of a value block
    static constexpr int kLoads = 2 * (kCodes / 1024) + 1;
    static constexpr int kMetaLanes = 2 * kMeta / 16;

    // Starts copying the tile of tokens tb .. tb + 31 (pages p0 and p1) into a slot.
    __device__ static void fetch(const PagedStore &st, int h, int lane, char *slot, int tb, int p0, int p1) {
        const int heads = st.heads, log_page = st.log_page, in_page = (1 << log_page) - 1;
        const int64_t row0 = (int64_t)max(p0, 0) * heads + h, row1 = (int64_t)max(p1, 0) * heads + h;
        const int off0 = tb & in_page, off1 = (tb + 16) & in_page;
#pragma unroll
        for (int i = 0; i < kCodes / 1024; ++i) {
            // place -> (row or block, piece) -> address
            const int place = i * 64 + lane;
            const int kt = place / kKP, kc = (place % kKP) ^ ((kt >> 3) % kKP);
            const bool second = D == 128 ? i == 1 : lane >= 32;
            const int64_t row = second ? row1 : row0;
            const int off = second ? off1 : off0;
            const uint32_t *k = st.k_codes + ((row << log_page) + off) * (D / 8);
            __builtin_amdgcn_global_load_lds(k + (kt % 16) * (D / 8) + kc * 4, as_lds<void>(slot + i * 1024), 16, 0, kNt);
            const int vb = place / kVP, vc = (place % kVP) ^ (((place % kVP) >> 4) & 1);
            const uint32_t *v = st.v_codes + (((row << log_page) + off) >> 3) * D;
            __builtin_amdgcn_global_load_lds(v + (vb % 2) * D + vc * 4, as_lds<void>(slot + kCodes + i * 1024), 16,
                                             0, kNt);
        }
        if (kMetaLanes == 64 || lane < kMetaLanes) {
            const int e = lane % (kMetaLanes / 2), mg = e / 8, t = e % 8 * 4;
            const int64_t row = t >= 16 ? row1 : row0;
            const int off = (t >= 16 ? off1 : off0) + t % 16;
            const uint32_t *m = lane < kMetaLanes / 2 ? st.k_meta : st.v_meta;
            __builtin_amdgcn_global_load_lds(m + ((row * G + mg) << log_page) + off,
                                             as_lds<void>(slot + 2 * kCodes), 16, 0, kNt);
        }
    }
};

// A word's eight codes as the four registers of an operand: pairs (0,1) and
// (4,5) times 2^-24, (2,3) and (6,7) times 2^-20.
__device__ __forceinline__ half8_t codes_operand(uint32_t w) {
    union {
        uint32_t u[4];
        half8_t h;
    } x;
    const uint32_t hi = w >> 8;
    x.u[0] = w & 0x000f000fu;
    x.u[1] = w & 0x00f000f0u;
    x.u[2] = hi & 0x000f000fu;
    x.u[3] = hi & 0x00f000f0u;
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

template <int N>
__device__ __forceinline__ float column_max(const float (&x)[N]) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
    return m;
}

// Over the four lanes of a column (lane%16 equal).
__device__ __forceinline__ float lanes4_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float lanes4_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Over the groups of a row (neighbouring columns).
template <int G>
__device__ __forceinline__ float groups_sum(float v) {
    if (G >= 2) v += dpp_mov<0xB1>(v);  // quad_perm [1,0,3,2]
    if (G >= 4) v += dpp_mov<0x4E>(v);  // quad_perm [2,3,0,1]
    return v;
}

// One workgroup: split blockIdx.x of the tokens of (request blockIdx.z, KV
// head), for NS column sets of 16/G query rows that share the stream.  Its
// waves take 32-token tiles in turn, the next tile's loads in flight while
// one is computed, and their results are joined through LDS at the end.
template <int D, int G, bool BF, int NS>
__global__ void __launch_bounds__(256, 2) paged_attn_kernel(const PagedAttn a) {
    constexpr int RS = 16 / G;       // rows of a column set
    constexpr int ROWS = RS * NS;    // rows of a workgroup
    constexpr int KS = D / 32;       // matrix steps over a head's dims
    constexpr int VT = D / 16;       // 16-dim tiles of the values
    constexpr int OP = D + 4;        // a row of the waves' results in LDS
    using TL = TileLds<D, G>;
    constexpr int kRing = kWaves * kStages * TL::kBytes, kJoin = kWaves * ROWS * (OP + 2) * 4;
    // the waves' tiles, then their results
    __shared__ __attribute__((aligned(16))) char lds[kRing > kJoin ? kRing : kJoin];
    float(*part)[ROWS][OP] = reinterpret_cast<float(*)[ROWS][OP]>(lds);
    float(*stats)[ROWS][2] = reinterpret_cast<float(*)[ROWS][2]>(lds + kWaves * ROWS * OP * 4);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int g = col % G;
    const bool in_group = quad * G / 4 == g;  // the lane's dims, and its rows of O, are in the column's group
    const int heads = a.st.heads, log_page = a.st.log_page, in_page = (1 << log_page) - 1;
    const int h = blockIdx.y % heads, r = blockIdx.z, split = blockIdx.x;
    const int blocks = gridDim.y / heads;

    if (a.zero_rest && r == a.n_req - 1 && split == 0 && (int)blockIdx.y < heads) {
        const int64_t from = max(0, table_read(a.starts, a.n_req));
        const int64_t per = (int64_t)a.rep * D;  // outputs of this KV head in a row, contiguous
        for (int64_t e = threadIdx.x; e < (a.n_tokens - from) * per; e += 256) {
            const int64_t t = e / per;
            store_from_f32(a.out, a.q_dtype, ((from + t) * a.hq + h * a.rep) * D + (e - t * per), 0.f);
        }
    }
    const Request rq = request(a, r);
    if (rq.rows == 0 || split >= rq.splits) return;
    const int begin = split * rq.chunk;
    const int end = (int)min((int64_t)begin + rq.chunk, (int64_t)rq.len);
    const int32_t *row_table = a.table + (int64_t)r * a.width;

    char *ring = lds + wave * kStages * TL::kBytes;
    // Page of the 16 tokens from `token`; -1 if the table names none of the pool.
    auto page_at = [&](int token) {
        const int p = table_read(row_table, min((int64_t)(token >> log_page), a.width - 1));
        return (uint32_t)p < (uint32_t)a.st.n_pages ? p : -1;
    };
    for (int rb = blockIdx.y / heads; rb * ROWS < rq.rows; rb += blocks) {
        // queries first: what is loaded later would hold them back
        int limit[NS];  // tokens that the column's row sees
        uint4 raw[NS][KS];
        bool live[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int row = rb * ROWS + s * RS + col / G;
            live[s] = row < rq.rows;
            const int i = live[s] ? row / a.rep : 0, hd = live[s] ? row % a.rep : 0;
            limit[s] = live[s] && a.causal ? max(0, min(rq.len, rq.len - rq.n_all + i + 1)) : rq.len;
            const uint16_t *q =
                static_cast<const uint16_t *>(a.q) + (rq.t0 + i) * a.q_st + (h * a.rep + hd) * a.q_sh + quad * (D / 4);
#pragma unroll
            for (int k = 0; k < KS; ++k) raw[s][k] = load_query8(q + 8 * k, a.vec);
        }
        int ahead = begin + kTile * wave;  // next tile to fetch
        int pages[kStages][2];             // of the tiles in flight, the oldest first
#pragma unroll
        for (int i = 0; i < kStages; ++i) {
            pages[i][0] = page_at(ahead), pages[i][1] = page_at(ahead + 16);
            if (i < kStages - 1 && ahead < end) TL::fetch(a.st, h, lane, ring + i * TL::kBytes, ahead, pages[i][0], pages[i][1]);
            ahead += kUnit;
        }
        int all_see = rq.len;
        half8_t qf[NS][KS];
        float qz[NS], factor[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            float x[KS][8], top = 0.f, sum = 0.f;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                float xh[8], xb[8];
                unpack16<__half>(raw[s][k], xh);
                unpack16<__hip_bfloat16>(raw[s][k], xb);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[k][e] = live[s] ? (a.q_dtype == SS_F16 ? xh[e] : xb[e]) : 0.f;
                    top = fmaxf(top, fabsf(x[k][e]));
                }
            }
            // a power of two brings the row into fp16's range: 16-bit
            // queries stay exact
            const int shift = row_exp_shift(lanes4_max(top));
            const float down = exp2i(-shift);
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float y = in_group ? x[k][e] * down : 0.f;
                    sum += y;
                    qf[s][k][e] = (_Float16)((e & 2) ? y * 0x1p-4f : y);
                }
            qz[s] = lanes4_sum(sum) * 0x1p-24f;
            factor[s] = a.scale * kLog2e * 0x1p24f * exp2i(shift);
        }
        // (limits grow with the row: the first row's is the smallest)
        if (a.causal) all_see = max(0, min(rq.len, rq.len - rq.n_all + rb * ROWS / a.rep + 1));

        float top[NS], l_even[NS], l_odd[NS], z_even[NS], z_odd[NS];
        float4_t o[NS][VT];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            top[s] = -INFINITY;
            l_even[s] = l_odd[s] = z_even[s] = z_odd[s] = 0.f;
#pragma unroll
            for (int j = 0; j < VT; ++j) o[s][j] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
        float vlim = 0.f;  // power of two, above every value scale seen in the column's group

        // masked: some row does not see some token of the tile
        auto compute = [&](const char *slot, int tb, bool ok, auto masked) {
            constexpr bool mask = decltype(masked)::value;
            uint32_t kw[2][KS], vw[VT], km[8], vm[8];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                // key tile y, row col: token 8*(col/4) + 4y + col%4
                const int t = 8 * (col >> 2) + 4 * y + (col & 3);
                if constexpr (KS == 4) {
                    read_words(slot + (t * TL::kKP + (quad ^ ((t >> 3) % TL::kKP))) * 16, kw[y]);
                } else {
                    read_words(slot + (t * TL::kKP + ((quad >> 1) ^ ((t >> 3) % TL::kKP))) * 16 + (quad & 1) * 8, kw[y]);
                }
            }
#pragma unroll
            for (int i = 0; i < VT / 4; ++i) {
                const int c = col * (VT / 4) + i;
                uint32_t w4[4];
                read_words(slot + TL::kCodes + (quad * TL::kVP + (c ^ ((c >> 4) & 1))) * 16, w4);
#pragma unroll
                for (int k = 0; k < 4; ++k) vw[4 * i + k] = w4[k];
            }
            read_words(slot + 2 * TL::kCodes + (g * kTile + 8 * quad) * 4, km);
            read_words(slot + 2 * TL::kCodes + TL::kMeta + (g * kTile + 8 * quad) * 4, vm);
            float ks[8], kz[8], vs[8], vz[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                ks[j] = from_bits16<BF>(km[j] & 0xffffu);
                kz[j] = from_bits16<BF>(km[j] >> 16);
                vs[j] = from_bits16<BF>(vm[j] & 0xffffu);
                vz[j] = from_bits16<BF>(vm[j] >> 16);
            }
            const int first = tb + 8 * quad;  // the lane's first token
            if (mask) {  // (behind the request's tokens a page may hold anything, NaN too)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!ok || first + j >= rq.len) vs[j] = 0.f;
            }
            // value scales enter the product times 2^10 / vlim
            const float vtop = column_max(vs);
            float vlim_was = vlim;
            if (__any(vtop > vlim)) {
                const float c = lanes4_max(vtop);
                if (c > vlim) {
                    const int e = (int)((__float_as_uint(c) >> 23) & 0xffu) - 126;  // c < 2^e
                    vlim = exp2i(max(-100, min(126, e)));
                }
                const float f = vlim_was > 0.f ? vlim_was / vlim : 1.f;
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int j = 0; j < VT; ++j) o[s][j] *= f;
            }
            const float vn = vlim > 0.f ? 0x1p10f / vlim : 0.f;
            half8_t p16[NS];
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                float x[8];
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < KS; ++k)
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_operand(kw[y][k]), qf[s][k], d, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = 4 * y + i;
                        x[j] = groups_sum<G>(fmaf(d[i], ks[j], kz[j] * qz[s])) * factor[s];
                    }
                }
                if (mask) {
                    const int see = ok ? limit[s] : 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (first + j >= see) x[j] = -INFINITY;
                }
                const float m = column_max(x);
                if (__any(m > top[s] + kLag)) {
                    const float now = fmaxf(top[s], lanes4_max(m));
                    const float f = now == top[s] ? 1.f : fast_exp2(top[s] - now);
                    top[s] = now;
                    l_even[s] *= f, l_odd[s] *= f, z_even[s] *= f, z_odd[s] *= f;
#pragma unroll
                    for (int j = 0; j < VT; ++j) o[s][j] *= f;
                }
                // pairs (2,3) and (6,7), whose codes count 16 times, at 2^-4
                const float even = top[s] == -INFINITY ? 0.f : top[s], odd = even + 4.f;
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float p = fast_exp2(x[j] - ((j & 2) ? odd : even));
                    // (a token that the row does not see adds nothing, whatever its value holds)
                    const bool off = mask && (!ok || first + j >= limit[s]);
                    const float z = off ? 0.f : vz[j];
                    if (j & 2) {
                        l_odd[s] += p;
                        z_odd[s] = fmaf(p, z, z_odd[s]);
                    } else {
                        l_even[s] += p;
                        z_even[s] = fmaf(p, z, z_even[s]);
                    }
                    w[j] = off ? 0.f : p * (vs[j] * vn);
                }
                // one rounding to fp16 (2^-11 of the term): the sums stay float32
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const half2_t hh = __builtin_convertvector(float2_t{w[j], w[j + 1]}, half2_t);
                    p16[s][j] = hh[0], p16[s][j + 1] = hh[1];
                }
            }
#pragma unroll
            for (int j = 0; j < VT; ++j) {
                const half8_t v = codes_operand(vw[j]);
#pragma unroll
                for (int s = 0; s < NS; ++s)
                    o[s][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p16[s], o[s][j], 0, 0, 0);
            }
        };

        // one tile: the next to fetch goes into `into`, the oldest is at `slot`
        auto step = [&](char *__restrict into, const char *__restrict slot, int tb, int p0, int p1, int next0,
                        int next1) {
            if (tb + (kStages - 1) * kUnit < end) {
                TL::fetch(a.st, h, lane, into, tb + (kStages - 1) * kUnit, next0, next1);
                wait_loads<(kStages - 1) * TL::kLoads>();
            } else {
                wait_loads<0>();
            }
            const bool ok = (quad < 2 ? p0 : p1) >= 0;
            if (tb + kTile > all_see || p0 < 0 || p1 < 0)
                compute(slot, tb, ok, std::true_type{});
            else
                compute(slot, tb, ok, std::false_type{});
        };
        int slot = 0;
        for (int tb = begin + kTile * wave; tb < end; tb += kUnit) {
            constexpr int last = kStages - 1;
            step(ring + (slot + last) % kStages * TL::kBytes, ring + slot * TL::kBytes, tb, pages[0][0], pages[0][1],
                 pages[last][0], pages[last][1]);
            slot = (slot + 1) % kStages;
#pragma unroll
            for (int i = 0; i < last; ++i) pages[i][0] = pages[i + 1][0], pages[i][1] = pages[i + 1][1];
            pages[last][0] = page_at(ahead), pages[last][1] = page_at(ahead + 16);
            ahead += kUnit;
        }
        __syncthreads();  // (the ring's memory takes the results)

        // the waves' results, joined
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const float l = lanes4_sum(l_even[s] + 16.f * l_odd[s]);
            const float z = lanes4_sum(z_even[s] + 16.f * z_odd[s]);
            const int row = s * RS + col / G;
            if (g == 0 && quad == 0) stats[wave][row][0] = top[s], stats[wave][row][1] = l;
            if (in_group) {
                // tile j, element i: dim (4 * quad + i) * D/16 + j
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < VT; ++j)
                        part[wave][row][(4 * quad + i) * VT + j] = o[s][j][i] * 0x1p14f * vlim + z;
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < ROWS * (D / 4); e += 256) {
            const int row = e / (D / 4), c = e % (D / 4) * 4, n = rb * ROWS + row;
            if (n >= rq.rows) break;
            float m = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) m = fmaxf(m, stats[w][row][0]);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float mw = stats[w][row][0];
                const float f = mw == m ? 1.f : fast_exp2(mw - m);
                l += f * stats[w][row][1];
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] += f * part[w][row][c + k];
            }
            if (rq.splits == 1) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const int64_t at = ((int64_t)(rq.t0 + n / a.rep) * a.hq + h * a.rep + n % a.rep) * D + c;
                store4_from_f32(a.out, a.q_dtype, at, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
            } else {
                const int64_t at = (((int64_t)r * heads + h) * a.row_cap + n) * a.splits + split;
                *reinterpret_cast<float4 *>(a.acc + at * D + c) = make_float4(x[0], x[1], x[2], x[3]);
                if (c == 0) *reinterpret_cast<float2 *>(a.ml + at * 2) = make_float2(m, l);
            }
        }
        __syncthreads();
    }
}

// The rows of requests that were split, one workgroup a row: every thread
// loads four dims of its splits at once, 8 (D 128) or 16 threads a dim.
template <int D>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedAttn a) {
    constexpr int CH = D / 4, PARTS = 256 / CH, PER = kMaxSplits / PARTS;
    __shared__ float red[PARTS][D + 4];
    __shared__ float weight[kMaxSplits];
    __shared__ float total;
    const int r = blockIdx.y, heads = a.st.heads;
    const Request rq = request(a, r);
    if (rq.splits == 1) return;
    const int c = threadIdx.x % CH * 4, p = threadIdx.x / CH;
    for (int e = blockIdx.x; e < rq.rows * heads; e += gridDim.x) {
        const int h = e % heads, n = e / heads;
        const int64_t at = (((int64_t)r * heads + h) * a.row_cap + n) * a.splits;
        float4 v[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i)
            v[i] = *reinterpret_cast<const float4 *>(a.acc + (at + min(p + i * PARTS, rq.splits - 1)) * D + c);
        if (threadIdx.x < 64) {
            const bool in = (int)threadIdx.x < rq.splits;
            const float2 s = *reinterpret_cast<const float2 *>(a.ml + (at + min((int)threadIdx.x, rq.splits - 1)) * 2);
            const float m = wave_max(in ? s.x : -INFINITY);
            const float f = in ? (s.x == m ? 1.f : fast_exp2(s.x - m)) : 0.f;
            weight[threadIdx.x] = f;
            const float l = wave_sum(in ? f * s.y : 0.f);
            if (threadIdx.x == 0) total = l;
        }
        __syncthreads();
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int s = p + i * PARTS;
            if (s >= rq.splits) break;
            const float f = weight[s];
            x[0] += f * v[i].x, x[1] += f * v[i].y, x[2] += f * v[i].z, x[3] += f * v[i].w;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) red[p][c + k] = x[k];
        __syncthreads();
        if (threadIdx.x < CH) {
            float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < PARTS; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] += red[i][c + k];
            const float inv = total == 0.f ? 0.f : 1.f / total;
            const int64_t o = ((int64_t)(rq.t0 + n / a.rep) * a.hq + h * a.rep + n % a.rep) * D + c;
            store4_from_f32(a.out, a.q_dtype, o, y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
        }
        __syncthreads();
    }
}

// -------------------------------------------------------------------- host

struct PagedPlan {
    int sets, blocks, splits, chunk, row_cap;
    size_t bytes;
};

// Launch shape from the hints.  Workgroups are cheap to leave, so the splits
// aim at enough of them to fill the device when every request is as long as
// the longest.
static PagedPlan paged_plan(const ss_paged_store *s, int64_t n_requests, int n_q_heads, int64_t max_new,
                            int64_t max_length) {
    PagedPlan p;
    const int rep = n_q_heads / s->n_kv_heads, rs = 16 / (s->head_dim / s->group_size);
    const int64_t rows = max_new * rep;
    p.sets = rows > rs ? 2 : 1;
    p.blocks = (int)max((int64_t)1, min((rows + p.sets * rs - 1) / (p.sets * rs), (int64_t)64));
    p.row_cap = p.blocks * p.sets * rs;
    const int64_t groups = n_requests * s->n_kv_heads * p.blocks;
    const int64_t want = (4 * device_cu_count() + groups - 1) / groups;
    const int64_t most = max((int64_t)1, min((int64_t)kMaxSplits, max_length / (2 * kUnit)));
    const int64_t n = max((int64_t)1, min(want, most));
    p.chunk = (int)(((max_length + n - 1) / n + kUnit - 1) / kUnit * kUnit);
    p.chunk = max(p.chunk, kUnit);
    p.splits = (int)n;
    p.bytes = p.splits > 1 ? (size_t)n_requests * s->n_kv_heads * p.row_cap * p.splits * (s->head_dim + 2) * 4 : 0;
    return p;
}

static int check_hints(const ss_paged_store *s, int64_t n_requests, int n_q_heads, int64_t max_new,
                       int64_t max_length) {
    SS_REQUIRE(n_requests >= 1 && n_requests <= 65535, "n_requests must be 1 .. 65535");
    SS_REQUIRE(n_q_heads >= 1 && n_q_heads % s->n_kv_heads == 0,
               "query heads must be a multiple of the KV heads");
    SS_UNSUPPORTED(n_q_heads <= 1024, "more than 1024 query heads");
    SS_REQUIRE(max_new >= 1 && max_new <= INT32_MAX / 1024 && max_length >= 1 && max_length <= INT32_MAX,
               "max_new and max_length must be positive");
    return SS_OK;
}

template <int D, int G, bool BF>
static void launch_paged(const PagedAttn &a, const PagedPlan &p, hipStream_t st) {
    const dim3 grid(p.splits, a.st.heads * p.blocks, a.n_req);
    if (p.sets == 1)
        hipLaunchKernelGGL((paged_attn_kernel<D, G, BF, 1>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((paged_attn_kernel<D, G, BF, 2>), grid, dim3(256), 0, st, a);
    if (p.splits > 1)
        hipLaunchKernelGGL(paged_merge_kernel<D>, dim3(p.row_cap * a.st.heads, a.n_req), dim3(256), 0, st, a);
}

}  // namespace ss

using namespace ss;

extern "C" size_t ss_paged_attn_workspace_bytes(const ss_paged_store *store, int64_t n_requests, int n_q_heads,
                                                int64_t max_new, int64_t max_length) {
    PagedStore ps;
    int log_page;
    if (check_paged_store(store, &ps, &log_page) || check_hints(store, n_requests, n_q_heads, max_new, max_length))
        return 0;
    return paged_plan(store, n_requests, n_q_heads, max_new, max_length).bytes;
}

extern "C" int ss_paged_attn(const ss_paged_store *store, const void *q, int q_dtype, int64_t n_tokens,
                             int64_t q_st, int64_t q_sh, int n_q_heads, const int32_t *block_table,
                             int64_t table_width, const int32_t *lengths, const int32_t *token_starts,
                             int64_t n_requests, float scale, int causal, int64_t max_new, int64_t max_length,
                             void *out, int zero_rest, void *workspace, size_t workspace_bytes, void *stream) {
    PagedAttn a;
    int log_page;
    if (int rc = check_paged_store(store, &a.st, &log_page)) return rc;
    if (int rc = check_hints(store, n_requests, n_q_heads, max_new, max_length)) return rc;
    SS_UNSUPPORTED(q_dtype == SS_F16 || q_dtype == SS_BF16, "queries must be float16 or bfloat16");
    SS_REQUIRE(n_tokens >= 0, "bad token count");
    if (n_tokens == 0) return SS_OK;
    SS_UNSUPPORTED(n_tokens <= INT32_MAX / n_q_heads, "too many query rows for one launch");
    SS_REQUIRE(q && out && block_table && lengths && token_starts, "null pointer argument");
    SS_REQUIRE(table_width >= 1, "bad block table width");
    SS_UNSUPPORTED(table_width <= (1 << 30) / store->page_size, "a table row of more than 2^30 tokens");
    const PagedPlan p = paged_plan(store, n_requests, n_q_heads, max_new, max_length);
    if (p.bytes > workspace_bytes || (p.bytes && !workspace)) {
        set_error("workspace of %zu bytes, %zu needed", workspace_bytes, p.bytes);
        return SS_ERR_WORKSPACE;
    }
    SS_REQUIRE(((uintptr_t)workspace & 15) == 0, "workspace must be 16-byte aligned");
    a.q = q, a.q_st = q_st, a.q_sh = q_sh, a.out = out;
    a.table = block_table, a.lengths = lengths, a.starts = token_starts;
    a.width = table_width, a.n_tokens = n_tokens, a.n_req = (int)n_requests;
    a.hq = n_q_heads, a.rep = n_q_heads / store->n_kv_heads;
    a.q_dtype = q_dtype, a.causal = causal, a.zero_rest = zero_rest, a.scale = scale;
    a.vec = ((uintptr_t)q & 15) == 0 && q_st % 8 == 0 && q_sh % 8 == 0;
    a.splits = p.splits, a.chunk = p.chunk, a.row_cap = p.row_cap;
    a.acc = static_cast<float *>(workspace);
    a.ml = a.acc + (size_t)n_requests * store->n_kv_heads * p.row_cap * p.splits * store->head_dim;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const bool bf = store->dtype == SS_BF16;
    const int key = store->head_dim * 1000 + store->group_size;
    if (key == 128032) bf ? launch_paged<128, 4, true>(a, p, st) : launch_paged<128, 4, false>(a, p, st);
    else if (key == 128064) bf ? launch_paged<128, 2, true>(a, p, st) : launch_paged<128, 2, false>(a, p, st);
    else if (key == 128128) bf ? launch_paged<128, 1, true>(a, p, st) : launch_paged<128, 1, false>(a, p, st);
    else if (key == 64032) bf ? launch_paged<64, 2, true>(a, p, st) : launch_paged<64, 2, false>(a, p, st);
    else bf ? launch_paged<64, 1, true>(a, p, st) : launch_paged<64, 1, false>(a, p, st);
    SS_LAUNCH_CHECK("paged_attn_kernel launch");
    return SS_OK;
}
