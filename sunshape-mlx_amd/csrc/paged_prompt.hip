// Attention over a paged cache of 4-bit keys and values: prompts, and chunks of
// long ones (paged_attn.hpp has the formulas).
//
// A workgroup takes 128 query rows of one KV head (its group's heads at
// consecutive positions), 32 a wave, over 64-token tiles.  Scores are exact:
// key codes enter v_mfma_f32_32x32x16_f16 unconverted, group by group, and
// every product sum is multiplied by its token's scale in float32; the zeros'
// part is one more product, of the zeros and the queries' sums, both split
// into bf16 parts.  Values are shared by all rows, so the workgroup
// dequantises each tile once, to fp16 in LDS, while the tile before it is
// computed; times a power of two a group that keeps the largest value met
// below 2^-6 (a code's factor then stays within fp16: code * 2^-24 times
// scale * 2^18).  Rounding them costs 2^-11 of a value, as the probabilities'
// rounding does; statistics and sums are float32.
#include "paged_attn.hpp"

namespace ss {

typedef float float16_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));

constexpr int kRows = 128;    // query rows of a workgroup
constexpr int kTokens = 64;   // of a tile

template <int D, int G>
struct PromptTile {
    // a tile's 16-token segments in LDS: key rows, value blocks, the keys' and
    // the values' (scale, zero) pairs [G][16].  16-byte piece c of key row t
    // sits at place c ^ (t / 4) % (pieces a row).
    static constexpr int kKeys = 8 * D, kMeta = 2 * G * 64;
    static constexpr int kSeg = 2 * kKeys + kMeta;
    static constexpr int kBytes = 4 * kSeg;
    static constexpr int kKP = D / 32;  // 16-byte pieces of a key row

    // Starts copying the segment of 16 tokens in page p (clamped by the
    // caller) from its token `off`.
    __device__ static void fetch(const PagedStore &st, int h, int lane, char *seg, int page, int off) {
        const int64_t row = (int64_t)page * st.heads + h;
        const uint32_t *k = st.k_codes + ((row << st.log_page) + off) * (D / 8);
        const uint32_t *v = st.v_codes + (((row << st.log_page) + off) >> 3) * D;
        const int place = lane % (kKeys / 16), t = place / kKP, c = (place % kKP) ^ ((t >> 2) % kKP);
        const uint32_t *from_k = k + t * (D / 8) + c * 4, *from_v = v + place * 4;
        if constexpr (D == 128) {
            __builtin_amdgcn_global_load_lds(from_k, as_lds<void>(seg), 16, 0, 0);
            __builtin_amdgcn_global_load_lds(from_v, as_lds<void>(seg + kKeys), 16, 0, 0);
        } else {
            __builtin_amdgcn_global_load_lds(lane < 32 ? from_k : from_v, as_lds<void>(seg), 16, 0, 0);
        }
        if (lane < kMeta / 16) {
            const int e = lane % (4 * G);
            const uint32_t *m = lane < 4 * G ? st.k_meta : st.v_meta;
            __builtin_amdgcn_global_load_lds(m + ((row * G + e / 4) << st.log_page) + off + e % 4 * 4,
                                             as_lds<void>(seg + 2 * kKeys), 16, 0, 0);
        }
    }
};

// Row tiles of a request that are this kernel's.
__device__ __forceinline__ int tiles_of(const PagedAttn &a, const Request &q) {
    return q.rows > a.most_rows ? (q.rows + kRows - 1) / kRows : 0;
}

__device__ __forceinline__ float half_max(float v) { return fmaxf(v, __shfl_xor(v, 32)); }

template <int D, int G, bool BF>
__global__ void __launch_bounds__(256, 2) paged_prompt_kernel(const PagedAttn a) {
    using PT = PromptTile<D, G>;
    constexpr int GW = D / 8 / G, HW = GW / 2;  // words of a group, and of a lane's half of it
    constexpr int NT = D / 32;                  // 32-dim tiles of the values
    constexpr int kValues = kTokens * D * 2;    // bytes of a tile's values as fp16
    __shared__ __attribute__((aligned(16))) char lds[3 * PT::kBytes + 2 * kValues];
    char *const raw = lds, *const vals = lds + 3 * PT::kBytes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int heads = a.st.heads, log_page = a.st.log_page, in_page = (1 << log_page) - 1;

    const int per = (a.n_req + 63) / 64, r0 = min(lane * per, a.n_req), r1 = min(r0 + per, a.n_req);
    int mine = 0;
    for (int i = r0; i < r1; ++i) mine += tiles_of(a, request(a, i));
    const int scan = wave_scan(mine);
    const int total = __builtin_amdgcn_readlane(scan, 63) * heads;

    for (int item = blockIdx.x; item < total; item += gridDim.x) {
        // (heads side by side: a head's tiles tend to meet in one L2)
        const int h = item % heads;
        int left = uniform_div(item, heads);
        const int holder = __ffsll((unsigned long long)__ballot(left < scan)) - 1;
        left -= holder ? __builtin_amdgcn_readlane(scan, holder - 1) : 0;
        int r = holder * per;
        Request rq;
        for (;; ++r) {
            rq = request(a, r);
            const int n = tiles_of(a, rq);
            if (left < n) {
                left = n - 1 - left;  // the longest first
                break;
            }
            left -= n;
        }
        const int row0 = left * kRows + wave * 32;  // the wave's first row
        const int32_t *row_table = a.table + (int64_t)r * a.width;
        auto page_at = [&](int token) {
            const int p = table_read(row_table, min((int64_t)(token >> log_page), a.width - 1));
            return (uint32_t)p < (uint32_t)a.st.n_pages ? p : -1;
        };
        auto sees = [&](int row) {  // tokens that a row sees
            return a.causal ? max(0, min(rq.len, rq.len - rq.n_all + row / a.rep + 1)) : rq.len;
        };
        const int last_row = min(left * kRows + kRows, rq.rows) - 1;
        const int end = __builtin_amdgcn_readfirstlane(sees(last_row));          // of the workgroup
        const int wave_last = min(row0 + 31, rq.rows - 1);
        const int wave_end = row0 < rq.rows ? __builtin_amdgcn_readfirstlane(sees(wave_last)) : 0;
        const int all_see = row0 < rq.rows ? __builtin_amdgcn_readfirstlane(sees(row0)) : 0;
        const int row = row0 + col;
        const bool live = row < rq.rows;
        const int limit = live ? sees(row) : rq.len;
        const int n_tiles = (end + kTokens - 1) / kTokens;

        // queries: B operand of step s of group g: dims of word g*GW + half*HW + s
        uint4 rawq[G][HW];
        {
            const int i = live ? row / a.rep : 0, hd = live ? row % a.rep : 0;
            const uint16_t *q = static_cast<const uint16_t *>(a.q) + (rq.t0 + i) * a.q_st + (h * a.rep + hd) * a.q_sh;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int s = 0; s < HW; ++s) rawq[g][s] = load_query8(q + (g * GW + half * HW + s) * 8, a.vec);
        }
        // pages of tile i: the wave copies the segment of tokens 16 * wave ..
        auto fetch = [&](char *slot, int tile) {
            const int tb = tile * kTokens + 16 * wave;
            PT::fetch(a.st, h, lane, slot + wave * PT::kSeg, max(page_at(tb), 0), tb & in_page);
        };
        auto pages_ok = [&](int tile) {  // bit w: the page of tokens 16 w .. is in the pool
            int ok = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) ok |= (page_at(tile * kTokens + 16 * w) >= 0 ? 1 : 0) << w;
            return ok;
        };
        wait_loads<0>();  // the queries, before tiles are waited for with them
        if (n_tiles > 0) fetch(raw, 0);
        if (n_tiles > 1) fetch(raw + PT::kBytes, 1);

        half8_t qf[G][HW];
        bf8_t qz[(G + 1) / 2];
        float factor, lag;
        {
            float x[G][HW][8], top = 0.f;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int s = 0; s < HW; ++s) {
                    float xh[8], xb[8];
                    unpack16<__half>(rawq[g][s], xh);
                    unpack16<__hip_bfloat16>(rawq[g][s], xb);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[g][s][e] = live ? (a.q_dtype == SS_F16 ? xh[e] : xb[e]) : 0.f;
                        top = fmaxf(top, fabsf(x[g][s][e]));
                    }
                }
            const int shift = row_exp_shift(half_max(top));
            const float down = a.scale < 0.f ? -exp2i(-shift) : exp2i(-shift);
            factor = fmaxf(fabsf(a.scale) * kLog2e * 0x1p24f * exp2i(shift), 1e-30f);
            lag = kLag / factor;
            float sums[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float sum = 0.f;
#pragma unroll
                for (int s = 0; s < HW; ++s)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float y = x[g][s][e] * down;
                        sum += y;
                        qf[g][s][e] = (_Float16)((e & 2) ? y * 0x1p-4f : y);
                    }
                sums[g] = (sum + __shfl_xor(sum, 32)) * 0x1p-24f;
            }
            // the sum of group 2y + half as three bf16 parts, for the zero's two:
            // (zh, zh, zh, zl, zl) . (q1, q2, q3, q1, q2)
#pragma unroll
            for (int y = 0; y < (G + 1) / 2; ++y) {
                float v = half == 0 ? sums[2 * y] : (2 * y + 1 < G ? sums[2 * y + 1 < G ? 2 * y + 1 : 0] : 0.f);
                float part[3];
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    part[k] = __bfloat162float(__float2bfloat16(v));
                    v -= part[k];
                }
                const float b[8] = {part[0], part[1], part[2], part[0], part[1], 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 8; ++e) qz[y][e] = (__bf16)b[e];
            }
        }

        float16_t o[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) o[j] = float16_t{};
        float top = -INFINITY, l = 0.f;
        int vexp[G];  // the values met in group g are below 2^vexp
#pragma unroll
        for (int g = 0; g < G; ++g) vexp[g] = -60;

        // Element i of a product's 16: its value's group, as NT dims a row of
        // the A operand make neighbours (row m of tile j is dim NT*m + j).
        auto group_of = [](int i) { return i / 4 * G / 4; };
        // Moves the sums to powers of two that hold the tile's values; bit t of
        // bad[g]: token t's group g is NaN.
        auto meet = [&](const char *slot, int tb, int ok, uint64_t (&bad)[G]) {
            const bool real = tb + lane < rq.len && (ok >> (lane >> 4) & 1);
            const uint32_t *m = reinterpret_cast<const uint32_t *>(slot + (lane >> 4) * PT::kSeg + 2 * PT::kKeys + G * 64) + (lane & 15);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t u = m[16 * g];
                const float s = low16<BF>(u), z = high16<BF>(u);
                const float v = real ? fmaxf(fabsf(z), fabsf(fmaf(15.f, s, z))) : 0.f;
                bad[g] = __ballot(real && !(s < INFINITY && fabsf(z) < INFINITY));
                const float c = wave_max_dpp(v < INFINITY ? v : 0.f);
                const int e = (int)((__float_as_uint(c) >> 23) & 0xffu) - 126;  // c < 2^e
                if (e > vexp[g]) {
                    const int now = min(e, 126);
                    const float f = ldexpf(1.f, vexp[g] - now);
                    vexp[g] = now;
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (group_of(i) == g) o[j][i] *= f;
                }
            }
        };
        // The tile's values as fp16: [8 blocks][dims][8 tokens], dim NT*m + j at
        // place 32 j + m, so that neighbouring threads write neighbouring places.
        auto dequantise = [&](const char *__restrict slot, char *__restrict out, int tb, int ok) {
            const int blk = threadIdx.x >> 5, m = threadIdx.x & 31, g = m * NT * G / D;
            const char *seg = slot + (blk >> 1) * PT::kSeg;
            uint32_t meta[8], w[NT];
            read_words(seg + 2 * PT::kKeys + (G + g) * 64 + (blk & 1) * 32, meta);
            read_words(seg + PT::kKeys + ((blk & 1) * D + m * NT) * 4, w);
            int e = vexp[0];
#pragma unroll
            for (int k = 1; k < G; ++k) e = g == k ? vexp[k] : e;
            const float fs = ldexpf(1.f, 18 - e), fz = ldexpf(1.f, -6 - e);
            const bool page = (ok >> (blk >> 1)) & 1;
            half2_t s2[4], z2[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                float s[2], z[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t u = meta[2 * p + k];
                    s[k] = low16<BF>(u) * fs, z[k] = high16<BF>(u) * fz;
                    // (what no row sees, and what makes rows NaN further down)
                    if (!page || tb + blk * 8 + 2 * p + k >= rq.len || !(fabsf(s[k]) + fabsf(z[k]) < INFINITY)) s[k] = z[k] = 0.f;
                }
                const float odd = (p & 1) ? 0x1p-4f : 1.f;  // codes of odd pairs count 16 times
                s2[p] = __builtin_convertvector(float2_t{s[0] * odd, s[1] * odd}, half2_t);
                z2[p] = __builtin_convertvector(float2_t{z[0], z[1]}, half2_t);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                union {
                    half8_t h;
                    half2_t p[4];
                    uint4 u;
                } x;
                x.h = codes_operand(w[j]);
#pragma unroll
                for (int p = 0; p < 4; ++p) x.p[p] = __builtin_elementwise_fma(x.p[p], s2[p], z2[p]);
                *reinterpret_cast<uint4 *>(out + ((blk * D) + 32 * j + m) * 16) = x.u;
            }
        };

        // One tile: its scores from `cur` and values from `vin`; the next one's
        // values from `next` into `vout`; the copy of the one after that into
        // `into`.  (The pointers differ: no read here waits for that copy.)
        uint64_t bad[G], bad_next[G];
        auto step = [&](char *__restrict into, const char *__restrict cur, const char *__restrict next,
                        const char *__restrict vin, char *__restrict vout, int tile, int ok, int ok_next) {
            const int tb = tile * kTokens;
            if (tile + 2 < n_tiles) {
                const int t16 = tb + 2 * kTokens + 16 * wave;
                PT::fetch(a.st, h, lane, into + wave * PT::kSeg, max(page_at(t16), 0), t16 & in_page);
            }
            half8_t p16[4];
            const bool on = tb < wave_end;
            if (on) {
                float x[32];
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    // row col of the A operand: this token, so that a lane's 16
                    // results are two whole blocks of 8 tokens
                    const int t = 32 * y + 16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3);
                    const char *seg = cur + (t >> 4) * PT::kSeg;
                    float16_t z = float16_t{};
#pragma unroll
                    for (int k = 0; k < (G + 1) / 2; ++k) {
                        const int zg = min(2 * k + half, G - 1);
                        const float zf = high16<BF>(*reinterpret_cast<const uint32_t *>(seg + 2 * PT::kKeys + zg * 64 + (t & 15) * 4));
                        const uint32_t zh = __float_as_uint(zf) >> 16;
                        const uint32_t zl = __float_as_uint(zf - __uint_as_float(zh << 16)) >> 16;
                        union {
                            uint32_t u[4];
                            bf8_t b;
                        } za;
                        za.u[0] = zh | (zh << 16), za.u[1] = zh | (zl << 16), za.u[2] = zl, za.u[3] = 0;
                        z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(za.b, qz[k], z, 0, 0, 0);
                    }
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        uint32_t w[HW];
                        const int c = (g * GW + half * HW) / 4, sw = (t >> 2) % PT::kKP;
                        if constexpr (HW == 8) {
                            uint32_t w4[4];
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                read_words(seg + ((t & 15) * PT::kKP + ((c + k) ^ sw)) * 16, w4);
#pragma unroll
                                for (int e = 0; e < 4; ++e) w[4 * k + e] = w4[e];
                            }
                        } else if constexpr (HW == 4) {
                            read_words(seg + ((t & 15) * PT::kKP + (c ^ sw)) * 16, w);
                        } else {
                            read_words(seg + ((t & 15) * PT::kKP + (c ^ sw)) * 16 + half * 8, w);
                        }
                        float16_t d = float16_t{};
#pragma unroll
                        for (int s = 0; s < HW; ++s)
                            d = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_operand(w[s]), qf[g][s], d, 0, 0, 0);
                        // element i: token 32y + 16(i/8) + 8 half + i%8
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            uint32_t m[4];
                            const int t4 = 16 * (i / 8) + 8 * half + i % 8;
                            read_words(cur + (2 * y + (t4 >> 4)) * PT::kSeg + 2 * PT::kKeys + g * 64 + (t4 & 15) * 4, m);
#pragma unroll
                            for (int e = 0; e < 4; ++e) z[i + e] = fmaf(low16<BF>(m[e]), d[i + e], z[i + e]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[16 * y + i] = z[i];
                }
                if (tb + kTokens > all_see || ok != 15) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int t = 32 * (i / 16) + 16 * (i % 16 / 8) + 8 * half + i % 8;
                        if (tb + t >= limit || !((ok >> (t >> 4)) & 1)) x[i] = -INFINITY;
                    }
                }
                const float m = column_max(x);
                if (__any(m > top + lag)) {
                    const float now = fmaxf(top, half_max(m));
                    const float f = now == top ? 1.f : fast_exp2((top - now) * factor);
                    top = now;
                    l *= f;
#pragma unroll
                    for (int j = 0; j < NT; ++j) o[j] *= f;
                }
                // (times 2^10: a probability below 2^-24 of the largest is one fp16 step)
                const float off = 10.f - (top == -INFINITY ? 0.f : top * factor);
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float p0 = fast_exp2(fmaf(x[i], factor, off)), p1 = fast_exp2(fmaf(x[i + 1], factor, off));
                    l += p0 + p1;
                    const half2_t hh = __builtin_convertvector(float2_t{p0, p1}, half2_t);
                    p16[i / 8][i % 8] = hh[0], p16[i / 8][i % 8 + 1] = hh[1];
                }
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const half8_t v = *reinterpret_cast<const half8_t *>(vin + ((2 * b + half) * D + 32 * j + col) * 16);
                        o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p16[b], o[j], 0, 0, 0);
                    }
#pragma unroll
                for (int g = 0; g < G; ++g)
                    if (bad[g]) {
                        const int see = min(limit - tb, kTokens);
                        const uint64_t seen = see <= 0 ? 0 : see == 64 ? ~0ull : (1ull << see) - 1;
                        if (bad[g] & seen)
#pragma unroll
                            for (int j = 0; j < NT; ++j)
#pragma unroll
                                for (int i = 0; i < 16; ++i)
                                    if (group_of(i) == g) o[j][i] = NAN;
                    }
            }
            if (tile + 1 < n_tiles) {
                meet(next, tb + kTokens, ok_next, bad_next);
                dequantise(next, vout, tb + kTokens, ok_next);
            }
        };

        wait_loads<0>();
        __syncthreads();
        int ok = n_tiles > 0 ? pages_ok(0) : 0;
        if (n_tiles > 0) {
            meet(raw, 0, ok, bad);
            dequantise(raw, vals, 0, ok);
        }
        for (int i = 0, slot = 0; i < n_tiles; ++i) {
            const int ok_next = pages_ok(i + 1);
            wait_loads<0>();  // the next tile's segment
            __syncthreads();  // everyone's, and this tile's values
            const int next = slot == 2 ? 0 : slot + 1, after = next == 2 ? 0 : next + 1;
            step(raw + after * PT::kBytes, raw + slot * PT::kBytes, raw + next * PT::kBytes, vals + (i & 1) * kValues,
                 vals + (~i & 1) * kValues, i, ok, ok_next);
            slot = next, ok = ok_next;
#pragma unroll
            for (int g = 0; g < G; ++g) bad[g] = bad_next[g];
        }

        const float sum = l + __shfl_xor(l, 32);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if (live) {
            const int64_t at = ((int64_t)(rq.t0 + row / a.rep) * a.hq + h * a.rep + row % a.rep) * D;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int m = 8 * (i / 4) + 4 * half + i % 4;
                const int e = vexp[group_of(i)] + 6;
                if constexpr (NT == 4) {
                    store4_from_f32(a.out, a.q_dtype, at + NT * m, ldexpf(o[0][i] * inv, e), ldexpf(o[1][i] * inv, e),
                                    ldexpf(o[2][i] * inv, e), ldexpf(o[3][i] * inv, e));
                } else {
#pragma unroll
                    for (int j = 0; j < NT; ++j) store_from_f32(a.out, a.q_dtype, at + NT * m + j, ldexpf(o[j][i] * inv, e));
                }
            }
        }
        __syncthreads();  // (the next item's copies)
    }
}

template <int D, int G>
static void launch_prompt(const PagedAttn &a, bool bf, unsigned groups, hipStream_t st) {
    if (bf)
        hipLaunchKernelGGL((paged_prompt_kernel<D, G, true>), dim3(groups), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((paged_prompt_kernel<D, G, false>), dim3(groups), dim3(256), 0, st, a);
}

int launch_paged_prompt(const PagedAttn &a, const ss_paged_store *s, hipStream_t st) {
    // at most this many row tiles: whole ones, and one a request of more than most_rows rows
    const int64_t rows = a.n_tokens * a.rep;
    const int64_t tiles = rows / kRows + min((int64_t)a.n_req, rows / (a.most_rows + 1));
    const unsigned groups = (unsigned)min(tiles * a.st.heads, (int64_t)1 << 20);
    if (groups == 0) return SS_OK;
    const bool bf = s->dtype == SS_BF16;
    const int key = s->head_dim * 1000 + s->group_size;
    if (key == 128032) launch_prompt<128, 4>(a, bf, groups, st);
    else if (key == 128064) launch_prompt<128, 2>(a, bf, groups, st);
    else if (key == 128128) launch_prompt<128, 1>(a, bf, groups, st);
    else if (key == 64032) launch_prompt<64, 2>(a, bf, groups, st);
    else launch_prompt<64, 1>(a, bf, groups, st);
    SS_LAUNCH_CHECK("paged_prompt_kernel launch");
    return SS_OK;
}

}  // namespace ss
