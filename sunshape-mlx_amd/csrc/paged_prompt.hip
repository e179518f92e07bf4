// Attention over a paged cache of 4-bit keys and values: prompts, and chunks of
// long ones (paged_attn.hpp has the formulas).
//
// A workgroup of eight waves takes 256 query rows of one KV head (its group's
// heads at consecutive positions), 32 a wave, over 64-token tiles.  While a
// tile is computed the next one is prepared, once for all rows: its key codes
// become 16-bit operands (see paged_attn.hpp) and its values are dequantised
// to fp16, both in the operand order of v_mfma_f32_32x32x16_f16, and the one
// after that is copied from HBM.
//
// Scores are exact: code products are summed group by group and each sum is
// multiplied by its token's scale in float32; the zeros' part is one more
// product, of zero/64 - scale and the queries' sums, both split into bf16
// parts.  Values are rounded to fp16 (2^-11 of a value, as the probabilities'
// rounding costs), times a power of two a group that keeps the largest value
// met below 2^15: values keep all 11 bits down to 2^-29 of it, and below that
// are off by 2^-40 of it.  (Codes as they lie, fp16's subnormals, would save
// 4 operations a word, but hold values below 2^-4 and cost those below 1/256
// of the largest their bits.)  Statistics and sums are float32.
//
// The vector ALUs bound it (per 32 rows and 64 tokens: 2 x 32 products of
// scale and sum, 32 exponentials), so what does not depend on the row is done
// once a workgroup.  32 rows a wave and 64 tokens are what the 256 registers of
// two waves a SIMD hold.  A prompt of 4093 tokens, 32 heads, 137 GFLOP, takes
// 266 us back to back under the profiler, 230 us between other calls: 0.5 to
// 0.6 PFLOP/s, vector ALUs 49 % of the cycles, matrix cores 27 %.
#include "paged_attn.hpp"

namespace ss {

typedef float float16_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));

constexpr int kPWaves = 8;
constexpr int kRows = 32 * kPWaves;  // query rows of a workgroup
static_assert(kRows == kPromptTile, "the rows that launches are planned for");
constexpr int kTokens = 64;          // of a tile
constexpr int kSlots = 3;            // tiles in LDS as they come: one being prepared, two on their way
// Fewest tiles of a part, where a workgroup's column is cut (1024 tokens, 32
// heads: 54 us for 2 to 8, 62 us for 16).
constexpr int kMinTiles = 8;

template <int D, int G>
struct PromptTile {
    // A tile in LDS as it comes: 16-token segments of key rows, value blocks,
    // the keys' and the values' (scale, zero) pairs [G][16].  16-byte piece c of
    // key row t sits at place c ^ (t / 4) % (pieces a row).
    static constexpr int kKeys = 8 * D, kMeta = 2 * G * 64;
    static constexpr int kSeg = 2 * kKeys + kMeta;
    static constexpr int kBytes = 4 * kSeg;
    static constexpr int kKP = D / 32;  // 16-byte pieces of a key row
    // Prepared, 16 bytes each: keys [2 halves of 32 tokens][D/16 steps][2][32 rows],
    // values [8 blocks of tokens][D places], zeros [2 halves][group pairs][2][32 rows];
    // and the keys' scales, 16 bits each, [G][64].
    static constexpr int kOperands = kTokens * D * 2;
    static constexpr int kPairs = (G + 1) / 2;
    static constexpr int kZeros = 2 * kPairs * 1024, kScales = G * kTokens * 2;
    static constexpr int kPrepared = 2 * kOperands + kZeros + kScales;

    // Starts copying, of the segment of 16 tokens in page p from its token
    // `off`, the keys and the pairs (part 0) or the values (part 1).
    __device__ static void fetch(const PagedStore &st, int h, int lane, char *seg, int page, int off, int part) {
        const int64_t slot = (((int64_t)page * st.heads + h) << st.log_page) + off;
        if (part == 0) {
            const int t = lane % (kKeys / 16) / kKP, c = (lane % kKP) ^ ((t >> 2) % kKP);
            const char *k = reinterpret_cast<const char *>(st.k_codes) + slot * (D / 2);
            if (kKeys == 1024 || lane < kKeys / 16)
                __builtin_amdgcn_global_load_lds(k + (uint32_t)(t * (D / 2) + c * 16), as_lds<void>(seg), 16, 0, 0);
            if (lane < kMeta / 16) {
                const int e = lane % (4 * G);
                const uint32_t *m = lane < 4 * G ? st.k_meta : st.v_meta;
                m += (slot - off) * G + off;
                __builtin_amdgcn_global_load_lds(m + (uint32_t)(((e / 4) << st.log_page) + e % 4 * 4),
                                                 as_lds<void>(seg + 2 * kKeys), 16, 0, 0);
            }
        } else if (kKeys == 1024 || lane < kKeys / 16) {
            const char *v = reinterpret_cast<const char *>(st.v_codes) + slot * (D / 2);
            __builtin_amdgcn_global_load_lds(v + (uint32_t)(lane * 16), as_lds<void>(seg + kKeys), 16, 0, 0);
        }
    }
};

// A word's eight codes as fp16 numbers, pairs (0,1) and (4,5) as they are, (2,3)
// and (6,7) times 16: put into the low bits of 1024, which is taken off again.
// (The constants as in CodeBits.)
struct CodeNumber {
    uint32_t low = 0x000f000fu, high = 0x00f000f0u, base = 0x64006400u;
    __device__ CodeNumber() { asm volatile("" : "+s"(low), "+s"(high), "+v"(base)); }
};
__device__ __forceinline__ half8_t codes_number(uint32_t w, const CodeNumber &k) {
    union {
        uint32_t u[4];
        half8_t h;
    } x;
    const uint32_t hi = w >> 8;
    x.u[0] = (w & k.low) | k.base;
    x.u[1] = (w & k.high) | k.base;
    x.u[2] = (hi & k.low) | k.base;
    x.u[3] = (hi & k.high) | k.base;
    return x.h - (_Float16)1024.f;
}

// Row tiles of a request that are this kernel's.
__device__ __forceinline__ int tiles_of(const PagedAttn &a, const Request &q) {
    return q.rows > a.most_rows ? (q.rows + kRows - 1) / kRows : 0;
}

// Parts of a request's columns at `share` tiles a part.
__device__ __forceinline__ int parts_of_tiles(const Request &q, int share) {
    return max(1, (int)(((int64_t)(q.len + kTokens - 1) / kTokens + share - 1) / share));
}

// The bits of the 16-bit float 2^k, k >= -126 (positive ones compare as
// integers); above the finite ones those of infinity, below all of them 1.
template <bool BF>
__device__ __forceinline__ uint32_t bits_of_exp2(int k) {
    if (BF) return (uint32_t)min(k + 127, 255) << 7;
    return k >= -14 ? (uint32_t)min(k + 15, 31) << 10 : 1u << max(k + 24, 0);
}

// Largest low and largest high half of the lanes' pairs, N sets side by side.
template <int N>
__device__ __forceinline__ void pair_max(uint32_t (&v)[N]) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    auto most = [](uint32_t a, int b) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, b)));
    };
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = most(v[i], dpp_mov_i<0xB1>(v[i]));  // quad_perm [1,0,3,2]
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = most(v[i], dpp_mov_i<0x4E>(v[i]));  // quad_perm [2,3,0,1]
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = most(v[i], dpp_mov_i<0x141>(v[i]));  // row_half_mirror
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = most(v[i], dpp_mov_i<0x140>(v[i]));  // row_mirror
#pragma unroll
    for (int i = 0; i < N; ++i)  // row_bcast:15 -> rows 1, 3
        v[i] = most(v[i], __builtin_amdgcn_update_dpp(v[i], v[i], 0x142, 0xa, 0xf, false));
#pragma unroll
    for (int i = 0; i < N; ++i)  // row_bcast:31 -> rows 2, 3
        v[i] = most(v[i], __builtin_amdgcn_update_dpp(v[i], v[i], 0x143, 0xc, 0xf, false));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __builtin_amdgcn_readlane(v[i], 63);
}

// A barrier for what lies in LDS: unlike __syncthreads it leaves copies to LDS
// on their way (each wave waits for those it needs).
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
}

__device__ __forceinline__ float half_max(float v) { return fmaxf(v, __shfl_xor(v, 32)); }

template <int D, int G, bool BF>
__global__ void __launch_bounds__(64 * kPWaves, 2) paged_prompt_kernel(const PagedAttn a) {
    using PT = PromptTile<D, G>;
    constexpr int GW = D / 8 / G, HW = GW / 2;  // words of a group, and of a lane's half of it
    constexpr int NT = D / 32;                  // 32-dim tiles of the values
    __shared__ __attribute__((aligned(16))) char lds[kSlots * PT::kBytes + 2 * PT::kPrepared];
    char *const raw = lds, *const prepared = lds + kSlots * PT::kBytes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int heads = a.st.heads, log_page = a.st.log_page, in_page = (1 << log_page) - 1;

    // Columns are (request, row tile, KV head).  Where there are fewer than half
    // as many as workgroups, each is cut along its tokens into parts of at most
    // `share` tiles of the request's length.
    const int per = (a.n_req + 63) / 64, r0 = min(lane * per, a.n_req);
    int r1 = min(r0 + per, a.n_req), columns = 0;
    bool down = false;
    uint32_t all_tiles = 0;  // (up to 128 columns of 2^24; of more it is not used)
    for (int i = r0; i < r1; ++i) {
        const Request q = request(a, i);
        const int n = tiles_of(a, q) * heads;
        down |= descends(a, i);
        columns += n, all_tiles += (uint32_t)n * ((q.len + kTokens - 1) / kTokens);
    }
    if (__any(down)) columns = 0, all_tiles = 0, r1 = r0;
    int scan = wave_scan(columns);
    const int n_columns = __builtin_amdgcn_readlane(scan, 63);
    int share = INT32_MAX;
    if (a.cut && 2 * n_columns <= a.target) {
        // sum of ceil(n / share) is at most total / share + columns, and about
        // total / share + columns / 2
        const uint32_t total = __builtin_amdgcn_readlane(wave_scan((int)all_tiles), 63);
        for (int spare = n_columns / 2;; spare = n_columns) {
            const int free_groups = a.target - spare;
            share = max(uniform_div((int)(total + free_groups - 1), free_groups), kMinTiles);
            columns = 0;
            for (int i = r0; i < r1; ++i) {
                const Request q = request(a, i);
                columns += tiles_of(a, q) * heads * parts_of_tiles(q, share);
            }
            scan = wave_scan(columns);
            if (spare == n_columns || __builtin_amdgcn_readlane(scan, 63) <= a.target) break;
        }
    }
    const int n_items = __builtin_amdgcn_readlane(scan, 63);
    int4 cut = make_int4(0, 0, 0, 0);

    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
        const int holder = __ffsll((unsigned long long)__ballot(item < scan)) - 1;
        int left = item - (holder ? __builtin_amdgcn_readlane(scan, holder - 1) : 0);
        int r = holder * per, parts, row_tile;
        Request rq;
        for (;; ++r) {
            rq = request(a, r);
            const int n = tiles_of(a, rq);
            parts = __builtin_amdgcn_readfirstlane(parts_of_tiles(rq, share));
            if (left < n * heads * parts) {
                // the longest row tiles first; heads side by side, so that a head's
                // tiles tend to meet in one L2
                const int t = uniform_div(left, heads * parts);
                left -= t * heads * parts;
                row_tile = n - 1 - t;
                break;
            }
            left -= n * heads * parts;
        }
        const int part = uniform_div(left, heads), h = left - part * heads;
        const int row0 = row_tile * kRows + wave * 32;  // the wave's first row
        const int32_t *row_table = a.table + (int64_t)r * a.width;
        auto page_at = [&](int token) {
            const int p = table_read(row_table, min((int64_t)(token >> log_page), a.width - 1));
            return (uint32_t)p < (uint32_t)a.st.n_pages ? p : -1;
        };
        auto sees = [&](int row) {  // tokens that a row sees
            return a.causal ? max(0, min(rq.len, rq.len - rq.n_all + row / a.rep + 1)) : rq.len;
        };
        const int last_row = min(row_tile * kRows + kRows, rq.rows) - 1;
        const int seen_tiles =
            (__builtin_amdgcn_readfirstlane(sees(last_row)) + kTokens - 1) / kTokens;  // by the workgroup
        const int first_tile = part_begin(part, seen_tiles, parts);
        const int n_tiles = part_begin(part + 1, seen_tiles, parts);
        const int wave_last = min(row0 + 31, rq.rows - 1);
        const int wave_end = row0 < rq.rows ? __builtin_amdgcn_readfirstlane(sees(wave_last)) : 0;
        const int all_see = row0 < rq.rows ? __builtin_amdgcn_readfirstlane(sees(row0)) : 0;
        const int row = row0 + col;
        const bool live = row < rq.rows;
        const int limit = live ? sees(row) : rq.len;

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
        // A tile's four pages, of 16 tokens each; bit w of the mask: it is in the pool.
        auto pages_of = [&](int tile, int (&p)[4]) {
#pragma unroll
            for (int w = 0; w < 4; ++w) p[w] = page_at(tile * kTokens + 16 * w);
        };
        auto mask_of = [](const int (&p)[4]) {
            return (p[0] >= 0 ? 1 : 0) | (p[1] >= 0 ? 2 : 0) | (p[2] >= 0 ? 4 : 0) | (p[3] >= 0 ? 8 : 0);
        };
        // The wave copies a part of segment wave % 4 of a tile.
        const int seg = wave & 3;
        auto own = [&](const int (&p)[4]) {
            return max(seg == 0 ? p[0] : seg == 1 ? p[1] : seg == 2 ? p[2] : p[3], 0);
        };
        auto offset = [&](int tile) { return (tile * kTokens + 16 * seg) & in_page; };
        int pages[4], ok[kSlots + 1];  // ok: of the tile computed and those behind it
        wait_loads<0>();  // the queries, before tiles are waited for with them
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            pages_of(first_tile + i, pages);
            ok[i] = mask_of(pages);
            if (first_tile + i < n_tiles)
                PT::fetch(a.st, h, lane, raw + i * PT::kBytes + seg * PT::kSeg, own(pages), offset(first_tile + i),
                          wave >> 2);
        }
        pages_of(first_tile + kSlots, pages);

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
            const QueryScale by(half_max(top), a.scale);
            factor = by.factor;
            lag = kLag / factor;
            float sums[(G + 1) / 2];  // of group 2y + half
#pragma unroll
            for (int y = 0; y < (G + 1) / 2; ++y) sums[y] = 0.f;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float sum = 0.f;
#pragma unroll
                for (int s = 0; s < HW; ++s)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float y = x[g][s][e] * by.down;
                        sum += y;
                        qf[g][s][e] = (_Float16)y;
                    }
                sum += __shfl_xor(sum, 32);
                sums[g / 2] = half == g % 2 ? sum : sums[g / 2];
            }
            // the sum of group 2y + half as three bf16 parts, for the zero's three:
            // (z1, z1, z1, z2, z2, z3) . (q1, q2, q3, q1, q2, q1); the first pair's two
            // places that are left take the row's reference, times 1
#pragma unroll
            for (int y = 0; y < (G + 1) / 2; ++y) {
                float v = sums[y];
                float part[3];
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    part[k] = __bfloat162float(__float2bfloat16(v));
                    v -= part[k];
                }
                const float b[8] = {part[0], part[1], part[2], part[0], part[1], part[0], 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 8; ++e) qz[y][e] = (__bf16)b[e];
            }
        }

        float16_t o[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) o[j] = float16_t{};
        float top = -INFINITY, l = 0.f, ref = 0.f;
        // The values met in group g are below 2^vexp; the tile prepared last has
        // vnext, which the sums move to when they come to it.
        int vexp[G], vnext[G];
#pragma unroll
        for (int g = 0; g < G; ++g) vexp[g] = vnext[g] = -110;
        // The bits from which zeros and scales would pass 2^vnext: few tiles
        // after the first have any, and a look at a tile's largest is skipped.
        uint32_t zero_top[G], scale_top[G];
#pragma unroll
        for (int g = 0; g < G; ++g) zero_top[g] = scale_top[g] = 1;

        // Element i of a product's 16: its value's group, as NT dims a row of
        // the A operand make neighbours (row m of tile j is dim NT*m + j).
        auto group_of = [](int i) { return i / 4 * G / 4; };
        // The tile's prepared form, its values times a power of two that holds
        // them (a lane looks at one token's pairs); bit t of bad_next[g]: token
        // t's group g is not finite.
        uint64_t bad_next[G];
        auto prepare = [&](const char *__restrict slot, char *__restrict out, int tb, int ok) {
            const CodeBits code_bits;
            constexpr uint32_t kInf = BF ? 0x7f80u : 0x7c00u;
            constexpr int KW = D / 64, VW = NT / 2;  // words of keys and values that a lane takes
            // everything that is read first
            const char *mine = slot + (lane >> 4) * PT::kSeg;  // of token `lane`
            const uint32_t *m = reinterpret_cast<const uint32_t *>(mine + 2 * PT::kKeys + G * 64) + (lane & 15);
            uint32_t pair[G], kw[2], vw[2], vm[8], km = 0;
#pragma unroll
            for (int g = 0; g < G; ++g) pair[g] = m[16 * g];
            if (wave < G) km = m[16 * (wave - G)];  // the keys' pairs lie before the values'
            // key words KW * wave .. of token `lane`
            const int w0 = wave * KW;
            const char *kfrom = mine + ((lane & 15) * PT::kKP + ((w0 / 4) ^ ((lane >> 2) % PT::kKP))) * 16 + w0 % 4 * 4;
            // value block `wave`, dims NT * col + j of the lane's half
            const int j0 = half * VW, vg = col * NT * G / D;
            const char *vseg = slot + (wave >> 1) * PT::kSeg;
            const char *vfrom = vseg + PT::kKeys + ((wave & 1) * D + col * NT + j0) * 4;
            if constexpr (KW == 2)
                read_words(kfrom, kw), read_words(vfrom, vw);
            else
                kw[0] = *reinterpret_cast<const uint32_t *>(kfrom), vw[0] = *reinterpret_cast<const uint32_t *>(vfrom);
            read_words(vseg + 2 * PT::kKeys + (G + vg) * 64 + (wave & 1) * 32, vm);

            // keys: the A operand's row of a token, so chosen that a lane's 16
            // results are two whole blocks of 8 tokens
            const int t = lane & 31, row = (t & 16) | (t >> 3 & 1) << 2 | (t >> 2 & 1) << 3 | (t & 3);
#pragma unroll
            for (int k = 0; k < KW; ++k) {
                const int g = (w0 + k) / GW, in = (w0 + k) % GW;
                const int place = (((lane >> 5) * (D / 16) + g * HW + in % HW) * 2 + in / HW) * 32 + row;
                *reinterpret_cast<half8_t *>(out + place * 16) = codes_operand(kw[k], code_bits);
            }
            if (wave < 2 * PT::kPairs) {  // zeros and scales of the keys' group `wave` (one past an odd number: 0)
                // (truncated parts: what is left is exact)
                const float zero = fmaf(high16<BF>(km), 1.f / 64.f, -low16<BF>(km));
                const uint32_t z1 = __float_as_uint(zero) >> 16;
                const float rest = zero - __uint_as_float(z1 << 16);
                const uint32_t z2 = __float_as_uint(rest) >> 16;
                const uint32_t z3 = __float_as_uint(rest - __uint_as_float(z2 << 16)) >> 16;
                const int place = (((lane >> 5) * PT::kPairs + (wave >> 1)) * 2 + (wave & 1)) * 32 + row;
                *reinterpret_cast<uint4 *>(out + 2 * PT::kOperands + place * 16) =
                    make_uint4(z1 | (z1 << 16), z1 | (z2 << 16), z2 | (z3 << 16), wave < 2 ? 0x3f803f80u : 0);
                if (wave < G)
                    reinterpret_cast<uint16_t *>(out + 2 * PT::kOperands + PT::kZeros)[wave * kTokens + lane] = (uint16_t)km;
            }

            const bool real = tb + lane < rq.len && (ok >> (lane >> 4) & 1);
            bool odd_ones = tb + kTokens > rq.len || ok != 15;
            bool more = false;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                pair[g] = real ? pair[g] & 0x7fff7fffu : 0;
                bad_next[g] = 0;
                more |= pair[g] >= zero_top[g] << 16 || (pair[g] & 0x7fffu) >= scale_top[g];
            }
            if (__any(more)) {
                uint32_t most[G];
#pragma unroll
                for (int g = 0; g < G; ++g) most[g] = pair[g];
                pair_max(most);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    if ((most[g] & 0xffffu) >= kInf || (most[g] >> 16) >= kInf) {
                        const bool b = (pair[g] & 0x7fffu) >= kInf || (pair[g] >> 16) >= kInf;
                        bad_next[g] = __ballot(b);
                        odd_ones = true;
                        uint32_t rest[1] = {b ? 0 : pair[g]};
                        pair_max(rest);
                        most[g] = rest[0];
                    }
                    // |zero + 15 scale| < 2 max(|zero|, 16 scale)
                    const float c = fmaxf(16.f * low16<BF>(most[g]), high16<BF>(most[g]));
                    const int e = __builtin_amdgcn_readfirstlane((int)((__float_as_uint(c) >> 23) & 0xffu) - 125);
                    vnext[g] = max(vnext[g], e);
                    zero_top[g] = bits_of_exp2<BF>(vnext[g] - 1), scale_top[g] = bits_of_exp2<BF>(vnext[g] - 5);
                }
            }
            if (odd_ones) {  // (what no row sees, and what makes rows NaN further down)
                uint64_t keep = ~0ull;
#pragma unroll
                for (int g = 0; g < G; ++g) keep = vg == g ? ~bad_next[g] : keep;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (tb + 8 * wave + i >= rq.len || !((ok >> (wave >> 1)) & 1) || !((keep >> (8 * wave + i)) & 1))
                        vm[i] = 0;
            }
            // (read as scalars: as elements the compiler would index an array in memory)
            int e = __builtin_amdgcn_readfirstlane(vnext[0]);
#pragma unroll
            for (int g = 1; g < G; ++g) e = vg == g ? __builtin_amdgcn_readfirstlane(vnext[g]) : e;
            const float up = exp2i(15 - e), up_odd = exp2i(11 - e);  // (-110 <= e <= 130)
            const CodeNumber number;
            half8_t sc, ze;  // codes of odd pairs count 16 times
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float f = (i & 2) ? up_odd : up;
                const half2_t s2 = __builtin_convertvector(float2_t{low16<BF>(vm[i]) * f, low16<BF>(vm[i + 1]) * f}, half2_t);
                const half2_t z2 = __builtin_convertvector(float2_t{high16<BF>(vm[i]) * up, high16<BF>(vm[i + 1]) * up}, half2_t);
                sc[i] = s2[0], sc[i + 1] = s2[1], ze[i] = z2[0], ze[i + 1] = z2[1];
            }
#pragma unroll
            for (int k = 0; k < VW; ++k)  // dim NT * m + j at place 32 j + m
                *reinterpret_cast<half8_t *>(out + PT::kOperands + (wave * D + 32 * (j0 + k) + col) * 16) =
                    __builtin_elementwise_fma(codes_number(vw[k], number), sc, ze);
        };

        // One tile: computed from `cur`; the next one prepared from `next` into
        // `out`; the copy of a later one started into `into`.  (The pointers
        // differ: no read here waits for that copy.)
        auto step = [&](char *__restrict into, const char *__restrict next, const char *__restrict cur,
                        char *__restrict out, int tile) {
            const int tb = tile * kTokens;
            if (tile + kSlots < n_tiles)
                PT::fetch(a.st, h, lane, into + seg * PT::kSeg, own(pages), offset(tile + kSlots), wave >> 2);
            // Of the two waves of a SIMD, w and w + 4, one prepares first and one
            // last, so that one's products meet the other's softmax.  The wave that
            // prepares goes first: the other has matrix products on their way (4093
            // tokens 225 -> 221 us, two chunks of 512 at 8192 219 -> 213 us).
            uint64_t bad[G];
            int move[G];
#pragma unroll
            for (int g = 0; g < G; ++g) bad[g] = bad_next[g], move[g] = vexp[g] - vnext[g], vexp[g] = vnext[g];
            __builtin_amdgcn_s_setprio(1);
            if (tile + 1 < n_tiles && wave >= 4) prepare(next, out, tb + kTokens, ok[1]);
#pragma unroll
            for (int g = 0; g < G; ++g)
                if (move[g]) {
                    const float f = ldexpf(1.f, move[g]);
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (group_of(i) == g) o[j][i] *= f;
                }
            __builtin_amdgcn_s_setprio(0);
            if (tb < wave_end) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float16_t x = float16_t{}, d[G];
#pragma unroll
                    for (int k = 0; k < PT::kPairs; ++k) {
                        const bf8_t z = *reinterpret_cast<const bf8_t *>(
                            cur + 2 * PT::kOperands + (((y * PT::kPairs + k) * 2 + half) * 32 + col) * 16);
                        x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(z, qz[k], x, 0, 0, 0);
                    }
                    // the groups' sums side by side: a product waits for the one before it
#pragma unroll
                    for (int g = 0; g < G; ++g) d[g] = float16_t{};
#pragma unroll
                    for (int s = 0; s < HW; ++s)
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            const half8_t k = *reinterpret_cast<const half8_t *>(
                                cur + (((y * (D / 16) + g * HW + s) * 2 + half) * 32 + col) * 16);
                            d[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qf[g][s], d[g], 0, 0, 0);
                        }
                    // element i: token 32y + 16(i/8) + 8 half + i%8
#pragma unroll
                    for (int g = 0; g < G; ++g)
#pragma unroll
                        for (int i = 0; i < 16; i += 8) {
                            uint32_t m[4];
                            read_words(cur + 2 * PT::kOperands + PT::kZeros + (g * kTokens + 32 * y + 2 * i + 8 * half) * 2, m);
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                x[i + e] = fmaf((e & 1) ? high16<BF>(m[e / 2]) : low16<BF>(m[e / 2]), d[g][i + e], x[i + e]);
                        }
                    if (tb + 32 * y + 32 > all_see || ok[0] != 15) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int t = 32 * y + 16 * (i / 8) + 8 * half + i % 8;
                            if (tb + t >= limit || !((ok[0] >> (2 * y + i / 8)) & 1)) x[i] = -INFINITY;
                        }
                    }
                    float m = x[0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) m = fmaxf(m, x[i]);
                    if (__any(m > top + lag)) {
                        const float now = fmaxf(top, half_max(m));
                        const float f = now == top ? 1.f : fast_exp2((top - now) * factor);
                        top = now;
                        if (__any(is_far(now, factor))) {
                            const float move = is_far(now, factor) ? now : 0.f;
                            ref += move, top -= move;
#pragma unroll
                            for (int i = 0; i < 16; ++i) x[i] -= move;
                            // minus the reference as three bf16 parts, in the zeros' product
                            float part[3], rest = -ref;
#pragma unroll
                            for (int k = 0; k < 3; ++k) {
                                part[k] = __bfloat162float(__float2bfloat16(rest));
                                rest -= part[k];
                            }
                            qz[0][6] = (__bf16)(half ? part[2] : part[0]);
                            qz[0][7] = (__bf16)(half ? 0.f : part[1]);
                        }
                        l *= f;
#pragma unroll
                        for (int j = 0; j < NT; ++j) o[j] *= f;
                    }
                    // (times 2^10: a probability below 2^-24 of the largest is one fp16 step)
                    const float off = 10.f - (top == -INFINITY ? 0.f : top * factor);
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        half8_t p16;
#pragma unroll
                        for (int i = 0; i < 8; i += 2) {
                            const float p0 = fast_exp2(fmaf(x[8 * b + i], factor, off));
                            const float p1 = fast_exp2(fmaf(x[8 * b + i + 1], factor, off));
                            l += p0 + p1;
                            const half2_t hh = __builtin_convertvector(float2_t{p0, p1}, half2_t);
                            p16[i] = hh[0], p16[i + 1] = hh[1];
                        }
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            const int blk = 2 * (2 * y + b) + half;
                            const half8_t v = *reinterpret_cast<const half8_t *>(cur + PT::kOperands + (blk * D + 32 * j + col) * 16);
                            o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p16, o[j], 0, 0, 0);
                        }
                    }
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
            __builtin_amdgcn_s_setprio(1);
            if (tile + 1 < n_tiles && wave < 4) prepare(next, out, tb + kTokens, ok[1]);
        };

        wait_loads<0>();
        __syncthreads();
        if (first_tile < n_tiles) prepare(raw, prepared, first_tile * kTokens, ok[0]);
        int slot = 0, into = 1;  // raw slot and prepared form of the tile computed
        for (int i = first_tile; i < n_tiles; ++i) {
            // the wave's copies of the next tile (of the one after it, two loads or
            // one may be on their way), then everyone's, and this tile's operands
            if (i + 2 >= n_tiles)
                wait_loads<0>();
            else if (wave < 4)
                wait_loads<2>();
            else
                wait_loads<1>();
            lds_barrier();
            const int next = slot == kSlots - 1 ? 0 : slot + 1, from = into ^ 1;
            step(raw + slot * PT::kBytes, raw + next * PT::kBytes, prepared + from * PT::kPrepared,
                 prepared + into * PT::kPrepared, i);
            slot = next, into = from;
#pragma unroll
            for (int k = 0; k < kSlots; ++k) ok[k] = ok[k + 1];
            ok[kSlots - 1] = mask_of(pages);
            pages_of(i + kSlots + 1, pages);
        }

        const float sum = l + __shfl_xor(l, 32);
        if (parts == 1) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            if (live) {
                const int64_t at = ((int64_t)(rq.t0 + row / a.rep) * a.hq + h * a.rep + row % a.rep) * D;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int m = 8 * (i / 4) + 4 * half + i % 4;
                    const int e = vexp[group_of(i)] - 15;
                    if constexpr (NT == 4) {
                        store_out4(a, at + NT * m, ldexpf(o[0][i] * inv, e), ldexpf(o[1][i] * inv, e),
                                   ldexpf(o[2][i] * inv, e), ldexpf(o[3][i] * inv, e));
                    } else if (i % 2 == 0) {  // (two rows of the A operand are neighbours)
                        store_out4(a, at + NT * m, ldexpf(o[0][i] * inv, e), ldexpf(o[1][i] * inv, e),
                                   ldexpf(o[0][i + 1] * inv, e), ldexpf(o[1][i + 1] * inv, e));
                    }
                }
            }
        } else {
            // a part: the sums as they are (times 2^10), for prompt_merge_kernel
            if (part == 0) cut = make_int4(parts, r, h, row_tile);
            const int64_t at = (int64_t)item * kRows + wave * 32 + col;
            if (half == 0) *reinterpret_cast<float2 *>(a.ml + at * 2) = make_float2((ref + top) * factor, sum);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int m = 8 * (i / 4) + 4 * half + i % 4;
                const int e = vexp[group_of(i)] - 15;
#pragma unroll
                for (int j = 0; j < NT; ++j) a.acc[at * D + NT * m + j] = ldexpf(o[j][i], e);
            }
        }
        __syncthreads();  // (the next item's copies)
    }
    if (a.cut && (int)blockIdx.x < a.target && threadIdx.x == 0) a.cut[blockIdx.x] = cut;
}

// Joins the parts of the column that cut[blockIdx.y] names: part i is at item
// blockIdx.y + i * heads.  A thread takes four dims of a row.  The parts' sums
// bound it: 256 of 256 rows, 34 MB, 9 us.
template <int D>
__global__ void __launch_bounds__(256) prompt_merge_kernel(const PagedAttn a) {
    constexpr int CH = D / 4, AT_ONCE = 256 / CH;
    const int4 cut = a.cut[blockIdx.y];
    const int parts = cut.x, r = cut.y, h = cut.z, c = threadIdx.x % CH * 4;
    if (parts == 0) return;
    const Request rq = request(a, r);
    for (int row = blockIdx.x * AT_ONCE + threadIdx.x / CH; row < kRows; row += gridDim.x * AT_ONCE) {
        const int n = cut.w * kRows + row;
        if (n >= rq.rows) return;
        auto at = [&](int i) { return ((int64_t)blockIdx.y + (int64_t)i * a.st.heads) * kRows + row; };
        float m = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < parts; ++i) m = fmaxf(m, a.ml[at(i) * 2]);
#pragma unroll 4
        for (int i = 0; i < parts; ++i) {
            const float2 e = *reinterpret_cast<const float2 *>(a.ml + at(i) * 2);
            const float4 v = *reinterpret_cast<const float4 *>(a.acc + at(i) * D + c);
            const float f = e.x == m ? 1.f : fast_exp2(e.x - m);
            l += f * e.y;
            x[0] += f * v.x, x[1] += f * v.y, x[2] += f * v.z, x[3] += f * v.w;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int64_t o = ((int64_t)(rq.t0 + n / a.rep) * a.hq + h * a.rep + n % a.rep) * D + c;
        store_out4(a, o, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    }
}

template <int D, int G>
static void launch_prompt(const PagedAttn &a, bool bf, unsigned groups, hipStream_t st) {
    const dim3 block(64 * kPWaves);
    if (bf)
        hipLaunchKernelGGL((paged_prompt_kernel<D, G, true>), dim3(groups), block, 0, st, a);
    else
        hipLaunchKernelGGL((paged_prompt_kernel<D, G, false>), dim3(groups), block, 0, st, a);
    if (a.target) hipLaunchKernelGGL(prompt_merge_kernel<D>, dim3(16, a.target), dim3(256), 0, st, a);
}

// Workgroups that fill the device (one a compute unit) if the columns alone
// may not, else 0: then no column is cut.
static int cut_target(int64_t n_requests, int heads, int64_t rows, int most_rows) {
    const int64_t least = max((int64_t)0, rows - n_requests * most_rows) / kRows * heads;
    return 2 * least <= device_cu_count() ? device_cu_count() : 0;
}

size_t paged_prompt_bytes(const ss_paged_store *s, int64_t n_requests, int64_t rows, int most_rows) {
    return (size_t)cut_target(n_requests, s->n_kv_heads, rows, most_rows) * (16 + kRows * (s->head_dim + 2) * 4);
}

int launch_paged_prompt(PagedAttn a, const ss_paged_store *s, void *workspace, size_t workspace_bytes,
                        hipStream_t st) {
    // at most this many row tiles: whole ones, and one a request of more than most_rows rows
    const int64_t rows = a.n_tokens * a.rep;
    const int64_t tiles = rows / kRows + min((int64_t)a.n_req, rows / (a.most_rows + 1));
    if (tiles == 0) return SS_OK;
    a.target = cut_target(a.n_req, a.st.heads, rows, a.most_rows);
    if (paged_prompt_bytes(s, a.n_req, rows, a.most_rows) > workspace_bytes) a.target = 0;
    a.cut = a.target ? static_cast<int4 *>(workspace) : nullptr;
    a.acc = reinterpret_cast<float *>(a.cut + a.target);
    a.ml = a.acc + (size_t)a.target * kRows * s->head_dim;
    const unsigned groups = (unsigned)max(min(tiles * a.st.heads, (int64_t)1 << 20), (int64_t)a.target);
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
