// Attention over a paged cache of 4-bit keys and values: the few query rows
// of decode steps and speculative verification (paged_attn.hpp has the
// formulas, paged_prompt.hip the many rows of prompts).
//
// Scales stay out of the codes' operands: the 16 columns of both products are
// (row r, group g), a query entering column (r, g) with the dims of group g
// alone, a probability times the value's scale in g.  Keys are the A operand
// (16 tokens), so a lane holds, of one column, 4 tokens of each key tile; two
// key tiles whose token order is chosen so make exactly the lane's 8 tokens of
// the second product's B operand: the probabilities never leave the lane's
// registers.
#include "paged_attn.hpp"

namespace ss {

constexpr int kTile = 32;          // tokens a wave takes at a time
constexpr int kWaves = 4;          // waves of a workgroup
constexpr int kUnit = kTile * kWaves;
constexpr int kStages = 4;         // tiles of a wave in LDS, one computed while the others arrive
// Cache policy of the stream: non-temporal (8 requests of 32768 tokens: 66 us;
// cached: 75 us.  1 request: 20.6 and 21.1 us).
constexpr int kNt = 2;
// Requests of more than kPromptRows query rows a KV head are the prompt
// kernel's, where this one would have more than kPromptUnits units a compute
// unit (at 128 dims; half as much work each at 64) than that one: a column
// costs kColumnUnits beside its units (queries, tables, the join), and a unit of
// a tile of 256 rows there kTileUnits of those here.  Fitted to 888 shapes (1 to
// 32 requests of 17 to 1024 new tokens at up to 8192, 1 to 8 rows a token, all
// groups): the kernel that is taken is 1.5 % behind the better one in the mean
// (work alone, without columns and tiles: 8.6 %).  Here and there: 64 rows of 64
// (request, head) columns at 8192 tokens 88 and 113 us, 96 rows 131 and 114; a
// prompt of 128 tokens and 32 heads 8.8 and 21 us, 512 tokens 32 and 39, 640
// tokens 52 and 43; 32 prompts of 64 tokens 72 and 22; 24 tokens of 8 requests at
// 2048 39 and 49, at 8192 tokens of one 30 and 51.  Below kPromptRows 256-row tiles
// are mostly empty.
constexpr int kPromptRows = 64, kPromptUnits = 32, kColumnUnits = 6, kTileUnits = 3;
// Columns of at most kWhole units are not cut, twice that if there are enough
// of them to give every second compute unit one: a cut adds a launch and a
// pass over the parts.  1 request of 8 heads, 640 tokens: 9.8 us whole, 11.7
// cut; 1536 tokens: 15.8 and 11.7.  16 requests: 640 tokens 10.5 and 15.7,
// 1536 tokens 16.7 and 18.8, 4096 tokens 33.9 and 30.0.
constexpr int kWhole = 8;
// Units of a run that may hold several columns (1 and 8 differ by less than
// runs of the same code do).
constexpr int kMinRun = 4;

// Blocks of `rows` query rows a KV head of a request that are this kernel's,
// and units of its tokens.
__device__ __forceinline__ int blocks_of(const PagedAttn &a, const Request &q, int rows) {
    return q.rows > a.most_rows ? 0 : (q.rows + rows - 1) / rows;
}
__device__ __forceinline__ int units_of(const Request &q) { return max(1, (q.len + kUnit - 1) / kUnit); }

// Parts of a column of `units` units at `share` units a part.
__device__ __forceinline__ int parts_of(int units, int share) {
    return units <= kWhole ? 1 : (int)(((uint32_t)units + (uint32_t)share - 1) / (uint32_t)share);
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
    // (written so that the move is part of the addition)
    if (G >= 2) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, true));  // quad_perm [1,0,3,2]
    if (G >= 4) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, true));  // quad_perm [2,3,0,1]
    return v;
}

// A column is (request, KV head, block of query rows); its tokens are units of
// 128.  A workgroup takes a run of units: a part of one column, or, where
// there are many columns, an even share of all their units, which may hold
// several columns and end inside one.  Parts are joined by
// paged_merge_kernel.  So uneven requests load the device evenly, and the host
// need not know their lengths.
//
// In a part of a column the waves take 32-token tiles in turn, each
// through a ring of its own in LDS that HBM streams into while older tiles
// are computed; their results are joined through LDS at the end.  NS sets of
// 16/G query rows share the stream.
//
// Long caches are bound by HBM and, nearly as much, by the vector ALUs (65 % of
// the cycles): 8 requests of up to 32768 tokens, 8 heads, 195 MB, take 42 us,
// 4.6 TB/s.  One such request, 38 MB, takes 17 us: tables, queries, four tiles
// a wave and the join follow each other.
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
    const int heads = a.st.heads, log_page = a.st.log_page;
    // Rows but [first, last): those before the first request's and behind the last one's.
    auto zero_rows = [&](int first, int last) {
        const int64_t row = (int64_t)a.hq * D, from = min((int64_t)max(0, first), a.n_tokens) * row;
        const int64_t theirs = max(min((int64_t)max(0, last), a.n_tokens) * row - from, (int64_t)0);
        for (int64_t e = blockIdx.x * 256 + threadIdx.x; e < a.n_tokens * row - theirs; e += gridDim.x * 256)
            store_from_f32(a.out, a.q_dtype, e < from ? e : e + theirs, 0.f);
    };
    if (a.zero_rest) zero_rows(table_read(a.starts, 0), table_read(a.starts, a.n_req));

    // This workgroup's run of units [u, stop), and the request r it starts in,
    // whose units start at `base`: every wave works it out by itself, a few
    // requests a lane.
    const int groups = gridDim.x, per = (a.n_req + 63) / 64;
    const int r0 = min(lane * per, a.n_req);
    int r1 = min(r0 + per, a.n_req);
    int units = 0, columns = 0;  // of the lane's requests
    bool down = false;
    for (int i = r0; i < r1; ++i) {
        const Request q = request(a, i);
        down |= descends(a, i);
        const int n = blocks_of(a, q, ROWS) * heads;
        units += units_of(q) * n, columns += n;
    }
    if (__any(down)) {
        units = columns = 0, r1 = r0;
        if (a.zero_rest) zero_rows(0, 0);
    }
    const int units_scan = wave_scan(units);
    const int total = __builtin_amdgcn_readlane(units_scan, 63);
    const int columns_scan = wave_scan(columns);
    const int all_columns = __builtin_amdgcn_readlane(columns_scan, 63);
    int u, stop, base, r, share, parts = 0;
    // Columns to be joined are listed for the merge, (parts, request, first
    // workgroup, column of the request) at `list`: by column where they are few.
    const bool few = a.cut && all_columns <= groups / 2;
    int list = blockIdx.x;
    int4 cut = make_int4(0, 0, 0, 0);
    if (few) {
        // Few columns: each is cut into parts of its own, of at most `share`
        // units, so that no workgroup has more than one.  Sum of ceil(n/share)
        // is at most total/share + columns, and about total/share + columns/2.
        auto items = [&](int share) {
            int n = 0;
            for (int i = r0; i < r1; ++i) {
                const Request q = request(a, i);
                n += blocks_of(a, q, ROWS) * heads * parts_of(units_of(q), share);
            }
            return n;
        };
        share = max(uniform_div(total + groups - all_columns / 2 - 1, groups - all_columns / 2), 1);
        int scan = wave_scan(items(share));
        if (__builtin_amdgcn_readlane(scan, 63) > groups) {
            share = uniform_div(total + groups - all_columns - 1, groups - all_columns);
            scan = wave_scan(items(share));
        }
        const int item = blockIdx.x;
        if (item >= __builtin_amdgcn_readlane(scan, 63)) {
            u = stop = base = r = 0;
        } else {
            const int holder = __ffsll((unsigned long long)__ballot(item < scan)) - 1;
            int left = item - (holder ? __builtin_amdgcn_readlane(scan, holder - 1) : 0);
            base = holder ? __builtin_amdgcn_readlane(units_scan, holder - 1) : 0;
            list = holder ? __builtin_amdgcn_readlane(columns_scan, holder - 1) : 0;
            for (r = holder * per;; ++r) {
                const Request q = request(a, r);
                const int n = blocks_of(a, q, ROWS) * heads, n_units = units_of(q);
                parts = __builtin_amdgcn_readfirstlane(parts_of(n_units, share));
                if (left < n * parts) {
                    const int column = uniform_div(left, parts), part = left - column * parts;
                    u = base + column * n_units;
                    stop = u + part_begin(part + 1, n_units, parts);
                    u += part_begin(part, n_units, parts);
                    list += column;
                    if (part == 0 && threadIdx.x == 0)
                        a.cut[list] = make_int4(parts > 1 ? parts : 0, r, blockIdx.x, column);
                    break;
                }
                left -= n * parts, base += n * n_units, list += n;
            }
        }
    } else {
        // Many: the units of all columns in one row, shared out evenly; a run
        // may end inside a column and may hold several.  (Without `cut`: a
        // workgroup takes the columns that begin in its share, whole.)
        share = max(uniform_div(total + groups - 1, groups), a.cut ? kMinRun : 1);
        u = min((int64_t)blockIdx.x * share, (int64_t)total);
        stop = min((int64_t)u + share, (int64_t)total);
        const uint64_t holds = __ballot(u < units_scan);
        const int holder = holds ? __ffsll((unsigned long long)holds) - 1 : 0;
        base = holder ? __builtin_amdgcn_readlane(units_scan, holder - 1) : 0;
        r = holder * per;
    }
    const int first_unit = u;

    while (u < stop) {
        const Request rq = request(a, r);
        const int row_blocks = blocks_of(a, rq, ROWS), n_units = units_of(rq), in_request = row_blocks * heads * n_units;
        if (u >= base + in_request) {
            base += in_request, ++r;
            continue;
        }
        const int column = uniform_div(u - base, n_units);
        const int c0 = base + column * n_units, c1 = c0 + n_units;
        if (!a.cut && c0 < first_unit) {
            u = c1;
            continue;
        }
        const int h = uniform_div(column, row_blocks), rb = column - h * row_blocks;
        const int begin = (u - c0) * kUnit;
        const int part_end = a.cut ? min(stop, c1) : c1;
        const int end = min((part_end - c0) * kUnit, rq.len);
        const bool whole = c0 >= first_unit && (!a.cut || c1 <= stop);
        const int place = c0 < first_unit ? 0 : 1;  // of this part, if it is one
        if (!few && !whole && place == 1)
            cut = make_int4(uniform_div(c1 - 1, share) - (int)blockIdx.x + 1, r, blockIdx.x, column);
        u = part_end;
        const int32_t *row_table = a.table + (int64_t)r * a.width;

        char *ring = lds + wave * kStages * TL::kBytes;
        const int last_page = (int)min(a.width - 1, (int64_t)INT32_MAX);
        // Page of the 16 tokens from `token`; -1 if the table names none of the pool.
        auto in_pool = [&](int p) { return (uint32_t)p < (uint32_t)a.st.n_pages ? p : -1; };
        auto page_at = [&](int token) { return table_read(row_table, min(token >> log_page, last_page)); };
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
            pages[i][0] = in_pool(page_at(ahead)), pages[i][1] = in_pool(page_at(ahead + 16));
            ahead += kUnit;
        }
        // The queries, here and not where they are used: by then they would wait
        // for the tiles too.
        wait_loads<0>();
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) {
            const int t = begin + kTile * wave + i * kUnit;
            if (t < end) TL::fetch(a.st, h, lane, ring + i * TL::kBytes, t, pages[i][0], pages[i][1]);
        }
        int all_see = rq.len;
        half8_t qf[NS][KS];
        float qz[NS], factor[NS], lag[NS];
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
            const QueryScale by(lanes4_max(top), a.scale);
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float y = in_group ? x[k][e] * by.down : 0.f;
                    sum += y;
                    qf[s][k][e] = (_Float16)y;
                }
            qz[s] = lanes4_sum(sum);
            factor[s] = by.factor;
            lag[s] = kLag / factor[s];
        }
        // (limits grow with the row: the first row's is the smallest)
        if (a.causal) all_see = max(0, min(rq.len, rq.len - rq.n_all + rb * ROWS / a.rep + 1));

        // Probabilities are kept times 2^kProb, so that a sum of bfloat16's largest
        // values stays finite (up to 2^20 tokens) and values down to 2^-102 keep
        // their bits; p * scale enters the products times 2^(kScaled -
        // vexp): vexp is above every value scale (as a power of two) that the
        // column's group has met, so it stays within fp16 whatever the scales.
        // top is in units of S.
        constexpr int kProb = -24, kScaled = 10 - kProb;
        float top[NS], l[NS], z[NS];
        float back[NS];  // added to each group's sum: minus the row's reference / G
        float4_t o[NS][VT], ones[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            top[s] = -INFINITY;
            l[s] = z[s] = back[s] = 0.f;
            ones[s] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < VT; ++j) o[s][j] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
        int vexp = -92;  // (2^(kScaled - vexp) is a float)
        float up = exp2i(kScaled - vexp);
        float offset[NS];  // of the exponents: kProb less the maximum's
        auto set_offset = [&](int s) { offset[s] = kProb - (top[s] == -INFINITY ? 0.f : top[s] * factor[s]); };
#pragma unroll
        for (int s = 0; s < NS; ++s) set_offset(s);
        const CodeBits code_bits;
        auto rescale = [&](int s, float f) {  // (what is times up)
            ones[s] *= f;
#pragma unroll
            for (int j = 0; j < VT; ++j) o[s][j] *= f;
        };

        // mask: some row does not see some token of the tile
        auto compute = [&](const char *slot, int tb, bool ok, bool mask) {
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
            const int first = tb + 8 * quad;  // the lane's first token
            if (mask) {  // (behind the request's tokens a page may hold anything, NaN too)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!ok || first + j >= rq.len) vm[j] = 0;
            }
            float vs[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) vs[j] = low16<BF>(vm[j]);
            const float vtop = column_max(vs);
            if (__any(vtop > exp2i(vexp))) {
                const float c = lanes4_max(vtop);
                const int e = (int)((__float_as_uint(c) >> 23) & 0xffu) - 126;  // c < 2^e
                const int now = max(vexp, min(e, 126));
#pragma unroll
                for (int s = 0; s < NS; ++s) rescale(s, ldexpf(1.f, vexp - now));
                vexp = now, up = exp2i(kScaled - vexp);
            }
            // (sets inside: an operand's registers serve every set and are free again)
            float xs[NS][8];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float4_t d[NS];
#pragma unroll
                for (int s = 0; s < NS; ++s) d[s] = float4_t{-qz[s], -qz[s], -qz[s], -qz[s]};
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const half8_t key = codes_operand(kw[y][k], code_bits);
#pragma unroll
                    for (int s = 0; s < NS; ++s)
                        d[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, qf[s][k], d[s], 0, 0, 0);
                }
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t m = km[4 * y + i];
                        xs[s][4 * y + i] = groups_sum<G>(fmaf(low16<BF>(m), d[s][i], fmaf(high16<BF>(m), qz[s] / 64.f, back[s])));
                    }
            }
            half8_t p16[NS];
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                float(&x)[8] = xs[s];
                float v[8], mid[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = vs[j] * up, mid[j] = fmaf(vs[j], 7.5f, high16<BF>(vm[j]));
                if (mask) {  // what the row does not see adds nothing, whatever its value holds
                    const int see = ok ? limit[s] : 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (first + j >= see) x[j] = -INFINITY, v[j] = mid[j] = 0.f;
                }
                const float m = column_max(x);
                if (__any(m > top[s] + lag[s])) {
                    const float now = fmaxf(top[s], lanes4_max(m));
                    const float f = now == top[s] ? 1.f : fast_exp2((top[s] - now) * factor[s]);
                    l[s] *= f, z[s] *= f;
                    rescale(s, f);
                    top[s] = now;
                    if (__any(is_far(now, factor[s]))) {
                        const float move = is_far(now, factor[s]) ? now : 0.f;
                        back[s] -= move / G, top[s] -= move;
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] -= move;
                    }
                    set_offset(s);
                }
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float p = fast_exp2(fmaf(x[j], factor[s], offset[s]));
                    // the value's middle, zero + 7.5 scale, in float32: what is
                    // left for the product, (code - 7.5) scale, is small
                    l[s] += p;
                    z[s] = fmaf(p, mid[j], z[s]);
                    w[j] = p * v[j];
                }
                // one rounding to fp16, 2^-11 of w (code - 7.5): the sum of the
                // rounded w is taken off again at the end
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const half2_t hh = __builtin_convertvector(float2_t{w[j], w[j + 1]}, half2_t);
                    p16[s][j] = hh[0], p16[s][j + 1] = hh[1];
                }
                ones[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_operand(0, code_bits), p16[s], ones[s], 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < VT; ++j) {
                const half8_t v = codes_operand(vw[j], code_bits);
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
            compute(slot, tb, ok, tb + kTile > all_see || p0 < 0 || p1 < 0);
        };
        int slot = 0;
        for (int tb = begin + kTile * wave; tb < end; tb += kUnit) {
            constexpr int last = kStages - 1;
            // (read here and looked at below: their wait is then the codes' own)
            const int new0 = page_at(ahead), new1 = page_at(ahead + 16);
            step(ring + (slot + last) % kStages * TL::kBytes, ring + slot * TL::kBytes, tb, pages[0][0], pages[0][1],
                 pages[last][0], pages[last][1]);
            slot = (slot + 1) % kStages;
#pragma unroll
            for (int i = 0; i < last; ++i) pages[i][0] = pages[i + 1][0], pages[i][1] = pages[i + 1][1];
            pages[last][0] = in_pool(new0), pages[last][1] = in_pool(new1);
            ahead += kUnit;
        }
        __syncthreads();  // the ring's memory takes the results

        // the waves' results, joined
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const float lsum = lanes4_sum(l[s]), zsum = lanes4_sum(z[s]);
            const int row = s * RS + col / G;
            if (g == 0 && quad == 0) stats[wave][row][0] = (top[s] - G * back[s]) * factor[s], stats[wave][row][1] = lsum;
            if (in_group) {
                // tile j, element i: dim (4 * quad + i) * D/16 + j
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < VT; ++j)
                        part[wave][row][(4 * quad + i) * VT + j] = ldexpf(64.f * o[s][j][i] - 71.5f * ones[s][i], vexp - kScaled) + zsum;
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
            if (whole) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const int64_t at = ((int64_t)(rq.t0 + n / a.rep) * a.hq + h * a.rep + n % a.rep) * D + c;
                store_out4(a, at, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
            } else {
                const int64_t at = ((int64_t)blockIdx.x * 2 + place) * ROWS + row;
                *reinterpret_cast<float4 *>(a.acc + at * D + c) = make_float4(x[0], x[1], x[2], x[3]);
                if (c == 0) *reinterpret_cast<float2 *>(a.ml + at * 2) = make_float2(m, l);
            }
        }
        __syncthreads();
    }
    if (a.cut && threadIdx.x == 0) {
        if (!few) a.cut[blockIdx.x] = cut;
        if (blockIdx.x == 0) a.cut[groups] = make_int4(few ? all_columns : groups, 0, 0, 0);
    }
}

// Joins the parts of the columns listed (the second place of the workgroup
// that began one, the first place of those that follow), one row (blockIdx.x)
// a workgroup: every thread loads four dims of its parts at once, 8 (D 128) or
// 16 threads a dim.  The host knows how many columns there can be and launches
// no more workgroups than that: 4.4 us for 8 columns of 64 parts, of which the
// launch and four reads in a row are nearly all (a workgroup for each of 512
// possible parts: 4.9 us).
template <int D>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedAttn a, int rows_per_block,
                                                          int groups) {
    constexpr int CH = D / 4, PARTS = 256 / CH, PER = 8, STEP = PARTS * PER;
    __shared__ float red[PARTS][D + 4];
    __shared__ float total[PARTS], tops[kWaves];
    const int4 begin = a.cut[blockIdx.y];  // (not after the count: one wait for both)
    const int n_list = a.cut[groups].x;
    for (int k = blockIdx.y; k < n_list; k += gridDim.y) {
        const int4 cut = k == (int)blockIdx.y ? begin : a.cut[k];
        const int parts = cut.x, row = blockIdx.x;
        if (parts == 0) continue;
        const Request rq = request(a, cut.y);
        const int row_blocks = blocks_of(a, rq, rows_per_block);
        const int h = uniform_div(cut.w, row_blocks), n = (cut.w - h * row_blocks) * rows_per_block + row;
        if (n >= rq.rows) continue;
        auto at = [&](int i) { return (((int64_t)cut.z + i) * 2 + (i == 0 ? 1 : 0)) * rows_per_block + row; };
        const int c = threadIdx.x % CH * 4, p = threadIdx.x / CH, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        float4 v[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i)
            v[i] = *reinterpret_cast<const float4 *>(a.acc + at(min(p + i * PARTS, parts - 1)) * D + c);
        float m = -INFINITY;
        for (int i = threadIdx.x; i < parts; i += 256) m = fmaxf(m, a.ml[at(i) * 2]);
        m = wave_max(m);
        if (lane == 0) tops[wave] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, tops[w]);
        float x[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
        for (int from = 0; from < parts; from += STEP) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int s = from + p + i * PARTS;
                if (s >= parts) break;
                const float2 e = *reinterpret_cast<const float2 *>(a.ml + at(s) * 2);
                const float f = e.x == m ? 1.f : fast_exp2(e.x - m);
                l += f * e.y;
                x[0] += f * v[i].x, x[1] += f * v[i].y, x[2] += f * v[i].z, x[3] += f * v[i].w;
            }
            if (from + STEP < parts)
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    v[i] = *reinterpret_cast<const float4 *>(a.acc + at(min(from + STEP + p + i * PARTS, parts - 1)) * D + c);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) red[p][c + k] = x[k];
        if (c == 0) total[p] = l;
        __syncthreads();
        if (threadIdx.x < CH) {
            float y[4] = {0.f, 0.f, 0.f, 0.f}, t = 0.f;
#pragma unroll
            for (int i = 0; i < PARTS; ++i) {
                t += total[i];
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] += red[i][c + k];
            }
            const float inv = t == 0.f ? 0.f : 1.f / t;
            const int64_t o = ((int64_t)(rq.t0 + n / a.rep) * a.hq + h * a.rep + n % a.rep) * D + c;
            store_out4(a, o, y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
        }
        __syncthreads();  // (the next column's sums)
    }
}

// -------------------------------------------------------------------- host

struct PagedPlan {
    int sets, rows, groups;  // column sets, query rows a workgroup takes; workgroups
    int columns;             // that there can be, at most `groups`
    bool cut;                // whether columns may be cut
    bool prompts;            // whether requests of many rows are the prompt kernel's
    size_t bytes;
};

// Launch shape: as many workgroups as the device holds at once (two a compute
// unit), or as the hints' units need.
static PagedPlan paged_plan(const ss_paged_store *s, int64_t n_tokens, int64_t n_requests, int n_q_heads,
                            int64_t max_new, int64_t max_length) {
    PagedPlan p{};
    const int rep = n_q_heads / s->n_kv_heads, rs = 16 / (s->head_dim / s->group_size);
    int64_t rows = max_new * rep;
    p.sets = rows > rs ? 2 : 1;
    p.rows = p.sets * rs;
    const int64_t units = (max_length + kUnit - 1) / kUnit;
    // columns of requests of at most `rows` rows each
    auto columns_of = [&](int64_t rows) {
        return s->n_kv_heads * min((double)n_requests * ((rows + p.rows - 1) / p.rows),
                                   (double)(n_tokens * rep / p.rows) + (double)n_requests);
    };
    if (rows > kPromptRows) {
        // what is more than a token a request, in as few requests as it fits
        const double more = (double)max(n_tokens - n_requests, (int64_t)0) * rep;
        const double longs = min((double)n_requests, ceil(more / rows));
        const double columns = s->n_kv_heads * (more / p.rows + longs);
        const double tiles = s->n_kv_heads * longs * (double)((rows + kPromptTile - 1) / kPromptTile);
        p.prompts = kColumnUnits * columns + (columns - kTileUnits * tiles) * units * s->head_dim / 128. >
                    (double)kPromptUnits * device_cu_count();
    }
    if (p.prompts) rows = kPromptRows;
    const double columns = columns_of(rows);
    p.cut = units > (2 * columns < device_cu_count() ? kWhole : 2 * kWhole);
    p.groups = (int)min((double)(2 * device_cu_count()), columns * (p.cut ? (double)units : 1.));
    p.groups = max(p.groups, 1);
    p.columns = (int)min(columns, (double)p.groups);
    p.bytes = p.cut ? 16 + (size_t)p.groups * (16 + 2 * p.rows * (s->head_dim + 2) * 4) : 0;
    if (p.prompts)  // (one after the other: they share it)
        p.bytes = max(p.bytes, paged_prompt_bytes(s, n_requests, n_tokens * rep, kPromptRows));
    return p;
}

// Units that tables of this width can ask of the decode kernel, which counts
// them in 32 bits: a request of r rows, up to kPromptRows with the prompt
// kernel beside it, is (r + rows - 1) / rows blocks.
constexpr double kCounted = 2147483648.0;
static double most_units(const ss_paged_store *s, const PagedPlan &p, int64_t n_tokens, int64_t n_requests, int rep,
                         int64_t table_width) {
    const double requests = (double)min(n_requests, n_tokens);
    double blocks = requests + (double)n_tokens * rep / p.rows;
    if (p.prompts) blocks = min(blocks, requests * ((kPromptRows + p.rows - 1) / p.rows));
    return blocks * s->n_kv_heads * (double)((table_width * s->page_size + kUnit - 1) / kUnit);
}

static int check_hints(const ss_paged_store *s, int64_t n_requests, int n_q_heads, int64_t max_new,
                       int64_t max_length) {
    SS_REQUIRE(n_requests >= 1 && n_requests <= 65535, "n_requests must be 1 .. 65535");
    SS_REQUIRE(n_q_heads >= 1 && n_q_heads % s->n_kv_heads == 0,
               "query heads must be a multiple of the KV heads");
    SS_UNSUPPORTED(n_q_heads <= 1024, "more than 1024 query heads");
    SS_REQUIRE(max_new >= 1 && max_new <= INT32_MAX && max_length >= 1 && max_length <= INT32_MAX,
               "max_new and max_length must be 1 .. 2^31 - 1");
    return SS_OK;
}

template <int D, int G, bool BF>
static void launch_paged(const PagedAttn &a, const PagedPlan &p, hipStream_t st) {
    if (p.sets == 1)
        hipLaunchKernelGGL((paged_attn_kernel<D, G, BF, 1>), dim3(p.groups), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((paged_attn_kernel<D, G, BF, 2>), dim3(p.groups), dim3(256), 0, st, a);
    if (p.cut)
        hipLaunchKernelGGL(paged_merge_kernel<D>, dim3(p.rows, p.columns), dim3(256), 0, st, a, p.rows, p.groups);
}

}  // namespace ss

using namespace ss;

extern "C" size_t ss_paged_attn_workspace_bytes(const ss_paged_store *store, int64_t n_tokens, int64_t n_requests,
                                                int n_q_heads, int64_t max_new, int64_t max_length) {
    PagedStore ps;
    int log_page;
    if (check_paged_store(store, &ps, &log_page) || check_hints(store, n_requests, n_q_heads, max_new, max_length) ||
        n_tokens < 0 || n_tokens > INT32_MAX / n_q_heads)
        return 0;
    return paged_plan(store, n_tokens, n_requests, n_q_heads, max_new, max_length).bytes;
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
    SS_REQUIRE(((uintptr_t)out & 7) == 0, "out must be 8-byte aligned");
    SS_REQUIRE(table_width >= 1, "bad block table width");
    SS_UNSUPPORTED(table_width <= (1 << 30) / store->page_size, "a table row of more than 2^30 tokens");
    PagedPlan p = paged_plan(store, n_tokens, n_requests, n_q_heads, max_new, max_length);
    // (hints that are too low for the tables)
    const int rep = n_q_heads / store->n_kv_heads;
    p.prompts |= most_units(store, p, n_tokens, n_requests, rep, table_width) >= kCounted;
    SS_UNSUPPORTED(most_units(store, p, n_tokens, n_requests, rep, table_width) < kCounted,
                   "%lld requests, %lld tokens and %lld pages a table row: more blocks of query rows and of %d tokens "
                   "than 32 bits count",
                   (long long)n_requests, (long long)n_tokens, (long long)table_width, kUnit);
    if (p.bytes > workspace_bytes || (p.bytes && !workspace)) {
        set_error("workspace of %zu bytes, %zu needed", workspace_bytes, p.bytes);
        return SS_ERR_WORKSPACE;
    }
    SS_REQUIRE(((uintptr_t)workspace & 15) == 0, "workspace must be 16-byte aligned");
    a.q = q, a.q_st = q_st, a.q_sh = q_sh, a.out = out;
    a.table = block_table, a.lengths = lengths, a.starts = token_starts;
    a.width = table_width, a.n_tokens = n_tokens, a.n_req = (int)n_requests;
    a.hq = n_q_heads, a.rep = rep;
    a.q_dtype = q_dtype, a.causal = causal, a.zero_rest = zero_rest, a.scale = scale;
    a.vec = ((uintptr_t)q & 15) == 0 && q_st % 8 == 0 && q_sh % 8 == 0;
    a.most_rows = p.prompts ? kPromptRows : INT32_MAX;
    a.cut = p.cut ? static_cast<int4 *>(workspace) : nullptr;
    a.acc = reinterpret_cast<float *>(a.cut + p.groups + 1);
    a.ml = a.acc + (size_t)p.groups * 2 * p.rows * store->head_dim;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const bool bf = store->dtype == SS_BF16;
    const int key = store->head_dim * 1000 + store->group_size;
    if (key == 128032) bf ? launch_paged<128, 4, true>(a, p, st) : launch_paged<128, 4, false>(a, p, st);
    else if (key == 128064) bf ? launch_paged<128, 2, true>(a, p, st) : launch_paged<128, 2, false>(a, p, st);
    else if (key == 128128) bf ? launch_paged<128, 1, true>(a, p, st) : launch_paged<128, 1, false>(a, p, st);
    else if (key == 64032) bf ? launch_paged<64, 2, true>(a, p, st) : launch_paged<64, 2, false>(a, p, st);
    else bf ? launch_paged<64, 1, true>(a, p, st) : launch_paged<64, 1, false>(a, p, st);
    SS_LAUNCH_CHECK("paged_attn_kernel launch");
    return p.prompts ? launch_paged_prompt(a, store, workspace, workspace_bytes, st) : SS_OK;
}
