// Paged 4-bit key/value cache: block tables, the quantising append and its
// inverse.  The attention over these pages is paged_attn.hip.
//
// A page holds P tokens of every KV head.  Per (page, head):
//   k_codes u32 [P][D/8]     dims 8w .. 8w+7 of a token in word w
//   v_codes u32 [P/8][D]     tokens 8w .. 8w+7 at dim d in word [w][d]
//   k_meta, v_meta [G][P]    (scale, zero) pairs of 16-bit floats per group
// Element j of a word sits at bit 4*(j/2) + 16*(j%2) (the interleaving of the
// grouped value codes), so (w >> 4p) & 0x000f000f is the pair (2p, 2p+1) as
// two 16-bit halves: the operand order of the matrix cores.  Keys are packed
// along the head's dims and values along the tokens because those are the
// axes that Q.K^T and P.V sum over.
#include "paged_append.hpp"

namespace ss {

// ------------------------------------------------------------ block tables

// Requests in one workgroup's tables (starts and page offsets in LDS).
constexpr int kMaxRequests = 4096;
constexpr int kTableThreads = 1024;
// Tokens up to which the table kernel also writes the slots itself; more get
// a launch of their own over many workgroups.  With a request per 16th of the
// tokens: 16 tokens 6.5 us in one launch, 7.7 in two; 4096 tokens 8.3 and 8.6;
// 8192 tokens 10.3 and 8.6.
constexpr int64_t kSlotsInline = 4096;

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int log_page) {
    return (tokens + (1 << log_page) - 1) >> log_page;
}

// Request of token `tok`: the last r with starts[r] <= tok (requests without
// new tokens share their start with the next one and are passed over).
__device__ __forceinline__ int request_of(const int32_t *starts, int n_req, int tok) {
    int lo = 0, hi = n_req;  // starts[lo] <= tok < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= tok)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

__device__ __forceinline__ void write_slot(int64_t tok, const int32_t *starts, int n_req, const int32_t *ends,
                                           const int32_t *table, int64_t width, int log_page, int32_t *slots,
                                           int32_t *positions) {
    int32_t slot = -1, pos = -1;
    if (tok < starts[n_req]) {
        const int r = request_of(starts, n_req, (int)tok);
        // ends: lengths after the step; the request's new tokens are its last
        pos = ends[r] - (starts[r + 1] - (int)tok);
        // (a page whose slots 32 bits do not hold is in no pool: its tokens have none)
        const uint32_t page = table[r * width + (pos >> log_page)];
        if (page <= (uint32_t)INT32_MAX >> log_page) slot = (int32_t)(page << log_page) + (pos & ((1 << log_page) - 1));
    }
    slots[tok] = slot;
    if (positions) positions[tok] = pos;
}

// One workgroup.  Thread i owns requests [i*per, (i+1)*per); one scan of
// (new tokens, pages given back, pages taken) over the threads gives every
// request its token start and its place on the stack.  All checks come first:
// a step that cannot be done whole changes nothing and says why in `status`.
// lengths_out and n_free_out may be lengths and n_free: every thread rewrites
// only lengths that it alone still reads, behind the barriers.
// What bounds it is latency, not bytes: 5.2 us for one request, of which most
// is the launch and the scan's barriers.  One workgroup, as every request's
// place depends on all before it, and a grid-wide scan would be more launches.
// 256 requests of up to 2048 pages, 26 of which end: 12.7 us (a wave to a
// request at a time: 42 us, as the ended ones can fall to one wave); 61
// prompts of 8003 tokens: 7.7 us, and 3.8 us of slots_kernel.
__global__ void __launch_bounds__(kTableThreads)
    block_tables_kernel(const int32_t *lengths, const int32_t *added, int n_req, int32_t *table, int64_t width,
                        int32_t *free_pages, int64_t pool, const int32_t *n_free, int log_page, int64_t n_tok,
                        int32_t *lengths_out, int32_t *n_free_out, int32_t *token_starts, int32_t *slots,
                        int32_t *positions, int32_t *status, int inline_slots) {
    __shared__ int32_t starts[kMaxRequests + 1];
    __shared__ int32_t ends[kMaxRequests];
    // pages given back and taken by the requests before one
    __shared__ int32_t given[kMaxRequests + 1];
    __shared__ int32_t taken[kMaxRequests + 1];
    __shared__ int64_t sums[3][kTableThreads / kWave];
    __shared__ int bad;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (n_req + kTableThreads - 1) / kTableThreads;
    const int r0 = min(tid * per, n_req), r1 = min(r0 + per, n_req);
    const int64_t most = min(width << log_page, (int64_t)INT32_MAX);
    if (tid == 0) bad = 0;
    __syncthreads();

    int64_t s[3] = {0, 0, 0};  // tokens, pages given, pages taken of the thread's requests
    int wrong = 0;
    for (int r = r0; r < r1; ++r) {
        const int64_t len = lengths[r], end = len + added[r];
        if (len < 0 || end < 0) wrong |= 1;
        if (len > most || end > most) wrong |= 2;
        const int64_t d = pages_of(end, log_page) - pages_of(len, log_page);
        s[0] += max(end - len, (int64_t)0);
        s[1] += max(-d, (int64_t)0);
        s[2] += max(d, (int64_t)0);
    }
    int64_t before[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        int64_t x = s[k];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        before[k] = x - s[k];
        if (lane == 63) sums[k][wave] = x;
    }
    __syncthreads();
    int64_t total[3] = {0, 0, 0};
#pragma unroll
    for (int k = 0; k < 3; ++k)
        for (int w = 0; w < kTableThreads / kWave; ++w) {
            if (w < wave) before[k] += sums[k][w];
            total[k] += sums[k][w];
        }
    const int64_t avail = n_free[0];
    if (total[2] > max(avail, (int64_t)0) + total[1]) wrong |= 4;
    if (total[0] > n_tok) wrong |= 8;
    if (avail < 0 || avail + total[1] > pool) wrong |= 16;
    if (wrong) atomicOr(&bad, wrong);
    __syncthreads();
    const int failed = bad;
    for (int r = r0; r < r1; ++r) {
        const int32_t len = lengths[r], n = failed ? 0 : added[r];
        const int32_t d = failed ? 0 : (int32_t)(pages_of(len + n, log_page) - pages_of(len, log_page));
        starts[r] = failed ? 0 : (int32_t)before[0];
        ends[r] = len + n;
        given[r] = failed ? 0 : (int32_t)before[1];
        taken[r] = failed ? 0 : (int32_t)before[2];
        before[0] += max(n, 0);
        before[1] += max(-d, 0);
        before[2] += max(d, 0);
    }
    if (tid == 0) {
        starts[n_req] = failed ? 0 : (int32_t)total[0];
        given[n_req] = failed ? 0 : (int32_t)total[1];
        taken[n_req] = failed ? 0 : (int32_t)total[2];
    }
    __syncthreads();

    // Page i of those given back (taken) is the last request's with prefix <= i.
    // Every wave has an even run of these pages, whatever the requests, and
    // looks for the request only where the run leaves one; four at a time, so
    // that their reads overlap.
    auto each_page = [&](const int32_t *prefix, bool give, auto move) {
        const int n = prefix[n_req], run = (int)(((int64_t)n + kTableThreads - 1) / kTableThreads) * kWave;
        const int stop = min(n, (wave + 1) * run);
        int r = -1, next = 0;  // the request, and the first page behind its own
        int64_t at = 0;        // table entry of page i, less i
        for (int i0 = wave * run + lane; i0 < stop; i0 += 4 * kWave) {
            int64_t entry[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = i0 + u * kWave;
                if (i >= next && i < stop) {
                    if (prefix[++r + 1] <= i) r = request_of(prefix, n_req, i);
                    next = prefix[r + 1];
                    // those given back lie behind the pages kept, those taken end them
                    at = r * width + pages_of(ends[r], log_page) - (give ? prefix[r] : next);
                }
                entry[u] = at + i;
            }
            move(i0, stop, entry);
        }
    };
    each_page(given, true, [&](int i0, int stop, const int64_t (&entry)[4]) {
        int32_t page[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i0 + u * kWave < stop) page[u] = table[entry[u]];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i0 + u * kWave < stop) free_pages[avail + i0 + u * kWave] = page[u];
    });
    __syncthreads();  // (the stack is read back below)
    each_page(taken, false, [&](int i0, int stop, const int64_t (&entry)[4]) {
        const int64_t top = avail + total[1] - 1;
        int32_t page[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i0 + u * kWave < stop) page[u] = free_pages[top - i0 - u * kWave];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i0 + u * kWave < stop) table[entry[u]] = page[u];
    });
    for (int r = tid; r <= n_req; r += kTableThreads) {
        token_starts[r] = starts[r];
        if (r < n_req) lengths_out[r] = ends[r];
    }
    if (tid == 0) {
        n_free_out[0] = (int32_t)(failed ? avail : avail + total[1] - total[2]);
        status[0] = failed;
    }
    if (!inline_slots) return;
    __syncthreads();  // (the tables are read back)
    for (int64_t t = tid; t < n_tok; t += kTableThreads)
        write_slot(t, starts, n_req, ends, table, width, log_page, slots, positions);
}

__global__ void __launch_bounds__(256)
    slots_kernel(const int32_t *token_starts, int n_req, const int32_t *ends, const int32_t *table, int64_t width,
                 int log_page, int64_t n_tok, int32_t *slots, int32_t *positions) {
    __shared__ int32_t starts[kMaxRequests + 1];
    for (int r = threadIdx.x; r <= n_req; r += 256) starts[r] = token_starts[r];
    __syncthreads();
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t < n_tok) write_slot(t, starts, n_req, ends, table, width, log_page, slots, positions);
}

// ------------------------------------------------------------- shared plan

// Row of token `tok` in the group of its request's parent, and its position.
__device__ __forceinline__ void write_shared(int64_t tok, const int32_t *starts, int n_req, const int32_t *lengths,
                                             const int32_t *parents, const int32_t *offsets, int2 *rows,
                                             int32_t *positions) {
    int64_t pos = -1;
    if (tok >= starts[0] && tok < starts[n_req]) {
        const int r = request_of(starts, n_req, (int)tok), p = parents[r];
        const int own = lengths[r] - (starts[r + 1] - (int)tok);
        if (p >= 0) rows[offsets[r] + (int)tok - starts[r]] = make_int2((int)tok, own);
        pos = max((int64_t)own + (p >= 0 ? max(lengths[p], 0) : 0), (int64_t)-1);
    }
    if (positions) positions[tok] = (int32_t)min(pos, (int64_t)INT32_MAX);
}

// One workgroup sorts the requests by their parents, in the requests' order:
// each wave ranks 64 of them among themselves, then the 64s follow each other.
// Latency bounds it, as the block tables: everything is read first, and few
// requests take a workgroup of four waves, whose barriers are cheaper.
template <int THREADS>
__global__ void __launch_bounds__(THREADS)
    shared_plan_kernel(const int32_t *parents, const int32_t *lengths, const int32_t *token_starts, int n_req,
                       int64_t n_tok, int32_t *group_starts, int2 *rows, int32_t *parents_out, int32_t *offsets,
                       int32_t *positions, int inline_rows) {
    constexpr int MOST = THREADS == kTableThreads ? kMaxRequests : THREADS;
    __shared__ int32_t starts[MOST + 1];
    __shared__ int32_t parent[MOST];
    __shared__ int32_t length[MOST];
    __shared__ int32_t offset[MOST];     // of a request's rows among its parent's
    __shared__ int32_t count[MOST + 1];  // rows of a parent: so far, then all, then before it
    __shared__ int32_t sums[THREADS / kWave];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int down = 0;
    for (int r = tid; r <= n_req; r += THREADS) {
        const int32_t from = token_starts[r];
        if (r < n_req) {
            const int32_t to = token_starts[r + 1], p = parents[r], n = lengths[r];
            down |= to < from;
            parent[r] = (uint32_t)p < (uint32_t)n_req && p != r && from >= 0 ? p : -1;
            length[r] = n;
        }
        starts[r] = from, count[r] = 0;
    }
    const bool failed = __syncthreads_or(down);
    auto rows_of = [&](int r) {  // of those that exist
        return r >= n_req || failed || starts[r] < 0 ? 0 : (int)max(min((int64_t)starts[r + 1], n_tok) - starts[r], (int64_t)0);
    };
    for (int r0 = wave * kWave; r0 < n_req; r0 += THREADS) {
        const int r = r0 + lane, n = rows_of(r), p = r < n_req && !failed ? parent[r] : -1;
        int before = 0;
        for (uint64_t left = __ballot(p >= 0); left;) {  // (one parent after the other)
            const bool mine = p == __builtin_amdgcn_readlane(p, __ffsll((unsigned long long)left) - 1);
            const int rows = mine ? n : 0, sum = wave_scan(rows);
            if (mine) before = sum - rows;
            left &= ~__ballot(mine);
        }
        if (r < n_req) parent[r] = p, offset[r] = before;
    }
    __syncthreads();
    if (wave == 0)
        for (int r0 = 0; r0 < n_req; r0 += kWave) {
            const int r = r0 + lane, p = r < n_req ? parent[r] : -1;
            if (p >= 0) offset[r] += count[p];
            wave_lds_sync();
            if (p >= 0) atomicAdd(&count[p], rows_of(r));
            wave_lds_sync();
        }
    __syncthreads();
    // where each parent's rows start
    const int per = (n_req + THREADS - 1) / THREADS;
    const int p0 = min(tid * per, n_req), p1 = min(p0 + per, n_req);
    int s = 0;
    for (int p = p0; p < p1; ++p) s += count[p];
    int scan = wave_scan(s);
    if (lane == 63) sums[wave] = scan;
    __syncthreads();
    int from = scan - s;
    for (int w = 0; w < wave; ++w) from += sums[w];
    for (int p = p0; p < p1; ++p) {
        const int n = count[p];
        count[p] = from, group_starts[p] = from;
        from += n;
    }
    if (p1 == n_req && p0 < p1) group_starts[n_req] = from;
    __syncthreads();
    for (int r = tid; r < n_req; r += THREADS) {
        const int p = parent[r];
        if (p >= 0) offset[r] += count[p];
        parents_out[r] = p, offsets[r] = offset[r];
    }
    if (!inline_rows) return;
    __syncthreads();
    if (failed) {
        if (positions)
            for (int64_t t = tid; t < n_tok; t += THREADS) positions[t] = -1;
        return;
    }
    for (int64_t t = tid; t < n_tok; t += THREADS) write_shared(t, starts, n_req, length, parent, offset, rows, positions);
}

__global__ void __launch_bounds__(256)
    shared_rows_kernel(const int32_t *token_starts, int n_req, int64_t n_tok, const int32_t *lengths,
                       const int32_t *parents, const int32_t *offsets, int2 *rows, int32_t *positions) {
    __shared__ int32_t starts[kMaxRequests + 1];
    __shared__ int bad;
    if (threadIdx.x == 0) bad = 0;
    for (int r = threadIdx.x; r <= n_req; r += 256) starts[r] = token_starts[r];
    __syncthreads();
    for (int r = threadIdx.x; r < n_req; r += 256)
        if (starts[r + 1] < starts[r]) bad = 1;
    __syncthreads();
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= n_tok) return;
    if (bad) {
        if (positions) positions[t] = -1;
        return;
    }
    write_shared(t, starts, n_req, lengths, parents, offsets, rows, positions);
}

// ------------------------------------------------------------------ append

// A wave takes 8 consecutive new tokens of one KV head, 8 values a lane.
// Key words are whole per token; value words hold 8 tokens each, which the wave
// transposes through LDS.  Vector operations bound long prompts (some
// 11 to quantise a value, and the 8 x 8 transposes), the latency of load ->
// reduce -> store short ones: 8192 tokens of 8 heads x 128 dims take 16 us
// (43 MB, 2.7 TB/s; the bytes alone would take 8.3 us), 16 tokens 7 us.
template <int D, int GROUP, bool BF>
__global__ void __launch_bounds__(256)
    append_paged_kernel(PagedStore st, const void *keys, const void *values, int in_dtype, int vec, int64_t k_st,
                        int64_t k_sh, int64_t v_st, int64_t v_sh, const int32_t *slots, int64_t n_tok,
                        uint32_t n_items) {
    constexpr int LPR = D / 8;          // lanes a row
    constexpr int RPP = 64 / LPR;       // rows a pass
    constexpr int PASSES = 8 / RPP;
    constexpr int G = D / GROUP;
    __shared__ uint32_t tile[4][8][LPR + 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t item = blockIdx.x * 4 + wave;
    if (item >= n_items) return;  // whole waves leave; no barrier follows
    const uint32_t win = item / (uint32_t)st.heads;
    const int h = (int)(item - win * (uint32_t)st.heads);
    const int64_t t0 = (int64_t)win * 8;
    const int n_slots = st.n_pages << st.log_page;
    // lane e < 8 holds the slot of token t0 + e (-1: not stored)
    int my_slot = -1;
    if (lane < 8 && t0 + lane < n_tok) {
        my_slot = slots[t0 + lane];
        if ((uint32_t)my_slot >= (uint32_t)n_slots) my_slot = -1;
    }
    const int w = lane % LPR, g = (w * 8) / GROUP;
    float x[2][PASSES][8];
    int slot_of[PASSES];
    const bool half = in_dtype != SS_F32 && vec;  // one wide load for 8 values
    uint4 raw[2][PASSES];
    auto row_of = [&](int p) { return min(t0 + p * RPP + lane / LPR, n_tok - 1); };
    if (half) {  // (all before the first is looked at)
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            raw[0][p] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(keys) + row_of(p) * k_st + h * k_sh + w * 8);
            raw[1][p] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(values) + row_of(p) * v_st + h * v_sh + w * 8);
        }
    } else {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            load8_f32(keys, in_dtype, vec, row_of(p) * k_st + h * k_sh + w * 8, x[0][p]);
            load8_f32(values, in_dtype, vec, row_of(p) * v_st + h * v_sh + w * 8, x[1][p]);
        }
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) slot_of[p] = __shfl(my_slot, p * RPP + lane / LPR);
    if (half) {
        if (in_dtype == SS_F16)
#pragma unroll
            for (int i = 0; i < 2 * PASSES; ++i) unpack16<__half>(raw[i / PASSES][i % PASSES], x[i / PASSES][i % PASSES]);
        else
#pragma unroll
            for (int i = 0; i < 2 * PASSES; ++i) unpack16<__hip_bfloat16>(raw[i / PASSES][i % PASSES], x[i / PASSES][i % PASSES]);
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int e = p * RPP + lane / LPR, slot = slot_of[p];
        const int64_t row = (int64_t)(slot >> st.log_page) * st.heads + h;
        const int off = slot & ((1 << st.log_page) - 1);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            if (in_dtype != (BF ? SS_BF16 : SS_F16))
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const uint32_t u = pack16<BF>(x[kv][p][i], x[kv][p][i + 1]);
                    x[kv][p][i] = from_bits16<BF>(u & 0xffffu), x[kv][p][i + 1] = from_bits16<BF>(u >> 16);
                }
            uint32_t meta;
            const uint32_t word = quantize8<GROUP / 8, BF>(x[kv][p], meta);
            if (kv) tile[wave][e][w] = word;
            if (slot >= 0) {
                if (!kv) st.k_codes[((row << st.log_page) + off) * LPR + w] = word;
                if (w % (GROUP / 8) == 0) (kv ? st.v_meta : st.k_meta)[((row * G + g) << st.log_page) + off] = meta;
            }
        }
    }
    store_value_words<D>(st, tile[wave], h, lane, my_slot);
}

// -------------------------------------------------------------------- read

// A thread takes 8 dims of the keys and of the values of one token and head:
// value = zero + code * scale, one rounding to the cache's type.  Tokens
// without a slot read as zeros.  A value word's 8 tokens are 8 threads', whose
// reads of it meet in the caches; 8192 tokens of 8 heads x 128 dims take 11.3
// us (43 MB, 3.8 TB/s), a copy of as many bytes 8.3 us.
template <int D, bool BF>
__global__ void __launch_bounds__(256)
    read_paged_kernel(PagedStore st, const int32_t *slots, int log_group, uint32_t n_rows, uint16_t *keys,
                      uint16_t *values) {
    constexpr int W = D / 8;
    const uint32_t th = blockIdx.x * (256 / W) + threadIdx.x / W;  // (token, head)
    if (th >= n_rows) return;
    const int w = threadIdx.x % W;
    const uint32_t t = th / (uint32_t)st.heads;
    const int h = (int)(th - t * (uint32_t)st.heads);
    const int slot = slots[t];
    uint4 *const to_k = reinterpret_cast<uint4 *>(keys + (int64_t)th * D) + w;
    uint4 *const to_v = reinterpret_cast<uint4 *>(values + (int64_t)th * D) + w;
    if ((uint32_t)slot >= (uint32_t)(st.n_pages << st.log_page)) {
        *to_k = *to_v = make_uint4(0, 0, 0, 0);
        return;
    }
    const int64_t row = (int64_t)(slot >> st.log_page) * st.heads + h;
    const int off = slot & ((1 << st.log_page) - 1), bit = nibble_bit(off & 7);
    const int64_t at = ((((row * D) >> log_group) + ((w * 8) >> log_group)) << st.log_page) + off;
    const uint32_t km = st.k_meta[at], vm = st.v_meta[at];
    const uint32_t kw = st.k_codes[((row << st.log_page) + off) * W + w];
    const uint32_t *const p = st.v_codes + (((row << st.log_page) + off) >> 3) * D + w * 8;
    const uint4 a = *reinterpret_cast<const uint4 *>(p), b = *reinterpret_cast<const uint4 *>(p + 4);
    const float ks = from_bits16<BF>(km & 0xffffu), kz = from_bits16<BF>(km >> 16);
    const float vs = from_bits16<BF>(vm & 0xffffu), vz = from_bits16<BF>(vm >> 16);
    // even pairs' codes as the bytes (0, 4, 1, 5) of one word, odd ones' (2, 6, 3, 7)
    const uint32_t even = kw & 0x0f0f0f0fu, odd = (kw >> 4) & 0x0f0f0f0fu;
    auto byte = [](uint32_t u, int i) { return (float)((u >> (8 * i)) & 0xffu); };
    auto key = [&](uint32_t u, int i) { return pack16<BF>(fmaf(byte(u, i), ks, kz), fmaf(byte(u, i + 2), ks, kz)); };
    *to_k = make_uint4(key(even, 0), key(odd, 0), key(even, 1), key(odd, 1));
    auto value = [&](uint32_t u) { return fmaf((float)((u >> bit) & 15u), vs, vz); };
    *to_v = make_uint4(pack16<BF>(value(a.x), value(a.y)), pack16<BF>(value(a.z), value(a.w)),
                       pack16<BF>(value(b.x), value(b.y)), pack16<BF>(value(b.z), value(b.w)));
}

// -------------------------------------------------------------------- host

int check_paged_store(const ss_paged_store *s, PagedStore *out, int *log_page) {
    SS_REQUIRE(s, "null store");
    SS_REQUIRE(s->k_codes && s->v_codes && s->k_meta && s->v_meta, "null store tensor");
    SS_REQUIRE((((uintptr_t)s->k_codes | (uintptr_t)s->v_codes | (uintptr_t)s->k_meta | (uintptr_t)s->v_meta) & 15) == 0,
               "store tensors must be 16-byte aligned");
    SS_REQUIRE(s->n_pages >= 1 && s->n_kv_heads >= 1, "bad pool shape");
    SS_UNSUPPORTED(s->dtype == SS_F16 || s->dtype == SS_BF16, "store dtype must be float16 or bfloat16");
    SS_UNSUPPORTED(s->head_dim == 64 || s->head_dim == 128, "head_dim %d (64 or 128)", s->head_dim);
    SS_UNSUPPORTED((s->group_size == 32 || s->group_size == 64 || s->group_size == 128) && s->group_size <= s->head_dim,
                   "group_size %d (32, 64 or 128, at most head_dim)", s->group_size);
    SS_UNSUPPORTED(s->page_size >= 16 && s->page_size <= 1024 && (s->page_size & (s->page_size - 1)) == 0,
                   "page_size %d (a power of two from 16 to 1024)", s->page_size);
    SS_UNSUPPORTED(s->n_pages <= INT32_MAX / s->page_size && s->n_pages <= INT32_MAX / s->n_kv_heads,
                   "the pool has more slots than 32 bits count");
    *log_page = __builtin_ctz((unsigned)s->page_size);
    *out = {static_cast<uint32_t *>(s->k_codes), static_cast<uint32_t *>(s->v_codes),
            static_cast<uint32_t *>(s->k_meta),  static_cast<uint32_t *>(s->v_meta),
            (int)s->n_pages,                     s->n_kv_heads,
            *log_page};
    return SS_OK;
}

}  // namespace ss

using namespace ss;

extern "C" int ss_block_tables(const int32_t *lengths, const int32_t *new_lengths, int64_t n_requests,
                               int32_t *block_table, int64_t table_width, int32_t *free_pages, int64_t pool,
                               const int32_t *n_free, int page_size, int64_t n_tokens, int32_t *lengths_out,
                               int32_t *n_free_out, int32_t *token_starts, int32_t *slots, int32_t *positions,
                               int32_t *status, void *stream) {
    SS_REQUIRE(n_requests >= 1 && table_width >= 1 && pool >= 1 && n_tokens >= 0, "bad sizes");
    SS_REQUIRE(lengths && new_lengths && block_table && free_pages && n_free && lengths_out && n_free_out &&
                   token_starts && status && (slots || n_tokens == 0),
               "null pointer argument");
    SS_UNSUPPORTED(n_requests <= kMaxRequests, "%lld requests (at most %d)", (long long)n_requests, kMaxRequests);
    SS_UNSUPPORTED(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
                   "page_size %d (a power of two from 16 to 1024)", page_size);
    SS_UNSUPPORTED(pool <= INT32_MAX / page_size && n_tokens <= INT32_MAX && table_width <= INT32_MAX / n_requests,
                   "more slots, tokens or table entries than 32 bits count");
    const int log_page = __builtin_ctz((unsigned)page_size);
    const int in_one = n_tokens <= kSlotsInline;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(block_tables_kernel, dim3(1), dim3(kTableThreads), 0, st, lengths, new_lengths,
                       (int)n_requests, block_table, table_width, free_pages, pool, n_free, log_page, n_tokens,
                       lengths_out, n_free_out, token_starts, slots, positions, status, in_one);
    SS_LAUNCH_CHECK("block_tables_kernel launch");
    if (!in_one) {
        hipLaunchKernelGGL(slots_kernel, dim3((unsigned)((n_tokens + 255) / 256)), dim3(256), 0, st, token_starts,
                           (int)n_requests, lengths_out, block_table, table_width, log_page, n_tokens, slots,
                           positions);
        SS_LAUNCH_CHECK("slots_kernel launch");
    }
    return SS_OK;
}

extern "C" int ss_shared_plan(const int32_t *parents, const int32_t *lengths, const int32_t *token_starts,
                              int64_t n_requests, int64_t n_tokens, int32_t *group_starts, int32_t *group_rows,
                              int32_t *parents_out, int32_t *offsets, int32_t *positions, void *stream) {
    SS_REQUIRE(n_requests >= 1 && n_tokens >= 0, "bad sizes");
    SS_REQUIRE(parents && lengths && token_starts && group_starts && parents_out && offsets &&
                   (group_rows || n_tokens == 0),
               "null pointer argument");
    SS_REQUIRE(((uintptr_t)group_rows & 7) == 0, "group_rows must be 8-byte aligned");
    SS_UNSUPPORTED(n_requests <= kMaxRequests, "%lld requests (at most %d)", (long long)n_requests, kMaxRequests);
    SS_UNSUPPORTED(n_tokens <= INT32_MAX, "too many tokens for one launch");
    const int in_one = n_tokens <= kSlotsInline;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    int2 *const rows = reinterpret_cast<int2 *>(group_rows);
    auto launch = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, dim3(1), dim3(threads), 0, st, parents, lengths, token_starts, (int)n_requests,
                           n_tokens, group_starts, rows, parents_out, offsets, positions, in_one);
    };
    if (n_requests <= 256 && n_tokens <= 1024) launch(shared_plan_kernel<256>, 256);
    else launch(shared_plan_kernel<kTableThreads>, kTableThreads);
    SS_LAUNCH_CHECK("shared_plan_kernel launch");
    if (!in_one) {
        hipLaunchKernelGGL(shared_rows_kernel, dim3((unsigned)((n_tokens + 255) / 256)), dim3(256), 0, st,
                           token_starts, (int)n_requests, n_tokens, lengths, parents_out, offsets, rows, positions);
        SS_LAUNCH_CHECK("shared_rows_kernel launch");
    }
    return SS_OK;
}

extern "C" int ss_append_paged(const ss_paged_store *store, const void *keys, const void *values, int in_dtype,
                               int64_t n_tokens, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh,
                               const int32_t *slots, void *stream) {
    PagedStore ps;
    int log_page;
    if (int rc = check_paged_store(store, &ps, &log_page)) return rc;
    SS_REQUIRE(valid_dtype(in_dtype), "bad key/value dtype");
    SS_REQUIRE(n_tokens >= 0, "bad sizes");
    if (n_tokens == 0) return SS_OK;
    SS_REQUIRE(keys && values && slots, "null pointer argument");
    SS_UNSUPPORTED(n_tokens <= INT32_MAX, "too many tokens for one launch");
    const int64_t items = (n_tokens + 7) / 8 * ps.heads;
    SS_UNSUPPORTED((items + 3) / 4 <= kMostGroups, "%lld tokens of %d heads: too many for one launch",
                   (long long)n_tokens, ps.heads);
    // 16-byte loads where every row starts on 16 bytes
    const int per = in_dtype == SS_F32 ? 4 : 8;
    const int vec = (((uintptr_t)keys | (uintptr_t)values) & 15) == 0 && k_st % per == 0 && k_sh % per == 0 &&
                    v_st % per == 0 && v_sh % per == 0;
    const dim3 grid((unsigned)((items + 3) / 4));
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, ps, keys, values, in_dtype, vec, k_st, k_sh, v_st, v_sh,
                           slots, n_tokens, (uint32_t)items);
    };
    const bool bf = store->dtype == SS_BF16;
    const int key = store->head_dim * 1000 + store->group_size;
    if (key == 128032) bf ? launch(append_paged_kernel<128, 32, true>) : launch(append_paged_kernel<128, 32, false>);
    else if (key == 128064) bf ? launch(append_paged_kernel<128, 64, true>) : launch(append_paged_kernel<128, 64, false>);
    else if (key == 128128) bf ? launch(append_paged_kernel<128, 128, true>) : launch(append_paged_kernel<128, 128, false>);
    else if (key == 64032) bf ? launch(append_paged_kernel<64, 32, true>) : launch(append_paged_kernel<64, 32, false>);
    else bf ? launch(append_paged_kernel<64, 64, true>) : launch(append_paged_kernel<64, 64, false>);
    SS_LAUNCH_CHECK("append_paged_kernel launch");
    return SS_OK;
}

extern "C" int ss_read_paged(const ss_paged_store *store, const int32_t *slots, int64_t n_tokens, void *keys,
                             void *values, void *stream) {
    PagedStore ps;
    int log_page;
    if (int rc = check_paged_store(store, &ps, &log_page)) return rc;
    SS_REQUIRE(n_tokens >= 0, "bad sizes");
    if (n_tokens == 0) return SS_OK;
    SS_REQUIRE(keys && values && slots, "null pointer argument");
    SS_REQUIRE((((uintptr_t)keys | (uintptr_t)values) & 15) == 0, "outputs must be 16-byte aligned");
    const int rows = 256 / (store->head_dim / 8);  // of a workgroup
    SS_UNSUPPORTED(n_tokens <= kMostGroups * rows / ps.heads, "%lld tokens of %d heads: too many for one launch",
                   (long long)n_tokens, ps.heads);
    const dim3 grid((unsigned)((n_tokens * ps.heads + rows - 1) / rows));
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, ps, slots, __builtin_ctz((unsigned)store->group_size),
                           (uint32_t)(n_tokens * ps.heads), static_cast<uint16_t *>(keys),
                           static_cast<uint16_t *>(values));
    };
    const bool bf = store->dtype == SS_BF16;
    if (store->head_dim == 128) bf ? launch(read_paged_kernel<128, true>) : launch(read_paged_kernel<128, false>);
    else bf ? launch(read_paged_kernel<64, true>) : launch(read_paged_kernel<64, false>);
    SS_LAUNCH_CHECK("read_paged_kernel launch");
    return SS_OK;
}
