// arfq_plan.hip -- a step's rows, page tables and slots from the requests' lengths.
//
// Sums over the sequences first: of rows, then of pages given back and pages wanted (what a sequence wants depends on
// whether its rows fit).  With T the largest running sum of wanted pages that the free ones cover, a sequence gets its
// pages where its running sum is at most T, and its first one is its predecessors' sum: nothing depends on
// another sequence's outcome but through T.  Then each row looks up its sequence, and each new page falls to the
// row that is its first token, which writes the table's entry; the other rows of the page work the same id out
// for themselves.  Nothing that is read is written: counts have places of their own, entries of the stack are written
// above the free ones and entries of the tables behind the held ones.  Bound by latency, a chain of loads and
// barriers: 64 chats' decode step 4.4 us (a launch alone is 3.4 on the host), 1000 requests with 60000 rows 7.1.
#include "arfq_step.h"

namespace arfq {
namespace {

// A sequence as the call finds and leaves it.
struct Change {
    uint32_t now;     // tokens to be held
    int have, need;   // pages held, and needed
    bool ok, grows;   // held is a length; rows are asked for
};
__device__ __forceinline__ Change change_of(const arfq_kv_step &s, int add, int held) {
    Change c;
    c.ok = held >= 0 && held <= (int)(s.max_pages * s.page_size);  // (at most 2^29)
    c.grows = add > 0;
    c.now = (uint32_t)max((int64_t)held + add, (int64_t)0);
    const uint32_t p = (uint32_t)s.page_size;
    c.have = c.ok ? (int)(((uint32_t)held + p - 1) / p) : 0;
    c.need = c.ok ? (int)min((c.now + p - 1) / p, (uint32_t)INT32_MAX) : 0;  // (the sum is below 2^29 + 2^31 + 2^16)
    return c;
}
__device__ __forceinline__ uint32_t rows_of(int add) { return (uint32_t)max(add, 0); }
__device__ __forceinline__ uint32_t back_of(const Change &c) { return c.ok && !c.grows ? (uint32_t)(c.have - c.need) : 0; }
__device__ __forceinline__ bool fits(const arfq_kv_step &s, const Change &c, uint32_t end) {
    return c.ok && c.grows && end <= (uint32_t)s.tokens && c.need <= s.max_pages;
}
__device__ __forceinline__ uint32_t free_of(const arfq_kv_step &s) { return (uint32_t)min(max((int64_t)s.n_free[0], (int64_t)0), s.n_pages); }

// Sums that stay at 2^32 - 1 when they get there (rows: more than any call has; pages: batch * max_pages is below 2^31).
__device__ __forceinline__ uint32_t plus(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {  // running sum over the lanes
    v = plus(v, dpp<0x111, 0xf>(v));  // row_shr:1, 2, 4, 8
    v = plus(v, dpp<0x112, 0xf>(v));
    v = plus(v, dpp<0x114, 0xf>(v));
    v = plus(v, dpp<0x118, 0xf>(v));
    v = plus(v, dpp<0x142, 0xa>(v));  // row_bcast:15 into rows 1 and 3
    return plus(v, dpp<0x143, 0xc>(v));  // row_bcast:31 into rows 2 and 3
}
// The same over W waves: this thread's value counted; all: the last one's.  (sh is free again behind the next barrier.)
template <int W>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t (&sh)[W], uint32_t &all) {
    uint32_t inc = wave_scan(v);
    const int wave = threadIdx.x >> 6;
    if constexpr (W == 1) {
        all = (uint32_t)__builtin_amdgcn_readlane((int)inc, 63);
        return inc;
    }
    if ((threadIdx.x & 63) == 63) sh[wave] = inc;
    __syncthreads();
    uint32_t before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        if (w == wave) before = all;
        all = plus(all, sh[w]);
    }
    return plus(inc, before);
}
template <int W>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t (&sh)[W]) {
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) v = max(v, (uint32_t)__shfl_xor((int)v, d));
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; w++) v = max(v, sh[w]);
    }
    return v;
}

// The largest i in [0, n] with sums[i] <= v, of a running sum from 0 on.
template <class P>
__device__ __forceinline__ int place_in(P sums, int n, uint32_t v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((uint32_t)sums[mid] <= v) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// What the rows go by, in LDS or (P: pointers) in memory.
template <class P, class F>
struct Sums {
    P start, taken, freed;  // [batch + 1]
    F change;               // (b) -> Change, `grows` whether it got its rows
    uint32_t free0;
};

// The `i`-th page given back.
template <class S>
__device__ __forceinline__ int32_t given_back(const arfq_kv_step &s, const S &m, uint32_t i) {
    const int b = place_in(m.freed, (int)s.batch, i);  // (< batch: i is below the sum of all)
    return s.pages[(int64_t)b * s.max_pages + m.change(b).need + (i - (uint32_t)m.freed[b])];
}

// Rows and pages, `at` of `of` threads.
template <class S>
__device__ __forceinline__ void plan_rows(const arfq_kv_step &s, const S &m, uint32_t at, uint32_t of) {
    const int n = (int)s.batch;
    const uint32_t back = (uint32_t)m.freed[n], page = (uint32_t)s.page_size;
    for (uint32_t t = at; t < (uint32_t)s.tokens; t += of) {
        const int b = t < (uint32_t)m.start[n] ? place_in(m.start, n, t) : n;
        int32_t pos = -1;
        int64_t slot = -1;
        if (b < n) {
            const Change c = m.change(b);
            if (c.grows) {
                pos = (int32_t)(c.now - ((uint32_t)m.start[b + 1] - t));
                const uint32_t pg = (uint32_t)pos / page, in = (uint32_t)pos - pg * page;
                int32_t *entry = s.pages + (int64_t)b * s.max_pages + pg;
                int32_t id;
                if ((int)pg < c.have) {
                    id = *entry;
                } else {
                    const uint32_t i = (uint32_t)m.taken[b] + (pg - (uint32_t)c.have);
                    id = i < back ? given_back(s, m, i) : s.free_pages[m.free0 - 1 - (i - back)];
                    if (in == 0) *entry = id;  // (a new page begins with a row)
                }
                slot = (int64_t)id * page + in;
            }
        }
        s.positions[t] = pos;
        s.slots[t] = slot;
    }
    for (uint32_t i = (uint32_t)m.taken[n] + at; i < back; i += of) {
        const uint32_t to = m.free0 + back - 1 - i;
        if (to < (uint32_t)s.n_pages) s.free_pages[to] = given_back(s, m, i);
    }
}

// At most a sequence a thread: every workgroup forms the sums for itself, in LDS, and has its share of the rows; the first
// writes what there is of sequences.
template <int W>
__global__ __launch_bounds__(64 * W) void plan_few(arfq_kv_step s) {
    constexpr int T = 64 * W;
    __shared__ uint32_t start[T + 1], taken[T + 1], freed[T + 1], now[T], sums[4][W];
    __shared__ int have[T], need[T];
    const int n = (int)s.batch, b = threadIdx.x;
    const bool mine = b < n;
    const int add = mine ? s.add[b] : 0, held = mine ? s.held[b] : 0;
    const uint32_t free0 = free_of(s);
    const Change c = change_of(s, add, held);
    uint32_t all_rows, all_back, all_want;
    const uint32_t end = block_scan(rows_of(add), sums[0], all_rows);
    const bool fit = mine && fits(s, c, end);
    const uint32_t back = back_of(c), want = fit ? (uint32_t)(c.need - c.have) : 0;
    const uint32_t freed_to = block_scan(back, sums[1], all_back), upto = block_scan(want, sums[2], all_want);
    const uint32_t there = free0 + all_back;
    const uint32_t most = block_max(upto <= there ? upto : 0, sums[3]);  // the pages that are taken
    const bool got = fit ? want == 0 || upto <= most : c.ok && !c.grows;
    const uint32_t taken_from = min(upto - want, most);
    if (mine) {
        start[b + 1] = min(end, (uint32_t)s.tokens);
        freed[b + 1] = freed_to;
        taken[b] = taken_from;
        now[b] = c.now;
        have[b] = c.have;
        need[b] = fit && got ? c.need : c.grows ? -1 : c.need;
    }
    if (b == 0) {
        start[0] = freed[0] = 0;
        taken[n] = most;
    }
    if (blockIdx.x == 0) {
        if (mine) {
            s.start[b + 1] = (int32_t)min(end, (uint32_t)s.tokens);
            s.freed[b + 1] = (int32_t)freed_to;
            s.taken[b] = (int32_t)taken_from;
            s.held_next[b] = got ? (int32_t)c.now : held;
            s.len[b] = got ? (int32_t)c.now : 0;
        }
        if (b == 0) {
            s.start[0] = s.freed[0] = 0;
            s.taken[n] = (int32_t)most;
            s.n_free_next[0] = (int32_t)min((int64_t)(there - most), s.n_pages);
        }
    }
    __syncthreads();
    auto change = [&](int i) {  // (of a sequence with rows, need is -1 where it was refused)
        Change r;
        r.now = now[i];
        r.have = have[i];
        r.need = need[i];
        r.grows = need[i] >= 0;
        r.ok = true;
        return r;
    };
    const Sums<const uint32_t *, decltype(change)> m = {start, taken, freed, change, free0};
    plan_rows(s, m, blockIdx.x * T + threadIdx.x, gridDim.x * T);
}

// More sequences: one workgroup forms the sums, a run of neighbouring sequences a thread, and writes them; the rows are a
// launch of their own.
constexpr int MANY = 16;
__global__ __launch_bounds__(64 * MANY) void plan_many(arfq_kv_step s) {
    __shared__ uint32_t sums[4][MANY];
    const int n = (int)s.batch, per = (n + 64 * MANY - 1) / (64 * MANY);
    const int b0 = min((int)threadIdx.x * per, n), b1 = min(b0 + per, n);
    __shared__ uint32_t ends[64 * MANY];
    uint32_t rows = 0, back = 0, want = 0, all_rows, all_back, all_want;
    for (int b = b0; b < b1; b++) rows = plus(rows, rows_of(s.add[b]));
    // (the sum before a thread's run is its neighbour's: its own less its rows may have stayed at the largest)
    ends[threadIdx.x] = block_scan(rows, sums[0], all_rows);
    __syncthreads();
    const uint32_t row0 = threadIdx.x ? ends[threadIdx.x - 1] : 0;
    uint32_t end = row0;
    for (int b = b0; b < b1; b++) {
        const int add = s.add[b];
        const Change c = change_of(s, add, s.held[b]);
        end = plus(end, rows_of(add));
        back += back_of(c);
        if (fits(s, c, end)) want += (uint32_t)(c.need - c.have);
    }
    const uint32_t back0 = block_scan(back, sums[1], all_back) - back, want0 = block_scan(want, sums[2], all_want) - want;
    const uint32_t free0 = free_of(s), there = free0 + all_back;
    uint32_t most = 0, sum = want0;
    end = row0;
    for (int b = b0; b < b1; b++) {
        const int add = s.add[b];
        const Change c = change_of(s, add, s.held[b]);
        end = plus(end, rows_of(add));
        if (fits(s, c, end)) sum += (uint32_t)(c.need - c.have);
        if (sum <= there) most = sum;
    }
    most = block_max(most, sums[3]);  // the pages that are taken
    uint32_t freed = back0;
    sum = want0;
    end = row0;
    for (int b = b0; b < b1; b++) {
        const int add = s.add[b], held = s.held[b];
        const Change c = change_of(s, add, held);
        s.start[b] = (int32_t)min(end, (uint32_t)s.tokens);
        s.freed[b] = (int32_t)freed;
        s.taken[b] = (int32_t)min(sum, most);
        end = plus(end, rows_of(add));
        freed += back_of(c);
        bool got = c.ok && !c.grows;
        if (fits(s, c, end)) {
            const uint32_t more = (uint32_t)(c.need - c.have);
            sum += more;
            got = more == 0 || sum <= most;
        }
        s.held_next[b] = got ? (int32_t)c.now : held;
        s.len[b] = got ? (int32_t)c.now : 0;
    }
    if (threadIdx.x == 0) {
        s.start[n] = (int32_t)min(all_rows, (uint32_t)s.tokens);
        s.freed[n] = (int32_t)all_back;
        s.taken[n] = (int32_t)most;
        s.n_free_next[0] = (int32_t)min((int64_t)(there - most), s.n_pages);
    }
}
__global__ __launch_bounds__(256) void plan_many_rows(arfq_kv_step s) {
    auto change = [&](int b) {
        Change c = change_of(s, s.add[b], s.held[b]);
        c.grows = c.grows && s.len[b] > 0;
        return c;
    };
    const Sums<const int32_t *, decltype(change)> m = {s.start, s.taken, s.freed, change, free_of(s)};
    plan_rows(s, m, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

template <int W>
hipError_t few_launch(const arfq_kv_step &s, hipStream_t stream) {
    // (a thread for each row, and 1024 at least: pages given back are shared by them too; 64 chats of 8192, four of which
    // end, 4.3 us with 16 workgroups and 6.5 with one)
    const int64_t groups = std::min<int64_t>(std::max<int64_t>((s.tokens + 64 * W - 1) / (64 * W), 16 / W), 4096 / W);
    plan_few<W><<<dim3((unsigned)groups), 64 * W, 0, stream>>>(s);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_plan(const arfq_kv_step &s, hipStream_t stream) {
    if (s.batch <= 64) return few_launch<1>(s, stream);
    if (s.batch <= 256) return few_launch<4>(s, stream);
    if (s.batch <= 1024) return few_launch<16>(s, stream);
    plan_many<<<1, 64 * MANY, 0, stream>>>(s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t groups = std::min<int64_t>(std::max<int64_t>((s.tokens + 255) / 256, 64), 4096);
    plan_many_rows<<<dim3((unsigned)groups), 256, 0, stream>>>(s);
    return hipGetLastError();
}

}  // namespace arfq
