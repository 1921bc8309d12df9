// arfq_plan.hip -- a step's rows, page tables and slots from the requests' lengths.
//
// Sums over the sequences first: of rows, then of pages given back and pages wanted (what a sequence wants depends on
// whether its rows fit).  With T the largest running sum of wanted pages that the free ones cover, a sequence gets its
// pages where its running sum is at most T, and its first one is its predecessors' sum: nothing depends on
// another sequence's outcome but through T.  Then each row looks up its sequence, and each new page falls to the
// row that is its first token, which writes the table's entry; the other rows of the page work the same id out
// for themselves.  Nothing that is read is written: counts have places of their own, entries of the stack are written
// above the free ones and entries of the tables behind the held ones.  Bound by latency, a chain of loads and
// barriers.
#include "arfq_step.h"

namespace arfq {
namespace {

constexpr int THREADS = 1024, WAVES = THREADS / WAVE;

__device__ __forceinline__ int64_t wave_scan(int64_t v) {  // running sum over the lanes
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) {
        const int64_t u = __shfl_up(v, d);
        if (lane >= d) v += u;
    }
    return v;
}

// Sum of the threads' values before this one's, and of all.  (All threads call it; sh is free again at the next
// barrier behind it.)
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t (&sh)[WAVES], int64_t &all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t inc = wave_scan(v);
    if (lane == 63) sh[wave] = inc;
    __syncthreads();
    int64_t before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        if (w < wave) before += sh[w];
        all += sh[w];
    }
    return before + inc - v;
}

struct Change {
    int64_t held, now;   // tokens: held, and to be held
    int have, need;      // pages of both
    bool ok, grows;      // held is a length; rows are asked for
};
__device__ __forceinline__ Change change_of(const arfq_kv_step &s, int b) {
    Change c;
    const int64_t add = s.add[b], most = s.max_pages * s.page_size;
    c.held = s.held[b];
    c.ok = c.held >= 0 && c.held <= most;
    c.now = max(c.held + add, (int64_t)0);
    c.grows = add > 0;
    const int64_t p = s.page_size;
    c.have = c.ok ? (int)((c.held + p - 1) / p) : 0;
    c.need = c.ok ? (int)(min((c.now + p - 1) / p, (int64_t)INT32_MAX)) : 0;
    return c;
}
__device__ __forceinline__ int back_of(const Change &c) { return c.ok && !c.grows ? c.have - c.need : 0; }

// The largest i in [0, n] with sums[i] <= v, of a running sum from 0 on (v >= 0).
__device__ __forceinline__ int place_in(const int32_t *sums, int n, int64_t v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sums[mid] <= v) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ int64_t free_of(const arfq_kv_step &s) { return min(max((int64_t)s.n_free[0], (int64_t)0), s.n_pages); }

// The `i`-th page given back.
__device__ __forceinline__ int32_t given_back(const arfq_kv_step &s, int64_t i) {
    const int b = place_in(s.freed, (int)s.batch, i);  // (< batch: i is below the sum of all)
    return s.pages[(int64_t)b * s.max_pages + change_of(s, b).need + (i - s.freed[b])];
}

// Rows and pages, `at` of `of` threads.
__device__ __forceinline__ void plan_rows(const arfq_kv_step &s, int64_t at, int64_t of) {
    const int n = (int)s.batch;
    const int64_t back = s.freed[n], taken = s.taken[n], free0 = free_of(s);
    for (int64_t t = at; t < s.tokens; t += of) {
        const int b = t < s.start[n] ? place_in(s.start, n, t) : n;
        int64_t pos = -1, slot = -1;
        if (b < n && s.len[b] > 0) {
            const Change c = change_of(s, b);
            pos = c.now - (s.start[b + 1] - t);
            const int pg = (int)(pos / s.page_size);
            const int64_t in = pos - (int64_t)pg * s.page_size;
            int32_t *entry = s.pages + (int64_t)b * s.max_pages + pg;
            int32_t id;
            if (pg < c.have) {
                id = *entry;
            } else {
                const int64_t i = s.taken[b] + (int64_t)(pg - c.have);
                id = i < back ? given_back(s, i) : s.free_pages[free0 - 1 - (i - back)];
                if (in == 0) *entry = id;  // (a new page begins with a row)
            }
            slot = (int64_t)id * s.page_size + in;
        }
        s.positions[t] = (int32_t)pos;
        s.slots[t] = slot;
    }
    for (int64_t i = taken + at; i < back; i += of) {
        const int64_t to = free0 + back - 1 - i;
        if (to < s.n_pages) s.free_pages[to] = given_back(s, i);
    }
}

// One workgroup.  ROWS: it does the rows too.
template <bool ROWS>
__global__ __launch_bounds__(THREADS) void plan_kernel(arfq_kv_step s) {
    __shared__ int64_t sums[3][WAVES], top[WAVES];
    const int n = (int)s.batch, per = (n + THREADS - 1) / THREADS;
    const int b0 = min((int)threadIdx.x * per, n), b1 = min(b0 + per, n);
    int64_t rows = 0, all_rows, all_back, all_want;
    for (int b = b0; b < b1; b++) rows += max(s.add[b], 0);
    const int64_t row0 = block_scan(rows, sums[0], all_rows);
    auto fits = [&](const Change &c, int64_t end) { return c.ok && c.grows && end <= s.tokens && c.need <= s.max_pages; };
    int64_t back = 0, want = 0, end = row0;
    for (int b = b0; b < b1; b++) {
        const Change c = change_of(s, b);
        if (c.grows) end += s.add[b];
        back += back_of(c);
        if (fits(c, end)) want += c.need - c.have;
    }
    const int64_t back0 = block_scan(back, sums[1], all_back), want0 = block_scan(want, sums[2], all_want);
    const int64_t there = free_of(s) + all_back;
    // the pages that are taken
    int64_t most = 0, sum = want0;
    end = row0;
    for (int b = b0; b < b1; b++) {
        const Change c = change_of(s, b);
        if (c.grows) end += s.add[b];
        if (fits(c, end)) sum += c.need - c.have;
        if (sum <= there) most = sum;
    }
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) most = max(most, (int64_t)__shfl_xor(most, d));
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) most = max(most, top[w]);
    // (sums past 2^31 - 1 are of pages that do not fit: what is written is min(sum, most), and most <= 2^31)
    int64_t given_sum = back0;
    sum = want0;
    end = row0;
    for (int b = b0; b < b1; b++) {
        const Change c = change_of(s, b);
        s.start[b] = (int32_t)min(end, s.tokens);
        s.freed[b] = (int32_t)given_sum;
        s.taken[b] = (int32_t)min(sum, most);
        if (c.grows) end += s.add[b];
        given_sum += back_of(c);
        bool got = c.ok && !c.grows;
        if (fits(c, end)) {
            const int more = c.need - c.have;
            sum += more;
            got = more == 0 || sum <= most;
        }
        s.held_next[b] = (int32_t)(got ? c.now : c.held);
        s.len[b] = got ? (int32_t)c.now : 0;
    }
    if (threadIdx.x == 0) {
        s.start[n] = (int32_t)min(all_rows, s.tokens);
        s.freed[n] = (int32_t)all_back;
        s.taken[n] = (int32_t)most;
        s.n_free_next[0] = (int32_t)min(there - most, s.n_pages);
    }
    if constexpr (ROWS) {
        __syncthreads();
        plan_rows(s, threadIdx.x, THREADS);
    }
}

__global__ __launch_bounds__(256) void plan_rows_kernel(arfq_kv_step s) {
    plan_rows(s, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

constexpr int64_t ONE_GROUP_ROWS = 4096;

}  // namespace

hipError_t launch_kv_plan(const arfq_kv_step &s, hipStream_t stream) {
    if (s.tokens <= ONE_GROUP_ROWS) {
        plan_kernel<true><<<1, THREADS, 0, stream>>>(s);
        return hipGetLastError();
    }
    plan_kernel<false><<<1, THREADS, 0, stream>>>(s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    plan_rows_kernel<<<dim3((unsigned)std::min<int64_t>((s.tokens + 255) / 256, 4096)), 256, 0, stream>>>(s);
    return hipGetLastError();
}

}  // namespace arfq
