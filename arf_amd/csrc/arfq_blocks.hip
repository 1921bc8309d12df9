// arfq_blocks.hip -- attention over the blocks (pages) of the 4-bit cache that each query chooses.
//
// Bounds: of each channel of a page's keys the largest and smallest (arfq_kv_bounds), f16 and exact, as keys are.
// A call: the scores' keys of all blocks (blocks_score), the best of them for each row and K/V head and their pages
// (blocks_select), attention with those pages as the row's table (the tile of arfq_attn_rows16.h, a row a sequence
// of its own), and the joining of rows whose keys were cut into pieces.
#include <math.h>

#include "arfq_attn_join.h"
#include "arfq_attn_rows16.h"
#include "arfq_step.h"

namespace arfq {
namespace {

// ---- rows ------------------------------------------------------------------------------------

// The sequence of row t (the same in all lanes), a.batch behind the last; none of it has rows from where start
// decreases on.
__device__ __forceinline__ int seq_of_row(const KvArgs &a, int t) {
    if (!a.start) return min(t, a.batch);
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < a.batch; b0 += WAVE) {
        const bool mine = b0 + lane < a.batch;
        const int u = mine ? a.start[b0 + lane] : 0;
        int v = mine ? a.start[b0 + lane + 1] : INT32_MAX;
        const uint64_t falls = __ballot(v < u);
        if (falls && (falls & (((uint64_t)2 << lane) - 1))) v = INT32_MAX;  // (at this lane or one before)
        const int n = __popcll(__ballot(v <= t));
        if (n < WAVE) return b0 + n;
    }
    return a.batch;
}

// A row's place: its sequence (-1: of none), the blocks up to its own, the tokens up to its own (0: it attends to
// nothing).
struct Row {
    int b, seen, end;
};
__device__ __forceinline__ Row row_of(const KvArgs &a, int t) {
    Row r = {-1, 0, 0};
    const int b = seq_of_row(a, t);
    if (b >= a.batch) return r;
    int t0, n;
    kv_seq(a, b, t0, n);
    if (t < t0 || t >= t0 + n) return r;
    r.b = b;
    const int64_t pos = (int64_t)a.len[b] - ((int64_t)t0 + n - t);
    r.end = pos < 0 ? 0 : (int)min(pos + 1, (int64_t)a.max_pages * a.page);
    r.seen = (r.end + a.page - 1) / a.page;
    return r;
}

// ---- bounds ----------------------------------------------------------------------------------

// One page of a head: a lane has a dword column of K's codes (eight values of a key), 64 / (4 NG) keys side by side.
template <int NG>
__device__ __forceinline__ void page_bounds(const KvArgs &a, int id, int head, int keys, _Float16 *bounds) {
    constexpr int D = 32 * NG, COLS = 4 * NG, KL = WAVE / COLS;
    const int lane = threadIdx.x & 63, kk = lane / COLS, col = lane - kk * COLS, g = col % NG, h = col / NG;
    const uint8_t *reg = a.data + ((int64_t)id * a.heads + head) * a.region;
    const uint32_t *codes = (const uint32_t *)reg + col;
    const uint16_t *scales = (const uint16_t *)(reg + a.off_ks) + g;
    float hi[8], lo[8];
    bool nan = false;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        hi[e] = -INFINITY;
        lo[e] = INFINITY;
    }
    if (kk < KL) {
#pragma unroll 4
        for (int key = kk; key < keys; key += KL) {
            const uint32_t w = codes[key * COLS];
            const float d = h2f(scales[key * NG]);
            nan |= d != d;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = d * (float)((int)(w >> (4 * ((e >> 1) + 4 * (e & 1))) & 15u) - 8);
                hi[e] = fmaxf(hi[e], v);
                lo[e] = fminf(lo[e], v);
            }
        }
    }
    // over the keys side by side: a tree over any number of them
    int bad = nan;
    for (int s = KL; s > 1;) {
        const int half = (s + 1) / 2;
        const bool in = kk + half < s;
        const int from = in ? lane + half * COLS : lane;
        bad |= __shfl(bad, from);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            hi[e] = fmaxf(hi[e], __shfl(hi[e], from));
            lo[e] = fminf(lo[e], __shfl(lo[e], from));
        }
        s = half;
    }
    if (kk != 0) return;
    _Float16 *o = bounds + ((int64_t)id * a.heads + head) * (2 * D) + 32 * g + 8 * h;
    f16x8 vh, vl;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        vh[e] = (_Float16)(bad ? NAN : hi[e]);
        vl[e] = (_Float16)(bad ? NAN : lo[e]);
    }
    *(f16x8 *)o = vh;
    *(f16x8 *)(o + D) = vl;
}

// A wave: `per` rows of a head, and of those the pages that begin with one of them, or in which a sequence's first one
// lies.
template <int NG>
__global__ __launch_bounds__(256) void kv_bounds_kernel(KvArgs a, _Float16 *bounds, int per, int items) {
    const int item = __builtin_amdgcn_readfirstlane(block_of() * 4 + (int)(threadIdx.x >> 6));
    if (item >= items) return;
    const int head = item % a.heads, row0 = item / a.heads * per, row1 = min(row0 + per, a.tokens);
    for (int b = seq_of_row(a, row0); b < a.batch; b++) {
        int t0, n;
        kv_seq(a, b, t0, n);
        if (a.start ? a.start[b] >= row1 || a.start[b + 1] < a.start[b] : b >= row1) break;
        const int r0 = max(row0, t0), r1 = min(row1, t0 + n);
        if (r0 >= r1) continue;
        const int64_t len = a.len[b], pos0 = max(len - ((int64_t)t0 + n - r0), (int64_t)0), pos1 = len - ((int64_t)t0 + n - r1) - 1;
        const int64_t p0 = r0 == t0 ? pos0 / a.page : (pos0 + a.page - 1) / a.page;
        const int64_t p1 = pos1 < 0 ? -1 : min(pos1 / a.page, (int64_t)a.max_pages - 1);
        for (int64_t p = p0; p <= p1; p++) {
            const int id = a.table[(int64_t)b * a.max_pages + p];
            if ((uint32_t)id < (uint32_t)a.n_pages) page_bounds<NG>(a, id, head, (int)min((int64_t)a.page, len - p * a.page), bounds);
        }
    }
}

template <int NG>
hipError_t bounds_launch(const KvArgs &a, _Float16 *bounds, int cus, hipStream_t s) {
    // rows of a wave: one while that does not fill the chip several times over
    const int64_t rows = (int64_t)a.tokens * a.heads;
    const int per = (int)std::min<int64_t>(std::max<int64_t>(rows / (64 * (int64_t)cus), 1), 64);
    const int64_t items = ((int64_t)a.tokens + per - 1) / per * a.heads;
    kv_bounds_kernel<NG><<<grid_of((items + 3) / 4), 256, 0, s>>>(a, bounds, per, (int)items);
    return hipGetLastError();
}

// ---- scores ----------------------------------------------------------------------------------

typedef double f64x4 __attribute__((ext_vector_type(4)));

// Scores as whole numbers in their order.  Those of chosen blocks by rule are never formed; NaN comes first, pages
// that are not the cache's last.
constexpr uint64_t KEY_NAN = ~0ull, KEY_NONE = 0;
__device__ __forceinline__ uint64_t key_of(double v) {
    if (v != v) return KEY_NAN;
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);  // (-0 as 0)
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__shfl((int)(v >> 32), lane) << 32 | (uint32_t)__shfl((int)v, lane);
}

struct ScoreArgs {
    KvArgs c;
    const _Float16 *bounds;
    const void *q;
    int64_t q_stride;
    bool q_f16, negative;
    int group, count;
    int row0, rows;       // of the chunk
    int per_tile;         // rows of a tile
    int blocks;           // of a wave
    uint64_t *keys;       // [rows][heads][max_pages]
};

// 16 blocks by 16 columns with v_mfma_f64_16x16x4_f64: a column is a (row, q head of the K/V head), and the sum runs
// over [max(q, 0), min(q, 0)] times [hi, lo].  The products of an f32 and an f16 are exact in 64 bits, so that nothing but the
// order of the sum's last bits is left to chance: blocks' order is that of their scores.  A lane of the operands has
// the channels D / 4 * (lane / 16) .. of its block or column.
template <int NG>
__global__ __launch_bounds__(256) void blocks_score(ScoreArgs a) {
    constexpr int D = 32 * NG, DL = D / 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, kg = lane >> 4;
    const KvArgs &kv = a.c;
    const int parts = (kv.max_pages + 4 * a.blocks - 1) / (4 * a.blocks);
    int block = block_of();
    const int head = block % kv.heads;
    block /= kv.heads;
    const int j0 = (block % parts * 4 + wave) * a.blocks, row0 = block / parts * a.per_tile;
    if (row0 >= a.rows) return;
    // this lane's column
    const int rt = c / a.group;  // (0 where the group has more than 16 heads)
    Row mine = {-1, 0, 0};
    int most = 0;  // blocks of the tile's rows
    for (int r = 0; r < a.per_tile && row0 + r < a.rows; r++) {
        const Row x = row_of(kv, a.row0 + row0 + r);
        if (rt == r) mine = x;
        if (x.seen > a.count) most = max(most, x.seen);
    }
    if (j0 >= most) return;
    if (mine.seen <= a.count) mine.b = -1;  // (its blocks are all chosen)
    const int64_t t = (int64_t)a.row0 + row0 + rt;
    uint64_t done = __ballot(mine.b < 0);
    while (done != ~0ull) {
        const int b = __builtin_amdgcn_readlane(mine.b, __ffsll((unsigned long long)~done) - 1);
        const uint64_t same = __ballot(mine.b == b);
        done |= same;
        int last = mine.b == b ? mine.seen : 0;
#pragma unroll
        for (int d = 1; d < 16; d *= 2) last = max(last, __shfl_xor(last, d));
        last = min(__builtin_amdgcn_readfirstlane(last), j0 + a.blocks);
        const int32_t *table = kv.table + (int64_t)b * kv.max_pages;
        // (one pass over the columns, unless the group has more than 16 heads: then the blocks' loop is inside)
        for (int g0 = 0; g0 < a.group; g0 += 16) {
            const int gh = g0 + (a.group > 16 ? c : c - rt * a.group);
            const bool on = mine.b == b && gh < a.group;
            float q[DL];
#pragma unroll
            for (int i = 0; i < DL; i++) q[i] = 0.0f;
            if (on) {
                const int64_t at = t * a.q_stride + (int64_t)(head * a.group + gh) * D + DL * kg;
#pragma unroll
                for (int i = 0; i < DL; i += 8) {
                    if (a.q_f16) {
                        const f16x8 v = *(const f16x8 *)((const _Float16 *)a.q + at + i);
#pragma unroll
                        for (int e = 0; e < 8; e++) q[i + e] = (float)v[e];
                    } else {
                        const f32x4 v = *(const f32x4 *)((const float *)a.q + at + i), w = *(const f32x4 *)((const float *)a.q + at + i + 4);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            q[i + e] = v[e];
                            q[i + 4 + e] = w[e];
                        }
                    }
                }
                if (a.negative)
#pragma unroll
                    for (int i = 0; i < DL; i++) q[i] = -q[i];
            }
            for (int j = j0; j < last; j += 16) {
                const int id = j + c < last ? table[j + c] : -1;
                const bool page = (uint32_t)id < (uint32_t)kv.n_pages;
                const _Float16 *p = a.bounds + ((int64_t)(page ? id : 0) * kv.heads + head) * (2 * D) + DL * kg;
                f64x4 up = {0, 0, 0, 0}, down = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < DL; i += 8) {
                    f16x8 hi = {0, 0, 0, 0, 0, 0, 0, 0}, lo = hi;
                    if (page) {
                        hi = *(const f16x8 *)(p + i);
                        lo = *(const f16x8 *)(p + D + i);
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float v = q[i + e];  // (NaN goes into the first)
                        up = __builtin_amdgcn_mfma_f64_16x16x4f64((double)(float)hi[e], (double)(v < 0.0f ? 0.0f : v), up, 0, 0, 0);
                        down = __builtin_amdgcn_mfma_f64_16x16x4f64((double)(float)lo[e], (double)(v < 0.0f ? v : 0.0f), down, 0, 0, 0);
                    }
                }
                // a lane's four results: blocks kg, kg + 4, .. of the 16, its column
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int jj = j + kg + 4 * i;
                    const bool there = __shfl(page, kg + 4 * i) != 0;  // (lane n has block n's page)
                    uint64_t key = on && there ? key_of(up[i] + down[i]) : KEY_NONE;
                    // the largest of the row's heads, at the first of them
                    const int heads = a.group > 16 ? 16 : a.group, h = a.group > 16 ? c : c - rt * a.group;
                    for (int d = 1; d < heads; d *= 2) {
                        const uint64_t other = shfl64(key, (lane & 48) | ((c + d) & 15));
                        if (h + d < heads) key = max(key, other);
                    }
                    if (h == 0 && mine.b == b && jj < min(mine.seen, last)) {
                        uint64_t *o = a.keys + ((int64_t)(row0 + rt) * kv.heads + head) * kv.max_pages + jj;
                        *o = g0 == 0 ? key : max(key, *o);
                    }
                }
            }
        }
    }
}

// ---- choice ----------------------------------------------------------------------------------

struct SelectArgs {
    KvArgs c;
    int row0, rows, count, first, last, width;
    const uint64_t *keys;
    int32_t *table;   // [rows][heads][width]: pages
    int32_t *chosen;  // of the whole call, or null
};

constexpr int SEL = 256, SEL_WAVES = SEL / WAVE;

template <class T, class F>
__device__ __forceinline__ T wave_all(T v, F f) {
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) v = f(v, (T)__shfl_xor(v, d));
    return v;
}

// A workgroup: a row and K/V head.  A thread has a run of neighbouring blocks.  The keys' range [lo, hi] that the
// last chosen one lies in is cut into 256 parts and counted, until a part's keys are all chosen or all alike.
__global__ __launch_bounds__(SEL) void blocks_select(SelectArgs a) {
    __shared__ uint32_t bins[256];
    __shared__ unsigned long long wlo[SEL_WAVES], whi[SEL_WAVES];
    __shared__ uint32_t found[3], sums[2][SEL_WAVES];
    const KvArgs &kv = a.c;
    const int block = block_of(), head = block % kv.heads, row = block / kv.heads, tid = threadIdx.x;
    if (row >= a.rows) return;
    const Row r = row_of(kv, a.row0 + row);
    if (r.b < 0) return;
    const int32_t *pages = kv.table + (int64_t)r.b * kv.max_pages;
    const int64_t at = (int64_t)row * kv.heads + head;
    int32_t *table = a.table + at * a.width;
    int32_t *chosen = a.chosen ? a.chosen + (((int64_t)a.row0 + row) * kv.heads + head) * a.count : nullptr;
    const int n = r.seen, most = min(n, a.count);
    auto take = [&](int rank, int j) {
        table[rank] = pages[j];
        if (chosen) chosen[rank] = j;
    };
    if (chosen)
        for (int i = most + tid; i < a.count; i += SEL) chosen[i] = -1;
    if (n <= a.count) {
        for (int j = tid; j < n; j += SEL) take(j, j);
        return;
    }
    const uint64_t *keys = a.keys + at * kv.max_pages;
    const int per = (n + SEL - 1) / SEL, j0 = min(tid * per, n), j1 = min(j0 + per, n);
    const int f0 = a.first, f1 = n - a.last;  // blocks [f0, f1) go by their scores
    constexpr int KEPT = 8;  // keys in registers
    uint64_t kept[KEPT];
#pragma unroll
    for (int i = 0; i < KEPT; i++) kept[i] = j0 + i < j1 ? keys[j0 + i] : 0;
    auto each = [&](auto f) {  // f(block, key)
#pragma unroll
        for (int i = 0; i < KEPT; i++)
            if (j0 + i < j1) f(j0 + i, kept[i]);
        for (int j = j0 + KEPT; j < j1; j++) f(j, keys[j]);
    };
    unsigned long long lo = ~0ull, hi = 0;
    each([&](int j, uint64_t key) {
        if (j < f0 || j >= f1) return;
        lo = min(lo, (unsigned long long)key);
        hi = max(hi, (unsigned long long)key);
    });
    lo = wave_all(lo, [](unsigned long long x, unsigned long long y) { return min(x, y); });
    hi = wave_all(hi, [](unsigned long long x, unsigned long long y) { return max(x, y); });
    if ((tid & 63) == 0) {
        wlo[tid >> 6] = lo;
        whi[tid >> 6] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SEL_WAVES; w++) {
        lo = min(lo, wlo[w]);
        hi = max(hi, whi[w]);
    }
    // the `need` largest of the keys in [lo, hi]; those above hi are chosen
    uint32_t need = (uint32_t)(a.count - a.first - a.last);
    bool all = need == 0;
    while (need > 0 && lo < hi) {
        const int bits = 64 - __clzll((long long)(hi - lo)), shift = max(bits - 8, 0);
        bins[tid] = 0;
        __syncthreads();
        each([&](int j, uint64_t key) {
            if (j >= f0 && j < f1 && key >= lo && key <= hi) atomicAdd(&bins[(key - lo) >> shift], 1u);
        });
        __syncthreads();
        // the part that the last chosen key lies in: 256 counts summed from the top
        const uint32_t mine = bins[255 - tid];
        uint32_t inc = mine;
#pragma unroll
        for (int d = 1; d < WAVE; d *= 2) {
            const uint32_t u = __shfl_up(inc, d);
            if ((tid & 63) >= d) inc += u;
        }
        if ((tid & 63) == 63) sums[0][tid >> 6] = inc;
        __syncthreads();
        for (int w = 0; w < (tid >> 6); w++) inc += sums[0][w];
        if (inc >= need && inc - mine < need) {
            found[0] = 255 - tid;
            found[1] = need - (inc - mine);
            found[2] = mine;
        }
        __syncthreads();
        const unsigned long long part = found[0];
        need = found[1];
        all = found[2] == need;
        lo += part << shift;
        const unsigned long long wide = (1ull << shift) - 1;
        if (hi - lo > wide) hi = lo + wide;
        if (all) break;
    }
    // chosen: by rule, keys above hi, with `all` those from lo on, otherwise the `need` first of those that are lo
    uint32_t sure = 0, ties = 0;
    auto is_sure = [&](int j, uint64_t key) { return j < f0 || j >= f1 || key > hi || (all && need > 0 && key >= lo); };
    auto is_tie = [&](int j, uint64_t key) { return !all && j >= f0 && j < f1 && key == lo; };
    each([&](int j, uint64_t key) {
        sure += is_sure(j, key);
        ties += is_tie(j, key);
    });
    uint32_t sure_inc = sure, ties_inc = ties;
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) {
        const uint32_t u = __shfl_up(sure_inc, d), v = __shfl_up(ties_inc, d);
        if ((tid & 63) >= d) {
            sure_inc += u;
            ties_inc += v;
        }
    }
    __syncthreads();
    if ((tid & 63) == 63) {
        sums[0][tid >> 6] = sure_inc;
        sums[1][tid >> 6] = ties_inc;
    }
    __syncthreads();
    for (int w = 0; w < (tid >> 6); w++) {
        sure_inc += sums[0][w];
        ties_inc += sums[1][w];
    }
    uint32_t before = sure_inc - sure, tie = ties_inc - ties;
    each([&](int j, uint64_t key) {
        const bool s = is_sure(j, key), e = is_tie(j, key);
        const uint32_t rank = before + min(tie, need);
        if ((s || (e && tie < need)) && rank < (uint32_t)most) take((int)rank, j);
        before += s;
        tie += e;
    });
}

// ---- attention -------------------------------------------------------------------------------

// A row as a sequence of its own, whose pages are the chosen ones: all but its own are whole.
struct RowsArgs {
    AttnArgs a;   // c.table and c.max_pages: the chosen pages
    int most;     // of the call's tables: max_pages
    int count, row0, rows, tiles, pieces;
};
__device__ __forceinline__ int chosen_keys(const RowsArgs &r, int t) {
    KvArgs c = r.a.c;
    c.max_pages = r.most;
    const Row x = row_of(c, t);
    if (x.b < 0) return -1;
    return x.end - max(x.seen - r.count, 0) * c.page;
}
__device__ __forceinline__ int pieces_of(const RowsArgs &r, int keys) { return max(1, min(r.pieces, (keys + MIN_PIECE - 1) / MIN_PIECE)); }

template <int NG, int PARTS>
__global__ __launch_bounds__(256, rows16_waves(NG)) void blocks_attend(RowsArgs r) {
    extern __shared__ float lds[];
    int block = block_of();
    const int head = block % r.a.c.heads;
    block /= r.a.c.heads;
    const int piece = block % r.pieces, tile = block / r.pieces % r.tiles, row = block / r.pieces / r.tiles;
    if (row >= r.rows) return;
    const int keys = chosen_keys(r, r.row0 + row);
    Item it;
    it.pieces = pieces_of(r, keys);
    if (keys < 0 || piece >= it.pieces) return;
    it.s = {r.row0 + row, 1, keys, 0, keys, r.tiles};
    it.b = row * r.a.c.heads + head;
    it.tile = tile;
    it.piece = piece;
    it.keys = ((keys + STEP - 1) / STEP + it.pieces - 1) / it.pieces * STEP;
    it.cut = 0;
    it.part = (row * r.tiles + tile) * r.pieces + piece;
    rows16_k::rows16_item<NG, PARTS>(r.a, it, head, lds);
}

template <int NG>
__global__ __launch_bounds__(256) void blocks_join(RowsArgs r) {
    __shared__ JoinLds<NG> sh;
    const int block = block_of(), head = block % r.a.c.heads, slot = block / r.a.c.heads;
    const int piece = slot % r.pieces, tile = slot / r.pieces % r.tiles, row = slot / r.pieces / r.tiles;
    if (row >= r.rows) return;
    const int keys = chosen_keys(r, r.row0 + row), pieces = pieces_of(r, keys);
    if (keys < 0 || pieces == 1 || piece >= pieces) return;
    join_tile<NG, 16>(r.a, r.a.few, make_int4(pieces | piece << 16, tile * 16, r.a.group, r.row0 + row), slot, head, sh);
}

template <int NG, int PARTS>
hipError_t attend_launch(const RowsArgs &r, hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t lds = rows16_k::lds_bytes(NG);
    const hipError_t e = set_max_lds_once((const void *)blocks_attend<NG, PARTS>, lds, done);
    if (e != hipSuccess) return e;
    blocks_attend<NG, PARTS><<<grid_of((int64_t)r.rows * r.tiles * r.pieces * r.a.c.heads), 256, lds, s>>>(r);
    return hipGetLastError();
}

// Blocks that a wave scores: all of a short sequence's; of long ones so many that the chip is filled.
int score_blocks(int cus, int64_t tiles, int max_pages) {
    const int64_t want = 16 * (int64_t)cus / std::max<int64_t>(tiles, 1);  // waves of a tile
    int64_t n = (max_pages + std::max<int64_t>(want, 4) - 1) / std::max<int64_t>(want, 4);
    return (int)((n + 15) / 16 * 16);
}

template <int NG>
hipError_t dim_launch(const BlocksArgs &b, const BlocksPlan &p, int cus, hipStream_t s) {
    const KvArgs &c = b.a.c;
    uint64_t *keys = (uint64_t *)b.ws;
    int32_t *table = (int32_t *)(b.ws + p.off_table);
    const bool f16 = b.a.q_dtype == ARFQ_F16 && b.a.out_dtype == ARFQ_F16;
    for (int row0 = 0; row0 < c.tokens; row0 += p.rows) {
        const int rows = std::min(p.rows, c.tokens - row0);
        hipError_t e;
        if (c.max_pages > b.count) {
            ScoreArgs sc = {c, b.bounds, b.a.q, b.a.q_stride, b.a.q_dtype == ARFQ_F16, b.a.scale < 0.0f, b.a.group, b.count, row0, rows,
                            std::max(1, 16 / b.a.group), 0, keys};
            if (!c.start) sc.per_tile = 1;  // (no two rows have blocks in common)
            const int64_t tiles = (int64_t)((rows + sc.per_tile - 1) / sc.per_tile) * c.heads;
            sc.blocks = score_blocks(cus, tiles, c.max_pages);
            const int64_t parts = (c.max_pages + 4 * (int64_t)sc.blocks - 1) / (4 * (int64_t)sc.blocks);
            blocks_score<NG><<<grid_of(tiles * parts), 256, 0, s>>>(sc);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
        const SelectArgs sel = {c, row0, rows, b.count, b.first, b.last, p.width, keys, table, b.chosen};
        blocks_select<<<grid_of((int64_t)rows * c.heads), SEL, 0, s>>>(sel);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        RowsArgs r = {b.a, c.max_pages, b.count, row0, rows, p.tiles, p.pieces};
        r.a.c.table = table;
        r.a.c.max_pages = p.width;
        r.a.causal = 1;
        r.a.window = 0;
        r.a.few = {1, 0, rows * p.tiles * p.pieces, 1, (float *)(b.ws + p.off_part), nullptr};
        e = f16 ? attend_launch<NG, 1>(r, s) : attend_launch<NG, 2>(r, s);
        if (e != hipSuccess) return e;
        if (p.pieces > 1) {
            blocks_join<NG><<<grid_of((int64_t)rows * p.tiles * p.pieces * c.heads), 256, 0, s>>>(r);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_kv_bounds(const KvArgs &a, int dim, _Float16 *bounds, int cus, hipStream_t s) {
    switch (dim) {
    case 64: return bounds_launch<2>(a, bounds, cus, s);
    case 96: return bounds_launch<3>(a, bounds, cus, s);
    case 128: return bounds_launch<4>(a, bounds, cus, s);
    case 256: return bounds_launch<8>(a, bounds, cus, s);
    }
    return hipErrorInvalidValue;
}

// Workspace of a chunk's keys and pages, at most (one row's where that is more).
constexpr int64_t CHUNK_BYTES = (int64_t)256 << 20;

BlocksPlan blocks_plan(int cus, int heads, int dim, int page, int64_t tokens, int q_heads, int64_t max_pages, int64_t count) {
    BlocksPlan p;
    const int64_t group = q_heads / heads;
    p.tiles = (int)((group + 15) / 16);
    p.width = (int)std::max<int64_t>(1, std::min(count, max_pages));
    const int64_t keys = max_pages > count ? heads * max_pages * 8 : 0, table = (int64_t)heads * p.width * 4;
    p.rows = (int)std::min<int64_t>(std::max<int64_t>(CHUNK_BYTES / (keys + table), 1), std::max<int64_t>(tokens, 1));
    const int64_t items = (int64_t)p.rows * heads * p.tiles, target = (int64_t)rows16_waves(dim / KV_GROUP) * cus;
    const int64_t most = std::min((p.width * (int64_t)page + MIN_PIECE - 1) / MIN_PIECE, (int64_t)0x7fff);
    p.pieces = (int)std::min(std::max<int64_t>(target / items, 1), most);
    auto align = [](int64_t n) { return (n + 255) / 256 * 256; };
    p.off_table = (size_t)align(p.rows * keys);
    p.off_part = p.off_table + (size_t)align(p.rows * table);
    p.ws_bytes = p.off_part + (p.pieces > 1 ? (size_t)items * p.pieces * 16 * (dim + 4) * sizeof(float) : 0);
    return p;
}

hipError_t launch_blocks(const BlocksArgs &b, int dim, const BlocksPlan &p, int cus, hipStream_t s) {
    switch (dim) {
    case 64: return dim_launch<2>(b, p, cus, s);
    case 96: return dim_launch<3>(b, p, cus, s);
    case 128: return dim_launch<4>(b, p, cus, s);
    case 256: return dim_launch<8>(b, p, cus, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace arfq
