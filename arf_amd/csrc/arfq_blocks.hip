// arfq_blocks.hip -- attention over the blocks (pages) of the 4-bit cache that each query chooses.
//
// Bounds: of each channel of a page's keys the largest and smallest (arfq_kv_bounds), f16 and exact, as keys are.
// A call: the scores' keys of all blocks (blocks_score), the best of them for each row and K/V head and their pages
// (blocks_select, or choose() within the next), attention with those pages as the row's table (blocks_attend: the tile of
// arfq_attn_rows16.h, a row a sequence of its own), and the joining of rows whose keys were cut into pieces.
// One token at 131071, 64 of 2048 blocks of 64, 40 x 128 on 8, f32: bounds 4, scores 8, attention 13 (6 of it the choice), join
// 4 us: latency.  256 rows of a prompt, 32 of 520 blocks of 32, 32 x 64 on 8, f16: 5, 30 and 44 (four rows of 16 in a tile's
// products, whose operands are made for every row anew).
#include <math.h>

#include "arfq_attn_join.h"
#include "arfq_attn_rows16.h"
#include "arfq_step.h"

namespace arfq {
namespace {

constexpr int SEL = 256, SEL_WAVES = SEL / WAVE;  // threads that choose for a row
constexpr int KEPT = 8;                           // keys of a thread in registers
// The attention's workgroups choose for themselves, each its row's pages, into its LDS (a launch and a table's way through memory
// less) where a row is one workgroup's, or where the threads' registers have all keys: otherwise every piece of a row's keys reads them
// again and again.  us by a launch of its own and in LDS, pages of 16.  All keys in registers: 8 K/V heads of 128, f32, one token, 64 of
// 1024 blocks 27.5 and 26.8, 1024 of 2048 32.9 and 31.8; 16 sequences, 4 of 64, f16, 256 of 2048 42.5 and 44.  More: those 256 of 4096 66
// and 91, of 8192 106 and 194; one token, 64 of 4096 41.2 and 39.7, 2048 of 16384 131 and 196.  A row one workgroup's: prompts, 8 of
// 64, f16, 256 rows, 32 of 512 65.6 and 63.2, 32 of 4096 423 and 335, 256 of 8192 1235 and 1042 (64 rows, two pieces each, 124 and 138 at 256 of 4096).
constexpr int WIDTH_LDS = 2048, BLOCKS_KEPT = SEL * KEPT;  // (chosen pages that LDS has room for)

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
// Rows one after another: those of one sequence are found by its first.
struct Rows {
    int b = 0, t0 = 0, n = 0, len = 0;
    __device__ __forceinline__ Row operator()(const KvArgs &a, int t) {
        if (t < t0 || t >= t0 + n) {
            n = 0;
            b = seq_of_row(a, t);
            if (b < a.batch) {
                len = a.len[b];
                kv_seq(a, b, t0, n);
            }
            if (t < t0 || t >= t0 + n) return {-1, 0, 0};
        }
        const int64_t pos = (int64_t)len - ((int64_t)t0 + n - t);
        const int end = pos < 0 ? 0 : (int)min(pos + 1, (int64_t)a.max_pages * a.page);
        return {b, (end + a.page - 1) / a.page, end};
    }
};
__device__ __forceinline__ Row row_of(const KvArgs &a, int t) {
    Rows rows;
    return rows(a, t);
}

// ---- bounds ----------------------------------------------------------------------------------

// Keys [k0, k1) of a page of a head: a lane has a dword column of K's codes (eight values of a key), 64 / (4 NG) keys side by
// side, and of those every one behind the last again (no branch: an extreme does not mind).  The result is in the first
// 4 NG lanes.
template <int NG>
struct Extremes {
    static constexpr int COLS = 4 * NG, KL = WAVE / COLS;
    float hi[8], lo[8];
    int bad;  // a key that is NaN
    __device__ __forceinline__ void add(const float (&h)[8], const float (&l)[8], int b) {
        bad |= b;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            hi[e] = fmaxf(hi[e], h[e]);
            lo[e] = fminf(lo[e], l[e]);
        }
    }
    __device__ __forceinline__ Extremes(const uint8_t *reg, const KvArgs &a, int k0, int k1) : bad(0) {
        const int lane = threadIdx.x & 63, kk = min(lane / COLS, KL - 1), col = lane % COLS, g = col % NG;
        const uint32_t *codes = (const uint32_t *)reg + col;
        const uint16_t *scales = (const uint16_t *)(reg + a.off_ks) + g;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            hi[e] = -INFINITY;
            lo[e] = INFINITY;
        }
        constexpr int U = 8;
        for (int key = k0 + kk; key < k1 + kk; key += U * KL) {
            uint32_t w[U];
            uint16_t d[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int at = min(key + u * KL, k1 - 1);
                w[u] = codes[at * COLS];
                d[u] = scales[at * NG];
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float f = h2f(d[u]);
                bad |= f != f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float v = f * (float)((int)(w[u] >> (4 * ((e >> 1) + 4 * (e & 1))) & 15u) - 8);
                    hi[e] = fmaxf(hi[e], v);
                    lo[e] = fminf(lo[e], v);
                }
            }
        }
        // over the keys side by side: a tree over any number of them
#pragma unroll
        for (int s = KL; s > 1;) {
            const int half = (s + 1) / 2, from = kk + half < s ? lane + half * COLS : lane;
            float h[8], l[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                h[e] = __shfl(hi[e], from);
                l[e] = __shfl(lo[e], from);
            }
            add(h, l, __shfl(bad, from));
            s = half;
        }
    }
    __device__ __forceinline__ void store(_Float16 *bounds) const {
        const int lane = threadIdx.x & 63, g = lane % NG, h = lane / NG;
        f16x8 vh, vl;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            vh[e] = (_Float16)(bad ? NAN : hi[e]);
            vl[e] = (_Float16)(bad ? NAN : lo[e]);
        }
        *(f16x8 *)(bounds + 32 * g + 8 * h) = vh;
        *(f16x8 *)(bounds + 32 * NG + 32 * g + 8 * h) = vl;
    }
};

// `per` rows of a head, and of those the pages that begin with one of them, or in which a sequence's first one lies.  By a
// wave, or (WIDE) by a workgroup whose waves share a page's keys.
template <int NG, bool WIDE>
__global__ __launch_bounds__(256) void kv_bounds_kernel(KvArgs a, _Float16 *bounds, int per, int items) {
    constexpr int COLS = 4 * NG;
    __shared__ float sh[WIDE ? 3 : 1][COLS][17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int item = WIDE ? block_of() : block_of() * 4 + wave;
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
            if ((uint32_t)id >= (uint32_t)a.n_pages) continue;
            const uint8_t *reg = a.data + ((int64_t)id * a.heads + head) * a.region;
            _Float16 *out = bounds + ((int64_t)id * a.heads + head) * (64 * NG);
            const int keys = (int)min((int64_t)a.page, len - p * a.page);
            if constexpr (WIDE) {
                const int share = a.page / 4, k0 = min(wave * share, keys - 1);
                Extremes<NG> x(reg, a, k0, min(k0 + share, keys));
                if (wave && lane < COLS) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        sh[wave - 1][lane][e] = x.hi[e];
                        sh[wave - 1][lane][8 + e] = x.lo[e];
                    }
                    sh[wave - 1][lane][16] = (float)x.bad;
                }
                __syncthreads();
                if (wave == 0 && lane < COLS) {
#pragma unroll
                    for (int w = 0; w < 3; w++) {
                        float h[8], l[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            h[e] = sh[w][lane][e];
                            l[e] = sh[w][lane][8 + e];
                        }
                        x.add(h, l, sh[w][lane][16] != 0.0f);
                    }
                    x.store(out);
                }
                __syncthreads();
            } else {
                const Extremes<NG> x(reg, a, 0, keys);
                if (lane < COLS) x.store(out);
            }
        }
    }
}

template <int NG>
hipError_t bounds_launch(const KvArgs &a, _Float16 *bounds, int cus, hipStream_t s) {
    const int64_t rows = (int64_t)a.tokens * a.heads;
    // (a workgroup a page: 8 rows of 64 keys 3.6 us for 5.8 by a wave; 2048 rows, of which 64 have a page, 8.6 for 5.2)
    if (rows <= 2 * (int64_t)cus) {
        kv_bounds_kernel<NG, true><<<grid_of(rows), 256, 0, s>>>(a, bounds, 1, (int)rows);
        return hipGetLastError();
    }
    // rows of a wave: one while that does not fill the chip several times over
    const int per = (int)std::min<int64_t>(std::max<int64_t>(rows / (64 * (int64_t)cus), 1), 64);
    const int64_t items = ((int64_t)a.tokens + per - 1) / per * a.heads;
    kv_bounds_kernel<NG, false><<<grid_of((items + 3) / 4), 256, 0, s>>>(a, bounds, per, (int)items);
    return hipGetLastError();
}

// ---- scores ----------------------------------------------------------------------------------

typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

// Scores as whole numbers in their order.  Those of chosen blocks by rule are never formed; NaN comes first, pages
// that are not the cache's last.
constexpr uint64_t KEY_NAN = ~0ull, KEY_NONE = 0;
__device__ __forceinline__ uint64_t key_of(double v, bool number) {
    if (!number && v != v) return KEY_NAN;
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);  // (-0 as 0)
    const uint32_t hi = (uint32_t)(u >> 32), sign = (uint32_t)((int32_t)hi >> 31);
    return (uint64_t)(hi ^ (sign | 0x80000000u)) << 32 | ((uint32_t)u ^ sign);
}
// Of the lane N further on in the 16 lanes of a row, around its end.
template <int N, class T>
__device__ __forceinline__ T lane_on(T t) {
    constexpr int ror = 0x120 + 16 - N;
    const uint64_t v = __builtin_bit_cast(uint64_t, t);
    return __builtin_bit_cast(T, (uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), ror, 0xf, 0xf, false) << 32 |
                                     (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ror, 0xf, 0xf, false));
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
    int parts;            // workgroups of a tile's blocks
    int second;           // workgroups from this one on are likely the second ones of their compute units
    uint64_t *keys;       // [rows][heads][max_pages]
};

// 16 blocks by 16 columns with v_mfma_f64_16x16x4_f64: a column is a (row, q head of the K/V head), and the sum runs
// over [max(q, 0), min(q, 0)] times [hi, lo].  The products of an f32 and an f16 are exact in 64 bits, so that nothing but the
// order of the sum's last bits is left to chance: blocks' order is that of their scores.  A lane of the operands has
// the channels D / 4 * (lane / 16) .. of its block or column.  The workgroup's waves have other blocks of the same columns,
// whose q is in LDS as the products take it.  The vector unit's instructions do not overlap with these products (two waves
// a SIMD: 69 cycles a product alone, 85 with three of them between), so what is not a product is kept short: 256 rows of 520
// blocks, 32 x 64 on 8: 29.7 us, 14 of them products at 64 cycles (34.2 with operands made product by product, and keys of
// every column compared as whole numbers); one row of 2048 blocks, 40 x 128 on 8: 8, of which a tile's products are 1.7.
// Waves of a SIMD, which the split of the blocks counts on.  (Three / four of them at 64 channels a quarter slower.)
constexpr int score_waves(int ng) { return ng <= 4 ? 2 : 1; }
template <int NG>
__global__ __launch_bounds__(256, score_waves(NG)) void blocks_score(ScoreArgs a) {
    constexpr int D = 32 * NG, DL = D / 4;
    __shared__ f64x2 qs[DL][WAVE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, kg = lane >> 4;
    const KvArgs &kv = a.c;
    int block = block_of();
    const int head = block % kv.heads;
    block /= kv.heads;
    const int part = block % a.parts, row0 = block / a.parts * a.per_tile;
    if (row0 >= a.rows) return;
    // this lane's column
    const int rt = c / a.group;  // (0 where the group has more than 16 heads)
    Row mine = {-1, 0, 0};
    int most = 0;  // blocks of the tile's rows
    Rows rows;
    for (int r = 0; r < a.per_tile && row0 + r < a.rows; r++) {
        const Row x = rows(kv, a.row0 + row0 + r);
        if (rt == r) mine = x;
        if (x.seen > a.count) most = max(most, x.seen);
    }
    // this wave's blocks [j0, j1): shares of whole sixteens, one more for the last ones where they do not come out even (the
    // first ones of a second workgroup: a SIMD has both workgroups' wave of a number)
    const int sixteens = (most + 15) / 16, share = sixteens / (4 * a.parts), odd = 4 * a.parts - sixteens % (4 * a.parts);
    auto share_of = [&](int w) { return 16 * (w * share + max(w - odd, 0)); };
    if (share_of(4 * part) == share_of(4 * part + 4)) return;
    const int of = 4 * part + ((int)blockIdx.x >= a.second ? 3 - wave : wave), j0 = share_of(of), j1 = share_of(of + 1);
    if (mine.seen <= a.count) mine.b = -1;  // (its blocks are all chosen)
    const int64_t t = (int64_t)a.row0 + row0 + rt;
    // (one pass, unless the group has more than 16 heads)
    for (int g0 = 0; g0 < a.group; g0 += 16) {
        const int gh = g0 + (a.group > 16 ? c : c - rt * a.group);
        const bool on = mine.b >= 0 && gh < a.group;
        if (g0) __syncthreads();
        for (int ch = wave; ch < DL / 8; ch += 4) {
            float q[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (on) {
                const int64_t at = t * a.q_stride + (int64_t)(head * a.group + gh) * D + DL * kg + 8 * ch;
                if (a.q_f16) {
                    const f16x8 v = *(const f16x8 *)((const _Float16 *)a.q + at);
#pragma unroll
                    for (int e = 0; e < 8; e++) q[e] = (float)v[e];
                } else {
                    const f32x4 v = *(const f32x4 *)((const float *)a.q + at), w = *(const f32x4 *)((const float *)a.q + at + 4);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        q[e] = v[e];
                        q[4 + e] = w[e];
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = a.negative ? -q[e] : q[e];  // (NaN goes into the first)
                qs[8 * ch + e][lane] = f64x2{v < 0.0f ? 0.0 : (double)v, v < 0.0f ? (double)v : 0.0};
            }
        }
        __syncthreads();
        uint64_t done = __ballot(mine.b < 0);
        while (done != ~0ull) {
            const int b = __builtin_amdgcn_readlane(mine.b, __ffsll((unsigned long long)~done) - 1);
            done |= __ballot(mine.b == b);
            int last = mine.b == b ? mine.seen : 0;
#pragma unroll
            for (int d = 1; d < 16; d *= 2) last = max(last, __shfl_xor(last, d));
            last = min(__builtin_amdgcn_readfirstlane(last), j1);
            if (j0 >= last) continue;
            const int32_t *table = kv.table + (int64_t)b * kv.max_pages;
            // bounds a tile ahead of their use, pages 64 blocks at a time; keys are stored a tile later, so that no load's
            // wait is for a store
            f16x8 hi[DL / 8], lo[DL / 8];
            int ids = 0, from = j0 - WAVE;
            auto load = [&](int j) -> bool {  // (a tile lies in one 64: the waves' blocks are a multiple of 16)
                if (j >= from + WAVE) {
                    from += WAVE;
                    ids = table[min(from + lane, last - 1)];
                }
                const int id = __shfl(ids, j - from + c);
                const bool page = (uint32_t)id < (uint32_t)kv.n_pages;
                const _Float16 *p = a.bounds + ((int64_t)(page ? id : 0) * kv.heads + head) * (2 * D) + DL * kg;
#pragma unroll
                for (int i = 0; i < DL / 8; i++) {
                    hi[i] = *(const f16x8 *)(p + 8 * i);
                    lo[i] = *(const f16x8 *)(p + D + 8 * i);
                }
                return page;
            };
            const int heads = a.group > 16 ? 16 : a.group, h0 = a.group > 16 ? c : c - rt * a.group;
            const bool first = h0 == 0 && mine.b == b;
            const bool plain = a.group <= 16 || g0 + 16 <= a.group;  // every column of a row is one of its heads
            uint64_t *out = a.keys + ((int64_t)(row0 + rt) * kv.heads + head) * kv.max_pages;
            uint64_t key[4];
            const int to = first ? min(mine.seen, last) - kg : 0;
            auto store = [&](int j) {  // a lane's four results: blocks kg, kg + 4, .. of the 16, its column
                uint64_t *o = out + j + kg;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (j + 4 * i < to) o[4 * i] = g0 == 0 ? key[i] : max(key[i], o[4 * i]);
            };
            bool page = load(j0);
            for (int j = j0; j < last; j += 16) {
                f64x4 up = {0, 0, 0, 0}, down = {0, 0, 0, 0};
                f16x8 h[DL / 8], l[DL / 8];
#pragma unroll
                for (int i = 0; i < DL / 8; i++) {
                    h[i] = hi[i];
                    l[i] = lo[i];
                }
                const bool there = page;
                if (j + 16 < last) page = load(j + 16);
                if (j > j0) store(j - 16);
                // (operands of eight channels made together: each change between the two units costs some cycles more)
#pragma unroll
                for (int ch = 0; ch < DL / 8; ch++) {
                    f64x2 q[8];
                    double x[8], y[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) q[e] = qs[8 * ch + e][lane];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[e] = (double)(float)h[ch][e];
                        y[e] = (double)(float)l[ch][e];
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        up = __builtin_amdgcn_mfma_f64_16x16x4f64(x[e], q[e].x, up, 0, 0, 0);
                        down = __builtin_amdgcn_mfma_f64_16x16x4f64(y[e], q[e].y, down, 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                // the largest of the row's heads, at the first of them (of its lanes alone the results are stored)
                double v[4];
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = up[i] + down[i];
                const double all = (v[0] + v[1]) + (v[2] + v[3]);
                const uint64_t pages = __ballot(there);  // (lane n has block n's page)
                auto heads_max = [&](auto &best) {
                    auto wider = [&](auto step) {
                        constexpr int N = decltype(step)::value;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const auto k = lane_on<N>(best[i]);
                            if (h0 + N < heads && k > best[i]) best[i] = k;
                        }
                    };
                    if (heads > 1) wider(std::integral_constant<int, 1>());
                    if (heads > 2) wider(std::integral_constant<int, 2>());
                    if (heads > 4) wider(std::integral_constant<int, 4>());
                    if (heads > 8) wider(std::integral_constant<int, 8>());
                };
                if (plain && pages == ~0ull && __ballot(all != all) == 0) {  // numbers throughout
                    heads_max(v);
#pragma unroll
                    for (int i = 0; i < 4; i++) key[i] = key_of(v[i], true);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) key[i] = on && (pages >> (kg + 4 * i) & 1) ? key_of(v[i], false) : KEY_NONE;
                    heads_max(key);
                }
            }
            store(j0 + (last - 1 - j0) / 16 * 16);
        }
    }
}

// ---- choice ----------------------------------------------------------------------------------

struct SelLds {
    uint32_t bins[256], found[3], sums[2][SEL_WAVES];
};

// Largest value and running sum over a wave's lanes, and over the workgroup's threads (sh is free again behind the next
// barrier).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lane_of(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <class F>
__device__ __forceinline__ uint32_t wave_run(uint32_t v, F f) {
    v = f(v, lane_of<0x111, 0xf>(v));  // row_shr:1, 2, 4, 8
    v = f(v, lane_of<0x112, 0xf>(v));
    v = f(v, lane_of<0x114, 0xf>(v));
    v = f(v, lane_of<0x118, 0xf>(v));
    v = f(v, lane_of<0x142, 0xa>(v));  // row_bcast:15 into rows 1 and 3
    return f(v, lane_of<0x143, 0xc>(v));  // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ uint32_t run_sum(uint32_t v) { return wave_run(v, [](uint32_t x, uint32_t y) { return x + y; }); }
__device__ __forceinline__ uint32_t run_max(uint32_t v) { return wave_run(v, [](uint32_t x, uint32_t y) { return max(x, y); }); }

// The `count` blocks of n that are chosen: the `first` earliest, the `last` latest, and of the others those with the largest
// keys, the earlier one of two alike; in their order.  A thread has a run of neighbouring blocks.  The
// range of the keys' upper halves that the last chosen one lies in is cut into 256 parts and counted, until a
// part's keys are all chosen or all alike; then, where they are alike, that of their lower halves.  (n > count, the
// workgroup's threads all come here.)  take(rank, block, page).
// most: places of keys and pages.
struct Kept {
    uint64_t key[KEPT];
    // (before n is known: the loads do not wait for it)
    __device__ __forceinline__ Kept(const uint64_t *keys, int most) {
        if (most == 0) return;  // (all blocks are chosen)
        const int j0 = threadIdx.x * ((most + SEL - 1) / SEL);
#pragma unroll
        for (int i = 0; i < KEPT; i++) key[i] = keys[min(j0 + i, most - 1)];
    }
};
template <class Take>
__device__ __forceinline__ void choose(const uint64_t *keys, const Kept &kept, const int32_t *pages, int most, int n, int count,
                                       int first, int last, SelLds &sh, Take take) {
    const int tid = threadIdx.x, wave = tid >> 6;
    const int per = (most + SEL - 1) / SEL, j0 = min(tid * per, n), j1 = min(j0 + per, n);
    const int f0 = first, f1 = n - last;  // blocks [f0, f1) go by their keys
    int32_t page[KEPT];
#pragma unroll
    for (int i = 0; i < KEPT; i++) page[i] = pages[min(j0 + i, n - 1)];
    auto each = [&](auto f) {  // f(block, key)
#pragma unroll
        for (int i = 0; i < KEPT; i++)
            if (j0 + i < j1) f(j0 + i, kept.key[i]);
        for (int j = j0 + KEPT; j < j1; j++) f(j, keys[j]);
    };
    sh.bins[tid] = 0;
    // The `need` largest of the candidates' words: all from `at` on (true), or those above `at` and `need` more of those that
    // are `at`.
    auto narrow = [&](auto word, auto candidate, uint32_t &need, uint32_t &at) {
        uint32_t hi = 0, not_lo = 0;
        each([&](int j, uint64_t key) {
            if (!candidate(j, key)) return;
            hi = max(hi, word(key));
            not_lo = max(not_lo, ~word(key));
        });
        hi = run_max(hi);
        not_lo = run_max(not_lo);
        if ((tid & 63) == 63) {
            sh.sums[0][wave] = hi;
            sh.sums[1][wave] = not_lo;
        }
        __syncthreads();
        hi = not_lo = 0;
#pragma unroll
        for (int w = 0; w < SEL_WAVES; w++) {
            hi = max(hi, sh.sums[0][w]);
            not_lo = max(not_lo, sh.sums[1][w]);
        }
        uint32_t lo = ~not_lo;
        bool all = false;
        while (lo < hi) {
            const int shift = max(24 - __clz((int)(hi - lo)), 0);
            each([&](int j, uint64_t key) {
                if (candidate(j, key) && word(key) >= lo && word(key) <= hi) atomicAdd(&sh.bins[(word(key) - lo) >> shift], 1u);
            });
            __syncthreads();
            // the part that the last chosen one lies in: 256 counts summed from the top
            const uint32_t mine = sh.bins[255 - tid];
            sh.bins[255 - tid] = 0;
            uint32_t upto = run_sum(mine);
            if ((tid & 63) == 63) sh.sums[0][wave] = upto;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < SEL_WAVES - 1; w++) upto += w < wave ? sh.sums[0][w] : 0;
            if (upto >= need && upto - mine < need) {
                sh.found[0] = 255 - tid;
                sh.found[1] = need - (upto - mine);
                sh.found[2] = mine;
            }
            __syncthreads();
            const uint32_t wide = (1u << shift) - 1;
            need = sh.found[1];
            lo += sh.found[0] << shift;
            if (hi - lo > wide) hi = lo + wide;
            all = sh.found[2] == need;
            if (all) break;
        }
        at = lo;
        return all;
    };
    auto upper = [](uint64_t key) { return (uint32_t)(key >> 32); };
    auto lower = [](uint64_t key) { return (uint32_t)key; };
    uint32_t need = (uint32_t)(count - first - last), at = ~0u, at_lower = ~0u;
    bool all = false, all_lower = false;
    if (need > 0) {
        all = narrow(upper, [&](int j, uint64_t) { return j >= f0 && j < f1; }, need, at);
        if (!all) {
            __syncthreads();  // (the sums' places)
            all_lower = narrow(lower, [&](int j, uint64_t key) { return j >= f0 && j < f1 && upper(key) == at; }, need, at_lower);
        }
    }
    auto is_sure = [&](int j, uint64_t key) {
        const uint32_t u = upper(key), l = lower(key);
        return j < f0 || j >= f1 || u > at || (u == at && (all || l > at_lower || (all_lower && l == at_lower)));
    };
    auto is_tie = [&](int j, uint64_t key) {
        return j >= f0 && j < f1 && !all && !all_lower && upper(key) == at && lower(key) == at_lower;
    };
    uint32_t sure = 0, ties = 0;
    each([&](int j, uint64_t key) {
        sure += is_sure(j, key);
        ties += is_tie(j, key);
    });
    uint32_t before = run_sum(sure), tie = run_sum(ties);
    __syncthreads();
    if ((tid & 63) == 63) {
        sh.sums[0][wave] = before;
        sh.sums[1][wave] = tie;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SEL_WAVES - 1; w++) {
        before += w < wave ? sh.sums[0][w] : 0;
        tie += w < wave ? sh.sums[1][w] : 0;
    }
    before -= sure;
    tie -= ties;
    auto step = [&](int j, uint64_t key, auto page) {
        const bool s = is_sure(j, key), e = is_tie(j, key);
        const uint32_t rank = before + min(tie, need);
        if ((s || (e && tie < need)) && rank < (uint32_t)count) take((int)rank, j, page());
        before += s;
        tie += e;
    };
#pragma unroll
    for (int i = 0; i < KEPT; i++)
        if (j0 + i < j1) step(j0 + i, kept.key[i], [&] { return page[i]; });
    for (int j = j0 + KEPT; j < j1; j++) step(j, keys[j], [&] { return pages[j]; });
}

// What a row chooses.  A row's pages of a K/V head are put into `table` (LDS or memory); `write`: its blocks into chosen, too.
struct ChooseArgs {
    KvArgs c;
    const uint64_t *keys;  // [rows][heads][max_pages] of the chunk
    int32_t *table;        // [rows][heads][width], or null: in the workgroups' LDS
    int32_t *chosen;       // [tokens][heads][count] of the call, or null
    int row0, rows, count, first, last, width;
};
__device__ __forceinline__ const uint64_t *keys_of(const ChooseArgs &a, int row, int head) {
    return a.keys + ((int64_t)row * a.c.heads + head) * a.c.max_pages;
}
__device__ __forceinline__ void choose_row(const ChooseArgs &a, const Row &r, const Kept &kept, int row, int head, int32_t *table,
                                           bool write, SelLds &sh) {
    const int32_t *pages = a.c.table + (int64_t)r.b * a.c.max_pages;
    int32_t *chosen = a.chosen && write ? a.chosen + (((int64_t)a.row0 + row) * a.c.heads + head) * a.count : nullptr;
    auto take = [&](int rank, int j, int32_t page) {
        table[rank] = page;
        if (chosen) chosen[rank] = j;
    };
    if (r.seen <= a.count) {
        for (int j = threadIdx.x; j < r.seen; j += SEL) take(j, j, pages[j]);
    } else {
        choose(keys_of(a, row, head), kept, pages, a.c.max_pages, r.seen, a.count, a.first, a.last, sh, take);
    }
    if (chosen)
        for (int i = min(r.seen, a.count) + (int)threadIdx.x; i < a.count; i += SEL) chosen[i] = -1;
}

__global__ __launch_bounds__(SEL) void blocks_select(ChooseArgs a) {
    __shared__ SelLds sh;
    const int block = block_of(), head = block % a.c.heads, row = block / a.c.heads;
    if (row >= a.rows) return;
    const Kept kept(keys_of(a, row, head), a.c.max_pages > a.count ? a.c.max_pages : 0);
    const Row r = row_of(a.c, a.row0 + row);
    if (r.b < 0) return;
    choose_row(a, r, kept, row, head, a.table + ((int64_t)row * a.c.heads + head) * a.width, true, sh);
}

// ---- attention -------------------------------------------------------------------------------

// A row is a sequence of its own, whose pages are the chosen ones: all but its own, the last, are whole.
struct RowsArgs {
    AttnArgs a;       // max_pages: chosen pages
    ChooseArgs ch;
    int tiles, pieces;
};
struct RowItem {
    Row r;
    int row, tile, piece, pieces, keys, part;
    __device__ __forceinline__ RowItem(const RowsArgs &a, int slot) : part(slot) {
        piece = slot % a.pieces;
        tile = slot / a.pieces % a.tiles;
        row = slot / a.pieces / a.tiles;
        r = {-1, 0, 0};
        if (row < a.ch.rows) r = row_of(a.ch.c, a.ch.row0 + row);
        keys = r.end - max(r.seen - a.ch.count, 0) * a.ch.c.page;
        pieces = max(1, min(a.pieces, (keys + MIN_PIECE - 1) / MIN_PIECE));
    }
    __device__ __forceinline__ bool none() const { return r.b < 0 || piece >= pieces; }
};

// Waves of a SIMD that the registers are for: five at 64 channels and one part (256 rows of 32 chosen blocks 44.2 us, 45.6 with
// four; two parts would go to scratch).  At 256 channels and two parts 36 of the 256 registers do (148 bytes a lane): one token of each of
// eight sequences of up to 16384, 16 x 256 on 4, f32, 32 blocks of 64, 37 us in all.
constexpr int attend_waves(int ng, int parts) { return ng == 2 && parts == 1 ? 5 : rows16_waves(ng); }
// CHOOSE: every workgroup chooses for itself, into its LDS (behind the tile's).
template <int NG, int PARTS, bool CHOOSE>
__global__ __launch_bounds__(256, attend_waves(NG, PARTS)) void blocks_attend(RowsArgs r) {
    extern __shared__ float lds[];
    __shared__ SelLds sh;
    const int block = block_of(), head = block % r.a.c.heads, slot = block / r.a.c.heads;
    const Kept kept(keys_of(r.ch, min(slot / r.pieces / r.tiles, r.ch.rows - 1), head), CHOOSE && r.ch.c.max_pages > r.ch.count ? r.ch.c.max_pages : 0);
    const RowItem x(r, slot);
    if (x.none()) return;
    const int32_t *table;
    if constexpr (CHOOSE) {
        int32_t *own = (int32_t *)((uint8_t *)lds + rows16_k::lds_bytes(NG));
        choose_row(r.ch, x.r, kept, x.row, head, own, x.tile == 0 && x.piece == 0, sh);
        __syncthreads();
        table = own;
    } else {
        table = r.ch.table + ((int64_t)x.row * r.a.c.heads + head) * r.ch.width;
    }
    Item it;
    it.s = {r.ch.row0 + x.row, 1, x.keys, 0, x.keys, r.tiles};
    it.b = it.cut = 0;
    it.tile = x.tile;
    it.piece = x.piece;
    it.pieces = x.pieces;
    it.keys = ((x.keys + STEP - 1) / STEP + x.pieces - 1) / x.pieces * STEP;
    it.part = x.part;
    rows16_k::rows16_item<NG, PARTS>(r.a, it, table, head, lds);
}

template <int NG>
__global__ __launch_bounds__(256) void blocks_join(RowsArgs r) {
    __shared__ JoinLds<NG> sh;
    const int block = block_of(), head = block % r.a.c.heads, slot = block / r.a.c.heads;
    const RowItem x(r, slot);
    if (x.none() || x.pieces == 1) return;
    join_tile<NG, 16>(r.a, r.a.few, make_int4(x.pieces | x.piece << 16, x.tile * 16, r.a.group, r.ch.row0 + x.row), slot, head, sh);
}

template <int NG, int PARTS, bool CHOOSE>
hipError_t attend_launch(const RowsArgs &r, hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t lds = rows16_k::lds_bytes(NG);
    const size_t all = lds + (CHOOSE ? (size_t)r.ch.width * sizeof(int32_t) : 0);
    const hipError_t e = set_max_lds_once((const void *)blocks_attend<NG, PARTS, CHOOSE>, lds + (CHOOSE ? WIDTH_LDS * sizeof(int32_t) : 0), done);
    if (e != hipSuccess) return e;
    blocks_attend<NG, PARTS, CHOOSE><<<grid_of((int64_t)r.ch.rows * r.tiles * r.pieces * r.a.c.heads), 256, all, s>>>(r);
    return hipGetLastError();
}

// Workgroups of a tile's blocks, which its four waves share: several where one leaves SIMDs without their waves, as far as there
// are sixteen blocks for a wave.
int score_parts(int cus, int waves, int64_t tiles, int max_pages) {
    return (int)std::max<int64_t>(1, std::min(waves * (int64_t)cus / std::max<int64_t>(tiles, 1), ((int64_t)max_pages + 63) / 64));
}

template <int NG>
hipError_t dim_launch(const BlocksArgs &b, const BlocksPlan &p, int cus, hipStream_t s) {
    const KvArgs &c = b.a.c;
    uint64_t *keys = (uint64_t *)b.ws;
    const bool f16 = b.a.q_dtype == ARFQ_F16 && b.a.out_dtype == ARFQ_F16;
    for (int row0 = 0; row0 < c.tokens; row0 += p.rows) {
        const int rows = std::min(p.rows, c.tokens - row0);
        hipError_t e;
        if (c.max_pages > b.count) {
            ScoreArgs sc = {c, b.bounds, b.a.q, b.a.q_stride, b.a.q_dtype == ARFQ_F16, b.a.scale < 0.0f, b.a.group, b.count, row0, rows,
                            std::max(1, 16 / b.a.group), 1, cus, keys};
            if (!c.start) sc.per_tile = 1;  // (no two rows have blocks in common)
            const int64_t tiles = (int64_t)((rows + sc.per_tile - 1) / sc.per_tile) * c.heads;
            sc.parts = score_parts(cus, score_waves(NG), tiles, c.max_pages);
            blocks_score<NG><<<grid_of(tiles * sc.parts), 256, 0, s>>>(sc);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
        const ChooseArgs ch = {c, keys, p.in_lds ? nullptr : (int32_t *)(b.ws + p.off_table), b.chosen, row0, rows, b.count, b.first, b.last, p.width};
        if (!p.in_lds) {
            blocks_select<<<grid_of((int64_t)rows * c.heads), SEL, 0, s>>>(ch);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
        RowsArgs r = {b.a, ch, p.tiles, p.pieces};
        r.a.c.max_pages = p.width;
        r.a.few = {1, 0, rows * p.tiles * p.pieces, 1, (float *)(b.ws + p.off_part), nullptr};
        e = p.in_lds ? f16 ? attend_launch<NG, 1, true>(r, s) : attend_launch<NG, 2, true>(r, s)
                     : f16 ? attend_launch<NG, 1, false>(r, s) : attend_launch<NG, 2, false>(r, s);
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
    const int64_t keys = max_pages > count ? heads * max_pages * 8 : 0, pages = (int64_t)heads * p.width * 4;
    const int64_t target = (int64_t)rows16_waves(dim / KV_GROUP) * cus;
    const int64_t most = std::min((p.width * (int64_t)page + MIN_PIECE - 1) / MIN_PIECE, (int64_t)0x7fff);
    int64_t table = 0, items = 0;
    auto split = [&] {  // rows of a chunk, and pieces
        p.rows = (int)std::min<int64_t>(keys + table ? std::max<int64_t>(CHUNK_BYTES / (keys + table), 1) : INT32_MAX, std::max<int64_t>(tokens, 1));
        items = (int64_t)p.rows * heads * p.tiles;
        p.pieces = (int)std::min(std::max<int64_t>(target / items, 1), most);
    };
    split();
    p.in_lds = p.width <= WIDTH_LDS && (max_pages <= BLOCKS_KEPT || p.pieces * p.tiles == 1);
    if (!p.in_lds) {
        table = pages;
        split();
    }
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
