// arfq_rope.hip -- rotary positions of one to four axes.
//
// A workgroup forms the cosines of one to eight tokens once, in LDS, for all of its heads; a thread has four pairs of a row
// (or eight of the values behind them), its first row's on the way meanwhile.  An angle counts in turns: position times
// turns a position in 64 bits, of which the nearest quarter is taken off, and what is left, at most an eighth of a turn,
// goes into the series of sine and cosine in 32 bits (the first terms left out are below 2^-27 of a turn's radius).
// Bound by memory: 8191 tokens of 48 x 128, f32, 403 MB in 74 us, 5.4 TB/s; f16 neighbours, 201 MB, 39.  Few rows by
// the launch (64 tokens of 36 x 128 3.2 us on the device).
#include <string.h>

#include "arfq_step.h"

namespace arfq {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr int THREADS = 256, DEEP_MAX = 8, ROWS_THREAD = 4;

struct Turn {
    float c, s;
};
__device__ __forceinline__ Turn turn_of(double turns, float gain) {
    const double quarter = rint(turns * 4.0);
    const float a = (float)(turns - quarter * 0.25) * 6.283185307179586f, w = a * a;
    const float c = 1.0f + w * (-1.0f / 2 + w * (1.0f / 24 + w * (-1.0f / 720 + w * (1.0f / 40320 + w * (-1.0f / 3628800)))));
    const float s = a + a * w * (-1.0f / 6 + w * (1.0f / 120 + w * (-1.0f / 5040 + w * (1.0f / 362880))));
    const int q = (int)((int64_t)quarter & 3);
    const float x = q & 1 ? s : c, y = q & 1 ? c : s;
    return {(q == 1 || q == 2 ? -x : x) * gain, (q >= 2 ? -y : y) * gain};
}

template <bool F16>
__device__ __forceinline__ void load4(const void *p, int64_t i, float (&o)[4]) {
    if constexpr (F16) {
        const u32x2 w = *(const u32x2 *)((const _Float16 *)p + i);
        o[0] = h2f(w.x); o[1] = h2f(w.x >> 16); o[2] = h2f(w.y); o[3] = h2f(w.y >> 16);
    } else {
        const f32x4 w = *(const f32x4 *)((const float *)p + i);
        o[0] = w.x; o[1] = w.y; o[2] = w.z; o[3] = w.w;
    }
}
template <bool F16>
__device__ __forceinline__ void store4(void *p, int64_t i, const float (&o)[4]) {
    if constexpr (F16)
        *(u32x2 *)((_Float16 *)p + i) = u32x2{pack_f16x2(o[0], o[1]), pack_f16x2(o[2], o[3])};
    else
        *(f32x4 *)((float *)p + i) = f32x4{o[0], o[1], o[2], o[3]};
}

// A workgroup: `deep` tokens, `span` heads of each.  lanes: threads of a row (dim / 8); slots: rows side by side.
// PAIRS at most: the host copies a launch's arguments (64 rows a call with room for 128 pairs 5.4 us, for 64 5.2).
template <bool XF16, bool OF16, bool NEIGHBOURS, int PAIRS>
__global__ __launch_bounds__(THREADS) void rope_kernel(RopeArgs a, RopePairsOf<PAIRS> pairs, int lanes, int slots, int deep, int span, int groups) {
    __shared__ Turn turns[DEEP_MAX * PAIRS];
    const int slot = threadIdx.x / lanes, u = threadIdx.x - slot * lanes, half = a.rot / 2;
    const int tile = block_of() / groups, t0 = tile * deep, h0 = (block_of() - tile * groups) * span;
    if (t0 >= a.tokens) return;
    deep = min(deep, a.tokens - t0);
    span = min(span, a.heads - h0);
    // two runs of four values: a pair's halves, or eight neighbours
    const bool turned = u < a.rot / 8;
    const int first = NEIGHBOURS || !turned ? 8 * u : 4 * u, second = first + (NEIGHBOURS || !turned ? 4 : half);
    const int rows = slot < slots && (turned || a.x != a.out) ? deep * span : 0;
    float x[4], y[4];
    int row = slot, tok = row / span;
    auto load = [&] {
        const int64_t o = (t0 + tok) * a.x_stride + (int64_t)(h0 + row - tok * span) * a.dim;
        load4<XF16>(a.x, o + first, x);
        load4<XF16>(a.x, o + second, y);
    };
    if (row < rows) load();
    for (int i = threadIdx.x; i < deep * half; i += THREADS) {
        const int t = i / half, p = i - t * half;
        turns[i] = turn_of((double)a.positions[pairs.axis[p] * a.position_stride + t0 + t] * pairs.turns[p], a.gain);
    }
    lds_barrier();
    while (row < rows) {
        if (turned) {
            const Turn *w = turns + tok * half + 4 * u;
            auto rotate = [&](int i, float &p, float &q) {
                const float r = p * w[i].c - q * w[i].s;
                q = p * w[i].s + q * w[i].c;
                p = r;
            };
            if constexpr (NEIGHBOURS) {
                rotate(0, x[0], x[1]);
                rotate(1, x[2], x[3]);
                rotate(2, y[0], y[1]);
                rotate(3, y[2], y[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) rotate(i, x[i], y[i]);
            }
        }
        const int64_t o = (t0 + tok) * a.out_stride + (int64_t)(h0 + row - tok * span) * a.dim;
        store4<OF16>(a.out, o + first, x);
        store4<OF16>(a.out, o + second, y);
        row += slots;
        if (row >= rows) break;
        tok = row / span;
        load();
    }
}

template <bool XF16, bool OF16, bool NEIGHBOURS, int PAIRS>
hipError_t rope_launch(const RopeArgs &a, const RopePairs &all, int cus, hipStream_t s) {
    RopePairsOf<PAIRS> pairs;
    memcpy(pairs.turns, all.turns, sizeof(pairs.turns));
    memcpy(pairs.axis, all.axis, sizeof(pairs.axis));
    const int lanes = a.dim / 8, slots = THREADS / lanes;
    // heads of a workgroup: all of a token's, fewer where that leaves compute units idle; then tokens, so that a
    // thread has about four rows
    int span = a.heads;
    while (span > slots && (int64_t)a.tokens * ((a.heads + span - 1) / span) < 4 * cus) span = (span + 1) / 2;
    const int groups = (a.heads + span - 1) / span;
    int deep = 1;
    while (deep < DEEP_MAX && 2 * deep * span <= ROWS_THREAD * slots && (int64_t)a.tokens / (2 * deep) * groups >= 4 * cus) deep *= 2;
    const int64_t blocks = ((int64_t)a.tokens + deep - 1) / deep * groups;
    rope_kernel<XF16, OF16, NEIGHBOURS, PAIRS><<<grid_of(blocks), THREADS, 0, s>>>(a, pairs, lanes, slots, deep, span, groups);
    return hipGetLastError();
}

template <bool XF16, bool OF16>
hipError_t types_launch(const RopeArgs &a, const RopePairs &p, int cus, hipStream_t s) {
    constexpr int FEW = 32, MANY = ROPE_DIM_MAX / 2;
    if (a.neighbours)
        return a.rot <= 2 * FEW   ? rope_launch<XF16, OF16, true, FEW>(a, p, cus, s)
               : a.rot <= 4 * FEW ? rope_launch<XF16, OF16, true, 2 * FEW>(a, p, cus, s)
                                  : rope_launch<XF16, OF16, true, MANY>(a, p, cus, s);
    return a.rot <= 2 * FEW   ? rope_launch<XF16, OF16, false, FEW>(a, p, cus, s)
           : a.rot <= 4 * FEW ? rope_launch<XF16, OF16, false, 2 * FEW>(a, p, cus, s)
                              : rope_launch<XF16, OF16, false, MANY>(a, p, cus, s);
}

}  // namespace

hipError_t launch_rope(const RopeArgs &a, const RopePairs &p, int cus, hipStream_t s) {
    if (a.x_f16) return a.out_f16 ? types_launch<true, true>(a, p, cus, s) : types_launch<true, false>(a, p, cus, s);
    return a.out_f16 ? types_launch<false, true>(a, p, cus, s) : types_launch<false, false>(a, p, cus, s);
}

}  // namespace arfq
