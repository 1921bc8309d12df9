// arfq_attn_rows16.h -- attention for few rows a sequence (decode steps, verified drafts).
#pragma once
#include "arfq_attn.h"

namespace arfq {
namespace {
namespace rows16_k {

constexpr int TR = 16;    // rows of a tile
constexpr int WAVES = 4;  // of a workgroup
// ---- rows of 16, keys spread over the waves ------------------------------------------------
// S^T = K Q^T, O^T = V^T P^T with v_mfma_f32_16x16x32_f16: the 16 rows are matrix columns, so a
// lane's four results of a tile belong to one row, its statistics are a register, and P^T in
// the layout of a result is the layout of the next product's operand (which keys a lane's
// eight slots stand for is free, as V is loaded to match).  K's scales multiply the products of
// a group (32 values: one MFMA), V's its codes; both straight from memory to registers, a step ahead.
// PARTS: f16 parts of q and p (2: hi + lo, 22 bits, for f32 q or out; 1: an f16 q is exact in one, and p's 11
// bits add to an f16 out's own rounding, 2.2e-4 to 2.4e-4 against 64 bits in all, for 2.05e-4 of rounding alone).
//
// Bound between memory and the vector unit: turning 4-bit codes into operands takes 4 instructions a key and
// group, whatever the rows are.  Measured (the join's launch with it): 64 sequences of up to 8192 tokens, f32,
// 32 x 128 q heads on 4: 45 us for 153 MB, 3.4 TB/s (the vector unit issues half of the time, a third of
// a wave's time it waits for loads); one of 131071 tokens, 40 q heads on 8: 41 us, 3.7 TB/s; 16 of up
// to 4097, f16, 32 x 64 heads ungrouped: 25.8 us, 3.0 TB/s; a window of 1024, f16, 16 x 256 on 8, 32
// sequences: 27.7 us, 2.6 TB/s; 193 tokens of one: 7.3 us, all of it latency.  At 256 values and two parts 13 of the 256
// registers go to scratch: 64 sequences of up to 8192, 32 x 256 on 4, f32, 152 us for 2.7 TB/s (f16, one part, 32 of
// up to 4000, 16 x 256 on 8: 50 us, 4.1 TB/s; the same in f32 62, 3.0).
// block: (item, head), head fastest.
template <int NG, int PARTS>
__device__ __forceinline__ void rows16(const AttnArgs &a, int block, float *lds) {
    constexpr int D = 32 * NG, NT = 2 * NG;  // NT: 16-row tiles of O^T
    constexpr int OS = D + 4;                // LDS floats of a row of O: [WAVES][16][OS], then [WAVES][16][2]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, h = lane >> 4;
    const int head = block % a.c.heads;  // (fastest: the list's unused end comes last)
    Item it;
    if (!take_item<TR>(a, block, it)) return;
    const Seq &s = it.s;

    // keys [lo, hi) of the row of token tok
    auto row_hi = [&](int64_t pos) { return pos < 0 ? 0 : a.causal ? (int)min(pos + 1, (int64_t)s.end) : s.end; };
    auto row_lo = [&](int64_t pos) { return a.window ? (int)max((int64_t)0, min(pos - a.window + 1, (int64_t)s.end)) : 0; };
    const int rows = s.n * a.group, piece_lo = s.lo + it.piece * it.keys, piece_hi = min(s.end, piece_lo + it.keys);
    // the tile's keys in this piece, and those that every row has (both ends rise with the token)
    const int64_t pos0 = (int64_t)s.len - s.n + it.tile * TR / a.group;
    const int64_t pos1 = (int64_t)s.len - s.n + min(it.tile * TR + TR - 1, rows - 1) / a.group;
    const int first = max(row_lo(pos0) & ~(STEP - 1), piece_lo), last = min(row_hi(pos1), piece_hi);
    const int inner_lo = row_lo(pos1), inner_hi = min(row_hi(pos0), piece_hi);
    // this lane's row
    const int row = it.tile * TR + c;
    const bool valid = row < rows;
    const int tok = valid ? row / a.group : 0, gh = valid ? row - tok * a.group : 0;
    const int64_t pos = (int64_t)s.len - s.n + tok;
    const int lo = row_lo(pos), hi = min(valid ? row_hi(pos) : 0, piece_hi);

    constexpr int NEXT = WAVES * STEP;
    Steps<NEXT / KV_TILE> steps(a.c, it.b);
    const Offs<NG> offs = lane_offs<NG>();
    Raw<NG> r;
    int k0 = first + wave * STEP;
    bool in0 = false, in1 = false;  // whether this step's tiles are the cache's
    Place p0 = {a.c.data, 0, false}, p1 = p0;
    auto load_ks = [&]() {
        load_k(p0.reg, a.c, p0.sub, 0, offs, r);
        load_k(p1.reg, a.c, p1.sub, 1, offs, r);
    };
    auto load_vs = [&]() {
        load_v<NG>(p0.reg, a.c, p0.sub, 0, offs, r);
        load_v<NG>(p1.reg, a.c, p1.sub, 1, offs, r);
    };
    auto places = [&](int k) {
        const int l = steps.step(a.c, head, k);
        p0 = steps.at(a.c, l);
        p1 = steps.at(a.c, l + 1);
    };
    if (k0 < last) {  // (keys: the table has a page)
        places(k0);
        in0 = p0.in;
        in1 = p1.in;
        load_ks();
        load_vs();
        places(k0 + NEXT);
    }

    // q as operands: values 32g + 8h .. +7 of the row, times a power of two that puts the row's
    // largest into [2^14, 2^15): hi + lo hold 22 bits (an f16 q its 11)
    f16x8 q[PARTS][NG];
    const int64_t qo = ((int64_t)s.t0 + tok) * a.q_stride + (int64_t)(head * a.group + gh) * D + 8 * h;
    float sc = fabsf(a.scale);
    {
        float x[NG][8], top = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; g++) load8_q(a, qo + 32 * g, valid, x[g]);
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[g][e]));
        top = row_max(top);
        const RowScale rs = row_scale(top, a.scale);
        sc *= rs.down;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = x[g][e] * rs.up;
                const _Float16 t = (_Float16)v;
                q[0][g][e] = t;
                if constexpr (PARTS == 2) q[1][g][e] = (_Float16)(v - (float)t);
            }
    }
    const float cap = a.softcap;
    const float x_of_s = score_unit(sc, cap), x_of_t = cap * 1.4426950408889634f;

    f32x4 acc[NT], sum = {0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = f32x4{0, 0, 0, 0};
    float m = -INFINITY;
    Frag ones;
#pragma unroll
    for (int i = 0; i < 4; i++) ones.w[i] = f16x2{(_Float16)1, (_Float16)1};

    while (k0 < last) {
        // (here, not before the loop: at 256 values and two parts q would be read from scratch in it, 99 us for 60 at
        // one token of each of 32 sequences of up to 4000, 16 x 256 on 8)
        const uint32_t magic = magic_1024();
        const int k1 = k0 + NEXT;
        float x[8], unit = x_of_s;  // scores; a unit of them in log2
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const f32x4 z = {0, 0, 0, 0};
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const f16x8 kf = k_frag(r, half, g, magic);
                f32x4 t = z;
#pragma unroll
                for (int p = 0; p < PARTS; p++) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[p][g], t, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float d = (float)half_of(r.ks[half][(i * NG + g) / 2], (i * NG + g) & 1);
                    x[4 * half + i] = g == 0 ? t[i] * d : __builtin_fmaf(t[i], d, x[4 * half + i]);
                }
            }
            // the scores are formed here: K's registers are free for the next step's loads
            asm volatile("" : "+v"(x[4 * half]), "+v"(x[4 * half + 1]), "+v"(x[4 * half + 2]), "+v"(x[4 * half + 3]));
        }
        if (k1 < last) load_ks();
        if (cap > 0.0f) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = tanh_of(x[i] * x_of_s) * x_of_t;
            unit = 1.0f;
        }
        if (k0 < inner_lo || k0 + STEP > inner_hi || !in0 || !in1) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint32_t from = (uint32_t)(k0 + half * 16 + 4 * h - lo), width = (half ? in1 : in0) ? (uint32_t)max(hi - lo, 0) : 0u;
#pragma unroll
                for (int i = 0; i < 4; i++) x[4 * half + i] = from + i < width ? x[4 * half + i] : -INFINITY;
            }
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 8; i++) top = fmaxf(top, x[i]);
        top *= unit;
        if (__ballot(top > m + M_SLACK)) {
            const float mn = fmaxf(m, row_max(top));
            const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            sum *= f;
#pragma unroll
            for (int t = 0; t < NT; t++) acc[t] *= f;
        }
        const float mb = P_BIAS - (m == -INFINITY ? 0.0f : m);
        Frag p[PARTS];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float v0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * i], unit, mb));
            const float v1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * i + 1], unit, mb));
            if constexpr (PARTS == 2)
                split2(v0, v1, p[0].w[i], p[1].w[i]);
            else
                p[0].w[i] = f16x2{(_Float16)v0, (_Float16)v1};
        }
#pragma unroll
        for (int pp = 0; pp < PARTS; pp++) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones.v, p[pp].v, sum, 0, 0, 0);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            f16x8 vl, vh;
            v_frags<NG>(r, g, magic, vl, vh);
#pragma unroll
            for (int pp = 0; pp < PARTS; pp++) {
                acc[2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, p[pp].v, acc[2 * g], 0, 0, 0);
                acc[2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, p[pp].v, acc[2 * g + 1], 0, 0, 0);
            }
        }
        if (k1 < last) {
            load_vs();
            in0 = p0.in;
            in1 = p1.in;
            places(k1 + NEXT);
        }
        k0 = k1;
    }

    // the waves' parts of the tile
    float *ml = lds + WAVES * TR * OS;
    if (h == 0) {
        ml[(wave * TR + c) * 2] = m;
        ml[(wave * TR + c) * 2 + 1] = sum[0];
    }
#pragma unroll
    for (int t = 0; t < NT; t++) *(f32x4 *)(lds + (wave * TR + c) * OS + 16 * t + 4 * h) = acc[t];
    __syncthreads();
    // row er of the tile: 16 threads, 4 values at a time
    const int er = threadIdx.x >> 4, u = threadIdx.x & 15;
    float f[WAVES], mm = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; w++) mm = fmaxf(mm, ml[(w * TR + er) * 2]);
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        const float mw = ml[(w * TR + er) * 2];
        f[w] = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - mm);
        // (a NaN key leaves a wave's maximum at -inf and its sum NaN)
        const float lw = ml[(w * TR + er) * 2 + 1];
        if (lw != lw) f[w] = lw;
        l += f[w] * lw;
    }
    const int rr = it.tile * TR + er;
    if (rr >= s.n * a.group) return;
    const int rt = rr / a.group, rg = rr - rt * a.group;
    const bool whole = it.pieces == 1;
    if (!whole && (uint32_t)it.part >= (uint32_t)a.few.cut) return;
    float *part = a.few.part + (((int64_t)it.part * a.c.heads + head) * TR + er) * (D + 4);
    const int64_t o = ((int64_t)s.t0 + rt) * a.out_stride + (int64_t)(head * a.group + rg) * D;
    const float inv = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
#pragma unroll
    for (int d = 0; d < D; d += 64) {
        const int e = d + 4 * u;
        if (D % 64 && e >= D) break;
        f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < WAVES; w++) v += f[w] * *(const f32x4 *)(lds + (w * TR + er) * OS + e);
        v *= inv;
        if (whole) {
            store_out(a, o + e, v);
        } else {
            *(f32x4 *)(part + 4 + e) = v;
        }
    }
    if (!whole && u == 0) {
        part[0] = mm;
        part[1] = l;
    }
}

constexpr size_t lds_bytes(int ng) { return (size_t)WAVES * TR * (32 * ng + 4 + 2) * sizeof(float); }

}  // namespace rows16_k
}  // namespace
}  // namespace arfq
