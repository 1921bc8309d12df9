// arfq_attn_rows128.h -- attention for prompts: tiles of 128 rows.
//
// A workgroup's four waves take 32 rows each and step through the keys together, 32 at a time: they
// turn K and V of a step into f16 once, in LDS (two waves K's, two V's tiles), and every wave multiplies
// all of it.  As in the kernel of few rows, S^T = K Q^T and O^T = V^T P^T (v_mfma_f32_32x32x16_f16): a
// row is a lane's column throughout, so its maximum and sum are registers, and the scores' registers
// 8b .. 8b + 7 are, as they lie, the second product's operand for keys
//     16b + 4h + {0, 1, 2, 3} and 16b + 8 + 4h + {0, 1, 2, 3}      (h = lane / 32),
// the order in which V goes to LDS.
//
// Bound by the matrix cores and the softmax beside them, two waves a SIMD (the accumulators and q take 128 registers
// of 256 at D = 128 and one part, 192 at two; 6 go to scratch).  Measured at 40 x 128 q heads on 8: 8192 tokens of f16
// 776 us (885 TFLOP/s of the 1131 that a plain f16 product reaches), 2048 tokens 72 (597; its longest tile's
// 64 steps one after another take 60, as none of more tiles than workgroups is cut); 512 f32 tokens after 32356 others
// 622 to 656 (550 to 521, twice that of f16 products, as f32's two parts double them; matrix cores and vector unit busy
// half the time each).  f16 24 x 96 on 8, seven prompts of up to 777 tokens: 51 to 58 (380 to 335): 47 steps of the longest
// tile.  With a cap of scores 2048 tokens take 111, with a window of 512 57, with both 76.
#pragma once
#include <type_traits>

#include "arfq_attn.h"

namespace arfq {
namespace {
namespace rows128_k {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int TR = 128, WR = 32;  // rows of a tile, of a wave
constexpr int WAVES = TR / WR, THREADS = 64 * WAVES;

// LDS of a step: K [32][D + 8] f16 (rows 16 bytes apart in the banks), V [4][D][8] f16: lane
// half and key block, value, keys.
template <int NG>
struct Step {
    static constexpr int D = 32 * NG, KS = D + 8;
    static constexpr int K_BYTES = STEP * KS * 2, V_BYTES = STEP * D * 2;
};

// What a lane turns into f16: a wave has K or V of one of the step's two 16-key tiles, 64 units of NG
// dwords.  K: chunk lane % 4 of key lane / 4, and the key's scales; V: matrix row lane % 16 of the four
// keys lane / 16, and their scales in pairs.
template <int NG>
struct Part {
    uint32_t x[NG], s[2 * NG];
};

// block: (item, head), head fastest.
template <int NG, int PARTS>
__device__ __forceinline__ void rows128(const AttnArgs &a, int block, uint8_t *lds) {
    constexpr int D = 32 * NG, KS = Step<NG>::KS;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), c = lane & 31, h = lane >> 5;
    const int head = block % a.c.heads;
    Item it;
    if (!take_item<TR>(a, block, it)) return;
    const Seq &s = it.s;

    auto row_hi = [&](int64_t pos) { return pos < 0 ? 0 : a.causal ? (int)min(pos + 1, (int64_t)s.end) : s.end; };
    auto row_lo = [&](int64_t pos) { return a.window ? (int)max((int64_t)0, min(pos - a.window + 1, (int64_t)s.end)) : 0; };
    const int rows = s.n * a.group, piece_lo = s.lo + it.piece * it.keys, piece_hi = min(s.end, piece_lo + it.keys);
    auto pos_of = [&](int row) { return (int64_t)s.len - s.n + min(row, rows - 1) / a.group; };
    // keys of the tile in this piece, and those that every row of the wave has
    const int first = max(row_lo(pos_of(it.tile * TR)) & ~(STEP - 1), piece_lo);
    const int last = min(row_hi(pos_of(it.tile * TR + TR - 1)), piece_hi);
    const int row0 = it.tile * TR + wave * WR;
    const int64_t pos0 = pos_of(row0), pos1 = pos_of(row0 + WR - 1);
    const int inner_lo = row_lo(pos1), inner_hi = min(row_hi(pos0), piece_hi);
    const int row = row0 + c;
    const bool valid = row < rows;
    const int tok = valid ? row / a.group : 0, gh = valid ? row - tok * a.group : 0;
    const int64_t pos = (int64_t)s.len - s.n + tok;
    const int lo = row_lo(pos), hi = min(valid ? row_hi(pos) : 0, piece_hi);

    // ---- a step's K and V: from the cache to registers, and to LDS as f16 ----
    Steps<STEP / KV_TILE> steps(a.c.table + (int64_t)it.b * a.c.max_pages);
    const int half = wave >> 1;  // the wave's tile
    const bool is_v = wave & 1;
    const uint32_t x_off = lane * (4 * NG), s_off = is_v ? (lane >> 4) * (8 * NG) : (lane >> 2) * (2 * NG);
    constexpr int AL = NG % 4 == 0 ? 16 : NG % 2 == 0 ? 8 : 4;
    const uint32_t x_at = is_v ? a.c.off_v : 0, s_at = is_v ? a.c.off_vs : a.c.off_ks;
    // keys k0 .. of the wave's tile into registers (past the last: some of the cache's, unused; no branch, so that
    // a wait for one part leaves the next one's loads in flight); whether the step's tiles are the cache's, in
    // the lowest bits of `in`
    constexpr int AHEAD = PARTS == 1 ? 2 : 1;  // parts in flight
    Part<NG> parts[AHEAD];
    uint32_t in = 0;
    auto load = [&](auto v, Part<NG> &part, int k0) __attribute__((always_inline)) {
        const int l = steps.step(a.c, head, k0);
        in = in << 2 | (steps.in(l) ? 1u : 0u) | (steps.in(l + 1) ? 2u : 0u);
        const Place pl = steps.at(a.c, l + half);
        const uint8_t *x = at(pl.reg + (x_at + pl.sub * (256u * NG)), x_off);
        const uint8_t *sc = at(pl.reg + (s_at + pl.sub * (32u * NG)), s_off);
        load_aligned<NG, AL>(x, part.x);
        if constexpr (v) {
            load_aligned<2 * NG, 8>(sc, part.s);
        } else if constexpr (NG % 2) {
#pragma unroll
            for (int g = 0; g < NG; g++) part.s[g] = ((const uint16_t *)sc)[g];
        } else {
            uint32_t w[NG / 2];
            load_aligned<NG / 2, NG % 8 == 0 ? 16 : NG % 4 == 0 ? 8 : 4>(sc, w);
#pragma unroll
            for (int g = 0; g < NG / 2; g++) part.s[g] = w[g];
        }
        asm volatile("");  // (or the stores of K's and V's branch are made one, to memory)
    };
    const uint32_t magic = magic_1024();
    // (K's rows; V's (key block, half of a lane's eight keys) and matrix row)
    const uint32_t to = is_v ? ((half * 2 + ((lane >> 4) & 1)) * D + (lane & 15)) * 16 + (lane >> 5) * 8
                             : (half * 16 + (lane >> 2)) * (KS * 2) + (lane & 3) * 16;
    auto store = [&](auto v, const Part<NG> &part, uint8_t *buf) __attribute__((always_inline)) {
        uint8_t *o = buf + to;
        if constexpr (v) {
#pragma unroll
            for (int g = 0; g < NG; g++) {
                f16x2 l[2], u[2];
#pragma unroll
                for (int pr = 0; pr < 2; pr++) {
                    const uint32_t w = pair_bytes<NG>(part.x, pr, g);
                    const f16x2 d = __builtin_bit_cast(f16x2, part.s[2 * g + pr]);
                    l[pr] = codes_f16<true>(w, magic) * d;
                    u[pr] = codes_f16<false>(w, magic) * d;
                }
                *(u32x2 *)(o + g * 512) = u32x2{__builtin_bit_cast(uint32_t, l[0]), __builtin_bit_cast(uint32_t, l[1])};
                *(u32x2 *)(o + g * 512 + 256) = u32x2{__builtin_bit_cast(uint32_t, u[0]), __builtin_bit_cast(uint32_t, u[1])};
            }
        } else {
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const uint32_t w = part.x[g], w8 = w >> 8, d2 = part.s[NG % 2 ? g : g / 2];
                const f16x2 d = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(d2, d2, NG % 2 || g % 2 == 0 ? 0x01000100u : 0x03020302u));
                Frag f;
                f.w[0] = codes_f16<true>(w, magic) * d;
                f.w[1] = codes_f16<false>(w, magic) * d;
                f.w[2] = codes_f16<true>(w8, magic) * d;
                f.w[3] = codes_f16<false>(w8, magic) * d;
                *(f16x8 *)(o + g * 64) = f.v;
            }
        }
    };
    constexpr std::true_type V{};
    constexpr std::false_type K{};
    Part<NG> &part0 = parts[0];
    if (first < last) {
        if (is_v)
            load(V, part0, first);
        else
            load(K, part0, first);
    }

    // ---- q as operands, values 16i + 8h .. +7 of the row, scaled as in the kernel of few rows ----
    f16x8 q[PARTS][2 * NG];
    float sc = fabsf(a.scale);
    {
        float top = 0.0f;
        const int64_t qo = ((int64_t)s.t0 + tok) * a.q_stride + (int64_t)(head * a.group + gh) * D + 8 * h;
        float x[8];
        if constexpr (PARTS == 2) {
#pragma unroll
            for (int i = 0; i < 2 * NG; i++) {
                load8_q(a, qo + 16 * i, valid, x);
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[e]));
            }
            top = fmaxf(top, __shfl_xor(top, 32));
        }
        const RowScale rs = row_scale(PARTS == 2 ? top : 0.0f, a.scale);
        sc *= rs.down;
#pragma unroll
        for (int i = 0; i < 2 * NG; i++) {
            load8_q(a, qo + 16 * i, valid, x);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = x[e] * rs.up;
                const _Float16 f = (_Float16)v;
                q[0][i][e] = f;
                if constexpr (PARTS == 2) q[1][i][e] = (_Float16)(v - (float)f);
            }
        }
    }
    const float cap = a.softcap;
    const float x_of_s = score_unit(sc, cap), x_of_t = cap * 1.4426950408889634f;

    f32x16 acc[NG];
    const f32x16 zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < NG; i++) acc[i] = zero;
    float m = -INFINITY, sum = 0.0f;

    // K's step is one ahead of V's: while the softmax of step i is computed, its p entering V's products, the
    // matrix cores multiply K of step i + 1, and in the shadow of V's products the wave turns its
    // part of the step after into operands.  LDS: K of two steps, V of two.
    uint8_t *const kb = lds, *const vb = lds + 2 * Step<NG>::K_BYTES;
    auto scores = [&](const uint8_t *b, f32x16 &x) __attribute__((always_inline)) {
        f16x8 kf[2 * NG];
#pragma unroll
        for (int i = 0; i < 2 * NG; i++) kf[i] = *(const f16x8 *)(b + c * (KS * 2) + (2 * i + h) * 16);
        x = zero;
#pragma unroll
        for (int i = 0; i < 2 * NG; i++)
#pragma unroll
            for (int p = 0; p < PARTS; p++) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i], q[p][i], x, 0, 0, 0);
    };
    f32x16 x = zero;
    auto step = [&](auto v, int k0, int odd) __attribute__((always_inline)) {
        const uint32_t was = in >> 2 * (AHEAD + (v ? 0 : 1));  // (of this step: as many loads ago)
        float unit = x_of_s;
        if (cap > 0.0f) {
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = tanh_of(x[i] * x_of_s) * x_of_t;
            unit = 1.0f;
        }
        if (k0 < inner_lo || k0 + STEP > inner_hi || (was & 3) != 3) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint32_t from = (uint32_t)(k0 + u * 16 + 4 * h - lo), width = (was >> u & 1) ? (uint32_t)max(hi - lo, 0) : 0u;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int at = (i >> 2) * 8 + (i & 3);
                    x[8 * u + i] = from + at < width ? x[8 * u + i] : -INFINITY;
                }
            }
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 16; i++) top = fmaxf(top, x[i]);
        top *= unit;
        if (__ballot(top > m + M_SLACK)) {
            const float mn = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
            const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            sum *= f;
#pragma unroll
            for (int i = 0; i < NG; i++) acc[i] *= f;
        }
        const float mb = P_BIAS - (m == -INFINITY ? 0.0f : m);
        f32x16 y;
        // (past the last step: of what lies there, unused)
        if constexpr (PARTS == 1) scores(kb + (odd ^ 1) * Step<NG>::K_BYTES, y);
        f16x8 vf[2][NG];
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int i = 0; i < NG; i++) vf[b][i] = *(const f16x8 *)(vb + odd * Step<NG>::V_BYTES + ((b * 2 + h) * D + 32 * i + c) * 16);
        Frag p[2][PARTS];
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float v0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * b + 2 * i], unit, mb));
                const float v1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * b + 2 * i + 1], unit, mb));
                if constexpr (PARTS == 2) {
                    split2(v0, v1, p[b][0].w[i], p[b][1].w[i]);
                    sum += v0 + v1;
                } else {
                    // (what the values are multiplied with: a rounding of p then moves both alike)
                    const f16x2 f = {(_Float16)v0, (_Float16)v1};
                    p[b][0].w[i] = f;
                    sum = __builtin_amdgcn_fdot2(f, f16x2{(_Float16)1, (_Float16)1}, sum, false);
                }
            }
        // (the products of a wave that has them ahead go first, the other wave's softmax falls beside them: 634 us
        // down to 624 at 512 tokens of 32868, f32; with one part, where a wave overlaps its own, no gain)
        if constexpr (PARTS == 2) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int i = 0; i < NG; i++)
#pragma unroll
                for (int pp = 0; pp < PARTS; pp++)
                    acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[b][i], p[b][pp].v, acc[i], 0, 0, 0);
        if constexpr (PARTS == 2) {  // (no registers for both steps' scores)
            __builtin_amdgcn_sched_barrier(0);
            scores(kb + (odd ^ 1) * Step<NG>::K_BYTES, y);
        }
        Part<NG> &part = parts[odd % AHEAD];
        store(v, part, v ? vb + (odd ^ 1) * Step<NG>::V_BYTES : kb + odd * Step<NG>::K_BYTES);  // (past the last step: to where nothing is read)
        if constexpr (PARTS == 2) __builtin_amdgcn_s_setprio(0);
        x = y;
        load(v, part, k0 + ((v ? 1 : 2) + AHEAD) * STEP);
        lds_barrier();
    };
    auto loop = [&](auto v) __attribute__((always_inline)) {
        store(v, part0, v ? vb : kb);
        load(v, part0, first + STEP);
        if constexpr (!v) {
            store(v, part0, kb + Step<NG>::K_BYTES);
            load(v, part0, first + 2 * STEP);
        }
        if constexpr (AHEAD == 2) load(v, parts[1], first + (v ? 2 : 3) * STEP);
        lds_barrier();
        scores(kb, x);
        lds_barrier();
        for (int k0 = first; k0 < last; k0 += 2 * STEP) {
            step(v, k0, 0);
            step(v, k0 + STEP, 1);  // (without a branch, as the loads are; past the last: every key masked)
        }
    };
    if (first < last) {
        if (is_v)
            loop(V);
        else
            loop(K);
    }

    sum += __shfl_xor(sum, 32);
    if (!valid) return;
    const int64_t o = ((int64_t)s.t0 + tok) * a.out_stride + (int64_t)(head * a.group + gh) * D;
    const bool whole = it.pieces == 1;
    if (!whole && (uint32_t)it.part >= (uint32_t)a.many.cut) return;
    float *dst = a.many.part + (((int64_t)it.part * a.c.heads + head) * TR + wave * WR + c) * (D + 4);
    const float inv = whole ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
#pragma unroll
    for (int i = 0; i < NG; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            f32x4 v = {acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]};
            const int e = 32 * i + 8 * j + 4 * h;
            if (whole)
                store_out(a, o + e, v * inv);
            else
                *(f32x4 *)(dst + 4 + e) = v;
        }
    if (!whole && h == 0) *(float2 *)dst = make_float2(m, sum);
}

constexpr size_t lds_bytes(int ng) { return 2 * (size_t)STEP * ((32 * ng + 8) + 32 * ng) * 2; }

}  // namespace rows128_k
}  // namespace
}  // namespace arfq
