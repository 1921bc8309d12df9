// arfq_attn.h -- what the attention kernels share: the places of a wave's keys, the matrix operands
// made from the cache, and the rows' scaling.  (The work list: arfq_attn_list.h.)
#pragma once
#include <math.h>

#include "arfq_attn_list.h"

namespace arfq {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// p is held as exp2(x - m + P_BIAS), m behind the running maximum by at most M_SLACK: f16 (2^16)
// is not passed, and a part of p keeps its 11 bits down to 2^-27 of the largest p (below, half
// a step is 2^-38 of it).  The slack spares most steps the rescaling of the sums.
constexpr float P_BIAS = 13.0f, M_SLACK = 2.0f;

// Where a 16-key tile is: the (page, head) region (page 0's for a page that is not the cache's: loads stay in
// it, its keys are masked), its place there, and whether its page is the cache's.
struct Place {
    const uint8_t *reg;
    uint32_t sub;
    bool in;
};
// A wave's steps through a sequence, SS tiles apart: lane 2j + i has the place of tile i of step j, for 32 steps at
// a time.  A step takes its two from there: no scalar load (the wait for LDS data is for scalar
// loads too, and these miss the scalar cache), and few scalar instructions.
template <int SS>
struct Steps {
    const int32_t *table;
    int first;  // the tile of lane 0
    uint32_t lo, hi, sub;  // sub: bit 31 where the page is not the cache's
    // through the pages of a table, max_pages of them (k0 a multiple of 16; max_pages > 0)
    __device__ __forceinline__ Steps(const int32_t *table) : table(table), first(INT32_MIN / 2) { lo = hi = sub = 0; }
    // The lane of the step's first tile.
    __device__ __forceinline__ int step(const KvArgs &a, int head, int k0) {
        const int t0 = k0 / KV_TILE, j = (t0 - first) / SS;
        if (j < WAVE / 2) return 2 * j;
        // (past the table's end: of its last page)
        const int lane = threadIdx.x & 63, t = t0 + (lane >> 1) * SS + (lane & 1), pg = kv_page_of(a, t);
        const int id = table[min(pg, a.max_pages - 1)];
        const bool in = (uint32_t)id < (uint32_t)a.n_pages;
        const uint64_t p = (uint64_t)(uint32_t)(in ? id : 0) * a.page_bytes + (uint64_t)head * a.region;
        lo = (uint32_t)p;
        hi = (uint32_t)(p >> 32);
        sub = (uint32_t)(t - pg * a.tiles) | (in ? 0u : 0x80000000u);
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0) here, and not at each use
        first = t0;
        return 0;
    }
    // The tile of lane l.  (An offset, not an address, in the lanes: the loads stay global ones.)
    __device__ __forceinline__ Place at(const KvArgs &a, int l) const {
        const uint32_t s = __builtin_amdgcn_readlane(sub, l);
        return {a.data + ((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, l) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, l)),
                s & 0x7fffffffu, (int32_t)s >= 0};
    }
    __device__ __forceinline__ bool in(int l) const { return __builtin_amdgcn_readlane((int)sub, l) >= 0; }
};

// ---- operands ----------------------------------------------------------------------------

// Two codes + 8 in bits 0..3 (LO) or 4..7 of the halves -> the codes as f16: or-ed into 1024
// (2^10: a unit in the last place is 1) they read 1024 + c, or 1024 + 16 c; the steps that
// follow are exact.  `magic` is that 1024 twice in a vector register, which the compiler does
// not see through: with a literal there it splits v_and_or_b32 into two instructions.
__device__ __forceinline__ uint32_t magic_1024() {
    uint32_t m;
    asm("v_mov_b32 %0, 0x64006400" : "=v"(m));
    return m;
}
template <bool LO>
__device__ __forceinline__ f16x2 codes_f16(uint32_t w, uint32_t magic) {
    const f16x2 h = __builtin_bit_cast(f16x2, (w & (LO ? 0x000f000fu : 0x00f000f0u)) | magic);
    if constexpr (LO) return h - f16x2{(_Float16)1032, (_Float16)1032};
    return h * f16x2{(_Float16)0.0625f, (_Float16)0.0625f} - f16x2{(_Float16)72, (_Float16)72};
}

union Frag {
    f16x2 w[4];
    f16x8 v;
};

// v0 and v1 as two f16 parts each: hi rounded, lo what is left (one rounding each: v - hi is formed in f32
// on the way into lo's half).
__device__ __forceinline__ void split2(float v0, float v1, f16x2 &hi, f16x2 &lo) {
    hi = f16x2{(_Float16)v0, (_Float16)v1};
    asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(lo) : "v"(hi), "v"(v0));
    asm("v_fma_mixhi_f16 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(lo) : "v"(hi), "v"(v1));
}

// What a lane of the step's 32 keys loads: K of two 16-key tiles (key lane % 16, chunk lane / 16)
// and V of the keys 4 * (lane / 16) .. +3 of both (matrix rows lane % 16).
template <int NG>
struct Raw {
    uint32_t k[2][NG], v[2][NG];
    uint32_t ks[2][2 * NG];              // of keys 4 * (lane / 16) .. +3: [4][NG] f16
    uint32_t vs[2][2 * NG];              // of the same, in pairs: [NG][2]
};

// N dwords at an address that is a multiple of A bytes.
template <int N, int A>
__device__ __forceinline__ void load_aligned(const void *p, uint32_t (&o)[N]) {
    static_assert(A == 4 || A == 8 || A == 16, "");
    if constexpr (A == 16 && N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const u32x4 v = ((const u32x4 *)p)[i];
            o[4 * i] = v.x; o[4 * i + 1] = v.y; o[4 * i + 2] = v.z; o[4 * i + 3] = v.w;
        }
    } else if constexpr (A >= 8 && N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const u32x2 v = ((const u32x2 *)p)[i];
            o[2 * i] = v.x; o[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = ((const uint32_t *)p)[i];
    }
}

// Byte offsets of a lane's operands in a 16-key tile (from the region, its V codes, scales and V scales).
template <int NG>
struct Offs {
    uint32_t k, v, s;
};
template <int NG>
__device__ __forceinline__ Offs<NG> lane_offs() {
    const uint32_t lane = threadIdx.x & 63, c = lane & 15, h = lane >> 4;
    return {c * (16 * NG) + h * (4 * NG), h * (64 * NG) + c * (4 * NG), h * (8 * NG)};
}
// p + o with p uniform: hidden from the compiler, which would widen o once and keep it in two registers
// instead of the loads' scalar base and 32-bit offset.
__device__ __forceinline__ const uint8_t *at(const uint8_t *p, uint32_t o) {
    asm("" : "+v"(o));
    return p + o;
}
// reg (uniform): the tile's (page, head) region; sub: the 16-key tile within the page
template <int NG>
__device__ __forceinline__ void load_k(const uint8_t *reg, const KvArgs &a, uint32_t sub, int half, const Offs<NG> &o, Raw<NG> &r) {
    constexpr int AL = NG % 4 == 0 ? 16 : NG % 2 == 0 ? 8 : 4;
    load_aligned<NG, AL>(at(reg + sub * (256u * NG), o.k), r.k[half]);
    load_aligned<2 * NG, 8>(at(reg + (a.off_ks + sub * (32u * NG)), o.s), r.ks[half]);
}
template <int NG>
__device__ __forceinline__ void load_v(const uint8_t *reg, const KvArgs &a, uint32_t sub, int half, const Offs<NG> &o, Raw<NG> &r) {
    constexpr int AL = NG % 4 == 0 ? 16 : NG % 2 == 0 ? 8 : 4;
    load_aligned<NG, AL>(at(reg + (a.off_v + sub * (256u * NG)), o.v), r.v[half]);
    load_aligned<2 * NG, 8>(at(reg + (a.off_vs + sub * (32u * NG)), o.s), r.vs[half]);
}

// The f16 in half i of w.
__device__ __forceinline__ _Float16 half_of(uint32_t w, int i) {
    return __builtin_bit_cast(_Float16, (unsigned short)(i ? w >> 16 : w));
}

// MFMA operand of group g of the K tile: eight codes of one key.
template <int NG>
__device__ __forceinline__ f16x8 k_frag(const Raw<NG> &r, int half, int g, uint32_t magic) {
    const uint32_t w = r.k[half][g], w8 = w >> 8;
    Frag f;
    f.w[0] = codes_f16<true>(w, magic);
    f.w[1] = codes_f16<false>(w, magic);
    f.w[2] = codes_f16<true>(w8, magic);
    f.w[3] = codes_f16<false>(w8, magic);
    return f.v;
}

// V's bytes of group g of keys 2 pr and 2 pr + 1 of a four-key block (NG dwords: [4][NG] bytes), one in each half.
template <int NG>
__device__ __forceinline__ uint32_t pair_bytes(const uint32_t (&v)[NG], int pr, int g) {
    const int b0 = 2 * pr * NG + g, b1 = b0 + NG;
    const uint32_t sel = 0x0c000c00u | (uint32_t)((b1 & 3) + 4) << 16 | (uint32_t)(b0 & 3);
    return __builtin_amdgcn_perm(v[b1 >> 2], v[b0 >> 2], sel);
}
// MFMA operands of group g of the V tile: eight keys of the values 32g + lane % 16 (lo) and
// 32g + 16 + lane % 16 (hi).
template <int NG>
__device__ __forceinline__ void v_frags(const Raw<NG> &r, int g, uint32_t magic, f16x8 &lo, f16x8 &hi) {
    Frag l, h;
#pragma unroll
    for (int half = 0; half < 2; half++)
#pragma unroll
        for (int pr = 0; pr < 2; pr++) {
            const uint32_t t = pair_bytes<NG>(r.v[half], pr, g);
            const f16x2 d = __builtin_bit_cast(f16x2, r.vs[half][2 * g + pr]);
            l.w[2 * half + pr] = codes_f16<true>(t, magic) * d;
            h.w[2 * half + pr] = codes_f16<false>(t, magic) * d;
        }
    lo = l.v;
    hi = h.v;
}

// tanh to 2^-22 of its range: (1 - t) / (1 + t) with t = exp(-2 |v|), and its series below 1/4
// (the next term is 2^-27 of the value there), where 1 - t loses bits.
__device__ __forceinline__ float tanh_of(float v) {
    const float t = __builtin_amdgcn_exp2f(fabsf(v) * -2.8853900817779268f);
    const float w = v * v;
    const float s = v + v * w * (-1.0f / 3 + w * (2.0f / 15 + w * (-17.0f / 315 + w * (62.0f / 2835))));
    return fabsf(v) < 0.25f ? s : copysignf((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t), v);
}

// A power of two that puts a row's largest |q| into [2^14, 2^15), where two f16 parts hold 22 bits of it,
// with the sign of `scale` (the scores' sign goes into q: larger products, larger scores), and its inverse.
struct RowScale {
    float up, down;
};
__device__ __forceinline__ RowScale row_scale(float top, float scale) {
    const int ex = min(max(top > 0.0f ? 141 - (int)(__builtin_bit_cast(uint32_t, top) >> 23) : 0, -126), 126);
    return {__builtin_bit_cast(float, (uint32_t)(ex + 127) << 23) * (scale < 0.0f ? -1.0f : 1.0f),
            __builtin_bit_cast(float, (uint32_t)(127 - ex) << 23)};
}

// What a row's products t of q and K are multiplied by: t * this is a score's log2, or tanh's argument where there
// is a cap (below 2^64).  sc: a product's score.  Not below the smallest normal number (a masked score is -inf, and
// -inf * 0 would be NaN): |t| is below 2^40, so what that makes of smaller scores stays below 2^-22.  Nor
// beyond the largest (0 * inf).
__device__ __forceinline__ float score_unit(float sc, float cap) {
    return fminf(fmaxf(cap > 0.0f ? sc / cap : sc * 1.4426950408889634f, 1.1754944e-38f), 3.4028235e38f);
}

__device__ __forceinline__ float row_max(float v) {  // over the lanes of one matrix column
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

// Eight values of q from element i on (zeros where !on).
__device__ __forceinline__ void load8_q(const AttnArgs &a, int64_t i, bool on, float (&o)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) o[e] = 0.0f;
    if (!on) return;
    if (a.q_dtype == ARFQ_F16) {
        const f16x8 v = *(const f16x8 *)((const _Float16 *)a.q + i);
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (float)v[e];
    } else {
        const f32x4 v = *(const f32x4 *)((const float *)a.q + i), w = *(const f32x4 *)((const float *)a.q + i + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            o[e] = v[e];
            o[4 + e] = w[e];
        }
    }
}

__device__ __forceinline__ void store_out(const AttnArgs &a, int64_t i, f32x4 v) {
    if (a.out_dtype == ARFQ_F16)
        *(u32x2 *)((_Float16 *)a.out + i) = u32x2{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])};
    else
        *(f32x4 *)((float *)a.out + i) = v;
}

}  // namespace
}  // namespace arfq
