// arfq_attn.hip -- attention over the 4-bit K/V cache.
#include <math.h>

#include <algorithm>

#include "arfq_kv.h"

namespace arfq {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int TR = 16;        // rows of a tile: (token, head of the group) pairs, head fastest
constexpr int STEP = 32;      // keys of a step
constexpr int WAVES = 4;
constexpr int MIN_PIECE = 256;  // keys
// p is held as exp2(x - m + P_BIAS), m behind the running maximum by at most M_SLACK: f16 (2^16)
// is not passed, and a part of p keeps its 11 bits down to 2^-27 of the largest p (below, half
// a step is 2^-38 of it).  The slack spares most steps the rescaling of the sums.
constexpr float P_BIAS = 13.0f, M_SLACK = 2.0f;

// ---- the work list -----------------------------------------------------------------------
// A sequence with n tokens has ceil(n * group / 16) row tiles, and its keys [lo, end) are cut
// into pieces; a work item is a (tile, piece).  The piece length is what cuts the whole batch's
// (tile, key) area into about `target` pieces, so that a long sequence is spread over the chip
// whatever its neighbours are: decided here, from the lengths, which are on the device.

struct Seq {
    int t0, n, len;
    int lo, end;  // keys that some row may attend to; lo is a multiple of STEP
    int tiles;
};

__device__ __forceinline__ Seq seq_of(const AttnArgs &a, int b) {
    Seq s = {0, 0, 0, 0, 0, 0};
    if (b >= a.c.batch) return s;
    kv_seq(a.c, b, s.t0, s.n);
    s.len = a.c.len[b];
    s.end = (int)min((int64_t)max(s.len, 0), a.c.max_pages * a.c.page);
    if (a.window) s.lo = (int)max((int64_t)0, min((int64_t)s.len - s.n - a.window + 1, (int64_t)s.end)) & ~(STEP - 1);
    s.tiles = (int)(((int64_t)s.n * a.group + TR - 1) / TR);
    return s;
}

__device__ __forceinline__ int64_t wave_sum(int64_t v) {
#pragma unroll
    for (int x = 1; x < WAVE; x <<= 1) v += __shfl_xor(v, x);
    return v;
}

__device__ __forceinline__ int pieces_of(const Seq &s, int piece) {
    return max(1, (s.end - s.lo + piece - 1) / piece);
}

// Keys of a piece (a multiple of STEP), the same in every wave of the launch.
__device__ __forceinline__ int piece_len(const AttnArgs &a) {
    const int lane = threadIdx.x & 63;
    int64_t area = 0;
    for (int b0 = 0; b0 < a.c.batch; b0 += WAVE) {
        const Seq s = seq_of(a, b0 + lane);
        area += (int64_t)s.tiles * (s.end - s.lo);
    }
    area = wave_sum(area);
    const int64_t piece = ((area + a.target - 1) / a.target + STEP - 1) / STEP * STEP;
    return (int)min((int64_t)KV_KEYS_MAX, max((int64_t)MIN_PIECE, piece));
}

struct Item {
    Seq s;
    int b, tile, piece, pieces;
    int first;  // index of the (tile's) first piece in the list
};

// The `index`-th (tile, piece) of the batch, tiles of a sequence one after another, pieces
// fastest (PIECES false: the index-th tile, with the index of its first piece).  False: the
// list has fewer.
template <bool PIECES>
__device__ __forceinline__ bool find_item(const AttnArgs &a, int piece, int64_t index, Item &it) {
    const int lane = threadIdx.x & 63;
    int64_t before = 0, items = 0;
    for (int b0 = 0; b0 < a.c.batch; b0 += WAVE) {
        const Seq s = seq_of(a, b0 + lane);
        const int np = pieces_of(s, piece);
        const int64_t own = PIECES ? (int64_t)s.tiles * np : s.tiles, work = (int64_t)s.tiles * np;
        int64_t inc = own, winc = work;
#pragma unroll
        for (int x = 1; x < WAVE; x <<= 1) {
            const int64_t v = __shfl_up(inc, x), w = __shfl_up(winc, x);
            if (lane >= x) {
                inc += v;
                winc += w;
            }
        }
        const uint64_t past = __ballot(before + inc > index);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            it.s.t0 = __builtin_amdgcn_readlane(s.t0, l);
            it.s.n = __builtin_amdgcn_readlane(s.n, l);
            it.s.len = __builtin_amdgcn_readlane(s.len, l);
            it.s.lo = __builtin_amdgcn_readlane(s.lo, l);
            it.s.end = __builtin_amdgcn_readlane(s.end, l);
            it.s.tiles = __builtin_amdgcn_readlane(s.tiles, l);
            it.pieces = __builtin_amdgcn_readlane(np, l);
            it.b = b0 + l;
            const int rest = __builtin_amdgcn_readlane((int)(index - before - (inc - own)), l);
            const int64_t base = items + __shfl(winc - work, l);
            it.tile = PIECES ? rest / it.pieces : rest;
            it.piece = PIECES ? rest - it.tile * it.pieces : 0;
            it.first = (int)min((int64_t)INT32_MAX, base + (int64_t)it.tile * it.pieces);
            return true;
        }
        before += __shfl(inc, 63);
        items += __shfl(winc, 63);
    }
    return false;
}

// ---- operands ----------------------------------------------------------------------------

__device__ __forceinline__ uint32_t pk_mul(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, a) * __builtin_bit_cast(f16x2, b));
}
// Two codes + 8 in bits 0..3 (LO) or 4..7 of the halves -> the codes as f16: or-ed into 1024
// (2^10: a unit in the last place is 1) they read 1024 + c, or 1024 + 16 c; both steps are exact.
template <bool LO>
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
    const f16x2 h = __builtin_bit_cast(f16x2, (w & (LO ? 0x000f000fu : 0x00f000f0u)) | 0x64006400u);
    if constexpr (LO) return __builtin_bit_cast(uint32_t, h - f16x2{(_Float16)1032, (_Float16)1032});
    const f16x2 r = h * f16x2{(_Float16)0.0625f, (_Float16)0.0625f} - f16x2{(_Float16)72, (_Float16)72};
    return __builtin_bit_cast(uint32_t, r);
}

union Frag {
    uint32_t w[4];
    f16x8 v;
};

// What a lane of the step's 32 keys loads: K of two 16-key tiles (key lane % 16, chunk lane / 16)
// and V of the keys 4 * (lane / 16) .. +3 of both (matrix rows lane % 16).
template <int NG>
struct Raw {
    uint32_t k[2][NG], v[2][NG];
    uint32_t vs[2][2 * NG];  // pairs of keys: [NG][2]
    uint16_t ks[2][NG];
};

template <int N>
__device__ __forceinline__ void load_dwords(const void *p, uint32_t (&o)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = ((const uint32_t *)p)[i];
}

// The same for N dwords whose address is a multiple of A bytes.
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
        load_dwords(p, o);
    }
}

template <int NG>
__device__ __forceinline__ void load_tile(const uint8_t *reg, const KvArgs &a, int sub, int half, Raw<NG> &r) {
    constexpr int AL = NG % 4 == 0 ? 16 : NG % 2 == 0 ? 8 : 4;
    const int lane = threadIdx.x & 63, c = lane & 15, h = lane >> 4;
    // (sub: the 16-key tile within the page)
    load_aligned<NG, AL>(reg + (sub * 16 + c) * (16 * NG) + h * (4 * NG), r.k[half]);
    load_aligned<NG, AL>(reg + a.off_v + (sub * 4 + h) * (64 * NG) + c * (4 * NG), r.v[half]);
    load_aligned<2 * NG, 8>(reg + a.off_vs + (sub * 4 + h) * (8 * NG), r.vs[half]);
    const uint16_t *ks = (const uint16_t *)(reg + a.off_ks) + (sub * 16 + c) * NG;
    if constexpr (NG % 2 == 0) {
        uint32_t w[NG / 2];
        load_aligned<NG / 2, NG % 8 == 0 ? 16 : NG % 4 == 0 ? 8 : 4>(ks, w);
#pragma unroll
        for (int g = 0; g < NG; g++) r.ks[half][g] = (uint16_t)(w[g / 2] >> (16 * (g & 1)));
    } else {
#pragma unroll
        for (int g = 0; g < NG; g++) r.ks[half][g] = ks[g];
    }
}

// MFMA operand of group g of the K tile: eight values of one key.
template <int NG>
__device__ __forceinline__ f16x8 k_frag(const Raw<NG> &r, int half, int g) {
    const uint32_t w = r.k[half][g], w8 = w >> 8, d = r.ks[half][g] * 0x10001u;
    Frag f;
    f.w[0] = pk_mul(codes_f16<true>(w), d);
    f.w[1] = pk_mul(codes_f16<false>(w), d);
    f.w[2] = pk_mul(codes_f16<true>(w8), d);
    f.w[3] = pk_mul(codes_f16<false>(w8), d);
    return f.v;
}

// MFMA operands of group g of the V tile: eight keys of the values 32g + lane % 16 (lo) and
// 32g + 16 + lane % 16 (hi).
template <int NG>
__device__ __forceinline__ void v_frags(const Raw<NG> &r, int g, f16x8 &lo, f16x8 &hi) {
    Frag l, h;
#pragma unroll
    for (int half = 0; half < 2; half++)
#pragma unroll
        for (int pr = 0; pr < 2; pr++) {
            // bytes g of keys 2 pr and 2 pr + 1: one into each half
            const int b0 = 2 * pr * NG + g, b1 = b0 + NG;
            const uint32_t sel = 0x0c000c00u | (uint32_t)((b1 & 3) + 4) << 16 | (uint32_t)(b0 & 3);
            const uint32_t t = __builtin_amdgcn_perm(r.v[half][b1 >> 2], r.v[half][b0 >> 2], sel);
            const uint32_t d = r.vs[half][2 * g + pr];
            l.w[2 * half + pr] = pk_mul(codes_f16<true>(t), d);
            h.w[2 * half + pr] = pk_mul(codes_f16<false>(t), d);
        }
    lo = l.v;
    hi = h.v;
}

__device__ __forceinline__ float row_max(float v) {  // over the lanes of one matrix column
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ float q_at(const AttnArgs &a, int64_t i) {
    return a.q_dtype == ARFQ_F16 ? (float)((const _Float16 *)a.q)[i] : ((const float *)a.q)[i];
}

__device__ __forceinline__ void store_out(const AttnArgs &a, int64_t i, f32x4 v) {
    if (a.out_dtype == ARFQ_F16)
        *(u32x2 *)((_Float16 *)a.out + i) = u32x2{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])};
    else
        *(f32x4 *)((float *)a.out + i) = v;
}

// ---- rows of 16, keys spread over the waves ------------------------------------------------
// S^T = K Q^T, O^T = V^T P^T with v_mfma_f32_16x16x32_f16: the 16 rows are matrix columns, so a
// lane's four results of a tile belong to one row, its statistics are a register, and P^T in
// the layout of a result is the layout of the next product's operand (which keys a lane's
// eight slots stand for is free, as V is loaded to match).
// PARTS: f16 parts of q and p (2: hi + lo, 22 bits, for f32 q or out).
template <int NG, int PARTS>
__global__ __launch_bounds__(64 * WAVES) void attn_rows16(AttnArgs a) {
    constexpr int D = 32 * NG, NT = 2 * NG;  // NT: 16-row tiles of O^T
    constexpr int OS = D + 4;                // LDS floats of a row of O
    extern __shared__ float lds[];           // [WAVES][16][OS], then [WAVES][16][2]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, h = lane >> 4;
    const int head = blockIdx.y;
    const int piece = piece_len(a);
    Item it;
    if (!find_item<true>(a, piece, blockIdx.x, it)) return;
    const Seq &s = it.s;

    // this lane's row
    const int row = it.tile * TR + c;
    const bool valid = row < s.n * a.group;
    const int tok = valid ? row / a.group : 0, gh = valid ? row - tok * a.group : 0;
    const int64_t pos = (int64_t)s.len - s.n + tok;
    int hi = valid && pos >= 0 ? (a.causal ? (int)min(pos + 1, (int64_t)s.end) : s.end) : 0;
    int lo = a.window ? (int)max((int64_t)0, min(pos - a.window + 1, (int64_t)INT32_MAX)) : 0;
    hi = min(hi, min(s.end, s.lo + (it.piece + 1) * piece));
    // the tile's keys in this piece, and those that every row has
    int first = valid && lo < hi ? lo : INT32_MAX, last = valid && lo < hi ? hi : 0, inner_lo = valid ? lo : 0,
        inner_hi = valid ? hi : INT32_MAX;
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) {
        first = min(first, __shfl_xor(first, x));
        last = max(last, __shfl_xor(last, x));
        inner_lo = max(inner_lo, __shfl_xor(inner_lo, x));
        inner_hi = min(inner_hi, __shfl_xor(inner_hi, x));
    }
    first = __builtin_amdgcn_readfirstlane(max(first & ~(STEP - 1), s.lo + it.piece * piece));
    last = __builtin_amdgcn_readfirstlane(last);
    if (first >= last) first = last = 0;  // no key (first may be INT32_MAX: no sum with it)
    inner_lo = __builtin_amdgcn_readfirstlane(inner_lo);
    inner_hi = __builtin_amdgcn_readfirstlane(inner_hi);

    // q as operands: values 32g + 8h .. +7 of the row
    f16x8 q[PARTS][NG];
    const int64_t qo = ((int64_t)s.t0 + tok) * a.q_stride + (int64_t)(head * a.group + gh) * D + 8 * h;
    float sc = a.scale;
    {
        float x[NG][8], top = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[g][e] = valid ? q_at(a, qo + 32 * g + e) : 0.0f;
                top = fmaxf(top, fabsf(x[g][e]));
            }
        if constexpr (PARTS == 1) {
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int e = 0; e < 8; e++) q[0][g][e] = (_Float16)x[g][e];
        } else {
            // a power of two puts the row's largest into [2^14, 2^15): hi + lo hold 22 bits
            top = row_max(top);
            int ex = top > 0.0f ? 15 - (int)(__builtin_bit_cast(uint32_t, top) >> 23) + 126 : 0;
            ex = min(max(ex, -126), 126);
            const float up = __builtin_bit_cast(float, (uint32_t)(ex + 127) << 23);
            const float down = __builtin_bit_cast(float, (uint32_t)(127 - ex) << 23);
            sc *= down;
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float v = x[g][e] * up;
                    const _Float16 t = (_Float16)v;
                    q[0][g][e] = t;
                    q[PARTS - 1][g][e] = (_Float16)(v - (float)t);
                }
        }
    }
    constexpr float LOG2E = 1.4426950408889634f;
    const float cap = a.softcap, x_of_s = cap > 0.0f ? sc / cap : sc * LOG2E, x_of_t = cap * LOG2E;

    f32x4 acc[NT], sum = {0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = f32x4{0, 0, 0, 0};
    float m = -INFINITY;
    Frag ones;
#pragma unroll
    for (int i = 0; i < 4; i++) ones.w[i] = 0x3c003c00u;

    const int32_t *table = a.c.table + (int64_t)it.b * a.c.max_pages;
    // the 16-key tile t of the sequence: its region, or null when its page is not the cache's
    auto tile_at = [&](int t, int &sub) -> const uint8_t * {
        const int pg = kv_page_of(a.c, t);
        sub = t - pg * a.c.tiles;
        const int id = pg >= 0 && pg < a.c.max_pages ? table[pg] : -1;
        return id >= 0 && id < a.c.n_pages ? a.c.data + ((int64_t)id * a.c.heads + head) * a.c.region : nullptr;
    };
    auto load_step = [&](int k0, Raw<NG> &r, bool (&have)[2]) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            int sub;
            const uint8_t *reg = tile_at(k0 / KV_TILE + half, sub);
            have[half] = reg != nullptr;
            load_tile<NG>(reg ? reg : a.c.data, a.c, reg ? sub : 0, half, r);
        }
    };

    int k0 = first + wave * STEP;
    Raw<NG> cur;
    bool have[2];
    if (k0 < last) load_step(k0, cur, have);
    while (k0 < last) {
        const int k1 = k0 + WAVES * STEP;
        Raw<NG> nxt;
        bool nhave[2] = {false, false};
        if (k1 < last) load_step(k1, nxt, nhave);

        f32x4 st[2];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            st[half] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const f16x8 kf = k_frag<NG>(cur, half, g);
#pragma unroll
                for (int p = 0; p < PARTS; p++)
                    st[half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[p][g], st[half], 0, 0, 0);
            }
        }
        // scores in units of log2
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float v = st[i >> 2][i & 3] * x_of_s;
            x[i] = cap > 0.0f ? tanhf(v) * x_of_t : v;
        }
        if (k0 < inner_lo || k0 + STEP > inner_hi || !have[0] || !have[1]) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int key = k0 + (i >> 2) * 16 + 4 * h + (i & 3);
                if (key < lo || key >= hi || !have[i >> 2]) x[i] = -INFINITY;
            }
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 8; i++) top = fmaxf(top, x[i]);
        if (__ballot(top > m + M_SLACK)) {
            const float mn = fmaxf(m, row_max(top));
            const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            sum *= f;
#pragma unroll
            for (int t = 0; t < NT; t++) acc[t] *= f;
        }
        const float mb = m == -INFINITY ? 0.0f : m - P_BIAS;
        f16x8 p[PARTS];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float v = __builtin_amdgcn_exp2f(x[i] - mb);
            const _Float16 t = (_Float16)v;
            p[0][i] = t;
            if constexpr (PARTS == 2) p[1][i] = (_Float16)(v - (float)t);
        }
#pragma unroll
        for (int pp = 0; pp < PARTS; pp++) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones.v, p[pp], sum, 0, 0, 0);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            f16x8 vl, vh;
            v_frags<NG>(cur, g, vl, vh);
#pragma unroll
            for (int pp = 0; pp < PARTS; pp++) {
                acc[2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, p[pp], acc[2 * g], 0, 0, 0);
                acc[2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, p[pp], acc[2 * g + 1], 0, 0, 0);
            }
        }
        cur = nxt;
        have[0] = nhave[0];
        have[1] = nhave[1];
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
    // row r of the tile: 16 threads, 4 values at a time
    const int r = threadIdx.x >> 4, u = threadIdx.x & 15;
    float f[WAVES], mm = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; w++) mm = fmaxf(mm, ml[(w * TR + r) * 2]);
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        const float mw = ml[(w * TR + r) * 2];
        f[w] = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - mm);
        // (a NaN key leaves a wave's maximum at -inf and its sum NaN)
        const float lw = ml[(w * TR + r) * 2 + 1];
        if (lw != lw) f[w] = lw;
        l += f[w] * lw;
    }
    const int rr = it.tile * TR + r;
    if (rr >= s.n * a.group) return;
    const int rt = rr / a.group, rg = rr - rt * a.group;
    const bool whole = it.pieces == 1;
    const int64_t slot = (int64_t)it.first + it.piece;
    if (!whole && slot >= a.slots) return;
    float *part = a.part + ((slot * a.c.heads + head) * TR + r) * (D + 2);
    const int64_t o = ((int64_t)s.t0 + rt) * a.out_stride + (int64_t)(head * a.group + rg) * D;
    const float inv = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
#pragma unroll
    for (int d = 0; d < D; d += 64) {
        const int e = d + 4 * u;
        if (D % 64 && e >= D) break;
        f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < WAVES; w++) v += f[w] * *(const f32x4 *)(lds + (w * TR + r) * OS + e);
        v *= inv;
        if (whole) {
            store_out(a, o + e, v);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) part[2 + e + i] = v[i];
        }
    }
    if (!whole && u == 0) {
        part[0] = mm;
        part[1] = l;
    }
}

// Rows whose keys were cut into pieces: their parts joined.  A workgroup has one (tile, head).
template <int NG>
__global__ __launch_bounds__(256) void attn_join(AttnArgs a) {
    constexpr int D = 32 * NG;
    const int head = blockIdx.y;
    const int piece = piece_len(a);
    Item it;
    if (!find_item<false>(a, piece, blockIdx.x, it) || it.pieces == 1) return;
    const int r = threadIdx.x >> 4, u = threadIdx.x & 15, rr = it.tile * TR + r;
    if (rr >= it.s.n * a.group || (int64_t)it.first + it.pieces > a.slots) return;
    const float *part = a.part + (((int64_t)it.first * a.c.heads + head) * TR + r) * (D + 2);
    const int64_t next = (int64_t)a.c.heads * TR * (D + 2);
    float mm = -INFINITY, l = 0.0f;
    for (int p = 0; p < it.pieces; p++) mm = fmaxf(mm, part[p * next]);
    f32x4 v[(D + 63) / 64];
#pragma unroll
    for (int d = 0; d < (D + 63) / 64; d++) v[d] = f32x4{0, 0, 0, 0};
    for (int p = 0; p < it.pieces; p++) {
        const float mp = part[p * next], lp = part[p * next + 1];
        float f = mp == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mp - mm);
        if (lp != lp) f = lp;
        l += f * lp;
#pragma unroll
        for (int d = 0; d < (D + 63) / 64; d++) {
            const int e = 64 * d + 4 * u;
            if (D % 64 && e >= D) break;
#pragma unroll
            for (int i = 0; i < 4; i++) v[d][i] += f * part[p * next + 2 + e + i];
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int rt = rr / a.group, rg = rr - rt * a.group;
    const int64_t o = ((int64_t)it.s.t0 + rt) * a.out_stride + (int64_t)(head * a.group + rg) * D;
#pragma unroll
    for (int d = 0; d < (D + 63) / 64; d++) {
        const int e = 64 * d + 4 * u;
        if (D % 64 && e >= D) break;
        store_out(a, o + e, v[d] * inv);
    }
}

template <int NG, int PARTS>
hipError_t rows16_launch(const AttnArgs &a, unsigned tiles, hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t lds = (size_t)WAVES * TR * (32 * NG + 4 + 2) * sizeof(float);
    const hipError_t e = set_max_lds_once((const void *)attn_rows16<NG, PARTS>, lds, done);
    if (e != hipSuccess) return e;
    attn_rows16<NG, PARTS><<<dim3((unsigned)a.slots, a.c.heads), 64 * WAVES, lds, s>>>(a);
    attn_join<NG><<<dim3(tiles, a.c.heads), 256, 0, s>>>(a);
    return hipGetLastError();
}

int64_t tile_bound(int64_t batch, int64_t tokens, int group) {
    return std::min(tokens * group / TR + batch, tokens * ((group + TR - 1) / TR));
}

template <int NG>
hipError_t dim_launch(const AttnArgs &a, hipStream_t s) {
    const unsigned tiles = (unsigned)tile_bound(a.c.batch, a.c.tokens, a.group);
    return a.q_dtype == ARFQ_F16 && a.out_dtype == ARFQ_F16 ? rows16_launch<NG, 1>(a, tiles, s)
                                                            : rows16_launch<NG, 2>(a, tiles, s);
}

}  // namespace

bool attn_dim_ok(int dim) { return dim == 64 || dim == 96 || dim == 128 || dim == 256; }

AttnPlan attn_plan(int cus, int heads, int dim, int64_t batch, int64_t tokens, int q_heads) {
    AttnPlan p;
    const int group = q_heads / heads;
    p.target = std::max(1, 2 * cus / heads);
    // tiles * pieces: the area cut into `target` pieces, and at most one more for each tile
    p.slots = (int)(p.target + tile_bound(batch, tokens, group));
    p.ws_bytes = (size_t)p.slots * heads * TR * (dim + 2) * sizeof(float);
    return p;
}

hipError_t launch_attn(const AttnArgs &a, int dim, hipStream_t s) {
    switch (dim) {
    case 64: return dim_launch<2>(a, s);
    case 96: return dim_launch<3>(a, s);
    case 128: return dim_launch<4>(a, s);
    case 256: return dim_launch<8>(a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace arfq
