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
// waves of a SIMD (a workgroup has one on each): registers below 512 / that
constexpr int rows16_waves(int ng) { return ng <= 2 ? 4 : ng <= 4 ? 3 : 2; }
// p is held as exp2(x - m + P_BIAS), m behind the running maximum by at most M_SLACK: f16 (2^16)
// is not passed, and a part of p keeps its 11 bits down to 2^-27 of the largest p (below, half
// a step is 2^-38 of it).  The slack spares most steps the rescaling of the sums.
constexpr float BIAS_UNIT = 32768.0f;
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
    s.end = (int)min((int64_t)max(s.len, 0), (int64_t)a.c.max_pages * a.c.page);
    if (a.window) s.lo = (int)max((int64_t)0, min((int64_t)s.len - s.n - a.window + 1, (int64_t)s.end)) & ~(STEP - 1);
    s.tiles = (int)(((int64_t)s.n * a.group + TR - 1) / TR);
    return s;
}

__device__ __forceinline__ int pieces_of(const Seq &s, int piece) {
    return max(1, (s.end - s.lo + piece - 1) / piece);
}

// Running sums over the wave's lanes (six DPP additions: a row of 16 by shifts, then the rows).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int v) {
    v += dpp<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v += dpp<0x112, 0xf>(v);
    v += dpp<0x114, 0xf>(v);
    v += dpp<0x118, 0xf>(v);
    v += dpp<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    v += dpp<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    auto step = [&](int w) { v += __builtin_bit_cast(float, w); };
    step(dpp<0x111, 0xf>(__builtin_bit_cast(int, v)));
    step(dpp<0x112, 0xf>(__builtin_bit_cast(int, v)));
    step(dpp<0x114, 0xf>(__builtin_bit_cast(int, v)));
    step(dpp<0x118, 0xf>(__builtin_bit_cast(int, v)));
    step(dpp<0x142, 0xa>(__builtin_bit_cast(int, v)));
    step(dpp<0x143, 0xc>(__builtin_bit_cast(int, v)));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

struct Item {
    Seq s;
    int b, tile, piece, pieces;
    int keys;  // of a piece (a multiple of STEP): the sequence's keys in equal parts
    int slot;  // place of the (tile, piece) in the list of all
};

// The `index`-th (tile, piece) of the batch: sequences in order, their tiles one after another,
// pieces fastest; or (PIECES false) the first piece of the index-th tile.  False: the list has
// fewer.  The keys that make a new piece necessary are the same in every wave of the launch: the
// fewest that cut the area into at most `target` pieces, or nearly so (a target of workgroups that
// the chip holds at once: one more round for a few of them would take as long as the first).
// The area is summed in f32 in one fixed order; the 2^-16 added covers its rounding, so that the
// list has no more than target + tiles items.
template <bool PIECES>
__device__ __forceinline__ bool find_item(const AttnArgs &a, int index, Item &it) {
    const int lane = threadIdx.x & 63;
    const Seq s0 = seq_of(a, lane);  // (the whole batch, mostly)
    auto over_batch = [&](auto f) {
        float v = f(s0);
        for (int b0 = WAVE; b0 < a.c.batch; b0 += WAVE) v += f(seq_of(a, b0 + lane));
        return wave_sum(v);
    };
    const float area = over_batch([](const Seq &s) { return (float)s.tiles * (float)((s.end - s.lo + STEP - 1) / STEP); });
    const float target = (float)a.target;
    auto keys_of = [](float steps) { return (int)fminf(steps, (float)(KV_KEYS_MAX / STEP)) * STEP; };
    float steps = fmaxf(ceilf(area / target * (1.0f + 1.0f / 65536)), (float)(MIN_PIECE / STEP));
    if (a.c.batch > 1) {
        for (int i = 0; i < 3; i++) {
            const int piece = keys_of(steps);
            const float items = over_batch([&](const Seq &s) { return (float)s.tiles * (float)pieces_of(s, piece); });
            if (items <= target) break;
            // (tiles of one piece stay: the others' pieces shrink in number with their length)
            steps = ceilf(steps * fminf(items / target, 2.0f));
        }
    }
    const int piece = keys_of(steps);
    int before = 0, items = 0;
    for (int b0 = 0; b0 < a.c.batch; b0 += WAVE) {
        const Seq s = b0 ? seq_of(a, b0 + lane) : s0;
        const int np = pieces_of(s, piece), all = (int)min((int64_t)s.tiles * np, (int64_t)1 << 30);
        const int own = PIECES ? all : s.tiles, inc = wave_scan(own), sum = PIECES ? inc : wave_scan(all);
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
            it.keys = ((it.s.end - it.s.lo + STEP - 1) / STEP + it.pieces - 1) / it.pieces * STEP;
            const int rest = index - before - __builtin_amdgcn_readlane(inc - own, l);
            it.tile = PIECES ? rest / it.pieces : rest;
            it.piece = PIECES ? rest - it.tile * it.pieces : 0;
            it.slot = PIECES ? index : items + __builtin_amdgcn_readlane(sum - all, l) + it.tile * it.pieces;
            return rest >= 0 && it.tile < it.s.tiles && it.slot >= 0;
        }
        before += __builtin_amdgcn_readlane(inc, 63);
        items += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

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

// What a lane of the step's 32 keys loads: K of two 16-key tiles (key lane % 16, chunk lane / 16)
// and V of the keys 4 * (lane / 16) .. +3 of both (matrix rows lane % 16).
template <int NG>
struct Raw {
    uint32_t k[2][NG], v[2][NG];
    uint32_t ks[2][2 * NG];              // of keys 4 * (lane / 16) .. +3: [4][NG] f16
    uint32_t vs[2][2 * NG];              // of the same, in pairs: [NG][2]
    uint32_t ka[2][(NG + 1) / 2];        // of key lane % 16 (RAW)
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
    uint32_t k, v, s, a;
};
template <int NG>
__device__ __forceinline__ Offs<NG> lane_offs() {
    const uint32_t lane = threadIdx.x & 63, c = lane & 15, h = lane >> 4;
    return {c * (16 * NG) + h * (4 * NG), h * (64 * NG) + c * (4 * NG), h * (8 * NG), c * (2 * NG)};
}
// p + o with p uniform: hidden from the compiler, which would widen o once and keep it in two registers
// instead of the loads' scalar base and 32-bit offset.
__device__ __forceinline__ const uint8_t *at(const uint8_t *p, uint32_t o) {
    asm("" : "+v"(o));
    return p + o;
}
// reg (uniform): the tile's (page, head) region; sub: the 16-key tile within the page
template <bool RAW, int NG>
__device__ __forceinline__ void load_k(const uint8_t *reg, const KvArgs &a, uint32_t sub, int half, const Offs<NG> &o, Raw<NG> &r) {
    constexpr int AL = NG % 4 == 0 ? 16 : NG % 2 == 0 ? 8 : 4;
    load_aligned<NG, AL>(at(reg + sub * (256u * NG), o.k), r.k[half]);
    const uint8_t *ks = reg + (a.off_ks + sub * (32u * NG));
    load_aligned<2 * NG, 8>(at(ks, o.s), r.ks[half]);
    if constexpr (!RAW) {
    } else if constexpr (NG % 2 == 0) {
        load_aligned<NG / 2, NG % 8 == 0 ? 16 : NG % 4 == 0 ? 8 : 4>(at(ks, o.a), r.ka[half]);
    } else {
        const uint16_t *k1 = (const uint16_t *)at(ks, o.a);
#pragma unroll
        for (int i = 0; i < NG / 2; i++) r.ka[half][i] = k1[2 * i] | (uint32_t)k1[2 * i + 1] << 16;
        r.ka[half][NG / 2] = k1[NG - 1];
    }
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

// MFMA operand of group g of the K tile, eight codes of one key.
// RAW: as they lie, plus 8, as subnormal f16 numbers of c * 2^-24 (nibbles in bits 0..3) and 16 c * 2^-24
// (bits 4..7); q's values for the latter slots (2, 3, 6, 7) come divided by 16.  The matrix core
// multiplies subnormals, but aligns its sums by the exponent field: 2^-14 of the sum is lost,
// an eighth of an f16 q's own rounding and far above an f32 one's.
// Otherwise the codes themselves.
template <bool RAW, int NG>
__device__ __forceinline__ f16x8 k_frag(const Raw<NG> &r, int half, int g, uint32_t magic) {
    const uint32_t w = r.k[half][g], w8 = w >> 8;
    Frag f;
    if constexpr (RAW) {
        f.w[0] = __builtin_bit_cast(f16x2, w & 0x000f000fu);
        f.w[1] = __builtin_bit_cast(f16x2, w & 0x00f000f0u);
        f.w[2] = __builtin_bit_cast(f16x2, w8 & 0x000f000fu);
        f.w[3] = __builtin_bit_cast(f16x2, w8 & 0x00f000f0u);
    } else {
        f.w[0] = codes_f16<true>(w, magic);
        f.w[1] = codes_f16<false>(w, magic);
        f.w[2] = codes_f16<true>(w8, magic);
        f.w[3] = codes_f16<false>(w8, magic);
    }
    return f.v;
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
            // bytes g of keys 2 pr and 2 pr + 1: one into each half
            const int b0 = 2 * pr * NG + g, b1 = b0 + NG;
            const uint32_t sel = 0x0c000c00u | (uint32_t)((b1 & 3) + 4) << 16 | (uint32_t)(b0 & 3);
            const uint32_t t = __builtin_amdgcn_perm(r.v[half][b1 >> 2], r.v[half][b0 >> 2], sel);
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

// ---- rows of 16, keys spread over the waves ------------------------------------------------
// S^T = K Q^T, O^T = V^T P^T with v_mfma_f32_16x16x32_f16: the 16 rows are matrix columns, so a
// lane's four results of a tile belong to one row, its statistics are a register, and P^T in
// the layout of a result is the layout of the next product's operand (which keys a lane's
// eight slots stand for is free, as V is loaded to match).  K's scales multiply the products of
// a group (32 values: one MFMA), V's its codes.
// PARTS: f16 parts of q and p (2: hi + lo, 22 bits, for f32 q or out).
template <int NG, int PARTS>
__global__ __launch_bounds__(64 * WAVES, rows16_waves(NG)) void attn_rows16(AttnArgs a) {
    constexpr int D = 32 * NG, NT = 2 * NG;  // NT: 16-row tiles of O^T
    constexpr bool RAW = PARTS == 1;         // K's operands: see k_frag
    constexpr int OS = D + 4;                // LDS floats of a row of O
    extern __shared__ float lds[];           // [WAVES][16][OS], then [WAVES][16][2]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, h = lane >> 4;
    const int head = blockIdx.x % a.c.heads;  // (fastest: the list's unused end comes last)
    Item it;
    if (!find_item<true>(a, blockIdx.x / a.c.heads, it)) return;
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

    // the page ids of a step's two 16-key tiles (of the table's last page past its end: those keys are masked)
    const int32_t *table = a.c.table + (int64_t)it.b * a.c.max_pages;
    const uint8_t *base = a.c.data + head * a.c.region;
    const int64_t page_bytes = a.c.region * a.c.heads;
    auto ids_at = [&](int k, int (&o)[2]) {
#pragma unroll
        for (int half = 0; half < 2; half++) o[half] = table[min(kv_page_of(a.c, k / KV_TILE + half), a.c.max_pages - 1)];
    };
    auto in_cache = [&](int id) { return (uint32_t)id < (uint32_t)a.c.n_pages; };
    // a tile's region (of page 0 for an id that is not the cache's: the loads stay in it, the keys are masked)
    auto region = [&](int id) { return base + (in_cache(id) ? (int64_t)id * page_bytes : 0); };
    auto sub_of = [&](int k, int half) {
        const int t = k / KV_TILE + half;
        return (uint32_t)(t - kv_page_of(a.c, t) * a.c.tiles);
    };
    constexpr int NEXT = WAVES * STEP;
    const Offs<NG> offs = lane_offs<NG>();
    Raw<NG> r;
    int k0 = first + wave * STEP;
    int id[2] = {0, 0}, nid[2] = {0, 0};  // of this step, of the next one
    auto load_ks = [&](int k, const int (&i)[2]) {
#pragma unroll
        for (int half = 0; half < 2; half++) load_k<RAW>(region(i[half]), a.c, sub_of(k, half), half, offs, r);
    };
    auto load_vs = [&](int k, const int (&i)[2]) {
#pragma unroll
        for (int half = 0; half < 2; half++) load_v<NG>(region(i[half]), a.c, sub_of(k, half), half, offs, r);
    };
    if (k0 < last) {  // (keys: the table has a page)
        ids_at(k0, id);
        ids_at(k0 + NEXT, nid);
        load_ks(k0, id);
        load_vs(k0, id);
    }

    // q as operands: values 32g + 8h .. +7 of the row, times a power of two that puts the row's
    // largest into [2^14, 2^15): hi + lo hold 22 bits (an f16 q its 11)
    f16x8 q[PARTS][NG];
    // RAW codes come with 8 added: -8 times the sum of a group's q, in three f16 parts (lanes 0..15, 16..31,
    // 32..47 of a row's), times K's scales is one more product
    Frag bias;
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
        int ex = top > 0.0f ? 141 - (int)(__builtin_bit_cast(uint32_t, top) >> 23) : 0;
        ex = min(max(ex, -126), 126);
        // (the scores' sign goes into q: larger products, larger scores)
        const float up = __builtin_bit_cast(float, (uint32_t)(ex + 127) << 23) * (a.scale < 0.0f ? -1.0f : 1.0f);
        sc *= __builtin_bit_cast(float, (uint32_t)(127 - ex) << 23);
#pragma unroll
        for (int i = 0; i < 4; i++) bias.w[i] = f16x2{(_Float16)0, (_Float16)0};
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float all = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = x[g][e] * up * (RAW && (e & 2) ? 0.0625f : 1.0f);
                const _Float16 t = (_Float16)v, l = (_Float16)(v - (float)t);
                q[0][g][e] = t;
                if constexpr (PARTS == 2) q[1][g][e] = l;
                all += (float)t * (e & 2 ? 16.0f : 1.0f);
            }
            if constexpr (!RAW) continue;
            all += __shfl_xor(all, 16);
            all += __shfl_xor(all, 32);
            all *= -8.0f / 16777216 * BIAS_UNIT;  // at most 8 * 32 * 2^15 / 2^24 * 2^15 = 2^14
            const float b0 = (float)(_Float16)all, b1 = (float)(_Float16)(all - b0), b2 = all - b0 - b1;
            bias.w[g / 2][g % 2] = (_Float16)(h == 0 ? b0 : h == 1 ? b1 : h == 2 ? b2 : 0.0f);
        }
    }
    constexpr float LOG2E = 1.4426950408889634f;
    constexpr float UNIT = RAW ? 16777216.0f : 1.0f;  // of the products (RAW: of codes * 2^-24)
    // a product in the scores' log2, or in the cap (not below the smallest normal
    // number, where products of it are 0 beside p's 24 bits: a masked score is -inf, and -inf * 0 would be NaN)
    const float cap = a.softcap, x_of_s = fmaxf((cap > 0.0f ? sc / cap : sc * LOG2E) * UNIT, 1.1754944e-38f);
    const float x_of_t = cap * LOG2E;

    f32x4 acc[NT], sum = {0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = f32x4{0, 0, 0, 0};
    float m = -INFINITY;
    Frag ones;
#pragma unroll
    for (int i = 0; i < 4; i++) ones.w[i] = f16x2{(_Float16)1, (_Float16)1};
    const uint32_t magic = magic_1024();

    while (k0 < last) {
        const int k1 = k0 + NEXT;
        float x[8], unit = x_of_s;  // scores; a unit of them in log2
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const f32x4 z = {0, 0, 0, 0};
            if constexpr (RAW) {
                Frag ka;
#pragma unroll
                for (int i = 0; i < 4; i++) ka.w[i] = __builtin_bit_cast(f16x2, i < (NG + 1) / 2 ? r.ka[half][i] : 0u);
                const f32x4 o = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka.v, bias.v, z, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) x[4 * half + i] = o[i] * (1.0f / BIAS_UNIT);
            }
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const f16x8 kf = k_frag<RAW>(r, half, g, magic);
                f32x4 t = z;
#pragma unroll
                for (int p = 0; p < PARTS; p++) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[p][g], t, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float d = (float)half_of(r.ks[half][(i * NG + g) / 2], (i * NG + g) & 1);
                    x[4 * half + i] = !RAW && g == 0 ? t[i] * d : __builtin_fmaf(t[i], d, x[4 * half + i]);
                }
            }
            // the scores are formed here: K's registers are free for the next step's loads
            asm volatile("" : "+v"(x[4 * half]), "+v"(x[4 * half + 1]), "+v"(x[4 * half + 2]), "+v"(x[4 * half + 3]));
        }
        if (k1 < last) load_ks(k1, nid);
        if (cap > 0.0f) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = tanh_of(x[i] * x_of_s) * x_of_t;
            unit = 1.0f;
        }
        if (k0 < inner_lo || k0 + STEP > inner_hi || !in_cache(id[0]) || !in_cache(id[1])) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint32_t from = (uint32_t)(k0 + half * 16 + 4 * h - lo), width = in_cache(id[half]) ? (uint32_t)max(hi - lo, 0) : 0u;
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
        f16x8 p[PARTS];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], unit, mb));
            const _Float16 t = (_Float16)v;
            p[0][i] = t;
            if constexpr (PARTS == 2) p[1][i] = (_Float16)__builtin_fmaf((float)t, -1.0f, v);
        }
#pragma unroll
        for (int pp = 0; pp < PARTS; pp++) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones.v, p[pp], sum, 0, 0, 0);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            f16x8 vl, vh;
            v_frags<NG>(r, g, magic, vl, vh);
#pragma unroll
            for (int pp = 0; pp < PARTS; pp++) {
                acc[2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, p[pp], acc[2 * g], 0, 0, 0);
                acc[2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, p[pp], acc[2 * g + 1], 0, 0, 0);
            }
        }
        if (k1 < last) load_vs(k1, nid);
        id[0] = nid[0];
        id[1] = nid[1];
        if (k1 < last) ids_at(k1 + NEXT, nid);
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
        float *part = a.part + (((int64_t)it.slot * a.c.heads + head) * TR + er) * (D + 4);
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

// Rows whose keys were cut into pieces: their parts joined, in a fixed order.  A workgroup has one row in
// gridDim.z of a (tile, head); its threads take D / 4 columns of four values and 1024 / D
// pieces at a time.
template <int NG>
__global__ __launch_bounds__(256) void attn_join(AttnArgs a) {
    constexpr int D = 32 * NG, CT = D / 4, PT = 256 / CT;
    __shared__ f32x4 v_of[PT][CT];
    __shared__ float l_of[PT], m_of[PT];
    const int head = blockIdx.x % a.c.heads;
    Item it;
    if (!find_item<false>(a, blockIdx.x / a.c.heads, it) || it.pieces == 1) return;
    const int pt = threadIdx.x / CT, ct = threadIdx.x - pt * CT;
    const int rows = min(it.s.n * a.group - it.tile * TR, TR), pieces = min(it.pieces, a.slots - it.slot);
    const int64_t next = (int64_t)a.c.heads * TR * (D + 4);
    // the weight of a part (m, l) below a common maximum; NaN for a NaN part (a NaN key leaves
    // a wave's maximum at -inf and its sum NaN)
    auto weight = [](float m, float l, float top) { return l != l ? l : m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top); };
    for (int r = blockIdx.z; r < rows; r += gridDim.z) {
        const float *part = a.part + (((int64_t)it.slot * a.c.heads + head) * TR + r) * (D + 4);
        float mm = -INFINITY, l = 0.0f;
        f32x4 v = {0, 0, 0, 0};
        if (pt < PT) {
            constexpr int U = 8;  // loads in flight
            for (int p0 = pt; p0 < pieces; p0 += U * PT) {
                float m_p[U], l_p[U];
                f32x4 w[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int p = min(p0 + u * PT, pieces - 1);
                    const float2 ml = *(const float2 *)(part + p * next);
                    w[u] = *(const f32x4 *)(part + p * next + 4 + 4 * ct);
                    m_p[u] = p0 + u * PT < pieces ? ml.x : -INFINITY;
                    l_p[u] = p0 + u * PT < pieces ? ml.y : 0.0f;
                }
                float top = mm;
#pragma unroll
                for (int u = 0; u < U; u++) top = fmaxf(top, m_p[u]);
                const float f0 = weight(mm, l, top);
                l *= f0;
                v *= f0;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const float f = weight(m_p[u], l_p[u], top);
                    l += f * l_p[u];
                    v += f * w[u];
                }
                mm = top;
            }
            v_of[pt][ct] = v;
            if (ct == 0) {
                m_of[pt] = mm;
                l_of[pt] = l;
            }
        }
        __syncthreads();
        if (pt == 0) {
#pragma unroll
            for (int p = 0; p < PT; p++) mm = fmaxf(mm, m_of[p]);
            l = 0.0f;
            v = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < PT; p++) {
                const float f = weight(m_of[p], l_of[p], mm);
                l += f * l_of[p];
                v += f * v_of[p][ct];
            }
            const int rr = it.tile * TR + r, rt = rr / a.group, rg = rr - rt * a.group;
            store_out(a, ((int64_t)it.s.t0 + rt) * a.out_stride + (int64_t)(head * a.group + rg) * D + 4 * ct,
                      v * (l == 0.0f ? 0.0f : 1.0f / l));
        }
        __syncthreads();
    }
}

int64_t tile_bound(int64_t batch, int64_t tokens, int group) {
    return std::min(tokens * group / TR + batch, tokens * ((group + TR - 1) / TR));
}

template <int NG, int PARTS>
hipError_t rows16_launch(const AttnArgs &a, hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t lds = (size_t)WAVES * TR * (32 * NG + 4 + 2) * sizeof(float);
    const hipError_t e = set_max_lds_once((const void *)attn_rows16<NG, PARTS>, lds, done);
    if (e != hipSuccess) return e;
    attn_rows16<NG, PARTS><<<dim3((unsigned)a.slots * a.c.heads), 64 * WAVES, lds, s>>>(a);
    if (a.joins) attn_join<NG><<<dim3((unsigned)tile_bound(a.c.batch, a.c.tokens, a.group) * a.c.heads, 1, a.joins), 256, 0, s>>>(a);
    return hipGetLastError();
}

template <int NG>
hipError_t dim_launch(const AttnArgs &a, hipStream_t s) {
    return a.q_dtype == ARFQ_F16 && a.out_dtype == ARFQ_F16 ? rows16_launch<NG, 1>(a, s) : rows16_launch<NG, 2>(a, s);
}

}  // namespace

bool attn_dim_ok(int dim) { return dim == 64 || dim == 96 || dim == 128 || dim == 256; }

AttnPlan attn_plan(int cus, int heads, int dim, int64_t batch, int64_t tokens, int q_heads, int64_t max_keys) {
    AttnPlan p;
    const int64_t tiles = tile_bound(batch, tokens, q_heads / heads), most = (max_keys + MIN_PIECE - 1) / MIN_PIECE;
    p.target = std::max(1, rows16_waves(dim / KV_GROUP) * cus / heads);
    // the area cut into `target` pieces, and at most one more for each tile; none shorter than MIN_PIECE
    p.slots = (int)std::min(p.target + tiles, tiles * std::max<int64_t>(most, 1));
    if (most > 1) {
        p.ws_bytes = (size_t)p.slots * heads * TR * (dim + 4) * sizeof(float);
        // workgroups of a (tile, head): one for each row of it, while they are about the chip's
        const int64_t rows = std::min<int64_t>(TR, tokens > batch ? TR : q_heads / heads);
        p.joins = (int)std::max<int64_t>(1, std::min<int64_t>(rows, 4 * cus / (tiles * heads)));
    }
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
