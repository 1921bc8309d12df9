// arfq_kv.hip -- writing K and V rows into the 4-bit cache and reading them back.
//
// Four lanes have a group of 32 values, its K and its V, eight of each a lane: a group's extremes are two
// exchanges within a quad, and what a lane has is a dword of the cache.  Bound by memory, and by the chain of
// dependent loads in front of it (the row's sequence, its length, its page): f32 rows of three prompts,
// 18552 tokens of 8 x 128, written in 52 us (173 MB, 3.3 TB/s; the codes' exact quotients are a third of
// that time's vector work), read back in 32 (5.4 TB/s); 141000 tokens read as f16, 740 MB in
// all, in 189 (3.9 TB/s; a plain copy reaches 4.8).
// By width, 20700 tokens of 1536 values, at 64 / 96 / 128 / 256, us: f32 rows (290 MB with the codes) written in
// 94 / 111 / 90 / 89, read in 70 / 70 / 81 / 81; f16 rows (163 MB) written in 92 / 114 / 89 / 86 (the quotients, not
// the bytes), read in 38 / 37 / 31 / 31.  At 64 and 96 V goes byte by byte (VLane), at 96 a quarter of the
// lanes idles besides.
#include "arfq_kv.h"

namespace arfq {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// Lanes of a (token, head) row: four for each group of 32 values, up to a power of two
// (a row's lanes lie in one wave; D = 96 leaves four of its sixteen idle).
template <int NG>
constexpr int row_lanes() { return NG <= 2 ? 8 : NG <= 4 ? 16 : 32; }

// (non-temporal: each value is read once; 83 us for 85 at 18552 f32 rows written and read)
__device__ __forceinline__ void load4(const void *p, int64_t i, bool f16, float *o) {
    if (f16) {
        const u32x2 w = __builtin_nontemporal_load((const u32x2 *)((const _Float16 *)p + i));
        o[0] = h2f(w.x); o[1] = h2f(w.x >> 16); o[2] = h2f(w.y); o[3] = h2f(w.y >> 16);
    } else {
        const f32x4 w = __builtin_nontemporal_load((const f32x4 *)((const float *)p + i));
        o[0] = w.x; o[1] = w.y; o[2] = w.z; o[3] = w.w;
    }
}

// 16 bytes; PAST: not kept in the caches (see read_launch).
template <bool PAST, class T>
__device__ __forceinline__ void store16(void *p, T v) {
    if constexpr (PAST)
        __builtin_nontemporal_store(v, (T *)p);
    else
        *(T *)p = v;
}
__device__ __forceinline__ u32x4 pack8(const float *o) {
    return u32x4{pack_f16x2(o[0], o[1]), pack_f16x2(o[2], o[3]), pack_f16x2(o[4], o[5]), pack_f16x2(o[6], o[7])};
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(uint32_t, v)));
}

// Byte b of lane a of a quad <-> byte a of lane b: pairs of lanes, then pairs of those.
__device__ __forceinline__ uint32_t quad_transpose(uint32_t w) {
    const uint32_t lane = threadIdx.x, y = dpp<0xb1>(w);  // quad_perm:[1,0,3,2]
    w = __builtin_amdgcn_perm(y, w, lane & 1 ? 0x03070105u : 0x06020400u);
    const uint32_t z = dpp<0x4e>(w);  // quad_perm:[2,3,0,1]
    return __builtin_amdgcn_perm(z, w, lane & 2 ? 0x03020706u : 0x05040100u);
}

// Where a row's lane u has its V: values 4i .. +3 and 16 + 4i .. +3 of group g.  NG a multiple of 4: a dword of the
// cache has a matrix row's bytes of four groups, and a quad of lanes turns the dwords of four such
// rows into one group's bytes each; so g runs fastest over the lanes.  Otherwise byte by byte.
template <int NG>
struct VLane {
    static constexpr bool DWORDS = NG % 4 == 0;
    int g, i;
    __device__ __forceinline__ VLane(int u) : g(DWORDS ? (u & 3) + (u >> 4) * 4 : u >> 2), i(DWORDS ? (u >> 2) & 3 : u & 3) {}
    // what the lane of i ^ 1 has
    static __device__ __forceinline__ uint32_t pair(uint32_t v) {
        if constexpr (DWORDS) return (uint32_t)__builtin_amdgcn_ds_swizzle((int)v, 0x101f);  // lane ^ 4
        return dpp<0xb1>(v);
    }
    // over the lanes of a group (i)
    template <class F>
    static __device__ __forceinline__ float all(float v, F f) {
        if constexpr (DWORDS) {
            v = f(v, dpp<0x124>(v));  // row_ror:4, 8
            return f(v, dpp<0x128>(v));
        } else {
            v = f(v, dpp<0xb1>(v));
            return f(v, dpp<0x4e>(v));
        }
    }
};

// Scale of a group from its extremes: s is the value of largest magnitude, the positive one of
// two alike; d = s / -8 (a power of two: exact), at most 8160 so that 8 d is an f16, to 8
// significant bits (ties to even) and to f16, whose subnormals hold multiples of 2^-24.
__device__ __forceinline__ uint32_t group_scale(float hi, float lo) {
    const float s = hi >= -lo ? hi : lo;
    float d = fminf(fmaxf(s * -0.125f, -8160.0f), 8160.0f);
    uint32_t u = __builtin_bit_cast(uint32_t, d);
    u = (u + 0x7fffu + ((u >> 16) & 1u)) & 0xffff0000u;
    return __builtin_bit_cast(unsigned short, (_Float16)__builtin_bit_cast(float, u));
}

// Code + 8 of x: the nearest integer to x / d, ties to even, in [-8, 7].  The product with
// 1 / d lands on it or a neighbour; x - k d is exact (k d has 12 bits, and x and k d are
// multiples of a unit that their difference, at most 2 |d|, holds 24 bits of), so comparing it
// with d / 2 decides as the quotient in real numbers does.
__device__ __forceinline__ uint32_t code_of(float x, float d, float rd) {
    float k = rintf(fminf(fmaxf(x * rd, -9.0f), 9.0f));
    const float ad = fabsf(d), e = d < 0 ? -fmaf(-k, d, x) : fmaf(-k, d, x);  // (x / d - k) * |d|
    const bool odd = ((int)k & 1) != 0;
    if (e + e > ad || (odd && e + e == ad)) k += 1.0f;
    else if (-(e + e) > ad || (odd && -(e + e) == ad)) k -= 1.0f;
    return (uint32_t)((int)fminf(fmaxf(k, -8.0f), 7.0f) + 8);
}

// The places in the cache of the rows that a lane works on, S of them, a wave's rows (row0 + set * R + lane / RL)
// apart: regions (null: none), keys within the pages, tokens and heads.  Rows are (token, head) pairs,
// head fastest.  The searches of all sets go side by side, and so do their loads of lengths
// and page ids: one after another they take longer than the rows themselves.
template <int RL, int S>
struct Rows {
    static constexpr int R = WAVE / RL;  // rows of a wave in a set
    uint8_t *reg[S];
    int key[S], token[S], head[S];
    __device__ __forceinline__ Rows(const KvArgs &a, int row0, int rows) {
        const int lane = threadIdx.x & 63;
        int b[S];
#pragma unroll
        for (int s = 0; s < S; s++) {
            const int row = min(row0 + s * R + lane / RL, rows - 1);
            token[s] = row / a.heads;
            head[s] = row - token[s] * a.heads;
            b[s] = a.start ? 0 : token[s];
        }
        if (a.start) {
            // sequences b with start[b + 1] <= t come before t's, 64 compared at once; none from where start
            // decreases on (kv_seq then finds that one without rows)
            const int t0 = row0 / a.heads, t1 = min(row0 + S * R, rows) - 1;
            for (int b0 = 0; b0 < a.batch; b0 += WAVE) {
                const bool mine = b0 + lane < a.batch;
                const int u = mine ? a.start[b0 + lane] : 0;
                int v = mine ? a.start[b0 + lane + 1] : INT32_MAX;
                const uint64_t falls = __ballot(v < u);
                if (falls && (falls & (((uint64_t)2 << lane) - 1))) v = INT32_MAX;  // (at this lane or one before)
                for (int t = t0; t <= t1 / a.heads; t++) {
                    const int n = __popcll(__ballot(v <= t));
#pragma unroll
                    for (int s = 0; s < S; s++) b[s] += token[s] == t ? n : 0;
                }
                if (falls) break;
            }
        }
        int64_t pos[S];
        int pg[S], id[S];
#pragma unroll
        for (int s = 0; s < S; s++) {
            pos[s] = -1;
            if (row0 + s * R + lane / RL < rows && b[s] < a.batch) {
                int t0, n;
                kv_seq(a, b[s], t0, n);
                if (token[s] >= t0 && token[s] < t0 + n) pos[s] = (int64_t)a.len[b[s]] - ((int64_t)t0 + n - token[s]);
            }
        }
#pragma unroll
        for (int s = 0; s < S; s++) {
            pg[s] = kv_page_of(a, (int)(pos[s] >> 4));
            const bool in = pos[s] >= 0 && pos[s] <= INT32_MAX && pg[s] < a.max_pages;
            id[s] = in ? a.table[(int64_t)b[s] * a.max_pages + pg[s]] : -1;
        }
#pragma unroll
        for (int s = 0; s < S; s++) {
            key[s] = (int)(pos[s] - (int64_t)pg[s] * a.page);
            reg[s] = (uint32_t)id[s] < (uint32_t)a.n_pages ? a.data + ((int64_t)id[s] * a.heads + head[s]) * a.region : nullptr;
        }
    }
};

// A row: quantised and written.  (All lanes of the wave call it.)
template <int NG>
__device__ __forceinline__ void write_row(const KvArgs &a, const float (&xk)[8], const float (&xv)[8], uint8_t *reg, int key) {
    constexpr int RL = row_lanes<NG>(), D = 32 * NG;
    const int lane = threadIdx.x & 63;
    const int u = lane % RL, g = u >> 2, i = u & 3;
    const VLane<NG> vl(u);
    const bool on = reg && g < NG;
    // not finite: 0 * x is NaN
    float nk = 0.0f, nv = 0.0f, kh = xk[0], kl = xk[0], vh = xv[0], vlow = xv[0];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        nk += 0.0f * xk[e];
        nv += 0.0f * xv[e];
        kh = fmaxf(kh, xk[e]);
        kl = fminf(kl, xk[e]);
        vh = fmaxf(vh, xv[e]);
        vlow = fminf(vlow, xv[e]);
    }
    auto hi = [](float a, float b) { return fmaxf(a, b); };
    auto lo = [](float a, float b) { return fminf(a, b); };
    auto sum = [](float a, float b) { return a + b; };  // (NaN if one is)
    kh = hi(kh, dpp<0xb1>(kh));
    kh = hi(kh, dpp<0x4e>(kh));
    kl = lo(kl, dpp<0xb1>(kl));
    kl = lo(kl, dpp<0x4e>(kl));
    vh = VLane<NG>::all(vh, hi);
    vlow = VLane<NG>::all(vlow, lo);
    const uint64_t mine = ((1ull << RL) - 1) << (lane / RL * RL);
    const uint64_t bad = __ballot(nk != nk || nv != nv) & mine;
    nv = VLane<NG>::all(nv, sum);
    if (!on) return;
    const uint32_t dk = group_scale(kh, kl), dv = nv != nv ? 0u : group_scale(vh, vlow);
    const float fk = h2f(dk), fv = h2f(dv), rk = 1.0f / fk, rv = 1.0f / fv;
    uint32_t wk = 0, wv = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint32_t ck = fk == 0.0f || bad ? 8u : code_of(xk[e], fk, rk);
        const uint32_t cv = fv == 0.0f ? 8u : code_of(xv[e], fv, rv);
        wk |= ck << (4 * ((e >> 1) + 4 * (e & 1)));
        wv |= cv << (e < 4 ? 8 * e : 8 * (e - 4) + 4);
    }
    *(uint32_t *)(reg + (int64_t)key * (D / 2) + (i * NG + g) * 4) = wk;
    uint8_t *vc = reg + a.off_v + (key >> 2) * (64 * NG) + (key & 3) * NG;
    if constexpr (VLane<NG>::DWORDS) {
        *(uint32_t *)(vc + (u & 15) * (4 * NG) + (u >> 4) * 4) = quad_transpose(wv);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) vc[(4 * i + j) * 4 * NG + g] = (uint8_t)(wv >> (8 * j));
    }
    // a row with a value that is not finite: its key is NaN, as is what attends to it
    if (i == 0) ((uint16_t *)(reg + a.off_ks))[key * NG + g] = (uint16_t)(bad ? 0x7e00u : dk);
    if (vl.i == 0) ((uint16_t *)(reg + a.off_vs))[((key >> 2) * NG + vl.g) * 4 + (key & 3)] = (uint16_t)dv;
}

template <int NG>
__global__ __launch_bounds__(256) void kv_write_kernel(KvArgs a, const void *k, int64_t k_stride, const void *v,
                                                       int64_t v_stride, int f16, int rows) {
    constexpr int RL = row_lanes<NG>(), D = 32 * NG;
    const int row0 = __builtin_amdgcn_readfirstlane((block_of() * 4 + (threadIdx.x >> 6)) * (WAVE / RL));
    if (row0 >= rows) return;
    const Rows<RL, 1> r(a, row0, rows);
    const int u = threadIdx.x % RL, g = u >> 2, i = u & 3;
    const VLane<NG> vl(u);
    float xk[8], xv[8];
#pragma unroll
    for (int e = 0; e < 8; e++) xk[e] = xv[e] = 0.0f;
    if (r.reg[0] && g < NG) {
        const int64_t ok = r.token[0] * k_stride + r.head[0] * D + 32 * g, ov = r.token[0] * v_stride + r.head[0] * D + 32 * vl.g;
        load4(k, ok + 8 * i, f16, xk);
        load4(k, ok + 8 * i + 4, f16, xk + 4);
        load4(v, ov + 4 * vl.i, f16, xv);
        load4(v, ov + 4 * vl.i + 16, f16, xv + 4);
    }
    write_row<NG>(a, xk, xv, r.reg[0], r.key[0]);
}

template <int NG, int S, bool F16, bool PAST>
__global__ __launch_bounds__(256) void kv_read_kernel(KvArgs a, void *k, int64_t k_stride, void *v, int64_t v_stride,
                                                      int rows) {
    constexpr int RL = row_lanes<NG>(), D = 32 * NG;
    const int row0 = __builtin_amdgcn_readfirstlane((block_of() * 4 + (threadIdx.x >> 6)) * (WAVE / RL * S));
    if (row0 >= rows) return;
    const Rows<RL, S> r(a, row0, rows);
    const int u = threadIdx.x % RL, g = u >> 2, i = u & 3;
    const VLane<NG> vl(u);
    uint32_t wk[S], wv[S];
    uint16_t sk[S], sv[S];
#pragma unroll
    for (int s = 0; s < S; s++) {
        wk[s] = wv[s] = sk[s] = sv[s] = 0;
        if (!r.reg[s] || g >= NG) continue;
        const uint8_t *reg = r.reg[s];
        const int key = r.key[s];
        sk[s] = ((const uint16_t *)(reg + a.off_ks))[key * NG + g];
        sv[s] = ((const uint16_t *)(reg + a.off_vs))[((key >> 2) * NG + vl.g) * 4 + (key & 3)];
        wk[s] = *(const uint32_t *)(reg + (int64_t)key * (D / 2) + (i * NG + g) * 4);
        const uint8_t *vc = reg + a.off_v + (key >> 2) * (64 * NG) + (key & 3) * NG;
        if constexpr (VLane<NG>::DWORDS) {
            wv[s] = *(const uint32_t *)(vc + (u & 15) * (4 * NG) + (u >> 4) * 4);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) wv[s] |= (uint32_t)vc[(4 * i + j) * 4 * NG + g] << (8 * j);
        }
    }
#pragma unroll
    for (int s = 0; s < S; s++) {
        if (!r.reg[s] || g >= NG) continue;
        const float dk = h2f(sk[s]), dv = h2f(sv[s]);
        const uint32_t w = VLane<NG>::DWORDS ? quad_transpose(wv[s]) : wv[s];
        const int64_t ok = r.token[s] * k_stride + r.head[s] * D + 32 * g, ov = r.token[s] * v_stride + r.head[s] * D + 32 * vl.g;
        float xk[8], xv[8];
        // a quad stores 64 bytes of a group at a time: f16 as eight neighbours a lane, f32 as four, twice
        if constexpr (F16) {
            // V: of i and i ^ 1, the even one takes values 4i .. +7, the odd one 4i + 12 .. +7
            const uint32_t other = VLane<NG>::pair(w), odd = vl.i & 1;
            const uint32_t first = (odd ? other >> 4 : w) & 0x0f0f0f0fu, second = (odd ? w >> 4 : other) & 0x0f0f0f0fu;
#pragma unroll
            for (int e = 0; e < 8; e++) xk[e] = dk * (float)((int)(wk[s] >> (4 * ((e >> 1) + 4 * (e & 1))) & 15u) - 8);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                xv[e] = dv * (float)((int)byte_of(first, e) - 8);
                xv[4 + e] = dv * (float)((int)byte_of(second, e) - 8);
            }
            store16<PAST>((_Float16 *)k + ok + 8 * i, pack8(xk));
            store16<PAST>((_Float16 *)v + ov + 4 * vl.i + (odd ? 12 : 0), pack8(xv));
        } else {
            // K: values 4i .. +3 are half i % 2 of lane i / 2's, 16 + 4i .. +3 of lane 2 + i / 2's
            const uint32_t sh = (i & 1) * 8, wa = dpp<0x50>(wk[s]) >> sh, wb = dpp<0xfa>(wk[s]) >> sh;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int at = 4 * ((e >> 1) + 4 * (e & 1));
                xk[e] = dk * (float)((int)(wa >> at & 15u) - 8);
                xk[4 + e] = dk * (float)((int)(wb >> at & 15u) - 8);
                xv[e] = dv * (float)((int)byte_of(w & 0x0f0f0f0fu, e) - 8);
                xv[4 + e] = dv * (float)((int)byte_of(w >> 4 & 0x0f0f0f0fu, e) - 8);
            }
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                store16<PAST>((float *)k + ok + 4 * i + 4 * e, f32x4{xk[e], xk[e + 1], xk[e + 2], xk[e + 3]});
                store16<PAST>((float *)v + ov + 4 * vl.i + 4 * e, f32x4{xv[e], xv[e + 1], xv[e + 2], xv[e + 3]});
            }
        }
    }
}

// Sets of rows a wave reads: four where that still fills the chip (32 waves a compute unit), one otherwise
// (141000 tokens of f16 from eight sequences: one 253 us, four 194, eight 208, before the stores were non-temporal).  Writing keeps to one: its
// rows are wider in registers (345 MB in and out, f32: one 84 us, two 87, four 95).
constexpr int SETS = 4;
template <int NG, int S, class K, class... A>
hipError_t rows_launch(K kernel, const KvArgs &a, hipStream_t s, A... args) {
    const int64_t rows = (int64_t)a.tokens * a.heads, per = 4 * S * (WAVE / row_lanes<NG>());
    kernel<<<grid_of((rows + per - 1) / per), 256, 0, s>>>(a, args..., (int)rows);
    return hipGetLastError();
}
template <int NG, class... A>
hipError_t write_launch(const KvArgs &a, hipStream_t s, A... args) {
    return rows_launch<NG, 1>(kv_write_kernel<NG>, a, s, args...);
}
// f16 goes past the caches, f32 from PAST_BYTES on (the last cache has 256 MB; below, what follows finds it
// there).  us past them and not, 8 x 128, into three sets of rows in turn.  f16 alone: 2 MB 4.2 and 4.2, 20 MB 7.5
// and 9.1, 107 MB 29 and 31, 214 MB 52 and 65, 428 MB 92 and 148; with copies of the rows after it 43 MB 31.2 and
// 29.5, 107 MB 63 and 70.  f32 alone: 80 MB 23 and 20, 160 MB 52 and 34, 214 MB 67 and 48, 256 MB 79 and 78, 428 MB
// 129 and 145; with copies after it 80 MB 53 and 44, 128 MB 80 and 82, 256 MB 177 and 177.  Into the same rows
// again and again f32 gains from 214 MB on (56 and 77; 428 MB 127 and 144), which the border goes by; behind their
// writing 152 MB take 92 and 82 with it.
constexpr int64_t PAST_BYTES = (int64_t)192 << 20;
template <int NG, class... A>
hipError_t read_launch(const KvArgs &a, hipStream_t s, bool f16, A... args) {
    constexpr int64_t MANY = (int64_t)256 * 32 * SETS * (WAVE / row_lanes<NG>()), F32_BYTES = 2 * 32 * NG * sizeof(float);
    static_assert(MANY * F32_BYTES <= PAST_BYTES, "f32 rows that go past the caches are many");
    const int64_t rows = (int64_t)a.tokens * a.heads;
    if (f16)
        return rows >= MANY ? rows_launch<NG, SETS>(kv_read_kernel<NG, SETS, true, true>, a, s, args...)
                            : rows_launch<NG, 1>(kv_read_kernel<NG, 1, true, true>, a, s, args...);
    if (rows * F32_BYTES >= PAST_BYTES) return rows_launch<NG, SETS>(kv_read_kernel<NG, SETS, false, true>, a, s, args...);
    return rows >= MANY ? rows_launch<NG, SETS>(kv_read_kernel<NG, SETS, false, false>, a, s, args...)
                        : rows_launch<NG, 1>(kv_read_kernel<NG, 1, false, false>, a, s, args...);
}

}  // namespace

hipError_t launch_kv_write(const KvArgs &a, int dim, const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                           int dtype, hipStream_t s) {
    const int f16 = dtype == ARFQ_F16;
    switch (dim) {
    case 64: return write_launch<2>(a, s, k, k_stride, v, v_stride, f16);
    case 96: return write_launch<3>(a, s, k, k_stride, v, v_stride, f16);
    case 128: return write_launch<4>(a, s, k, k_stride, v, v_stride, f16);
    case 256: return write_launch<8>(a, s, k, k_stride, v, v_stride, f16);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_kv_read(const KvArgs &a, int dim, void *k, int64_t k_stride, void *v, int64_t v_stride, int dtype,
                          hipStream_t s) {
    const bool f16 = dtype == ARFQ_F16;
    switch (dim) {
    case 64: return read_launch<2>(a, s, f16, k, k_stride, v, v_stride);
    case 96: return read_launch<3>(a, s, f16, k, k_stride, v, v_stride);
    case 128: return read_launch<4>(a, s, f16, k, k_stride, v, v_stride);
    case 256: return read_launch<8>(a, s, f16, k, k_stride, v, v_stride);
    }
    return hipErrorInvalidValue;
}

}  // namespace arfq
