// arfq_kv.hip -- writing K and V rows into the 4-bit cache and reading them back.
#include "arfq_kv.h"

namespace arfq {
namespace {

// Lanes of a (token, head) row: four for each group of 32 values, up to a power of two
// (a row's lanes lie in one wave; D = 96 leaves four of its sixteen idle).
template <int NG>
constexpr int row_lanes() { return NG <= 2 ? 8 : NG <= 4 ? 16 : 32; }

__device__ __forceinline__ void load4(const void *p, int64_t i, bool f16, float *o) {
    if (f16) {
        const u32x2 w = *(const u32x2 *)((const _Float16 *)p + i);
        o[0] = h2f(w.x); o[1] = h2f(w.x >> 16); o[2] = h2f(w.y); o[3] = h2f(w.y >> 16);
    } else {
        const float4 w = *(const float4 *)((const float *)p + i);
        o[0] = w.x; o[1] = w.y; o[2] = w.z; o[3] = w.w;
    }
}

__device__ __forceinline__ void store4(void *p, int64_t i, bool f16, const float *o) {
    if (f16)
        *(u32x2 *)((_Float16 *)p + i) = u32x2{pack_f16x2(o[0], o[1]), pack_f16x2(o[2], o[3])};
    else
        *(float4 *)((float *)p + i) = make_float4(o[0], o[1], o[2], o[3]);
}

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

// Sequence of the wave's tokens t[0 .. R): sequences b with start[b + 1] <= t come before it,
// 64 compared at once.
template <int R>
__device__ __forceinline__ void find_seqs(const KvArgs &a, const int (&t)[R], int (&b)[R]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int r = 0; r < R; r++) b[r] = 0;
    for (int b0 = 0; b0 < a.batch; b0 += WAVE) {
        const int v = b0 + lane < a.batch ? a.start[b0 + lane + 1] : INT32_MAX;
#pragma unroll
        for (int r = 0; r < R; r++) b[r] += __popcll(__ballot(v <= t[r]));
    }
}

// The place in the cache of the row that this lane works on: its region (null: none) and its
// key within the page.  Rows are (token, head) pairs, head fastest.
template <int RL>
__device__ __forceinline__ uint8_t *place(const KvArgs &a, int64_t row0, int64_t rows, int &token, int &head, int &key) {
    constexpr int R = WAVE / RL;  // rows of a wave
    const int lane = threadIdx.x & 63;
    int ts[R], bs[R];
#pragma unroll
    for (int r = 0; r < R; r++) ts[r] = (int)(min(row0 + r, rows - 1) / a.heads);
    const int mine = lane / RL;
    const int64_t row = row0 + mine;
    token = (int)(min(row, rows - 1) / a.heads);
    head = (int)(min(row, rows - 1) - (int64_t)token * a.heads);
    int b = token;
    if (a.start) {
        find_seqs<R>(a, ts, bs);
        b = bs[0];
#pragma unroll
        for (int r = 1; r < R; r++) b = mine == r ? bs[r] : b;
    }
    if (row >= rows || b >= a.batch) return nullptr;
    int t0, n;
    kv_seq(a, b, t0, n);
    const int64_t pos = (int64_t)a.len[b] - ((int64_t)t0 + n - token);
    if (token < t0 || token >= t0 + n || pos < 0 || pos > INT32_MAX) return nullptr;
    const int tile = (int)(pos >> 4), pg = kv_page_of(a, tile);
    if (pg >= a.max_pages) return nullptr;
    const int id = a.table[(int64_t)b * a.max_pages + pg];
    if (id < 0 || id >= a.n_pages) return nullptr;
    key = (int)(pos - (int64_t)pg * a.page);
    return a.data + ((int64_t)id * a.heads + head) * a.region;
}

template <int NG>
__global__ __launch_bounds__(256) void kv_write_kernel(KvArgs a, const void *k, int64_t k_stride, const void *v,
                                                       int64_t v_stride, int f16, int64_t rows) {
    constexpr int RL = row_lanes<NG>(), D = 32 * NG;
    const int lane = threadIdx.x & 63;
    const int64_t row0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * (WAVE / RL);
    if (row0 >= rows) return;
    int token, head, key = 0;
    uint8_t *reg = place<RL>(a, row0, rows, token, head, key);
    const int u = lane % RL, g = u >> 2, i = u & 3;
    const bool on = reg && g < NG;
    float xk[8], xv[8];
#pragma unroll
    for (int e = 0; e < 8; e++) xk[e] = xv[e] = 0.0f;
    if (on) {
        const int64_t ok = token * k_stride + head * D + 32 * g, ov = token * v_stride + head * D + 32 * g;
        load4(k, ok + 8 * i, f16, xk);
        load4(k, ok + 8 * i + 4, f16, xk + 4);
        load4(v, ov + 4 * i, f16, xv);
        load4(v, ov + 4 * i + 16, f16, xv + 4);
    }
    // not finite: 0 * x is NaN
    float nk = 0.0f, nv = 0.0f, kh = xk[0], kl = xk[0], vh = xv[0], vl = xv[0];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        nk += 0.0f * xk[e];
        nv += 0.0f * xv[e];
        kh = fmaxf(kh, xk[e]);
        kl = fminf(kl, xk[e]);
        vh = fmaxf(vh, xv[e]);
        vl = fminf(vl, xv[e]);
    }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
        kh = fmaxf(kh, __shfl_xor(kh, x));
        kl = fminf(kl, __shfl_xor(kl, x));
        vh = fmaxf(vh, __shfl_xor(vh, x));
        vl = fminf(vl, __shfl_xor(vl, x));
    }
    const uint64_t quad = 0xfull << (lane & ~3);
    const uint64_t mine = (RL == 64 ? ~0ull : ((1ull << RL) - 1)) << (lane / RL * RL);
    const uint64_t bad_v = __ballot(nv != 0.0f || nv != nv), bad = (__ballot(nk != 0.0f || nk != nk) | bad_v) & mine;
    if (!on) return;
    uint32_t dk = group_scale(kh, kl), dv = bad_v & quad ? 0u : group_scale(vh, vl);
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
    uint8_t *vc = reg + a.off_v + (key >> 2) * (64 * NG) + (key & 3) * NG + g;
#pragma unroll
    for (int j = 0; j < 4; j++) vc[(4 * i + j) * 4 * NG] = (uint8_t)(wv >> (8 * j));
    if (i == 0) {
        // a row with a value that is not finite: its key is NaN, as is what attends to it
        const int at = ((key >> 2) * NG + g) * 4 + (key & 3);
        ((uint16_t *)(reg + a.off_ks))[key * NG + g] = (uint16_t)(bad ? 0x7e00u : dk);
        ((uint16_t *)(reg + a.off_vs))[at] = (uint16_t)dv;
    }
}

template <int NG>
__global__ __launch_bounds__(256) void kv_read_kernel(KvArgs a, void *k, int64_t k_stride, void *v, int64_t v_stride,
                                                      int f16, int64_t rows) {
    constexpr int RL = row_lanes<NG>(), D = 32 * NG;
    const int lane = threadIdx.x & 63;
    const int64_t row0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * (WAVE / RL);
    if (row0 >= rows) return;
    int token, head, key = 0;
    const uint8_t *reg = place<RL>(a, row0, rows, token, head, key);
    const int u = lane % RL, g = u >> 2, i = u & 3;
    if (!reg || g >= NG) return;
    const int at = ((key >> 2) * NG + g) * 4 + (key & 3);
    const float dk = h2f(((const uint16_t *)(reg + a.off_ks))[key * NG + g]), dv = h2f(((const uint16_t *)(reg + a.off_vs))[at]);
    const uint32_t wk = *(const uint32_t *)(reg + (int64_t)key * (D / 2) + (i * NG + g) * 4);
    const uint8_t *vc = reg + a.off_v + (key >> 2) * (64 * NG) + (key & 3) * NG + g;
    float xk[8], xv[8];
#pragma unroll
    for (int e = 0; e < 8; e++) xk[e] = dk * (float)((int)(wk >> (4 * ((e >> 1) + 4 * (e & 1))) & 15u) - 8);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t b = vc[(4 * i + j) * 4 * NG];
        xv[j] = dv * (float)((int)(b & 15u) - 8);
        xv[4 + j] = dv * (float)((int)(b >> 4) - 8);
    }
    const int64_t ok = token * k_stride + head * D + 32 * g, ov = token * v_stride + head * D + 32 * g;
    store4(k, ok + 8 * i, f16, xk);
    store4(k, ok + 8 * i + 4, f16, xk + 4);
    store4(v, ov + 4 * i, f16, xv);
    store4(v, ov + 4 * i + 16, f16, xv + 4);
}

template <int NG, class K, class... A>
hipError_t rows_launch(K kernel, const KvArgs &a, hipStream_t s, A... args) {
    const int64_t rows = (int64_t)a.tokens * a.heads, per = 4 * (WAVE / row_lanes<NG>());
    kernel<<<dim3((unsigned)((rows + per - 1) / per)), 256, 0, s>>>(a, args..., rows);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_write(const KvArgs &a, int dim, const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                           int dtype, hipStream_t s) {
    const int f16 = dtype == ARFQ_F16;
    switch (dim) {
    case 64: return rows_launch<2>(kv_write_kernel<2>, a, s, k, k_stride, v, v_stride, f16);
    case 96: return rows_launch<3>(kv_write_kernel<3>, a, s, k, k_stride, v, v_stride, f16);
    case 128: return rows_launch<4>(kv_write_kernel<4>, a, s, k, k_stride, v, v_stride, f16);
    case 256: return rows_launch<8>(kv_write_kernel<8>, a, s, k, k_stride, v, v_stride, f16);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_kv_read(const KvArgs &a, int dim, void *k, int64_t k_stride, void *v, int64_t v_stride, int dtype,
                          hipStream_t s) {
    const int f16 = dtype == ARFQ_F16;
    switch (dim) {
    case 64: return rows_launch<2>(kv_read_kernel<2>, a, s, k, k_stride, v, v_stride, f16);
    case 96: return rows_launch<3>(kv_read_kernel<3>, a, s, k, k_stride, v, v_stride, f16);
    case 128: return rows_launch<4>(kv_read_kernel<4>, a, s, k, k_stride, v, v_stride, f16);
    case 256: return rows_launch<8>(kv_read_kernel<8>, a, s, k, k_stride, v, v_stride, f16);
    }
    return hipErrorInvalidValue;
}

}  // namespace arfq
