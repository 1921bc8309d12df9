// arfq_lora.hip -- low-rank adapters of many requests beside a shared projection:
// out[t] = base[t] + scale_e B_e (A_e x[t]), e = ids[t].
//
// Two launches, where A_e x takes little one.  The first forms parts of h = A_e x over ranges of k, [splits][rows][rank] in
// f32; the second adds the parts in order, and B_e h to base.  Few rows: a workgroup has one row (and a range of k, or of n)
// on the vector unit, products in f32.  Many rows: tiles of neighbouring rows on the matrix cores, once for each adapter that the
// tile's rows name; an f32 x goes through v_mfma_f32_16x16x4_f32 as it is, an f16 x is exact in f16 operands, and h
// enters the second product as two f16 parts of 22 bits of the row's largest.  Every adapter has accumulators of its own: a NaN
// in one does not reach another's rows.  Bound by memory and latency: 64 rows of 32 adapters, 5120 x 7168, rank 16, 17.6 MB
// in 8.6 us (4.1 and 5.2 of it on the device: the row's id, then what it names); 2048 rows of four, 5120 x 17408, rank 64,
// f16, 318 MB in 84: 18, of which the f16 products are 3, and 68 for base and out at 4.5 TB/s (rank 16: 10 and 55).
#include "arfq_step.h"

#include <math.h>

#include <type_traits>

namespace arfq {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

constexpr int K_PART = 512;  // values of k of a workgroup with one row: eight a lane

__device__ __forceinline__ int id_of(const LoraArgs &a, int t) {
    const int e = a.ids[t];
    return e >= 0 && e < a.l.adapters ? e : -1;
}

__device__ __forceinline__ f16x8 zero8() { return f16x8{0, 0, 0, 0, 0, 0, 0, 0}; }

// Eight values of x from element i on.
template <bool F16>
__device__ __forceinline__ void load8(const void *x, int64_t i, float (&o)[8]) {
    if constexpr (F16) {
        const f16x8 v = *(const f16x8 *)((const _Float16 *)x + i);
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (float)v[e];
    } else {
        const f32x4 v = *(const f32x4 *)((const float *)x + i), w = *(const f32x4 *)((const float *)x + i + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            o[e] = v[e];
            o[4 + e] = w[e];
        }
    }
}

// The same as a vector.  (x is 16-byte aligned, an f32x8 would have to be 32.)
__device__ __forceinline__ f16x8 eight(const _Float16 *x) { return *(const f16x8 *)x; }
__device__ __forceinline__ f32x8 eight(const float *x) {
    const f32x4 v = *(const f32x4 *)x, w = *(const f32x4 *)(x + 4);
    return __builtin_shufflevector(v, w, 0, 1, 2, 3, 4, 5, 6, 7);
}

// ---- few rows ----

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
// Sum over N neighbouring lanes, in each of them.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (N >= 2) v += dpp<0xb1>(v);    // quad_perm:[1,0,3,2]
    if constexpr (N >= 4) v += dpp<0x4e>(v);    // quad_perm:[2,3,0,1]
    if constexpr (N >= 8) v += dpp<0x141>(v);   // row_half_mirror
    if constexpr (N >= 16) v += dpp<0x140>(v);  // row_mirror
    if constexpr (N >= 32) v += __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401f));  // lane ^ 16
    if constexpr (N == 64)
        v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 0)) +
            __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 32));
    return v;
}

template <bool F16>
__global__ __launch_bounds__(256) void lora_rows_a(LoraArgs a, int splits) {
    const int block = block_of(), t = block / splits, part = block - t * splits;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= a.rows) return;
    const int rank = (int)a.l.rank;
    const int64_t k = (int64_t)part * K_PART + 8 * lane;
    const bool on = k < a.l.k;
    const int e = id_of(a, t);
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (on) load8<F16>(a.x, t * a.l.k + k, x);
    if (e < 0) return;
    const _Float16 *A = (const _Float16 *)a.l.a + (int64_t)e * rank * a.l.k + k;
    float *h = a.h + ((int64_t)part * a.rows + t) * rank;
    constexpr int U = 4;  // (a wave has every fourth run of as many ranks: 8 divides the rank)
    for (int r0 = wave * U; r0 < rank; r0 += 4 * U) {
        f16x8 w[U];
#pragma unroll
        for (int u = 0; u < U; u++) w[u] = on ? *(const f16x8 *)(A + (r0 + u) * a.l.k) : zero8();
        float s[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            s[u] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) s[u] = __builtin_fmaf((float)w[u][i], x[i], s[u]);
            s[u] = lanes_sum<64>(s[u]);
        }
        if (lane == 0) *(f32x4 *)(h + r0) = f32x4{s[0], s[1], s[2], s[3]};
    }
}

// Outputs n0 .. of a row, 64 W of them: LP lanes have an output, eight ranks each.  B and base of the first eight that a lane
// has a part in are loaded by begin(), before h is known.
template <int LP, int W>
struct Outputs {
    static constexpr int U = LP < 8 ? LP : 8, APART = 64 * W / LP;  // outputs of LP lanes at once; of a lane and the next
    const float *base;
    float *out;
    const _Float16 *B;
    int64_t n, n0;
    int rank, u;
    bool on;
    f16x8 w[U];
    float own[U];
    __device__ __forceinline__ void load(int j0) {
#pragma unroll
        for (int j = 0; j < U; j++) {
            const int64_t at = n0 + (j0 + j) * APART + threadIdx.x / LP;
            w[j] = on && at < n ? *(const f16x8 *)(B + at * rank) : zero8();
            own[j] = base && u == 0 && at < n ? base[at] : 0.0f;
        }
    }
    __device__ __forceinline__ Outputs(const LoraArgs &a, int t, int e, int64_t n0)
        : base(a.base ? a.base + t * a.base_stride : nullptr), out(a.out + t * a.out_stride), n(a.l.n), n0(n0), rank((int)a.l.rank),
          u(threadIdx.x % LP), on(8 * u < rank) {
        B = (const _Float16 *)a.l.b + (int64_t)e * n * rank + 8 * u;
    }
    // (a row without an adapter)
    __device__ __forceinline__ void copy() {
        const int64_t at = n0 + threadIdx.x;
        if (at < n && base != out) out[at] = base ? base[at] : 0.0f;
    }
    __device__ __forceinline__ void finish(const float *sh) {
        float h[8];
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = on ? sh[8 * u + i] : 0.0f;
#pragma unroll 1
        for (int j0 = 0; j0 < LP; j0 += U) {
            if (j0 > 0) load(j0);
#pragma unroll
            for (int j = 0; j < U; j++) {
                float v = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) v = __builtin_fmaf((float)w[j][i], h[i], v);
                v = lanes_sum<LP>(v);
                const int64_t at = n0 + (j0 + j) * APART + threadIdx.x / LP;
                if (u == 0 && at < n) out[at] = own[j] + v;
            }
        }
    }
};

template <int LP>
__global__ __launch_bounds__(256) void lora_rows_b(LoraArgs a, int splits, int parts) {
    __shared__ float sh[LORA_RANK_MAX];
    const int block = block_of(), t = block / parts, part = block - t * parts;
    if (t >= a.rows) return;
    const int e = id_of(a, t), rank = (int)a.l.rank;
    Outputs<LP, 4> o(a, t, e, (int64_t)part * 256);
    if (e < 0) return o.copy();
    float s = 0.0f;
    if ((int)threadIdx.x < rank) {
#pragma unroll 8
        for (int p = 0; p < splits; p++) s += a.h[((int64_t)p * a.rows + t) * rank + threadIdx.x];
        if (a.l.scale) s *= a.l.scale[e];
    }
    o.load(0);
    if ((int)threadIdx.x < rank) sh[threadIdx.x] = s;
    lds_barrier();
    o.finish(sh);
}

// Both products in one launch, where A_e x takes little: each workgroup forms it for itself.  The waves share the ranks, four
// a wave, and where these are fewer, k.  (Four waves for sixteen: 0.1 us slower at the smallest sizes, twice the time at the
// largest.)
constexpr int ONE_WAVES = 16, ONE_OUT = 64 * ONE_WAVES;  // outputs of a workgroup
template <int LP>
__global__ __launch_bounds__(64 * ONE_WAVES) void lora_rows_ab(LoraArgs a, int parts) {
    constexpr int W = ONE_WAVES;
    constexpr int R = 2 * LP < W ? 2 * LP : W;  // waves side by side on ranks (LP lanes: 8 LP ranks at most)
    constexpr int K = W / R;
    __shared__ __align__(16) float sh[K][LORA_RANK_MAX];
    const int block = block_of(), t = block / parts, part = block - t * parts;
    if (t >= a.rows) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rw = wave % R, kw = wave / R;
    const int e = id_of(a, t), rank = (int)a.l.rank;
    Outputs<LP, W> o(a, t, e, (int64_t)part * 64 * W);
    if (e < 0) return o.copy();
    const _Float16 *A = (const _Float16 *)a.l.a + (int64_t)e * rank * a.l.k;
    const float scale = a.l.scale ? a.l.scale[e] : 1.0f;
    o.load(0);
    constexpr int U = 4;
    for (int r0 = rw * U; r0 < rank; r0 += R * U) {
        float s[U] = {0, 0, 0, 0};
#pragma unroll 2
        for (int64_t k = 512 * kw + 8 * lane; k < a.l.k; k += 512 * K) {
            float x[8];
            if (a.x_f16) load8<true>(a.x, t * a.l.k + k, x);
            else load8<false>(a.x, t * a.l.k + k, x);
            f16x8 w[U];
#pragma unroll
            for (int u = 0; u < U; u++) w[u] = *(const f16x8 *)(A + (r0 + u) * a.l.k + k);
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < 8; i++) s[u] = __builtin_fmaf((float)w[u][i], x[i], s[u]);
        }
#pragma unroll
        for (int u = 0; u < U; u++) s[u] = lanes_sum<64>(s[u]);
        if (lane == 0) *(f32x4 *)&sh[kw][r0] = f32x4{s[0], s[1], s[2], s[3]};
    }
    lds_barrier();
    if ((int)threadIdx.x < rank) {
        float s = sh[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < K; i++) s += sh[i][threadIdx.x];
        sh[0][threadIdx.x] = s * scale;
    }
    lds_barrier();
    o.finish(sh[0]);
}

// ---- many rows ----

constexpr int TR = 16;  // rows of a tile: a matrix instruction's columns

// Workgroups go to the eight XCDs in turn: this numbering gives each of them a run of neighbouring items instead, so that an
// adapter's A or B is fetched into few L2s.
__device__ __forceinline__ int xcd_run(int block, int blocks) {
    const int per = blocks / 8;
    return block < 8 * per ? block % 8 * per + block / 8 : block;
}

// The adapters that the rows of tiles name, one after another (`mine`: those of this lane's rows; the same in all lanes of
// a row; -1: none).  Returns the next one, or -2 behind the last; done: the lanes whose rows are served.
template <int N>
__device__ __forceinline__ int next_id(const int (&mine)[N], uint64_t (&done)[N]) {
    int e = -2;
#pragma unroll
    for (int s = 0; s < N; s++)
        if (e == -2 && done[s] != ~0ull) e = __builtin_amdgcn_readlane(mine[s], __ffsll((unsigned long long)~done[s]) - 1);
#pragma unroll
    for (int s = 0; s < N; s++) done[s] |= __ballot(mine[s] == e);
    return e;
}
__device__ __forceinline__ int next_id(int mine, uint64_t &done) {
    if (done == ~0ull) return -2;
    const int e = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)~done) - 1);
    done |= __ballot(mine == e);
    return e;
}

// RT 16-rank tiles of h, two tiles of rows, a part of k in four by the waves, whose sums are added through LDS.  A step is
// 32 values of k: eight neighbouring ones a lane.
constexpr int A_WAVES = 4, A_TILES = 2;
template <int RT, class X>
struct Operands {
    f16x8 w[RT];
    X x[A_TILES];
};
template <int RT, bool F16>
__global__ __launch_bounds__(64 * A_WAVES, 2) void lora_tiles_a(LoraArgs a, int splits, int k_part, int ranks, int shares, int groups) {
    __shared__ f32x4 sh[A_WAVES][A_TILES][RT][64];
    int block = block_of();
    const int share = block / groups;  // (slowest: those with nothing to do come last)
    block -= share * groups;
    block = xcd_run(block, groups);
    const int rb = block % ranks;
    block /= ranks;
    const int part = block % splits, t0 = block / splits * (A_TILES * TR);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    if (share >= shares) return;
    const int rank = (int)a.l.rank, r0 = rb * RT * 16;
    const int64_t k = a.l.k;
    // the wave's range, in steps of 32: eight values a lane
    const int64_t lo = (int64_t)part * k_part + (int64_t)wave * (k_part / A_WAVES), hi = min(lo + k_part / A_WAVES, k);
    int mine[A_TILES];
#pragma unroll
    for (int s = 0; s < A_TILES; s++) mine[s] = t0 + 16 * s + c < a.rows ? id_of(a, t0 + 16 * s + c) : -1;
    using T = std::conditional_t<F16, _Float16, float>;
    using X = std::conditional_t<F16, f16x8, f32x8>;
    const T *xp[A_TILES];
#pragma unroll
    for (int s = 0; s < A_TILES; s++) xp[s] = (const T *)a.x + min(t0 + 16 * s + c, a.rows - 1) * k + lo + 8 * g;
    uint64_t done[A_TILES] = {};
    for (int e, turn = 0; (e = next_id(mine, done)) != -2;) {
        if (e < 0 || turn++ % shares != share) continue;
        f32x4 acc[A_TILES][RT];
#pragma unroll
        for (int s = 0; s < A_TILES; s++)
#pragma unroll
            for (int i = 0; i < RT; i++) acc[s][i] = f32x4{0, 0, 0, 0};
        const _Float16 *A = (const _Float16 *)a.l.a + (int64_t)e * rank * k;
        const _Float16 *wp[RT];
#pragma unroll
        for (int i = 0; i < RT; i++) wp[i] = A + min(r0 + 16 * i + c, rank - 1) * k + lo + 8 * g;
        constexpr int DEPTH = 4;
        Operands<RT, X> ring[DEPTH];
        auto load = [&](Operands<RT, X> &o, int64_t at, bool on) {
#pragma unroll
            for (int i = 0; i < RT; i++) o.w[i] = on ? *(const f16x8 *)(wp[i] + at) : zero8();
#pragma unroll
            for (int s = 0; s < A_TILES; s++) o.x[s] = on ? eight(xp[s] + at) : X{};
        };
        auto add = [&](const Operands<RT, X> &o) {
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int s = 0; s < A_TILES; s++) {
                    if constexpr (F16) {
                        acc[s][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(o.w[i], o.x[s], acc[s][i], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            acc[s][i] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)o.w[i][j], o.x[s][j], acc[s][i], 0, 0, 0);
                    }
                }
        };
        // loads DEPTH steps ahead of their use; the range's last, shorter step by itself
        const int64_t whole = max(hi - lo, (int64_t)0) & ~(int64_t)31;
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
            if (32 * d < whole) load(ring[d], 32 * d, true);
#pragma unroll 1
        for (int64_t at = 0; at < whole; at += 32 * DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                if (at + 32 * d < whole) add(ring[d]);
                if (at + 32 * (d + DEPTH) < whole) load(ring[d], at + 32 * (d + DEPTH), true);
            }
        }
        if (lo + whole < hi) {
            load(ring[0], whole, lo + whole + 8 * g < hi);
            add(ring[0]);
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < A_TILES; s++)
#pragma unroll
            for (int i = 0; i < RT; i++) sh[wave][s][i][lane] = acc[s][i];
        __syncthreads();
        // a lane's four results: ranks 4g .. +3 of a tile, row c
#pragma unroll
        for (int s = 0; s < A_TILES; s++)
            for (int i = wave; i < RT; i += A_WAVES) {
                f32x4 v = sh[0][s][i][lane];
#pragma unroll
                for (int u = 1; u < A_WAVES; u++) v += sh[u][s][i][lane];
                const int r = r0 + 16 * i + 4 * g;
                if (mine[s] == e && r < rank) *(f32x4 *)(a.h + ((int64_t)part * a.rows + t0 + 16 * s + c) * rank + r) = v;
            }
    }
}

// TileB::ROWS rows at most, of KS runs of 32 ranks.  Their h first, into LDS: the parts added, and as two f16 parts of it times a power of
// two that puts a row's largest into [2^14, 2^15).  Then each wave has 16 NT outputs and goes over the rows' tiles: B_e
// stays in registers while the adapter does, base is loaded a tile ahead.
// A lane's results are four outputs of each of NT tiles, its neighbours' those of the next rows; they are exchanged
// for a piece of as many rows, so that a load of base or a store has 64 NT contiguous bytes of a row (2048 rows of 17408 outputs,
// rank 16: 59 us for 66 with 64 bytes).
constexpr int B_WAVES = 4;
template <int CTRL>
__device__ __forceinline__ void exchange(f32x4 &a, f32x4 &b, bool upper) {  // b of the lower lane for a of the upper
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float got = dpp<CTRL>(upper ? a[i] : b[i]);
        if (upper) a[i] = got;
        else b[i] = got;
    }
}
// Of NT neighbouring lanes: v[j] of lane p becomes v[p] of lane j.
template <int NT>
__device__ __forceinline__ void turn_lanes(f32x4 (&v)[NT]) {
    const int p = threadIdx.x;
#pragma unroll
    for (int i = 0; i < NT; i += 2) exchange<0xb1>(v[i], v[i + 1], p & 1);  // quad_perm:[1,0,3,2]
    if constexpr (NT == 4) {
        exchange<0x4e>(v[0], v[2], p & 2);  // quad_perm:[2,3,0,1]
        exchange<0x4e>(v[1], v[3], p & 2);
    }
}
template <int KS>
struct TileB {
    static constexpr int ROWS = KS <= 4 ? 64 : 32, NT = KS <= 4 ? 4 : 2, RANK = 32 * KS, LD = RANK + 8, OUT = B_WAVES * NT * 16;
};
// Base and out four at a time, at any address of a float.  PAST: past the caches.  `span`: rows of a workgroup, up to ROWS.
// (Three waves a SIMD at two runs, whose registers would be two's: 2048 rows of 17408 outputs 70 us for 80.)
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
template <int KS, bool PAST>
__global__ __launch_bounds__(64 * B_WAVES, KS == 2 ? 3 : 1) void lora_tiles_b(LoraArgs a, int splits, int parts, int span) {
    using T = TileB<KS>;
    constexpr int NT = T::NT, ROWS = T::ROWS;
    __shared__ __align__(16) _Float16 sh[2][ROWS][T::LD];
    __shared__ __align__(16) float unit[ROWS];
    __shared__ __align__(16) int ids[ROWS];
    const int block = block_of(), part = block % parts, t0 = block / parts * span;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    if (t0 >= a.rows) return;
    const int rank = (int)a.l.rank, rows = min(span, a.rows - t0);
    const int64_t n = a.l.n, n0 = (int64_t)part * T::OUT + wave * (NT * 16);
    // behind the exchange: rows c0 .. of a tile, outputs `own` ..
    const int c0 = c & ~(NT - 1);
    const int64_t own = n0 + 16 * (c & (NT - 1)) + 4 * g;
    const int left = (int)max((int64_t)0, min(n - own, (int64_t)4));  // of its four outputs
    f32x4 next[NT];  // base of the tile to come
    auto load_base = [&](int s) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int at = 16 * s + c0 + j;
            next[j] = f32x4{0, 0, 0, 0};
            if (!a.base || at >= rows) continue;
            const float *from = a.base + (int64_t)(t0 + at) * a.base_stride + own;
            if (left == 4) {
                next[j] = PAST ? __builtin_nontemporal_load((const f32x4_any *)from) : *(const f32x4_any *)from;
            } else {
#pragma unroll
                for (int i = 0; i < 3; i++)
                    if (i < left) next[j][i] = from[i];
            }
        }
    };
    f16x8 w[NT][KS];
    auto load_b = [&](int e) {
        const _Float16 *B = (const _Float16 *)a.l.b + (int64_t)e * n * rank;
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int q = 0; q < KS; q++)
                w[i][q] = 32 * q + 8 * g < rank ? *(const f16x8 *)(B + min(n0 + 16 * i + c, n - 1) * rank + 32 * q + 8 * g) : zero8();
    };
    // (loads in the order of their use: ids, h, B of the first row, base)
    constexpr int LANES = 4 * KS, ITEMS = ROWS * LANES / (64 * B_WAVES);  // eight ranks of a row
    int of[ITEMS];
    float h[ITEMS][8];
    const int u = threadIdx.x % LANES, row0 = threadIdx.x / LANES;
    constexpr int APART = 64 * B_WAVES / LANES;
#pragma unroll
    for (int it = 0; it < ITEMS; it++) {
        of[it] = row0 + it * APART < rows ? id_of(a, t0 + row0 + it * APART) : -1;
#pragma unroll
        for (int j = 0; j < 8; j++) h[it][j] = 0.0f;
    }
    int loaded = id_of(a, t0);
#pragma unroll 2
    for (int p = 0; p < splits; p++)
#pragma unroll
        for (int it = 0; it < ITEMS; it++) {
            if (it * APART >= rows) continue;
            float v[8];
            load8<false>(a.h, ((int64_t)p * a.rows + min(t0 + row0 + it * APART, a.rows - 1)) * rank + min(8 * u, rank - 8), v);
#pragma unroll
            for (int j = 0; j < 8; j++) h[it][j] += v[j];
        }
    loaded = __builtin_amdgcn_readfirstlane(loaded);
    if (loaded >= 0) load_b(loaded);
    load_base(0);
#pragma unroll
    for (int it = 0; it < ITEMS; it++) {
        const int row = row0 + it * APART, e = of[it];
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (e < 0 || 8 * u >= rank) h[it][j] = 0.0f;  // (what was loaded is not this row's)
            top = fmaxf(top, fabsf(h[it][j]));
        }
#pragma unroll
        for (int d = 1; d < LANES; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
        const int ex = min(max(top > 0.0f ? 141 - (int)(__builtin_bit_cast(uint32_t, top) >> 23) : 0, -126), 126);
        const float up = __builtin_bit_cast(float, (uint32_t)(ex + 127) << 23);
        f16x8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float v = h[it][j] * up;
            hi[j] = (_Float16)v;
            lo[j] = fabsf(v) == INFINITY ? (_Float16)0 : (_Float16)(v - (float)hi[j]);
        }
        *(f16x8 *)&sh[0][row][8 * u] = hi;
        *(f16x8 *)&sh[1][row][8 * u] = lo;
        if (u == 0) {
            ids[row] = e;
            unit[row] = __builtin_bit_cast(float, (uint32_t)(127 - ex) << 23) * (e >= 0 && a.l.scale ? a.l.scale[e] : 1.0f);
        }
    }
    lds_barrier();
    if (n0 >= n) return;
#pragma unroll 1
    for (int s = 0; 16 * s < rows; s++) {
        f32x4 base[NT];
#pragma unroll
        for (int i = 0; i < NT; i++) base[i] = next[i];
        if (16 * (s + 1) < rows) load_base(s + 1);
        const int mine = ids[16 * s + c];
        uint64_t done = 0;
        for (int e; (e = next_id(mine, done)) != -2;) {
            f32x4 acc[NT];
#pragma unroll
            for (int i = 0; i < NT; i++) acc[i] = f32x4{0, 0, 0, 0};
            if (e >= 0) {
                if (e != loaded) load_b(e);
                loaded = e;
#pragma unroll
                for (int q = 0; q < KS; q++)
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        const f16x8 h = *(const f16x8 *)&sh[p][16 * s + c][32 * q + 8 * g];
#pragma unroll
                        for (int i = 0; i < NT; i++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[i][q], h, acc[i], 0, 0, 0);
                    }
            }
            if (e >= 0) turn_lanes<NT>(acc);
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const int at = 16 * s + c0 + j;
                if (at >= rows || ids[at] != e) continue;
                float *o = a.out + (int64_t)(t0 + at) * a.out_stride;
                if (e < 0 && a.base && a.base + (int64_t)(t0 + at) * a.base_stride == o) continue;
                const f32x4 v = e < 0 ? base[j] : base[j] + acc[j] * unit[at];
                if (left == 4) {
                    if (PAST) __builtin_nontemporal_store(v, (f32x4_any *)(o + own));
                    else *(f32x4_any *)(o + own) = v;
                } else {
#pragma unroll
                    for (int i = 0; i < 3; i++)
                        if (i < left) o[own + i] = v[i];
                }
            }
        }
    }
}

// rows * (k + n) * (rank + 8) above which rows are taken in tiles; twice that for an f32 x, whose products there are eight for an f16
// x's one, and twice that again where k passes 3 / 2 n, as a tile forms A_e x anew for each adapter that it names.  The ids are on
// the device: the border stands where rows in runs lose about as large a factor one by one as mixed rows lose in tiles.  us one by one and in
// tiles, rows of two adapters in two runs / rows of 32 in any order; 5120 x 7168, f16 x: rank 16, 512 rows (1.5e8) 29 and 18 / 30
// and 61, 1024 rows (3.02e8) 51 and 23 / 52 and 111; rank 64, 256 rows (2.3e8) 29 and 18.6 / 44 and 65, 512 rows (4.5e8) 48 and
// 23.5 / 74 and 111; rank 128, 128 rows (2.1e8) 29 and 20 / 46 and 70, 256 rows (4.3e8) 50 and 25.5 / 91 and 114; f32 x, rank 16, 1024 rows
// 51 and 25 / 52 and 148, 2048 rows (6.04e8) 113 and 47 / 115 and 273.  4096 x 1024, rank 64, f16, 1024 rows (3.8e8) 36 and 19 /
// 38 and 104, 2048 rows (7.5e8) 64 and 26 / 67 and 193.  Over 377 sizes the factors are at most 1.5 apart on the side that is taken for an f16 x; for an
// f32 x with k far above n mixed rows lose more there (2048 rows of 8192 x 512, rank 64, 100 and 51 / 107 and 549).
constexpr int64_t TILE_WORK = 300 * 1000 * 1000;
bool in_tiles(const arfq_lora &l, int64_t rows, bool x_f16) {
    const int64_t most = TILE_WORK * (x_f16 ? 1 : 2) * (2 * l.k > 3 * l.n ? 2 : 1);
    return rows * (l.k + l.n) > most / (l.rank + 8);
}

// Values of A_e, and of it over all workgroups, up to which both products of rows one by one are one launch.  us in one and
// in two: k = n = 512, rank 16, any rows up to 256 4.3 and 6.8; k = n = 2048, rank 64 (2^17 of A), one row 7.1 and 8.2;
// k = 5120, n = 17408, rank 16, 8 rows (11 M) 5.4 and 6.6; k = n = 2048, rank 64, 64 rows (17 M) 9.1 and 8.8; k = 1024,
// n = 4096, rank 16, 256 rows (17 M) 12.3 and 9.6; k = 17408, rank 16 (2^18), one row 8.7 and 6.7.
// And not in more workgroups than two a compute unit, one above rank 32 (a unit's registers hold one at a time): 512 of them at k = n =
// 512, rank 16 6.5 and 7.6, 1024 11.3 and 7.7; k = n = 64, rank 8, 2048 17 and 7.6; rank 64, k = n = 256, 256 5.7 and 7.7, 512 9.7 and 7.9.
constexpr int64_t ONE_A = 1 << 17, ONE_READ = 12 << 20;

template <int LP>
hipError_t rows_b(const LoraArgs &a, const LoraPlan &p, hipStream_t s) {
    const int64_t parts = (a.l.n + (p.one ? ONE_OUT : 256) - 1) / (p.one ? ONE_OUT : 256);
    const dim3 grid = grid_of(a.rows * parts);
    if (p.one) lora_rows_ab<LP><<<grid, 64 * ONE_WAVES, 0, s>>>(a, (int)parts);
    else lora_rows_b<LP><<<grid, 256, 0, s>>>(a, p.splits, (int)parts);
    return hipGetLastError();
}

template <int RT>
hipError_t tiles_a(const LoraArgs &a, const LoraPlan &p, hipStream_t s) {
    const int ranks = (int)((a.l.rank + RT * 16 - 1) / (RT * 16));
    const int64_t groups = (int64_t)((a.rows + A_TILES * TR - 1) / (A_TILES * TR)) * p.splits * ranks;
    // a tile's adapters are shared by workgroups, two at least (those with nothing to do end at once): otherwise the tile in
    // which one adapter's rows end and another's begin takes twice as long as any other
    const int shares = (int)std::min<int64_t>(std::max<int64_t>(512 / groups, 2), A_TILES * TR);
    const dim3 grid = grid_of(groups * shares);
    if (a.x_f16) lora_tiles_a<RT, true><<<grid, 64 * A_WAVES, 0, s>>>(a, p.splits, p.k_part, ranks, shares, (int)groups);
    else lora_tiles_a<RT, false><<<grid, 64 * A_WAVES, 0, s>>>(a, p.splits, p.k_part, ranks, shares, (int)groups);
    return hipGetLastError();
}

// Bytes of base and out from which on they go past the caches.  us past them / through: rank 64, k = 5120, 2048 rows of 17408
// outputs (285 MB) 86 / 92, 1024 rows (143) 56.5 / 59; 2048 rows of 5120 (84) 43 / 39, 512 rows of 17408 (71) 37 / 34.
constexpr int64_t PAST_BYTES = (int64_t)112 << 20;

template <int KS>
hipError_t tiles_b(const LoraArgs &a, const LoraPlan &p, int cus, hipStream_t s) {
    const int parts = (int)((a.l.n + TileB<KS>::OUT - 1) / TileB<KS>::OUT);
    // fewer rows a workgroup where these would not fill the chip (701 rows of 138 outputs, rank 40: 9.3 us for 27)
    int span = TileB<KS>::ROWS;
    while (span > 16 && (int64_t)((a.rows + span - 1) / span) * parts <= cus) span /= 2;
    const dim3 grid = grid_of((int64_t)((a.rows + span - 1) / span) * parts);
    const bool past = a.rows * a.l.n * (int64_t)sizeof(float) * (a.base ? 2 : 1) >= PAST_BYTES;
    if (past) lora_tiles_b<KS, true><<<grid, 64 * B_WAVES, 0, s>>>(a, p.splits, parts, span);
    else lora_tiles_b<KS, false><<<grid, 64 * B_WAVES, 0, s>>>(a, p.splits, parts, span);
    return hipGetLastError();
}

}  // namespace

LoraPlan lora_plan(int cus, const arfq_lora &l, int64_t rows, bool x_f16) {
    LoraPlan p;
    p.tiles = in_tiles(l, rows, x_f16);
    if (p.tiles) {
        // a workgroup a compute unit, and not fewer than four steps a wave
        const int64_t tiles = (rows + A_TILES * TR - 1) / (A_TILES * TR);
        const int64_t splits = std::max<int64_t>(1, std::min(cus / tiles, l.k / (4 * 32 * A_WAVES)));
        p.k_part = (int)(((l.k + splits - 1) / splits + 32 * A_WAVES - 1) / (32 * A_WAVES) * (32 * A_WAVES));
        p.splits = (int)((l.k + p.k_part - 1) / p.k_part);
    } else {
        p.k_part = K_PART;
        p.splits = (int)((l.k + K_PART - 1) / K_PART);
        const int64_t groups = rows * ((l.n + ONE_OUT - 1) / ONE_OUT), a_e = l.k * l.rank;
        p.one = a_e <= ONE_A && groups <= cus * (l.rank <= 32 ? 2 : 1) && groups * a_e <= ONE_READ;
    }
    p.ws_bytes = p.one ? 0 : (size_t)p.splits * rows * l.rank * sizeof(float);
    return p;
}

hipError_t launch_lora(const LoraArgs &a, const LoraPlan &p, int cus, hipStream_t s) {
    if (p.tiles) {
        hipError_t e = a.l.rank <= 16 ? tiles_a<1>(a, p, s) : a.l.rank <= 32 ? tiles_a<2>(a, p, s) : tiles_a<4>(a, p, s);
        if (e != hipSuccess) return e;
        const int64_t runs = (a.l.rank + 31) / 32;
        return runs <= 1 ? tiles_b<1>(a, p, cus, s) : runs <= 2 ? tiles_b<2>(a, p, cus, s) :
               runs <= 4 ? tiles_b<4>(a, p, cus, s) : tiles_b<8>(a, p, cus, s);
    }
    if (!p.one) {
        const dim3 grid = grid_of((int64_t)a.rows * p.splits);
        if (a.x_f16) lora_rows_a<true><<<grid, 256, 0, s>>>(a, p.splits);
        else lora_rows_a<false><<<grid, 256, 0, s>>>(a, p.splits);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    const int64_t lanes = a.l.rank / 8;
    return lanes <= 1 ? rows_b<1>(a, p, s) : lanes <= 2 ? rows_b<2>(a, p, s) : lanes <= 4 ? rows_b<4>(a, p, s) :
           lanes <= 8 ? rows_b<8>(a, p, s) : lanes <= 16 ? rows_b<16>(a, p, s) : rows_b<32>(a, p, s);
}

}  // namespace arfq
