// arfq_lora.hip -- low-rank adapters of many requests beside a shared projection:
// out[t] = base[t] + scale_e B_e (A_e x[t]), e = ids[t].
//
// Two launches.  The first forms parts of h = A_e x over ranges of k, [splits][rows][rank] in f32; the second adds the
// parts in order, and B_e h to base.  Few rows: a workgroup has one row (and a range of k, or of n) on the vector unit,
// products in f32.  Many rows: tiles of 16 or 32 neighbouring rows on the matrix cores, once for each adapter that the
// tile's rows name; an f32 x goes through v_mfma_f32_16x16x4_f32 as it is, an f16 x is exact in f16 operands, and h
// enters the second product as two f16 parts of 22 bits of the row's largest.  Every adapter has accumulators of its
// own: a NaN in one does not reach another's rows.  Bound by memory: the adapters' bytes for few rows, base and out for
// many.
#include "arfq_step.h"

#include <math.h>

namespace arfq {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

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

// ---- few rows ----

template <int N>
__device__ __forceinline__ float lanes_sum(float v) {  // over N neighbouring lanes
#pragma unroll
    for (int d = 1; d < N; d *= 2) v += __shfl_xor(v, d);
    return v;
}

template <bool F16>
__global__ __launch_bounds__(256) void lora_rows_a(LoraArgs a, int splits) {
    const int block = block_of(), t = block / splits, part = block - t * splits;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (t >= a.rows) return;
    const int e = id_of(a, t);
    if (e < 0) return;
    const int rank = (int)a.l.rank;
    const int64_t k = (int64_t)part * K_PART + 8 * lane;
    const bool on = k < a.l.k;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (on) load8<F16>(a.x, t * a.l.k + k, x);
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

// LP lanes have an output, eight ranks each.
constexpr int N_PART = 256;  // outputs of a workgroup
template <int LP>
__global__ __launch_bounds__(256) void lora_rows_b(LoraArgs a, int splits, int parts) {
    __shared__ float sh[LORA_RANK_MAX];
    const int block = block_of(), t = block / parts, part = block - t * parts;
    if (t >= a.rows) return;
    const int e = id_of(a, t), rank = (int)a.l.rank;
    const float *base = a.base ? a.base + t * a.base_stride : nullptr;
    float *out = a.out + t * a.out_stride;
    const int64_t n0 = (int64_t)part * N_PART;
    if (e < 0) {
        const int64_t n = n0 + threadIdx.x;
        if (n < a.l.n && base != out) out[n] = base ? base[n] : 0.0f;
        return;
    }
    if ((int)threadIdx.x < rank) {
        float s = 0.0f;
        for (int p = 0; p < splits; p++) s += a.h[((int64_t)p * a.rows + t) * rank + threadIdx.x];
        sh[threadIdx.x] = a.l.scale ? s * a.l.scale[e] : s;
    }
    __syncthreads();
    const int u = threadIdx.x % LP, r0 = 8 * u;
    const bool on = r0 < rank;
    float h[8];
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = on ? sh[r0 + i] : 0.0f;
    const _Float16 *B = (const _Float16 *)a.l.b + (int64_t)e * a.l.n * rank + r0;
#pragma unroll
    for (int j = 0; j < LP; j++) {
        const int64_t n = n0 + j * (256 / LP) + threadIdx.x / LP;
        const f16x8 w = on && n < a.l.n ? *(const f16x8 *)(B + n * rank) : zero8();
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) s = __builtin_fmaf((float)w[i], h[i], s);
        s = lanes_sum<LP>(s);
        if (u == 0 && n < a.l.n) out[n] = (base ? base[n] : 0.0f) + s;
    }
}

// ---- many rows ----

constexpr int TR = 16;  // rows of a tile: a matrix instruction's columns

// The adapters that a tile's rows name, one after another (`mine`: this lane's row's; the same in all lanes of a row).
// Returns the next one, or -2 behind the last; done: the lanes whose rows are served.
__device__ __forceinline__ int next_id(int mine, uint64_t &done) {
    if (done == ~0ull) return -2;
    const int e = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)~done) - 1);
    done |= __ballot(mine == e);
    return e;
}

// RT 16-rank tiles of h, TR rows, a part of k in four by the waves.
template <int RT, bool F16>
__global__ __launch_bounds__(256) void lora_tiles_a(LoraArgs a, int splits, int k_part, int ranks) {
    __shared__ f32x4 sh[4][RT][64];
    int block = block_of();
    const int rb = block % ranks;
    block /= ranks;
    const int part = block % splits, t0 = block / splits * TR;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    if (t0 >= a.rows) return;
    const int rank = (int)a.l.rank, r0 = rb * RT * 16, t = min(t0 + c, a.rows - 1);
    const int64_t k = a.l.k;
    // the wave's range, in steps of 32: eight values a lane
    const int64_t lo = (int64_t)part * k_part + (int64_t)wave * (k_part / 4), hi = min(lo + k_part / 4, k);
    const int mine = t0 + c < a.rows ? id_of(a, t0 + c) : -1;
    uint64_t done = 0;
    for (int e; (e = next_id(mine, done)) != -2;) {
        if (e < 0) continue;
        f32x4 acc[RT];
#pragma unroll
        for (int i = 0; i < RT; i++) acc[i] = f32x4{0, 0, 0, 0};
        const _Float16 *A = (const _Float16 *)a.l.a + (int64_t)e * rank * k;
        for (int64_t k0 = lo; k0 < hi; k0 += 32) {
            const int64_t kk = k0 + 8 * g;
            const bool on = kk < hi;
            f16x8 w[RT];
#pragma unroll
            for (int i = 0; i < RT; i++) w[i] = on ? *(const f16x8 *)(A + min(r0 + 16 * i + c, rank - 1) * k + kk) : zero8();
            if constexpr (F16) {
                const f16x8 x = on ? *(const f16x8 *)((const _Float16 *)a.x + t * k + kk) : zero8();
#pragma unroll
                for (int i = 0; i < RT; i++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[i], x, acc[i], 0, 0, 0);
            } else {
                float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (on) load8<false>(a.x, t * k + kk, x);
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int i = 0; i < RT; i++)
                        acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)w[i][j], x[j], acc[i], 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < RT; i++) sh[wave][i][lane] = acc[i];
        __syncthreads();
        // a lane's four results: ranks 4g .. +3 of a tile, row c
        for (int i = wave; i < RT; i += 4) {
            const f32x4 s = sh[0][i][lane] + sh[1][i][lane] + sh[2][i][lane] + sh[3][i][lane];
            const int r = r0 + 16 * i + 4 * g;
            if (mine == e && r < rank) *(f32x4 *)(a.h + ((int64_t)part * a.rows + t0 + c) * rank + r) = s;
        }
        __syncthreads();
    }
}

// A wave: CT tiles of rows, NT tiles of 16 outputs, ranks in runs of 64.
constexpr int CT = 2, NT = 4;
template <bool VEC>
__global__ __launch_bounds__(256) void lora_tiles_b(LoraArgs a, int splits, int parts) {
    const int block = block_of(), part = block % parts, t0 = block / parts * (CT * TR);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    if (t0 >= a.rows) return;
    const int rank = (int)a.l.rank;
    const int64_t n = a.l.n, n0 = (int64_t)part * (4 * NT * 16) + wave * (NT * 16);
    if (n0 >= n) return;
    int mine[CT];
#pragma unroll
    for (int s = 0; s < CT; s++) mine[s] = t0 + 16 * s + c < a.rows ? id_of(a, t0 + 16 * s + c) : -1;
    uint64_t done[CT] = {};
    for (;;) {
        // the next adapter, or none, that one of the tiles' rows is still to be served with
        int e = -2;
#pragma unroll
        for (int s = 0; s < CT; s++)
            if (e == -2 && done[s] != ~0ull) e = __builtin_amdgcn_readlane(mine[s], __ffsll((unsigned long long)~done[s]) - 1);
        if (e == -2) break;
#pragma unroll
        for (int s = 0; s < CT; s++) done[s] |= __ballot(mine[s] == e);
        f32x4 sum[CT][NT];
#pragma unroll
        for (int s = 0; s < CT; s++)
#pragma unroll
            for (int i = 0; i < NT; i++) sum[s][i] = f32x4{0, 0, 0, 0};
        if (e >= 0) {
            const _Float16 *B = (const _Float16 *)a.l.b + (int64_t)e * n * rank;
            const float scale = a.l.scale ? a.l.scale[e] : 1.0f;
            for (int r0 = 0; r0 < rank; r0 += 64) {
                f16x8 w[NT][2];
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        const int r = r0 + 32 * q + 8 * g;
                        w[i][q] = r < rank ? *(const f16x8 *)(B + min(n0 + 16 * i + c, n - 1) * rank + r) : zero8();
                    }
#pragma unroll
                for (int s = 0; s < CT; s++) {
                    // h of the row: its parts added, and as two f16 parts of it times a power of two
                    float h[2][8], top = 0.0f;
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        const int r = r0 + 32 * q + 8 * g;
#pragma unroll
                        for (int j = 0; j < 8; j++) h[q][j] = 0.0f;
                        if (mine[s] == e && r < rank)
                            for (int p = 0; p < splits; p++) {
                                float v[8];
                                load8<false>(a.h, ((int64_t)p * a.rows + t0 + 16 * s + c) * rank + r, v);
#pragma unroll
                                for (int j = 0; j < 8; j++) h[q][j] += v[j];
                            }
#pragma unroll
                        for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(h[q][j]));
                    }
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const int ex = min(max(top > 0.0f ? 141 - (int)(__builtin_bit_cast(uint32_t, top) >> 23) : 0, -126), 126);
                    const float up = __builtin_bit_cast(float, (uint32_t)(ex + 127) << 23);
                    const float down = __builtin_bit_cast(float, (uint32_t)(127 - ex) << 23);
                    f16x8 hi[2], lo[2];
#pragma unroll
                    for (int q = 0; q < 2; q++)
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const float v = h[q][j] * up;
                            hi[q][j] = (_Float16)v;
                            lo[q][j] = fabsf(v) == INFINITY ? (_Float16)0 : (_Float16)(v - (float)hi[q][j]);
                        }
#pragma unroll
                    for (int i = 0; i < NT; i++) {
                        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[i][q], hi[q], acc, 0, 0, 0);
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[i][q], lo[q], acc, 0, 0, 0);
                        }
                        sum[s][i] += acc * (down * scale);
                    }
                }
            }
        }
#pragma unroll
        for (int s = 0; s < CT; s++) {
            const int t = t0 + 16 * s + c;
            if (mine[s] != e || t >= a.rows) continue;
            const float *base = a.base ? a.base + t * a.base_stride : nullptr;
            float *out = a.out + t * a.out_stride;
            if (e < 0 && base == out) continue;
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const int64_t at = n0 + 16 * i + 4 * g;
                if constexpr (VEC) {
                    if (at >= n) continue;
                    f32x4 v = sum[s][i];
                    if (base) v += *(const f32x4 *)(base + at);
                    *(f32x4 *)(out + at) = v;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (at + j < n) out[at + j] = (base ? base[at + j] : 0.0f) + sum[s][i][j];
                }
            }
        }
    }
}

// Rows from which on tiles are faster.
constexpr int64_t TILE_ROWS = 64;

template <int LP>
hipError_t rows_b(const LoraArgs &a, const LoraPlan &p, hipStream_t s) {
    const int parts = (int)((a.l.n + N_PART - 1) / N_PART);
    lora_rows_b<LP><<<grid_of((int64_t)a.rows * parts), 256, 0, s>>>(a, p.splits, parts);
    return hipGetLastError();
}

template <int RT>
hipError_t tiles_a(const LoraArgs &a, const LoraPlan &p, hipStream_t s) {
    const int ranks = (int)((a.l.rank + RT * 16 - 1) / (RT * 16));
    const dim3 grid = grid_of((int64_t)((a.rows + TR - 1) / TR) * p.splits * ranks);
    if (a.x_f16) lora_tiles_a<RT, true><<<grid, 256, 0, s>>>(a, p.splits, p.k_part, ranks);
    else lora_tiles_a<RT, false><<<grid, 256, 0, s>>>(a, p.splits, p.k_part, ranks);
    return hipGetLastError();
}

}  // namespace

LoraPlan lora_plan(int cus, const arfq_lora &l, int64_t rows) {
    LoraPlan p;
    p.tiles = rows > TILE_ROWS;
    if (p.tiles) {
        // two workgroups a compute unit, and not fewer than 128 values of k a wave
        const int64_t tiles = (rows + TR - 1) / TR;
        const int64_t want = std::max<int64_t>(1, 2 * cus / tiles), most = std::max<int64_t>(1, l.k / 512);
        const int64_t splits = std::min(want, most);
        p.k_part = (int)(((l.k + splits - 1) / splits + 127) / 128 * 128);
        p.splits = (int)((l.k + p.k_part - 1) / p.k_part);
    } else {
        p.k_part = K_PART;
        p.splits = (int)((l.k + K_PART - 1) / K_PART);
    }
    p.ws_bytes = (size_t)p.splits * rows * l.rank * sizeof(float);
    return p;
}

hipError_t launch_lora(const LoraArgs &a, const LoraPlan &p, hipStream_t s) {
    if (p.tiles) {
        hipError_t e = a.l.rank <= 16 ? tiles_a<1>(a, p, s) : a.l.rank <= 32 ? tiles_a<2>(a, p, s) : tiles_a<4>(a, p, s);
        if (e != hipSuccess) return e;
        const int parts = (int)((a.l.n + 4 * NT * 16 - 1) / (4 * NT * 16));
        const dim3 grid = grid_of((int64_t)((a.rows + CT * TR - 1) / (CT * TR)) * parts);
        const bool vec = a.l.n % 4 == 0 && a.out_stride % 4 == 0 && (uintptr_t)a.out % 16 == 0 &&
                         (!a.base || (a.base_stride % 4 == 0 && (uintptr_t)a.base % 16 == 0));
        if (vec) lora_tiles_b<true><<<grid, 256, 0, s>>>(a, p.splits, parts);
        else lora_tiles_b<false><<<grid, 256, 0, s>>>(a, p.splits, parts);
        return hipGetLastError();
    }
    const dim3 grid = grid_of((int64_t)a.rows * p.splits);
    if (a.x_f16) lora_rows_a<true><<<grid, 256, 0, s>>>(a, p.splits);
    else lora_rows_a<false><<<grid, 256, 0, s>>>(a, p.splits);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t lanes = a.l.rank / 8;
    return lanes <= 1 ? rows_b<1>(a, p, s) : lanes <= 2 ? rows_b<2>(a, p, s) : lanes <= 4 ? rows_b<4>(a, p, s) :
           lanes <= 8 ? rows_b<8>(a, p, s) : lanes <= 16 ? rows_b<16>(a, p, s) : rows_b<32>(a, p, s);
}

}  // namespace arfq
