// arfq_attn_join.h -- the parts of rows whose keys were cut into pieces, joined.
#pragma once
#include "arfq_attn.h"

namespace arfq {
namespace {

// Rows whose keys were cut into pieces: their parts joined, in a fixed order.  As many workgroups share a
// tile's rows as it has pieces.  A thread has four columns of a row: of the parts it takes them all, 1024 / D rows
// a workgroup side by side, or (few rows, many pieces) the workgroup's threads share a row's.  Bound by
// latency: 4 to 5 us, two loads that follow one another after the launch.
template <int NG>
struct JoinLds {
    static constexpr int D = 32 * NG, CT = D / 4, PT = 256 / CT;
    f32x4 v[PT][CT];
    float l[PT], m[PT];
};
template <int NG, int TR>
__device__ __forceinline__ void join_tile(const AttnArgs &a, const AttnList &list, int4 j, int slot, int head, JoinLds<NG> &sh) {
    constexpr int D = 32 * NG, CT = JoinLds<NG>::CT, PT = JoinLds<NG>::PT;
    if (j.x == 0) return;
    const int pt = threadIdx.x / CT, ct = threadIdx.x - pt * CT;
    const int rows = min(j.z - j.y, TR), pieces = j.x & 0xffff, piece = j.x >> 16, slot0 = slot - piece;
    if (slot0 < 0 || slot0 + pieces > list.cut) return;
    const int64_t next = (int64_t)a.c.heads * TR * (D + 4);
    // the weight of a part (m, l) below a common maximum; NaN for a NaN part (a NaN key leaves
    // a wave's maximum at -inf and its sum NaN)
    auto weight = [](float m, float l, float top) { return l != l ? l : m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top); };
    constexpr int U = 8;  // pieces loaded at a time
    // pieces p0, p0 + by, .. (U of them at most) of a row, onto its (mm, l, v) so far
    auto add = [&](const float *part, int p0, int by, float &mm, float &l, f32x4 &v) {
        float m_p[U], l_p[U];
        f32x4 w[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int p = min(p0 + u * by, pieces - 1);
            const float2 ml = *(const float2 *)(part + p * next);
            w[u] = *(const f32x4 *)(part + p * next + 4 + 4 * ct);
            m_p[u] = p0 + u * by < pieces ? ml.x : -INFINITY;
            l_p[u] = p0 + u * by < pieces ? ml.y : 0.0f;
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
    };
    auto part_of = [&](int r) { return list.part + (((int64_t)slot0 * a.c.heads + head) * TR + r) * (D + 4); };
    auto put = [&](int r, float l, f32x4 v) {
        const int rr = j.y + r, rt = rr / a.group, rg = rr - rt * a.group;
        store_out(a, ((int64_t)j.w + rt) * a.out_stride + (int64_t)(head * a.group + rg) * D + 4 * ct, v * (l == 0.0f ? 0.0f : 1.0f / l));
    };
    // the loads that follow one another: rows side by side, or one by one (with the LDS sum as one more).  (8 rows in
    // 512 pieces: 63 us with the attention side by side, 21 one by one; 512 rows in 16: 44 and 111.)
    const int beside = (rows + pieces * PT - 1) / (pieces * PT) * ((pieces + U - 1) / U);
    const int each = (rows + pieces - 1) / pieces * ((pieces + U * PT - 1) / (U * PT) + 1);
    if (beside <= each) {  // a row for each CT threads
        if (pt >= PT) return;
        for (int r = piece * PT + pt; r < rows; r += pieces * PT) {
            float mm = -INFINITY, l = 0.0f;
            f32x4 v = {0, 0, 0, 0};
            for (int p0 = 0; p0 < pieces; p0 += U) add(part_of(r), p0, 1, mm, l, v);
            put(r, l, v);
        }
        return;
    }
    for (int r = piece; r < rows; r += pieces) {  // all threads on a row
        float mm = -INFINITY, l = 0.0f;
        f32x4 v = {0, 0, 0, 0};
        if (pt < PT) {
            for (int p0 = pt; p0 < pieces; p0 += U * PT) add(part_of(r), p0, PT, mm, l, v);
            sh.v[pt][ct] = v;
            if (ct == 0) {
                sh.m[pt] = mm;
                sh.l[pt] = l;
            }
        }
        __syncthreads();
        if (pt == 0) {
#pragma unroll
            for (int p = 0; p < PT; p++) mm = fmaxf(mm, sh.m[p]);
            l = 0.0f;
            v = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < PT; p++) {
                const float f = weight(sh.m[p], sh.l[p], mm);
                l += f * sh.l[p];
                v += f * sh.v[p][ct];
            }
            put(r, l, v);
        }
        __syncthreads();
    }
}

template <int NG, int TR>
__device__ __forceinline__ void join_rows(const AttnArgs &a, int slot, int head, JoinLds<NG> &sh) {
    const AttnList &list = list_of<TR>(a);
    join_tile<NG, TR>(a, list, list.join[slot], slot, head, sh);
}

}  // namespace
}  // namespace arfq
