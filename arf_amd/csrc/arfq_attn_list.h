// arfq_attn_list.h -- the attention's work list: the host's bound on it, and the kernels' search for a
// workgroup's item.
#pragma once
#include <algorithm>

#include "arfq_kv.h"

namespace arfq {

constexpr int STEP = 32;  // keys of a step

// Rows of a sequence that the 16-row tiles take.  Each tile turns K and V into operands for itself; a 128-row tile
// does so once, but takes its time for few rows too (sequences x rows x keys, us with the 16-row tiles and with
// the 128-row ones: f16 16 x 36 x 4096 56 and 53, 1 x 56 x 8192 19 and 25, f32 16 x 56 x 4096 65 and 71;
// above, 16 x 80 x 4096 86 and 58, f32 16 x 128 x 4096 122 and 92, 1 x 128 x 8192 24 and 27).
constexpr int64_t FEW_ROWS = 64;

// waves of a SIMD (a workgroup has one on each): registers below 512 / that.  (One fewer, us: the 64 sequences below
// 52 for 45, the window 33 for 27, the ungrouped heads 29 for 25.)
constexpr int rows16_waves(int ng) { return ng <= 2 ? 4 : ng <= 4 ? 3 : 2; }

// the kernel of both lists: workgroups that a compute unit holds (a wave each on every SIMD), at ng groups of 32 values
constexpr int mixed_waves(int ng) { return ng <= 4 ? 2 : 1; }

// Keys of the shortest piece: below, its set-up and the joining of its rows take longer than its keys.  (128 of them /
// 256 / 512, us: 2048 keys of one head for 8 rows 10.8 / 10.9 / 12.6; 4096 keys of two heads, eight
// sequences 13.6 / 13.0 / 13.5; 131072 of one head 25 / 21 / 18.  Of prompts 256 / 512 / 1024: 640 rows of
// 2048 keys 27.9 / 29.3 / 43.8, 1024 rows of 4096 keys 42.4 / 42.4 / 44.7.)
constexpr int MIN_PIECE = 256;

// max_keys: of a sequence; one_each: a token of every sequence (no start)
inline AttnPlan attn_plan(int cus, int heads, int dim, int64_t batch, int64_t tokens, int q_heads, int64_t max_keys, bool one_each) {
    AttnPlan p;
    const int64_t group = q_heads / heads, rows = tokens * group;
    const int ng = dim / KV_GROUP;
    p.few_rows = FEW_ROWS;
    // a list's items: the area cut into `target` pieces, and at most one more for each tile; none of its
    // pieces shorter than MIN_PIECE
    auto plan = [&](AttnListPlan &l, int tr, int waves, int64_t tiles) {
        const int64_t most = std::max<int64_t>(1, (max_keys + MIN_PIECE - 1) / MIN_PIECE);
        l.target = std::max(1, waves * cus / heads);
        l.round = std::max(1, cus / heads);
        l.slots = (int)std::min(l.target + tiles, tiles * most);
        if (most > 1) {
            l.cut = std::min(l.slots, 2 * l.target);
            l.part_bytes = (size_t)l.cut * heads * tr * (dim + 4) * sizeof(float);
            l.join_bytes = (size_t)l.cut * sizeof(int4);
            p.ws_bytes += l.part_bytes + l.join_bytes;
        }
    };
    // sequences of at most FEW_ROWS rows, and the longer ones
    const bool many = (one_each ? group : rows) > FEW_ROWS;
    if (group <= FEW_ROWS)
        plan(p.few, 16, many ? std::min(mixed_waves(ng), rows16_waves(ng)) : rows16_waves(ng),
             std::min({rows / 16 + batch, batch * ((FEW_ROWS + 15) / 16), tokens * ((group + 15) / 16)}));
    if (many) plan(p.many, 128, mixed_waves(ng), rows / 128 + std::min(batch, rows / (FEW_ROWS + 1)));
    return p;
}

namespace {

// A row is a (token, head of the group) pair, head fastest.  Sequences with at most few_rows rows
// are in the list of 16-row tiles (a decode step), others in that of 128-row tiles (prompts); a
// kernel works through each.  A sequence's keys [lo, end) are cut into pieces; a work item is a
// (tile, piece).  The piece length is what cuts the whole batch's
// (tile, key) area into about `target` pieces, so that a long sequence is spread over the chip
// whatever its neighbours are: decided here, from the lengths, which are on the device.

struct Seq {
    int t0, n, len;
    int lo, end;  // keys that some row may attend to; lo is a multiple of STEP
    int tiles;
};

template <int TR>
__device__ __forceinline__ const AttnList &list_of(const AttnArgs &a) { return TR == 16 ? a.few : a.many; }

// (of 64 sequences, b in each lane of the wave; ended: kv_seq64)
template <int TR>
__device__ __forceinline__ Seq seq_of(const AttnArgs &a, int b, bool &ended) {
    Seq s = {0, 0, 0, 0, 0, 0};
    kv_seq64(a.c, b, ended, s.t0, s.n);
    if (b >= a.c.batch) return s;
    s.len = a.c.len[b];
    s.end = (int)min((int64_t)max(s.len, 0), (int64_t)a.c.max_pages * a.c.page);
    if (a.window) s.lo = (int)max((int64_t)0, min((int64_t)s.len - s.n - a.window + 1, (int64_t)s.end)) & ~(STEP - 1);
    const int64_t rows = (int64_t)s.n * a.group;
    if ((TR == 16) == (rows <= a.few_rows)) s.tiles = (int)((rows + TR - 1) / TR);
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
    int cut;   // items of the list that are pieces of several
    int part;  // this one's place among them
};

// The `index`-th (tile, piece) of the batch: sequences in order, their tiles one after another,
// pieces fastest.  False: the list has fewer.  The keys that make a new piece necessary are the same
// in every wave of the launch: the fewest that cut the area into at most `target` pieces, or
// nearly so (a target of workgroups that the chip holds at once: one more round for a few of
// them would take as long as the first).  The area is summed in f32 in one fixed order; the 2^-16
// added covers its rounding, so that the list has no more than target + tiles items, and no more than
// 2 target of them are pieces of several (ceil(x) < 2 x for x > 1).
template <int TR>
__device__ __forceinline__ bool find_item(const AttnArgs &a, int index, Item &it) {
    const int lane = threadIdx.x & 63;
    bool ended0 = false;
    const Seq s0 = seq_of<TR>(a, lane, ended0);  // (the whole batch, mostly)
    auto over_batch = [&](auto f) {
        float v = f(s0);
        bool ended = ended0;
        for (int b0 = WAVE; b0 < a.c.batch; b0 += WAVE) v += f(seq_of<TR>(a, b0 + lane, ended));
        return wave_sum(v);
    };
    const float area = over_batch([](const Seq &s) { return (float)s.tiles * (float)((s.end - s.lo + STEP - 1) / STEP); });
    const float target = (float)list_of<TR>(a).target;
    auto keys_of = [](float steps) { return (int)fminf(steps, (float)(KV_KEYS_MAX / STEP)) * STEP; };
    float steps = fmaxf(ceilf(area / target * (1.0f + 1.0f / 65536)), (float)(MIN_PIECE / STEP));
    for (int i = 0; i < 3; i++) {
        const int piece = keys_of(steps);
        const float items = over_batch([&](const Seq &s) { return (float)s.tiles * (float)pieces_of(s, piece); });
        if (items <= target) break;
        // (tiles of one piece stay: the others' pieces shrink in number with their length)
        steps = ceilf(steps * fminf(items / target, 2.0f));
    }
    const int piece = keys_of(steps);
    it.cut = (int)over_batch([&](const Seq &s) {
        const int np = pieces_of(s, piece);
        return np > 1 ? (float)s.tiles * (float)np : 0.0f;
    });
    int before = 0, cut_before = 0;
    bool ended = ended0;
    for (int b0 = 0; b0 < a.c.batch; b0 += WAVE) {
        const Seq s = b0 ? seq_of<TR>(a, b0 + lane, ended) : s0;
        const int np = pieces_of(s, piece), own = (int)min((int64_t)s.tiles * np, (int64_t)1 << 30), inc = wave_scan(own);
        const int cut = np > 1 ? own : 0, cut_inc = wave_scan(cut);
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
            it.part = cut_before + __builtin_amdgcn_readlane(cut_inc - cut, l) + rest;
            it.tile = rest / it.pieces;
            it.piece = rest - it.tile * it.pieces;
            // Prompts: the longest tile first, and every other round of workgroups (one a compute unit)
            // backwards, so that a unit's first and second tile are long and short (3000 tokens, 8 x 4
            // heads of 64, f32: 102 us, in plain order 105).
            if (TR == 128 && a.causal) {
                const int round = list_of<TR>(a).round, tiles = it.s.tiles;
                if (it.pieces == 1 && a.c.batch == 1 && (it.tile / round & 1)) {
                    const int lo = it.tile / round * round, hi = min(lo + round, tiles);
                    it.tile = hi - 1 - (it.tile - lo);
                }
                it.tile = tiles - 1 - it.tile;
            }
            return rest >= 0 && it.tile >= 0 && it.tile < it.s.tiles;
        }
        before += __builtin_amdgcn_readlane(inc, 63);
        cut_before += __builtin_amdgcn_readlane(cut_inc, 63);
    }
    return false;
}

// The workgroup's item, and what the join has to know of it (every place is written: the list has no more items
// than list.slots, the workgroups of a head, as no two sequences share a row): the tile's pieces (bits 0..15) and which of them it is, its rows, the sequence's first token.
template <int TR>
__device__ __forceinline__ bool take_item(const AttnArgs &a, int block, Item &it) {
    const AttnList &list = list_of<TR>(a);
    const int slot = block / a.c.heads;
    const bool got = find_item<TR>(a, slot, it);
    if (list.join && block % a.c.heads == 0 && threadIdx.x == 0) {
        if (slot >= it.cut && slot < list.cut) list.join[slot] = make_int4(0, 0, 0, 0);
        if (got && it.pieces > 1 && (uint32_t)it.part < (uint32_t)list.cut)
            list.join[it.part] = make_int4(it.pieces | it.piece << 16, it.tile * TR, it.s.n * a.group, it.s.t0);
    }
    return got;
}

}  // namespace
}  // namespace arfq
