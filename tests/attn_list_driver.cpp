// The attention's work list (arf_amd/csrc/arfq_attn_list.h) on the CPU: every workgroup that a call
// launches takes its item, over a wave of coroutines (host_wave).  Reads calls from stdin, a line each:
//     cus heads dim q_heads page max_pages window causal tokens batch has_start start... len...
// and prints for each, a line for a list (16-row tiles, 128-row tiles):
//     rows_of_a_tile slots cut items joins bad
// items: workgroups that got one.  joins: entries of the join that name a piece.  bad: what must not be, as
// bits: 1 an entry of the join that no workgroup wrote, 2 an entry whose rows or pieces do not lie in the call, 4 a
// piece of several without an entry of its own, 8 a (tile, head) with a piece missing or twice, 16 a sequence's rows
// not all in tiles, or those of two sequences overlapping.
#include "arfq_attn_list.h"

#include <map>
#include <set>
#include <stdio.h>
#include <vector>

using namespace arfq;

template <int TR>
static void check(const AttnArgs &a, const AttnListPlan &plan, std::vector<int> &owner) {
    const AttnList &list = list_of<TR>(a);
    const int heads = a.c.heads;
    int items = 0, joins = 0, bad = 0;
    std::map<std::pair<int, int>, std::set<int>> pieces;  // of a sequence's tile
    std::map<std::pair<int, int>, int> of;
    std::set<int> parts;
    for (int slot = 0; slot < list.slots; slot++) {
        Item got = {};
        bool has = false;
        host_wave::run([&] {
            Item it = {};
            const bool mine = take_item<TR>(a, slot * heads, it);
            if (threadIdx.x == 0) {
                got = it;
                has = mine;
            }
        });
        if (!has) continue;
        items++;
        const auto key = std::make_pair(got.b, got.tile);
        if (!pieces[key].insert(got.piece).second || got.piece < 0 || got.piece >= got.pieces) bad |= 8;
        of[key] = got.pieces;
        if (got.pieces > 1 && (got.part < 0 || got.part >= list.cut || !parts.insert(got.part).second)) bad |= 4;
    }
    for (const auto &t : pieces) {
        if ((int)t.second.size() != of[t.first]) bad |= 8;
        if (*t.second.begin() != 0) continue;
        const int b = t.first.first, t0 = a.c.start ? a.c.start[b] : b, n = a.c.start ? a.c.start[b + 1] - t0 : 1;
        for (int r = t.first.second * TR; r < std::min(n * a.group, (t.first.second + 1) * TR); r++) {
            const int64_t o = (int64_t)t0 * a.group + r;
            if (t0 < 0 || o >= (int64_t)a.c.tokens * a.group || owner[o] >= 0) bad |= 16;
            else owner[o] = b;
        }
    }
    for (int i = 0; i < list.cut && list.join; i++) {
        const int4 j = list.join[i];
        if (j.x == INT32_MIN) {
            bad |= 1;
            continue;
        }
        if (j.x == 0) continue;
        joins++;
        const int np = j.x & 0xffff, p = j.x >> 16;
        if (np < 2 || p < 0 || p >= np || i < p || i - p + np > list.cut || j.y < 0 || j.y >= j.z || j.w < 0 ||
            (int64_t)j.w * a.group + j.z > (int64_t)a.c.tokens * a.group)
            bad |= 2;
        if (!parts.count(i)) bad |= 2;
    }
    printf("%d %d %d %d %d %d\n", TR, plan.slots, plan.cut, items, joins, bad);
}

int main() {
    int cus, heads, dim, q_heads, page, max_pages, window, causal, tokens, batch, has_start;
    while (scanf("%d %d %d %d %d %d %d %d %d %d %d", &cus, &heads, &dim, &q_heads, &page, &max_pages, &window, &causal,
                 &tokens, &batch, &has_start) == 11) {
        std::vector<int32_t> start(batch + 1), len(batch);
        for (int i = 0; has_start && i <= batch; i++)
            if (scanf("%d", &start[i]) != 1) return 1;
        for (int i = 0; i < batch; i++)
            if (scanf("%d", &len[i]) != 1) return 1;
        const AttnPlan p = attn_plan(cus, heads, dim, batch, tokens, q_heads, (int64_t)max_pages * page, !has_start);
        AttnArgs a = {};
        a.c.heads = heads;
        a.c.page = page;
        a.c.batch = batch;
        a.c.tokens = tokens;
        a.c.start = has_start ? start.data() : nullptr;
        a.c.len = len.data();
        a.c.max_pages = max_pages;
        a.group = q_heads / heads;
        a.window = window;
        a.causal = causal;
        a.few_rows = p.few_rows;
        std::vector<int4> few(p.few.cut, int4{INT32_MIN, 0, 0, 0}), many(p.many.cut, int4{INT32_MIN, 0, 0, 0});
        a.few = {p.few.target, p.few.slots, p.few.cut, p.few.round, nullptr, p.few.join_bytes ? few.data() : nullptr};
        a.many = {p.many.target, p.many.slots, p.many.cut, p.many.round, nullptr, p.many.join_bytes ? many.data() : nullptr};
        std::vector<int> owner((size_t)tokens * a.group, -1);
        check<16>(a, p.few, owner);
        check<128>(a, p.many, owner);
        // every row of a sequence that has rows
        int left = 0;
        bool broken = false;
        for (int b = 0; b < batch; b++) {
            const int t0 = has_start ? start[b] : b, t1 = has_start ? start[b + 1] : b < tokens ? b + 1 : b;
            broken = broken || t1 < t0;
            if (broken || t0 < 0 || t1 > tokens) continue;
            for (int64_t r = (int64_t)t0 * a.group; r < (int64_t)t1 * a.group; r++) left += owner[r] != b;
        }
        printf("rows left out: %d\n", left);
        fflush(stdout);
    }
    return 0;
}
