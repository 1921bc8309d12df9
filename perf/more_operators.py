"""What stands around the K/V cache in a serving step of many requests, as measurable cases:

  plan    a step's rows, page tables and slots from the requests' lengths       Context.kv_plan
  adapt   every request's own low-rank adapter beside a shared projection       Context.lora_add
  rotate  rotary positions of one to four axes, on the rows of q and k          Context.rope
  blocks  the bounds of the step's own blocks of the 4-bit cache's keys, and    Context.kv_bounds,
          attention over the blocks whose bounds say the most to each query     Context.kv_attention_blocks

In a plain form (`own` false) each is written with elementary torch operations, in 32 bits (angles and the scores that
choose blocks in 64); otherwise the calls are those of arf_amd.Context.

plan: sequence b holds `held` tokens and is to hold `add` more, or that many fewer (all of its own at most).  A page has
`page` tokens.  Pages that a sequence no longer needs are given back, those that it needs more are taken: first from
what this call gives back, sequence after sequence, then from the top of the stack of free ones.  A sequence whose pages
no longer fit the free ones (those before it counted), whose pages pass the table, or whose rows pass `tokens` gets
nothing.
rotate: pair (a, b) of a row becomes (a cos - b sin, a sin + b cos) * gain, its angle the row's position on the pair's axis
times the pair's frequency; pairs are i and i + rot / 2, or 2i and 2i + 1.
blocks: a block is a page.  With hi and lo the largest and smallest of each channel of its keys, a block's score for a
query's K/V head is the largest of sum_d max(q_d hi_d, q_d lo_d) over the head's group; a query attends to its `last` latest
blocks, its `first` earliest and the best others, `count` of them in all (ties: the earlier block).
adapt: out_t = base_t + scale_e B_e (A_e x_t), e the row's adapter (-1: none).
"""
import math

import numpy as np
import torch

own = False

GROUP = 32
DTYPE = {"f32": torch.float32, "f16": torch.float16}
SIZE = {"f32": 4, "f16": 2}


def listed():
    return [
        # the bookkeeping of a decode step: a token of every chat, some ended, some with rejected drafts
        dict(name="plan decode", op="plan", batch=64, page=64, len=8192, new=1, drop=8, short=False),
        # of a step that takes in prompts beside the chats, with fewer free pages than they want
        dict(name="plan prompts", op="plan", batch=1000, page=16, len=3000, new=150, drop=16, short=True),
        # one chat with its own adapter on a projection
        dict(name="adapt one", op="adapt", rows=1, k=5120, n=5120, rank=16, adapters=8, runs=False, none=False, x="f32"),
        # a decode step of 64 chats on 32 adapters, some with none, beside a fused qkv product
        dict(name="adapt decode", op="adapt", rows=64, k=5120, n=7168, rank=16, adapters=32, runs=False, none=True, x="f32"),
        # prompts of four tenants beside the widest projection
        dict(name="adapt prompts", op="adapt", rows=2048, k=5120, n=17408, rank=64, adapters=4, runs=True, none=False, x="f16"),
        # q and k of a decode step, text: f32 products to f16 rows
        dict(name="rotate decode", op="rotate", tokens=64, heads=36, dim=128, rot=128, sections="64", layout="chunks",
             pairs="halves", inverse=False, strided=True, x="f32", out="f16", far=131072),
        # a video's rows: time, height and width share the pairs
        dict(name="rotate video", op="rotate", tokens=8191, heads=48, dim=128, rot=128, sections="16 24 24", layout="cycle",
             pairs="halves", inverse=False, strided=False, x="f32", out="f32", far=4096),
        # an image's, two axes with frequencies of their own, turned back
        dict(name="rotate image", op="rotate", tokens=1369, heads=16, dim=96, rot=64, sections="16 16", layout="own",
             pairs="neighbours", inverse=True, strided=False, x="f16", out="f16", far=64),
        # a short chat: everything that it has is chosen
        dict(name="blocks short", op="blocks", batch=1, new=1, len=193, ragged=False, idle=False, q_heads=16, kv_heads=8,
             dim=256, page=16, count=32, first=1, last=2, softcap=50.0, x="f16"),
        # one token at the end of a long document
        dict(name="blocks one long", op="blocks", batch=1, new=1, len=131071, ragged=False, idle=False, q_heads=40, kv_heads=8,
             dim=128, page=64, count=64, first=1, last=2, softcap=0.0, x="f32"),
        # a serving step over long chats of every age, one slot idle
        dict(name="blocks batch", op="blocks", batch=32, new=1, len=16384, ragged=True, idle=True, q_heads=32, kv_heads=4,
             dim=128, page=64, count=32, first=1, last=2, softcap=0.0, x="f32"),
        # the next piece of a long prompt: each of its tokens chooses for itself
        dict(name="blocks prompt", op="blocks", batch=1, new=256, len=16640, ragged=False, idle=False, q_heads=32, kv_heads=8,
             dim=64, page=32, count=32, first=1, last=4, softcap=0.0, x="f16"),
    ]


# bounds of a drawn case: the listed ones' largest values in memory and sums
MAX_CACHE = 1.4e8   # cached values of K
MAX_GATHER = 1.4e8  # values of K that the queries choose
MAX_SCORED = 2.8e8  # of the bounds that they look through
MAX_OUT = 3.6e7     # outputs of a product
MAX_FLOPS = 1.2e10
MAX_ROWS = 5.1e7    # rotated values


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_plan(rng):
    return dict(op="plan", batch=_log(rng, 1, 1000), page=rng.choice([16, 32, 48, 64, 128, 256]), len=_log(rng, 1, 32768),
                new=rng.choice([1, _log(rng, 1, 150)]), drop=_log(rng, 1, 64), short=rng.choice([True, False]))


def _draw_adapt(rng):
    runs = rng.choice([True, False])
    return dict(op="adapt", rows=_log(rng, 1, 2048 if runs else 128), k=8 * _log(rng, 4, 2176), n=_log(rng, 16, 17408),
                rank=8 * _log(rng, 1, 16), adapters=_log(rng, 1, 64), runs=runs, none=rng.choice([True, False]),
                x=rng.choice(["f32", "f16"]))


def _draw_rotate(rng):
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    rot = rng.choice([dim, dim, dim // 16 * 8])
    axes = rng.choice([1, 1, 2, 3, 4])
    cut = sorted(rng.sample(range(1, rot // 2), axes - 1))
    return dict(op="rotate", tokens=_log(rng, 1, 8192), heads=_log(rng, 1, 64), dim=dim, rot=rot,
                sections=" ".join(str(b - a) for a, b in zip([0] + cut, cut + [rot // 2])), layout=rng.choice(["chunks", "cycle", "own"]),
                pairs=rng.choice(["halves", "neighbours"]), inverse=rng.choice([True, False]), strided=rng.choice([True, False]),
                x=rng.choice(["f32", "f16"]), out=rng.choice(["f32", "f16"]), far=_log(rng, 1, 1 << 20))


def _draw_blocks(rng):
    kind = rng.choice(["decode", "decode", "drafts", "prompt"])
    c = dict(op="blocks", kv_heads=rng.choice([1, 2, 4, 8, 16]), dim=rng.choice([64, 96, 128, 128, 256]),
             page=rng.choice([16, 32, 48, 64, 128]), ragged=rng.choice([True, False]), idle=rng.choice([False, False, True]),
             count=_log(rng, 4, 128), first=rng.randint(0, 2), last=rng.randint(1, 2), softcap=rng.choice([0.0, 0.0, 30.0]),
             x=rng.choice(["f32", "f16"]))
    c["q_heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 16])
    if kind == "decode":
        c.update(batch=_log(rng, 1, 64), new=1, len=_log(rng, 1, 131072))
    elif kind == "drafts":
        c.update(batch=_log(rng, 1, 32), new=rng.randint(2, 16), len=_log(rng, 16, 32768))
    else:
        n = _log(rng, 17, 256)
        c.update(batch=_log(rng, 1, 4), new=n, len=n + _log(rng, 1, 32768))
    if c["batch"] == 1:
        c["idle"] = False
    return c


def _bounded(c):
    if c["op"] == "plan":
        return c["batch"] * c["new"] <= 150000
    if c["op"] == "adapt":
        plain = 2.0 * c["rows"] * c["adapters"] * c["rank"] * (c["k"] + c["n"])
        return (c["rows"] * c["n"] <= MAX_OUT and work(c)["flops"] <= MAX_FLOPS and plain <= 4 * MAX_FLOPS and
                c["adapters"] * c["rank"] * (c["k"] + c["n"]) <= 5.0e7)
    if c["op"] == "rotate":
        return c["tokens"] * c["heads"] * c["dim"] <= MAX_ROWS
    row, most = c["kv_heads"] * c["dim"], -(-c["len"] // c["page"])
    queries = c["batch"] * c["new"]
    return (c["batch"] * c["len"] * row <= MAX_CACHE and queries * min(c["len"], c["count"] * c["page"]) * row <= MAX_GATHER and
            queries * most * row <= MAX_SCORED and c["q_heads"] <= 128)


def draw(rng):
    """One more case: sizes spread over their logarithm, any head layout."""
    while True:
        c = rng.choice([_draw_plan, _draw_adapt, _draw_rotate, _draw_blocks, _draw_blocks])(rng)
        if _bounded(c):
            return c


def _seqs(case):
    """(new, len) of each sequence; the order they come in is the seed's."""
    n, length, got = case["new"], case["len"], []
    for b in range(case["batch"]):
        if not case["ragged"] or b == 0:
            got.append((n, max(n, length)))
            continue
        new = 1 + int((n - 1) * ((b * 0.7548776662) % 1.0))
        got.append((new, new + int(max(0, length - n) * ((b * 0.6180339887) % 1.0))))
    if case["idle"]:
        got[-1] = (1, 0)  # an idle slot: its token is nobody's
    return got


def _changes(case):
    """(held, add) of each sequence of a plan."""
    got = []
    for b in range(case["batch"]):
        held = int(case["len"] * ((b * 0.6180339887 + 0.37) % 1.0))
        add = 1 + int((case["new"] - 1) * ((b * 0.7548776662 + 0.5) % 1.0))
        kind = b % 16
        if kind == 3:
            add = -min(held, case["drop"])   # drafts that were rejected
        elif kind == 7:
            add = -held                      # ended
        elif kind == 11:
            add = 0                          # waits
        elif kind == 13 and case["new"] > 1:
            held = 0                         # a prompt
        got.append((held, add))
    return got


def _sections(case):
    """Pairs of each axis."""
    return [int(n) for n in case["sections"].split()]


def work(case):
    """Each input read once and each output written once; what the result needs to be computed."""
    op = case["op"]
    if op == "plan":
        rows = sum(max(a, 0) for _, a in _changes(case))
        # lengths and changes in, lengths, starts and page counts out; a page id taken or given back is read and
        # written; a row's position, slot and page
        moved = sum(abs(-(-(h + a) // case["page"]) + -h // case["page"]) for h, a in _changes(case))
        return {"bytes": 28.0 * case["batch"] + 8.0 * moved + 16.0 * rows, "flops": 4.0 * rows + 8.0 * case["batch"]}
    if op == "adapt":
        used = min(case["adapters"], case["rows"])
        held = 2.0 * used * case["rank"] * (case["k"] + case["n"])
        return {"bytes": held + case["rows"] * (case["k"] * SIZE[case["x"]] + 8.0 * case["n"]),
                "flops": 2.0 * case["rows"] * case["rank"] * (case["k"] + case["n"])}
    if op == "rotate":
        values = float(case["tokens"] * case["heads"] * case["dim"])
        return {"bytes": values * (SIZE[case["x"]] + SIZE[case["out"]]) + 4.0 * len(_sections(case)) * case["tokens"],
                "flops": 3.0 * values * case["rot"] / case["dim"]}
    row, page, count = case["kv_heads"] * case["dim"], case["page"], case["count"]
    held, flops, io = 0.0, 0.0, 0.0
    for n, ln in _seqs(case):
        if ln == 0:
            continue
        blocks, keys = -(-ln // page), min(ln, count * page)
        # keys of the blocks that some row of the sequence chooses (each on its own)
        union = ln * (1 - (1 - keys / ln) ** n)
        bounds = blocks * row * 4 if blocks > count else 0  # (all are chosen: nothing to score)
        touched = min(ln, n + page) * row * 9 / 16 + -(-n // page) * row * 4
        held += union * row * 9 / 8 + bounds + touched
        flops += n * case["q_heads"] * case["dim"] * (4.0 * keys + (4.0 * blocks if blocks > count else 0))
        io += 2.0 * n * case["q_heads"] * case["dim"] * SIZE[case["x"]] + 4.0 * n * case["kv_heads"] * count
    return {"bytes": held + io, "flops": flops}


# ---- a program's state ----------------------------------------------------------------


def _gen(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 64 + stream)
    return g


def _host_gen(seed, stream):
    g = torch.Generator()
    g.manual_seed(int(seed) * 64 + stream)
    return g


def _shuffled(items, seed):
    return [items[i] for i in torch.randperm(len(items), generator=_host_gen(seed, 1)).tolist()]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


class Buffer:
    """A torch tensor as the binding takes device buffers: address, dtype, shape and size."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes, self.shape = t, t.data_ptr(), t.numel() * t.element_size(), tuple(t.shape)
        self.dtype = np.dtype({torch.float32: np.float32, torch.float16: np.float16, torch.int32: np.int32,
                               torch.int64: np.int64}[t.dtype])


_context = None


def context():
    """One context for the process, as a program keeps one per device, on torch's current stream: what is
    prepared, run and read of the results follows in order.  (torch's default stream has no address to
    give: another is made the current one.)"""
    global _context
    if _context is None:
        import arf_amd
        stream = torch.cuda.Stream()
        torch.cuda.set_stream(stream)
        _context = arf_amd.Context(0, stream.cuda_stream)
    return _context


def _plan_inputs(case, seed):
    """add, held [batch], pages [batch, max_pages], the stack of free pages, their number, the step's rows."""
    page, seqs = case["page"], _shuffled(_changes(case), seed)
    held_pages = [-(-h // page) for h, _ in seqs]
    need = [-(-(h + a) // page) for h, a in seqs]
    most = max(1, max(max(a, b) for a, b in zip(held_pages, need)))
    used, wanted = sum(held_pages), sum(max(0, b - a) for a, b in zip(held_pages, need))
    back = sum(max(0, a - b) for a, b in zip(held_pages, need))
    free = max(0, wanted - back)
    free = free // 2 if case["short"] else free + 7
    total = max(1, used + free)
    ids = torch.randperm(total, generator=_host_gen(seed, 6)).to(torch.int32)
    pages = torch.full((len(seqs), most), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(held_pages):
        pages[b, :n] = ids[at:at + n]
        at += n
    stack = torch.full((total,), -1, dtype=torch.int32)
    stack[:free] = ids[at:at + free]
    return ([a for _, a in seqs], [h for h, _ in seqs], pages, stack, free, max(1, sum(max(a, 0) for _, a in seqs)))


def _adapt_inputs(case, seed):
    rows, e = case["rows"], case["adapters"]
    if case["runs"]:
        cut = sorted(torch.randint(0, rows + 1, (min(e, rows) - 1,), generator=_host_gen(seed, 2)).tolist())
        which = torch.randperm(e, generator=_host_gen(seed, 3))
        ids = torch.cat([torch.full((b - a,), int(which[i]), dtype=torch.int32)
                         for i, (a, b) in enumerate(zip([0] + cut, cut + [rows]))])
    else:
        ids = torch.randint(0, e, (rows,), generator=_host_gen(seed, 2), dtype=torch.int32)
    if case["none"]:
        ids[torch.rand(rows, generator=_host_gen(seed, 4)) < 0.125] = -1
    a = torch.randn(e, case["rank"], case["k"], generator=_gen(seed, 5), device="cuda") / math.sqrt(case["k"])
    b = torch.randn(e, case["n"], case["rank"], generator=_gen(seed, 6), device="cuda") / 8
    x = torch.randn(rows, case["k"], generator=_gen(seed, 7), device="cuda").to(DTYPE[case["x"]])
    base = torch.randn(rows, case["n"], generator=_gen(seed, 8), device="cuda")
    scale = torch.rand(e, generator=_gen(seed, 9), device="cuda") + 0.5
    return ids.cuda(), a.half(), b.half(), scale, x, base


def _rotate_inputs(case, seed):
    """positions [axes, tokens] and rows [tokens, heads, dim] (strided: the columns of wider rows)."""
    heads, wide = case["heads"], case["heads"] + (4 if case["strided"] else 0)
    pos = torch.randint(0, case["far"], (len(_sections(case)), case["tokens"]), generator=_gen(seed, 2), device="cuda",
                        dtype=torch.int32)
    x = torch.randn(case["tokens"], wide, case["dim"], generator=_gen(seed, 3), device="cuda").to(DTYPE[case["x"]])
    return pos, x[:, :heads]


def _freqs(case):
    """(axis, frequency) of each pair.  chunks: the axes' sections one after another; cycle: the axes in turn while
    they have pairs left; the frequency falls with the pair.  own: each axis from its own highest one on."""
    sections, half = _sections(case), case["rot"] // 2
    if case["layout"] == "cycle":
        left, axes = list(sections), []
        while len(axes) < half:
            for a in range(len(left)):
                if left[a]:
                    left[a] -= 1
                    axes.append(a)
    else:
        axes = [a for a, n in enumerate(sections) for _ in range(n)]
    if case["layout"] == "own":
        return [(a, 10000.0 ** (-i / n)) for a, n in enumerate(sections) for i in range(n)]
    return [(a, 10000.0 ** (-i / half)) for i, a in enumerate(axes)]


GAIN = 1.0


def _cached(case, seed):
    """K and V of every cached token, sequence after sequence: [rows, kv_heads, dim].  Keys have a few
    channels eight times larger, as those of language models do, and drift along the sequence."""
    rows, shape = sum(ln for _, ln in _seqs(case)), (case["kv_heads"], case["dim"])
    k = torch.randn(rows, *shape, generator=_gen(seed, 2), device="cuda", dtype=torch.float16)
    v = torch.randn(rows, *shape, generator=_gen(seed, 3), device="cuda", dtype=torch.float16)
    k += torch.randn(rows // 64 + 1, *shape, generator=_gen(seed, 7), device="cuda", dtype=torch.float16).repeat_interleave(64, 0)[:rows]
    k *= torch.where(torch.rand(shape, generator=_gen(seed, 4), device="cuda") < 1 / 32, 8.0, 1.0).half()
    return k, v


def _queries(case, seed):
    toks = sum(n for n, _ in _seqs(case))
    q = torch.randn(toks, case["q_heads"], case["dim"], generator=_gen(seed, 5), device="cuda")
    return q.to(DTYPE[case["x"]])


def _tables(case, seed, seqs):
    """start [batch + 1], len [batch] and pages [batch, max_pages] (int32), and the number of pages."""
    need = [-(-ln // case["page"]) for _, ln in seqs]
    total, most = max(1, sum(need)), max(1, max(need))
    ids = torch.randperm(total, generator=_host_gen(seed, 6)).to(torch.int32)
    pages = torch.full((len(seqs), most), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        pages[b, :n] = ids[at:at + n]
        at += n
    cum = [0]
    for n, _ in seqs:
        cum.append(cum[-1] + n)
    return _int32(cum), _int32([ln for _, ln in seqs]), pages.cuda(), total


def _whole(lens):
    """start [batch + 1] of a step whose tokens are all that is cached."""
    return torch.cat([lens.new_zeros(1), torch.cumsum(lens, 0).to(torch.int32)])


def prepare(case, seed):
    if own:
        context()
    s = {"plan": _prepare_plan, "adapt": _prepare_adapt, "rotate": _prepare_rotate, "blocks": _prepare_blocks}[case["op"]](case, seed)
    s["case"] = case
    torch.cuda.synchronize()
    return s


def _prepare_plan(case, seed):
    add, held, pages, stack, free, tokens = _plan_inputs(case, seed)
    n = case["batch"]
    s = dict(add=_int32(add), held=_int32(held), pages=pages.cuda(), free=stack.cuda(), n_free=_int32([free]),
             held_next=_int32([0] * n), n_free_next=_int32([0]), start=_int32([0] * (n + 1)), lens=_int32([0] * n),
             taken=_int32([0] * (n + 1)), freed=_int32([0] * (n + 1)), positions=_int32([0] * tokens),
             slots=torch.zeros(tokens, dtype=torch.int64, device="cuda"))
    if own:
        import arf_amd
        s["step"] = arf_amd.KVStep(case["page"], **{name: Buffer(t) for name, t in s.items()})
    return s


def _prepare_adapt(case, seed):
    ids, a, b, scale, x, base = _adapt_inputs(case, seed)
    s = dict(ids=ids, a=a, b=b, scale=scale, x=x, base=base)
    if own:
        import arf_amd
        s["lora"] = arf_amd.Lora(Buffer(a), Buffer(b), Buffer(scale))
        s["buf"] = {n: Buffer(s[n]) for n in ("ids", "x", "base")}
        s["out"] = Buffer(torch.empty_like(base))
    return s


def _prepare_rotate(case, seed):
    pos, x = _rotate_inputs(case, seed)
    s = dict(pos=pos, x=x)
    if own:
        import arf_amd
        pairs = _freqs(case)
        s["rope"] = arf_amd.Rope([f for _, f in pairs], [a for a, _ in pairs], pairs=case["pairs"], gain=GAIN)
        s["buf"] = {"pos": Buffer(pos), "x": Buffer(x)}
        if case["strided"]:  # (the rows' first columns: what lies from there to the array's end)
            s["buf"]["x"].nbytes = x.untyped_storage().nbytes()
        s["out"] = Buffer(torch.empty(x.shape, device="cuda", dtype=DTYPE[case["out"]]))
    return s


def _prepare_blocks(case, seed):
    seqs = _shuffled(_seqs(case), seed)
    start, lens, pages, n_pages = _tables(case, seed, seqs)
    toks = sum(n for n, _ in seqs)
    s = dict(start=start, lens=lens, pages=pages, tokens=toks, q=_queries(case, seed))
    k, v = _cached(case, seed)
    whole, d, kvh, page = _whole(lens), case["dim"], case["kv_heads"], case["page"]
    if own:
        import arf_amd
        ctx = context()
        s["kv"] = ctx.kv_cache(kvh, d, page, n_pages)
        s["bounds"] = torch.zeros(n_pages, kvh, 2, d, device="cuda", dtype=torch.float16)
        buf = {n: Buffer(s[n]) for n in ("start", "lens", "pages", "q", "bounds")}
        s["buf"], s["seqs"] = buf, arf_amd.KVSeqs(buf["pages"], buf["lens"], buf["start"] if case["new"] > 1 else None, toks)
        s["out"] = Buffer(torch.empty_like(s["q"]))
        s["chosen"] = Buffer(torch.full((toks, kvh, case["count"]), -1, dtype=torch.int32, device="cuda"))
        # the cache and its bounds as earlier steps left them
        every = arf_amd.KVSeqs(buf["pages"], buf["lens"], Buffer(whole), k.shape[0])
        ctx.kv_write(s["kv"], every, Buffer(k), Buffer(v))
        ctx.kv_bounds(s["kv"], every, buf["bounds"])
        return s
    # a page behind the others takes what has no place
    for name, t in (("k", k), ("v", v)):
        s[name + "c"] = torch.zeros(n_pages + 1, page, kvh, d // 2, device="cuda", dtype=torch.uint8)
        s[name + "s"] = torch.zeros(n_pages + 1, page, kvh, d // GROUP, device="cuda", dtype=torch.float16)
        b, pos = _places(whole, lens, t.shape[0])
        at = pages[b, pos // page].long()
        s[name + "c"][at, pos % page], s[name + "s"][at, pos % page] = _quantise(t)
    s["bounds"] = torch.zeros(n_pages + 1, kvh, 2, d, device="cuda", dtype=torch.float16)
    b = torch.arange(pages.shape[0], device="cuda").repeat_interleave(pages.shape[1])
    block = torch.arange(pages.shape[1], device="cuda").repeat(pages.shape[0])
    chunk = max(1, int(2.0e8) // (page * kvh * d))
    for i in range(0, b.numel(), chunk):
        _bounds(s, page, b[i:i + chunk], block[i:i + chunk])
    return s


# ---- the plain forms ------------------------------------------------------------------


def _plan(s):
    page, add, held = s["case"]["page"], s["add"].long(), s["held"].long()
    pages, stack, n, most = s["pages"], s["free"], s["add"].shape[0], s["pages"].shape[1]
    tokens, cap = s["positions"].shape[0], s["free"].shape[0]
    zero = held.new_zeros(1)
    ends = torch.cumsum(add.clamp(min=0), 0)
    new = (held + add).clamp(min=0)
    have, need = (held + page - 1) // page, (new + page - 1) // page
    fits = (add > 0) & (ends <= tokens) & (need <= most)
    want = torch.where(fits, need - have, 0)
    back = torch.where(add < 0, have - need, 0)
    freed = torch.cat([zero, torch.cumsum(back, 0)])
    upto = torch.cumsum(want, 0)
    there = s["n_free"].long() + freed[-1]
    given = fits & ((want == 0) | (upto <= there))
    taken = torch.cat([zero, torch.cumsum(torch.where(given, want, 0), 0)])
    # the pages given back, in the order of sequences and their pages (what has none goes behind the last)
    j = torch.arange(most, device=pages.device)
    gone = (j >= need[:, None]) & (j < have[:, None]) & (add < 0)[:, None]
    order = torch.where(gone, freed[:-1, None] + j - need[:, None], n * most)
    released = torch.zeros(n * most + 1, device=pages.device, dtype=torch.int32)
    released[order.reshape(-1)] = pages.reshape(-1)
    # the step's rows
    t = torch.arange(tokens, device=pages.device)
    start = torch.cat([zero, ends]).clamp(max=tokens)
    b = torch.searchsorted(start[1:], t, right=True).clamp(max=n - 1)
    on = given[b] & (t < ends[b])
    pos = torch.where(on, new[b] - (ends[b] - t), 0)
    i = taken[b] + pos // page - have[b]
    fresh = on & (pos // page >= have[b])
    from_stack = s["n_free"].long() - 1 - (i - freed[-1])
    id_new = torch.where(i < freed[-1], released[i.clamp(0, n * most)], stack[from_stack.clamp(0, cap - 1)])
    id_old = pages[b, (pos // page).clamp(max=most - 1)]
    ids = torch.where(fresh, id_new, id_old)
    s["positions"] = torch.where(on, pos, -1).int()
    s["slots"] = torch.where(on, ids.long() * page + pos % page, -1)
    # the tables' new entries, and the stack's
    flat = torch.cat([pages.reshape(-1), pages.new_zeros(1)])
    flat[torch.where(fresh, b * most + pos // page, n * most)] = torch.where(fresh, ids, 0)
    s["pages"] = flat[:-1].reshape(n, most)
    rank = torch.arange(n * most, device=pages.device)
    left = (rank >= taken[-1]) & (rank < freed[-1])
    at = s["n_free"].long() + freed[-1] - 1 - rank
    wide = torch.cat([stack, stack.new_zeros(1)])
    wide[torch.where(left, at.clamp(0, cap), cap)] = released[:-1]
    s["free"] = wide[:-1]
    s["held_next"] = torch.where((add <= 0) | given, new, held).int()
    s["n_free_next"] = (there - taken[-1]).int()
    s["start"], s["taken"], s["freed"] = start.int(), taken.int(), freed.int()
    s["lens"] = torch.where((add <= 0) | given, new, 0).int()
    return _plan_outputs(s)


PLAN_OUT = ("held_next", "n_free_next", "pages", "free", "start", "lens", "taken", "freed", "positions", "slots")


def _plan_outputs(s):
    return {name: s[name] for name in PLAN_OUT}


def _adapt(s):
    ids, x = s["ids"].long(), s["x"].float()
    e, r, k = s["a"].shape
    h = torch.matmul(x, s["a"].float().reshape(e * r, k).t()).reshape(-1, e, r)
    mine = (ids[:, None] == torch.arange(e, device=ids.device)).float() * s["scale"]
    h = (h * mine[:, :, None]).reshape(-1, e * r)
    b = s["b"].float().permute(0, 2, 1).reshape(e * r, -1)
    return s["base"] + torch.matmul(h, b)


def _rotate(s):
    c, x = s["case"], s["x"].float()
    pairs = _freqs(c)
    axes = torch.tensor([a for a, _ in pairs], device=x.device)
    freq = torch.tensor([f for _, f in pairs], device=x.device, dtype=torch.float64)
    angle = s["pos"].double()[axes].t() * freq * (-1.0 if c["inverse"] else 1.0)
    cos, sin = ((f(angle) * GAIN).float()[:, None] for f in (torch.cos, torch.sin))
    half = c["rot"] // 2
    a, b = (x[..., :half], x[..., half:c["rot"]]) if c["pairs"] == "halves" else (x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([ra, rb], -1) if c["pairs"] == "halves" else torch.stack([ra, rb], -1).flatten(-2)
    return torch.cat([turned, x[..., c["rot"]:]], -1).to(DTYPE[c["out"]])


def _places(start, lens, toks):
    """Each token's sequence and its position there."""
    t = torch.arange(toks, device=start.device, dtype=torch.int32)
    b = torch.searchsorted(start[1:], t, right=True)
    return b, (lens[b] - (start[b + 1] - t)).long()


def _quantise(x):
    """Codes (two a byte: value i and i + 16 of a group) and scales of [..., dim]."""
    g = x.float().reshape(*x.shape[:-1], -1, GROUP)
    hi, lo = g.amax(-1), g.amin(-1)
    s = torch.where(hi >= -lo, hi, lo)
    d = (s / -8).clamp(-8160, 8160).bfloat16().half()
    wide = d.double()[..., None]
    q = torch.where(wide == 0, 0.0, torch.round(g.double() / torch.where(wide == 0, 1.0, wide))).clamp(-8, 7)
    q = (q + 8).to(torch.uint8)
    return (q[..., :16] | q[..., 16:] << 4).reshape(*x.shape[:-1], -1), d


def _values(codes, scales):
    """[..., dim] in 32 bits."""
    c = codes.reshape(*scales.shape, 16)
    q = torch.cat([c & 15, c >> 4], -1).float() - 8
    return (q * scales.float()[..., None]).reshape(*scales.shape[:-1], -1)


def _bounds(s, page, b, block):
    """hi and lo of the blocks of sequences b."""
    keys = (s["lens"][b] - block * page).clamp(0, page)
    at = torch.where(keys > 0, s["pages"][b, block.clamp(min=0)].long(), s["bounds"].shape[0] - 1)
    k = _values(s["kc"][at], s["ks"][at])
    no = torch.arange(page, device=k.device) >= keys[:, None]
    s["bounds"][at] = torch.stack([k.masked_fill(no[..., None, None], -math.inf).amax(1),
                                   k.masked_fill(no[..., None, None], math.inf).amin(1)], 2).half()


def _blocks(s):
    c, q, lens, pages = s["case"], s["q"], s["lens"], s["pages"]
    toks, heads, dim = q.shape
    kvh, page, count, most = c["kv_heads"], c["page"], c["count"], pages.shape[1]
    g = heads // kvh
    b, pos = _places(s["start"], lens, toks)
    _bounds(s, page, b, torch.where(pos >= 0, pos // page, -1))
    out, chosen = torch.empty_like(q), torch.full((toks, kvh, count), -1, device=q.device, dtype=torch.int32)
    width = min(count, most)
    step = max(1, int(1.2e8) // max(most * kvh * dim, width * page * kvh * dim))
    j = torch.arange(most, device=q.device)
    for t in range(0, toks, step):
        bb, pp = b[t:t + step], pos[t:t + step]
        n = bb.shape[0]
        x = q[t:t + step].float().reshape(n, kvh, g, dim)
        seen = torch.where(pp >= 0, pp // page + 1, 0)
        ids = pages[bb].clamp(min=0).long()
        wide = x.double()
        hi, lo = (s["bounds"][:, :, i][ids].double().permute(0, 2, 3, 1).contiguous() for i in (0, 1))
        score = (torch.matmul(wide.clamp(min=0), hi) + torch.matmul(wide.clamp(max=0), lo)).amax(2)
        forced = (j < c["first"]) | (j >= seen[:, None] - c["last"])
        score = torch.where(forced[:, None], math.inf, score).masked_fill((j >= seen[:, None])[:, None], -math.inf)
        best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :width]
        best = torch.where(best < seen[:, None, None], best, most)  # what is not seen comes last
        best = torch.sort(best, dim=-1).values
        got = torch.where(best < most, best, -1)
        chosen[t:t + step, :, :width] = got.int()
        at = torch.gather(ids[:, None].expand(n, kvh, most), 2, best.clamp(max=most - 1))
        h = torch.arange(kvh, device=q.device)[:, None, None]
        off = torch.arange(page, device=q.device)
        k, v = (_values(s[y + "c"][at[..., None], off, h], s[y + "s"][at[..., None], off, h]).reshape(n, kvh, -1, dim) for y in "kv")
        w = torch.matmul(x, k.transpose(2, 3).contiguous()) * (1 / math.sqrt(dim))
        if c["softcap"]:
            w = c["softcap"] * torch.tanh(w / c["softcap"])
        ok = (got[..., None] >= 0) & (got[..., None] * page + off <= pp[:, None, None, None])
        w = w.masked_fill(~ok.reshape(n, kvh, 1, -1), -math.inf)
        top = w.amax(-1, keepdim=True)
        p = torch.exp(w - torch.where(torch.isfinite(top), top, 0.0))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
        out[t:t + step] = o.reshape(n, heads, dim).to(q.dtype)
    return {"out": out, "chosen": chosen, "bounds": s["bounds"][:-1]}


def run(s):
    c = s["case"]
    if not own:
        return {"plan": _plan, "adapt": _adapt, "rotate": _rotate, "blocks": _blocks}[c["op"]](s)
    ctx = context()
    if c["op"] == "plan":
        ctx.kv_plan(s["step"])
        return _plan_outputs(s)
    buf = s["buf"]
    if c["op"] == "adapt":
        ctx.lora_add(s["lora"], buf["ids"], buf["x"], c["rows"], s["out"], base=buf["base"])
        return s["out"].t
    if c["op"] == "rotate":
        stride = s["x"].stride(0)
        ctx.rope(s["rope"], buf["pos"], buf["x"], s["out"], c["tokens"], c["heads"], c["dim"], x_stride=stride, inverse=c["inverse"])
        return s["out"].t
    ctx.kv_bounds(s["kv"], s["seqs"], buf["bounds"])
    ctx.kv_attention_blocks(s["kv"], s["seqs"], buf["bounds"], buf["q"], s["out"], c["q_heads"], 1 / math.sqrt(c["dim"]),
                            c["count"], first=c["first"], last=c["last"], softcap=c["softcap"], chosen=s["chosen"])
    return {"out": s["out"].t, "chosen": s["chosen"].t, "bounds": s["bounds"]}


# ---- the same in 64 bits --------------------------------------------------------------


def _exact_plan(case, seed):
    """Sequence after sequence, page after page."""
    add, held, pages, stack, free, tokens = _plan_inputs(case, seed)
    page, pages, stack = case["page"], pages.tolist(), stack.tolist()
    most = len(pages[0])
    pool = []  # what is given back, in order
    freed, taken, start = [0], [0], [0]
    for h, a, row in zip(held, add, pages):
        if a < 0:
            left = max(0, h + a)
            pool += row[(left + page - 1) // page:(h + page - 1) // page]
        freed.append(len(pool))
        start.append(start[-1] + max(a, 0))
    there = free + len(pool)
    wanted, next_held, lens, positions, slots = 0, [], [], [], []
    took = 0
    for h, a, row in zip(held, add, pages):
        new = max(0, h + a)
        if a > 0:
            more = (new + page - 1) // page - (h + page - 1) // page
            wanted += more
            if more and wanted > there:
                next_held.append(h)
                lens.append(0)
                positions += [-1] * a
                slots += [-1] * a
                taken.append(took)
                continue
            for i in range((h + page - 1) // page, (new + page - 1) // page):
                row[i] = pool[took] if took < len(pool) else stack[free - 1 - (took - len(pool))]
                took += 1
            for p in range(h, new):
                positions.append(p)
                slots.append(row[p // page] * page + p % page)
        next_held.append(new)
        lens.append(new)
        taken.append(took)
    for rank in range(took, len(pool)):
        stack[free + len(pool) - 1 - rank] = pool[rank]
    positions += [-1] * (tokens - len(positions))
    slots += [-1] * (tokens - len(slots))
    got = dict(held_next=next_held, n_free_next=[there - took], pages=pages, free=stack, start=start, lens=lens, taken=taken,
               freed=freed, positions=positions)
    got = {name: _int32(v) for name, v in got.items()}
    got["slots"] = torch.tensor(slots, dtype=torch.int64).cuda()
    return {name: got[name] for name in PLAN_OUT}


def _exact_adapt(case, seed):
    ids, a, b, scale, x, base = _adapt_inputs(case, seed)
    out = base.double()
    for e in ids.unique().tolist():
        if e >= 0:
            rows = torch.nonzero(ids == e)[:, 0]
            h = x[rows].double() @ a[e].double().t().contiguous()
            out[rows] += scale[e].double() * (h @ b[e].double().t().contiguous())
    return out


def _exact_rotate(case, seed):
    pos, x = _rotate_inputs(case, seed)
    half, out = case["rot"] // 2, x.double()
    for i, (axis, freq) in enumerate(_freqs(case)):
        turn = torch.polar(torch.full((case["tokens"],), GAIN, dtype=torch.float64, device="cuda"), pos[axis].double() * freq)
        if case["inverse"]:
            turn = turn.conj()
        i, j = (i, i + half) if case["pairs"] == "halves" else (2 * i, 2 * i + 1)
        z = torch.complex(x[..., i].double(), x[..., j].double()) * turn[:, None]
        out[..., i], out[..., j] = z.real, z.imag
    return out


def _stored(x):
    """What the cache holds for x, from the definition."""
    g = x.double().unflatten(-1, (-1, GROUP))
    top, low = g.max(-1).values, g.min(-1).values
    s = torch.where(top + low >= 0, top, low)
    m, e = torch.frexp(torch.clamp(-s / 8, -8160, 8160))
    two = (e.long() - 8 + 1023).bitwise_left_shift(52).view(torch.float64)  # 2^(e - 8), to the bit
    d = torch.round(m * 256) * two  # 8 significant bits
    d = torch.where(d.abs() < 2.0 ** -14, torch.round(d * 2.0 ** 24) * 2.0 ** -24, d)[..., None]
    q = torch.clamp(torch.round(torch.nan_to_num(g / d, nan=0.0, posinf=0.0, neginf=0.0)), -8, 7)
    return (q * d).flatten(-2)


def _exact_blocks(case, seed):
    seqs = _shuffled(_seqs(case), seed)
    k, v = _cached(case, seed)
    q = _queries(case, seed).double()
    kvh, dim, page, count = case["kv_heads"], case["dim"], case["page"], case["count"]
    g, toks = case["q_heads"] // kvh, q.shape[0]
    out = torch.zeros_like(q)
    chosen = torch.full((toks, kvh, count), -1, dtype=torch.int32, device="cuda")
    _, _, pages, n_pages = _tables(case, seed, seqs)
    bounds = torch.zeros(n_pages, kvh, 2, dim, dtype=torch.float64, device="cuda")
    t = end = 0
    for b, (n, ln) in enumerate(seqs):
        end += ln
        if ln == 0:
            t += n
            continue
        x = q[t:t + n].reshape(n, kvh, g, dim)
        blocks = (ln + page - 1) // page
        for h in range(kvh):
            ks, vs = _stored(k[end - ln:end, h]), _stored(v[end - ln:end, h])
            rest = blocks * page - ln
            hi = torch.cat([ks, ks[-1:].expand(rest, dim)]).reshape(blocks, page, dim).max(1).values
            lo = torch.cat([ks, ks[-1:].expand(rest, dim)]).reshape(blocks, page, dim).min(1).values
            bounds[pages[b, :blocks].long(), h] = torch.stack([hi, lo], 1)
            for i in range(n):
                y, pos = x[i, h], ln - n + i
                seen = pos // page + 1
                if seen > count:
                    score = (y.relu() @ hi.t().contiguous() - (-y).relu() @ lo.t().contiguous()).max(0).values[:seen]
                    score[:case["first"]] = math.inf
                    score[max(0, seen - case["last"]):] = math.inf
                    picked = torch.sort(score, descending=True, stable=True).indices[:count].sort().values
                else:
                    picked = torch.arange(seen, device="cuda")
                chosen[t + i, h, :picked.numel()] = picked.int()
                keys = (picked[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)
                keep = keys <= pos
                keys = keys.clamp(max=ln - 1)
                w = (y @ ks[keys].t().contiguous()) / math.sqrt(dim)
                if case["softcap"]:
                    w = case["softcap"] * torch.tanh(w / case["softcap"])
                p = torch.softmax(w.masked_fill(~keep, -math.inf), -1)
                out[t + i, h * g:(h + 1) * g] = p @ vs[keys]
        t += n
    return {"out": out, "chosen": chosen, "bounds": bounds}


def exact(case, seed):
    return {"plan": _exact_plan, "adapt": _exact_adapt, "rotate": _exact_rotate, "blocks": _exact_blocks}[case["op"]](case, seed)
