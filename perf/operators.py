"""Timed cases of the paged-cache operators (rai_b200.paged, rai_b200.beams)
and their plain forms in elementary torch operations.

Four operators that one serving step runs one after the other:
  rope    rotary positions of a chunk's q and k, k and v stored in the pages
  attend  attention of a ragged chunk of new tokens over a paged cache
  beams   beam search's choice over beams and vocabulary
  pages   forking, growing (copy on write) and compacting the cache's pages
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# (query heads, KV heads, head size): the framework's model shapes (Qwen2.5-0.5B, TinyLlama, Llama-3.1-8B, OLMoE),
# and generic ones with an odd group or head size.
SHAPES = [(14, 2, 64), (32, 4, 64), (32, 8, 128), (16, 16, 128), (8, 2, 32), (15, 5, 80), (6, 1, 96), (4, 2, 256)]


# ---------------------------------------------------------------- cases

def listed():
    return [
        # One stream's next token early in a chat: latency alone.
        attend("attend one token", "bf16", 1, 1, 1, 130, 130, 2, 0, 16),
        # A batch of streams that decode one token each.
        attend("attend decode batch", "bf16", 64, 1, 1, 300, 2300, 1, 1, 16),
        # Draft verification (up to 8 drafts and the last token) over long documents, the most bytes.
        attend("attend verify long", "bf16", 8, 1, 9, 20000, 33000, 2, 2, 64),
        # The same over the framework's own f32 rows.
        attend("attend verify f32", "f32", 16, 5, 9, 500, 1300, 1, 3, 16),
        # Prompts, whole, the most operations.
        attend("attend prompts", "bf16", 3, 1900, 4096, 0, 0, 2, 4, 64),
        # Chunks of prompts beside streams that decode, capped scores and a sliding window.
        attend("attend mixed capped", "f16", 8, 1, 700, 200, 3000, 3, 5, 32, softcap=30.0, window=1024),
        # One token each of a batch of streams.
        rope("rope decode batch", "f32", "bf16", 64, 1, 1, 300, 2300, 2, 6, 16, rot=128),
        # Prompts' rows, interleaved pairs on a part of the head, far positions.
        rope("rope prompts", "bf16", "bf16", 4, 1500, 2300, 0, 90000, 3, 7, 64, rot=64, interleaved=True),
        # Four beams of one request.
        beams("beams one request", "f32", 1, 4, 32000, 8),
        # A batch of requests over the largest vocabulary.
        beams("beams batch", "bf16", 32, 8, 151936, 9),
        # A beam step's reordering: tables forked, shared last pages copied before one more token.
        pages("pages beam step", "fork", "bf16", 64, 100, 1100, 16, 4, 64, 4, 10),
        # Defragmenting a pool after many streams have ended.
        pages("pages compact", "compact", "bf16", 96, 100, 2000, 16, 4, 64, 8, 11),
    ]


def attend(name, dtype, seqs, rows_lo, rows_hi, past_lo, past_hi, shape, ragged, page, softcap=0.0, window=0):
    h, g, d = SHAPES[shape]
    return dict(name=name, op="attend", dtype=dtype, seqs=seqs, rows_lo=rows_lo, rows_hi=rows_hi, past_lo=past_lo, past_hi=past_hi, heads=h, kv_heads=g,
                head_dim=d, page=page, softcap=softcap, window=window, ragged=ragged)


def rope(name, dtype, cache, seqs, rows_lo, rows_hi, past_lo, past_hi, shape, ragged, page, rot, interleaved=False, theta=500000.0, mscale=1.0):
    h, g, d = SHAPES[shape]
    return dict(name=name, op="rope", dtype=dtype, cache=cache, seqs=seqs, rows_lo=rows_lo, rows_hi=rows_hi, past_lo=past_lo, past_hi=past_hi, heads=h,
                kv_heads=g, head_dim=d, page=page, rot=rot, interleaved=interleaved, theta=theta, mscale=mscale, ragged=ragged)


def beams(name, dtype, batch, n, vocab, ragged):
    return dict(name=name, op="beams", dtype=dtype, batch=batch, beams=n, vocab=vocab, ragged=ragged)


def pages(name, what, dtype, seqs, len_lo, len_hi, page, kv_heads, head_dim, layers, ragged):
    return dict(name=name, op="pages", what=what, dtype=dtype, seqs=seqs, len_lo=len_lo, len_hi=len_hi, page=page, kv_heads=kv_heads, head_dim=head_dim,
                layers=layers, ragged=ragged)


def spread(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "rope", "beams", "pages"])
    ragged = rng.randrange(1000, 1 << 20)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 100, 128])
    shape = rng.randrange(len(SHAPES))
    if op == "attend":
        kind = rng.choice(["decode", "verify", "chunk"])
        top = {"decode": 1, "verify": spread(rng, 2, 33), "chunk": spread(rng, 34, 1200)}[kind]
        past = spread(rng, 1, 30000 if kind != "chunk" else 4000)
        seqs = spread(rng, 1, 96 if kind != "chunk" else 8)
        seqs = max(1, min(seqs, 300000 // past, 8000000 // (top * (past + top))))
        c = attend("", dtype, seqs, rng.choice([1, max(1, top // 2), top]), top, past // rng.choice([1, 2, 8]), past, shape, ragged, page,
                   softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), window=rng.choice([0, 0, spread(rng, 1, 5000)]))
    elif op == "rope":
        top = spread(rng, 1, 2000)
        seqs = spread(rng, 1, max(1, min(128, 8000 // top)))
        past = spread(rng, 1, 400000 // seqs)
        d = SHAPES[shape][2]
        c = rope("", dtype, rng.choice(["bf16", "f16", "f32"]), seqs, max(1, top // 3), top, past // 3, past, shape, ragged, page,
                 rot=rng.choice([d, d, d // 2, d // 4]), interleaved=rng.random() < 0.5, theta=rng.choice([10000.0, 500000.0, 1000000.0]),
                 mscale=rng.choice([1.0, 1.0, 1.25]))
    elif op == "beams":
        vocab = spread(rng, 100, 160000)
        n = spread(rng, 1, 16)
        c = beams("", dtype, spread(rng, 1, max(1, min(64, 30000000 // (n * vocab * (2 if dtype == "f32" else 1))))), n, vocab, ragged)
    else:
        seqs = spread(rng, 1, 256)
        top = spread(rng, 1, min(4000, 150000 // seqs))
        _, g, d = SHAPES[shape]
        layers = max(1, min(spread(rng, 1, 16), int(1.5e8 / (2 * SIZE[dtype] * g * d * seqs * (top + page)))))
        c = pages("", rng.choice(["fork", "compact"]), dtype, seqs, max(1, top // 4), top, page, g, d, layers, ragged)
    del c["name"]
    return c


def chunk_of(c):
    """(new rows, tokens in the cache with them) of each sequence."""
    r = random.Random(c["ragged"])
    rows = [r.randint(c["rows_lo"], c["rows_hi"]) for _ in range(c["seqs"])]
    return rows, [n + r.randint(c["past_lo"], c["past_hi"]) for n in rows]


def beam_state(c):
    """Pages of `seqs` beams in groups of up to four that share their prompt's whole pages: (table of page numbers, lengths, parents, page count, order)."""
    r = random.Random(c["ragged"])
    n, ps = c["seqs"], c["page"]
    lens, table, used = [], [], 0
    for at in range(0, n, 4):
        size = min(4, n - at)
        base = r.randint(c["len_lo"], c["len_hi"])
        shared = r.randint(0, base // ps)
        head = list(range(used, used + shared))
        used += shared
        for _ in range(size):
            more = -(-base // ps) - shared
            lens.append(base)
            table.append(head + list(range(used, used + more)))
            used += more
    parents = [at // 4 * 4 + r.randrange(min(4, n - at // 4 * 4)) for at in range(n)]
    total = 2 * used + n + 8
    order = list(range(total))
    r.shuffle(order)
    return table, lens, parents, total, order


# ---------------------------------------------------------------- inputs

def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = {"attend": make_attend, "rope": make_rope, "beams": make_beams, "pages": make_pages}[c["op"]]
    s = make(c, gen, random.Random(seed))
    s["c"] = c
    return s


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make_chunk(c, rnd, dtype, gen):
    """A pool of pages in random order that holds the sequences' tokens, its tables and lengths."""
    rows, lens = chunk_of(c)
    ps = c["page"]
    need = [-(-n // ps) for n in lens]
    total = sum(need) + 3
    order = list(range(total))
    rnd.shuffle(order)
    width = max(need)
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    shape = (total, c["kv_heads"], ps, c["head_dim"])
    return dict(table=ints(table), kv_len=ints(lens), q_start=ints(starts), max_rows=max(rows), rows=starts[-1], k=normal(shape, dtype, gen),
                v=normal(shape, dtype, gen))


def normal(shape, dtype, gen, scale=1.0):
    x = torch.empty(shape, dtype=DT[dtype], device="cuda")
    x.normal_(0.0, scale, generator=gen)
    return x


def make_attend(c, gen, rnd):
    s = make_chunk(c, rnd, c["dtype"], gen)
    s["q"] = normal((s["rows"], c["heads"], c["head_dim"]), c["dtype"], gen, 1.5)
    s["scale"] = c["head_dim"] ** -0.5
    return s


def make_rope(c, gen, rnd):
    s = make_chunk(c, rnd, c["cache"], gen)
    h, g, d = c["heads"], c["kv_heads"], c["head_dim"]
    qkv = normal((s["rows"], (h + 2 * g) * d), c["dtype"], gen)  # as the projection leaves it
    s["q_in"], s["k_in"], s["v_in"] = (x.view(s["rows"], -1, d) for x in qkv.split([h * d, g * d, g * d], 1))
    i = torch.arange(0, c["rot"], 2, dtype=torch.float64)
    s["inv_freq"] = (c["theta"] ** -(i / c["rot"])).float().cuda()
    return s


def make_beams(c, gen, rnd):
    b, n, v = c["batch"], c["beams"], c["vocab"]
    logits = normal((b, n, v), c["dtype"], gen, 2.5)
    banned = torch.randint(0, v, (max(1, v // 50),), generator=gen, device="cuda")
    logits[:, :, banned] = -math.inf  # what a grammar or a bad-words list takes out
    scores = -20.0 * torch.rand((b, n), generator=gen, device="cuda")
    return dict(logits=logits, scores=scores, eos=v // 3)


def make_pages(c, gen, rnd):
    table, lens, parents, total, order = beam_state(c)
    width = -(-max(lens) // c["page"]) + 2
    refs = [0] * total
    for row in table:
        for p in row:
            refs[order[p]] += 1
    shape = (c["layers"], total, c["kv_heads"], c["page"], c["head_dim"])
    return dict(table=ints([[order[p] for p in row] + [-1] * (width - len(row)) for row in table]), lens=ints(lens), refs=ints(refs), parents=ints(parents),
                k=normal(shape, c["dtype"], gen), v=normal(shape, c["dtype"], gen))


# ---------------------------------------------------------------- one pass

def run(s):
    return {"attend": run_attend, "rope": run_rope, "beams": run_beams, "pages": run_pages}[s["c"]["op"]](s)


def run_attend(s):
    c = s["c"]
    if own:
        from rai_b200 import paged
        return paged.attention(s["q"], s["k"], s["v"], s["table"], s["kv_len"], s["q_start"], s["max_rows"], scale=s["scale"], softcap=c["softcap"],
                               window=c["window"])
    n, g, d = c["seqs"], c["kv_heads"], c["head_dim"]
    j, ps, wide = c["heads"] // g, c["page"], s["max_rows"]
    start, rows = s["q_start"][:-1].long(), (s["q_start"][1:] - s["q_start"][:-1]).long()
    i = torch.arange(wide, device="cuda")
    q = s["q"][(start[:, None] + i).clamp(max=s["rows"] - 1)].float()  # n, wide, heads, d
    q = q.view(n, wide, g, j, d).permute(0, 2, 3, 1, 4).reshape(n, g, j * wide, d)
    t = torch.arange(s["table"].shape[1] * ps, device="cuda")
    page = s["table"].long()[:, t // ps].clamp(min=0)
    there = t < s["kv_len"][:, None]
    k = s["k"][page, :, t % ps].float()  # n, t, g, d
    v = torch.where(there[:, :, None, None], s["v"][page, :, t % ps].float(), 0.0)
    x = (q @ k.permute(0, 2, 3, 1)).mul_(s["scale"]).view(n, g, j, wide, -1)
    if c["softcap"]:
        x = x.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    pos = s["kv_len"].long()[:, None] - rows[:, None] + i  # n, wide
    seen = there[:, None] & (t <= pos[:, :, None])
    if c["window"]:
        seen = seen & (t > pos[:, :, None] - c["window"])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    out = x.view(n, g, j * wide, -1) @ v.permute(0, 2, 1, 3)
    out = out.view(n, g, j, wide, d) / torch.where(total == 0, 1.0, total)
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["q_start"][1:].long(), row, right=True)
    return out.permute(0, 3, 1, 2, 4)[seq, row - start[seq]].reshape(s["rows"], c["heads"], d).to(DT[c["dtype"]])


def run_rope(s):
    c = s["c"]
    if own:
        from rai_b200 import paged
        q = paged.rope_append(s["q_in"], s["k_in"], s["v_in"], s["k"], s["v"], s["table"], s["kv_len"], s["q_start"], s["inv_freq"],
                              interleaved=c["interleaved"], mscale=c["mscale"])
        return [q, s["k"], s["v"]]
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["q_start"][1:].long(), row, right=True)
    pos = (s["kv_len"][seq] - (s["q_start"][seq + 1] - row)).long()
    angle = pos[:, None].double() * s["inv_freq"].double()  # far positions lose their angle in 32 bits
    cos, sin = ((f(angle) * c["mscale"]).float()[:, None] for f in (torch.cos, torch.sin))
    q, k = (turned(x.float(), cos, sin, c["rot"], c["interleaved"]).to(DT[c["cache"]]) for x in (s["q_in"], s["k_in"]))
    page, slot = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    s["k"][page, :, slot] = k
    s["v"][page, :, slot] = s["v_in"].to(DT[c["cache"]])
    return [q, s["k"], s["v"]]


def turned(x, cos, sin, rot, interleaved):
    half = rot // 2
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :half], x[..., half:rot])
    u, w = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1), x[..., rot:]], -1)


def run_beams(s):
    c = s["c"]
    if own:
        from rai_b200 import beams as ops
        r = ops.select(s["logits"], s["scores"], eos=s["eos"])
        return [r.cand_scores, r.cand_beams, r.cand_tokens, r.scores, r.parents, r.tokens]
    b, n, v = c["batch"], c["beams"], c["vocab"]
    x = s["logits"].double()  # near scores of different beams change places in 32 bits
    x = x - x.amax(-1, keepdim=True)
    total = s["scores"].double()[:, :, None] + (x - x.exp().sum(-1, keepdim=True).log())
    raw = s["logits"].reshape(b, n * v)
    by_raw = torch.sort(raw, dim=1, descending=True, stable=True)[1]
    by_score = torch.sort(total.view(b, n * v).gather(1, by_raw), dim=1, descending=True, stable=True)[1]
    at = by_raw.gather(1, by_score[:, : 2 * n])
    score = total.view(b, n * v).gather(1, at).float()
    beam, token = at // v, at % v
    going = torch.sort((token == s["eos"]).to(torch.int8), dim=1, stable=True)[1][:, :n]  # the first n that do not end
    parent = beam.gather(1, going) + n * torch.arange(b, device="cuda")[:, None]
    return [score, beam.int(), token.int(), score.gather(1, going), parent.int(), token.gather(1, going).int()]


def run_pages(s):
    c = s["c"]
    refs = s["refs"].clone()  # the calls update them in place
    if own:
        from rai_b200 import paged
        if c["what"] == "fork":
            table, lens = paged.fork(s["table"], s["lens"], refs, s["parents"], c["page"])
            short = paged.resize(table, lens, refs, s["k"], s["v"], delta=1)
            return [table, lens, refs, short, s["k"], s["v"]]
        table = s["table"].clone()
        used = paged.compact(table, s["lens"], refs, s["k"], s["v"])
        return [table, refs, used, s["k"], s["v"]]
    if c["what"] == "compact":
        page = torch.arange(refs.numel(), device="cuda")
        held = refs > 0
        used = held.sum()
        src, dst = page[held & (page >= used)], page[~held & (page < used)]
        to = page.clone()
        to[src] = dst
        s["k"][:, dst], s["v"][:, dst] = s["k"][:, src], s["v"][:, src]
        refs[dst] = refs[src]
        refs[src] = 0
        table = torch.where(s["table"] >= 0, to.int()[s["table"].clamp(min=0).long()], s["table"])
        return [table, refs, used.int().view(1), s["k"], s["v"]]
    ps, n = c["page"], c["seqs"]
    parents = s["parents"].long()
    table, lens = s["table"][parents], s["lens"][parents]
    children = torch.bincount(parents, minlength=n)
    flat = s["table"].clamp(min=0).long()
    change = torch.where(s["table"] >= 0, children[:, None] - 1, 0).int()
    refs.index_add_(0, flat.view(-1), change.view(-1))
    # One more token: a new page where the last is full, a copy of it where others hold it too (all but the last holder).
    last = (lens - 1) // ps
    tail = table.gather(1, last[:, None].long())[:, 0]
    part = lens % ps != 0
    order = torch.arange(n, device="cuda")
    before = ((tail[:, None] == tail[None]) & part[:, None] & part[None] & (order[None] < order[:, None])).sum(1)
    copied = part & (before < refs[tail.long()] - 1)
    takes = copied | ~part
    rank = torch.cumsum(takes, 0) - 1
    free = torch.nonzero(refs == 0)[:, 0].int()
    short = (takes.sum() - free.numel()).clamp(min=0)
    got = free[rank.clamp(min=0)]
    src, dst = tail[copied].long(), got[copied].long()
    s["k"][:, dst], s["v"][:, dst] = s["k"][:, src], s["v"][:, src]
    refs.index_add_(0, src, torch.full_like(src, -1, dtype=torch.int32))
    refs[got[takes].long()] = 1
    spot = (last + (~part).int())[:, None].long()
    table.scatter_(1, spot, torch.where(takes, got, tail)[:, None])
    return [table, lens + 1, refs, short.int().view(1), s["k"], s["v"]]


# ---------------------------------------------------------------- what a pass cannot do without

def pairs_of(c):
    """(query, key) pairs that a causal mask with the case's window leaves, and the cached tokens that any row sees."""
    pairs = keys = 0
    for n, t in zip(*chunk_of(c)):
        w = c["window"] or t
        first = t - n
        pairs += sum(min(p + 1, w) for p in range(first, t))
        keys += min(t, n - 1 + w)
    return pairs, keys


def work(c):
    if c["op"] == "beams":
        rows = c["batch"] * c["beams"]
        return {"bytes": rows * (c["vocab"] * SIZE[c["dtype"]] + 4 + 24 + 12), "flops": 3 * rows * c["vocab"]}
    if c["op"] == "pages":
        table, lens, parents, total, order = beam_state(c)
        size = 2 * c["layers"] * c["kv_heads"] * c["page"] * c["head_dim"] * SIZE[c["dtype"]]
        cells = sum(len(row) for row in table)
        if c["what"] == "compact":
            held = {order[p] for row in table for p in row}
            moved = sum(p >= len(held) for p in held)
            return {"bytes": 2 * moved * size + 8 * cells + 8 * total, "flops": 0}
        copies = sum(parents.count(p) - 1 for p in set(parents) if lens[p] % c["page"])
        return {"bytes": 2 * copies * size + 8 * cells + 8 * total, "flops": 0}
    h, g, d, rows = c["heads"], c["kv_heads"], c["head_dim"], sum(chunk_of(c)[0])
    if c["op"] == "rope":
        return {"bytes": rows * (h + 2 * g) * d * (SIZE[c["dtype"]] + SIZE[c["cache"]]), "flops": 3 * rows * (h + g) * c["rot"]}
    pairs, keys = pairs_of(c)
    return {"bytes": SIZE[c["dtype"]] * d * (2 * rows * h + 2 * keys * g), "flops": 4 * pairs * h * d}


# ---------------------------------------------------------------- in 64 bits, from the definitions

def exact(c, seed):
    s = prepare(c, seed)
    return {"attend": exact_attend, "rope": exact_rope, "beams": exact_beams, "pages": exact_pages}[c["op"]](c, s)


def tokens_of(pool, row, n, page):
    """A sequence's n cached vectors per KV head, in order: kv_heads, n, head_dim."""
    kept = row[: -(-n // page)]
    return torch.cat([pool[p] for p in kept], 1)[:, :n].double()


def exact_attend(c, s):
    rows, lens = chunk_of(c)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    j, at = c["heads"] // c["kv_heads"], 0
    for n, t, line in zip(rows, lens, s["table"].tolist()):
        k, v = (tokens_of(s[x], line, t, c["page"]) for x in "kv")
        where = torch.arange(t - n, t, device="cuda")[:, None]
        key = torch.arange(t, device="cuda")[None]
        hide = (key > where) | ((key <= where - c["window"]) if c["window"] else False)
        for h in range(c["heads"]):
            x = s["scale"] * (s["q"][at:at + n, h].double() @ k[h // j].T)
            if c["softcap"]:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            x[hide] = -math.inf
            out[at:at + n, h] = torch.softmax(x, 1) @ v[h // j]
        at += n
    return out


def exact_rope(c, s):
    rows, lens = chunk_of(c)
    q = s["q_in"].double().clone()
    k, v = s["k"].double(), s["v"].double()
    half, at = c["rot"] // 2, 0
    pair = torch.arange(half)
    one = 2 * pair if c["interleaved"] else pair
    two = one + 1 if c["interleaved"] else pair + half
    one, two = one.cuda(), two.cuda()
    for n, t, line in zip(rows, lens, s["table"].tolist()):
        pos = torch.arange(t - n, t, device="cuda")
        turn = torch.polar(torch.full((n, half), c["mscale"], dtype=torch.float64, device="cuda"), pos.double()[:, None] * s["inv_freq"].double())[:, None]
        fresh = []
        for x in (s["q_in"], s["k_in"]):
            x = x[at:at + n].double().clone()
            z = torch.complex(x[..., one], x[..., two]) * turn
            x[..., one], x[..., two] = z.real, z.imag
            fresh.append(x)
        q[at:at + n] = fresh[0]
        page, slot = torch.tensor(line, device="cuda")[pos // c["page"]], pos % c["page"]
        k[page, :, slot] = fresh[1]
        v[page, :, slot] = s["v_in"][at:at + n].double()
        at += n
    return [q, k, v]


def exact_beams(c, s):
    cand, kept = [], []
    for x, score in zip(s["logits"], s["scores"]):
        best = []
        for beam in range(c["beams"]):
            logp = torch.log_softmax(x[beam].double(), 0) + score[beam].double()
            top = torch.topk(logp, min(c["vocab"], 2 * c["beams"]))
            best += [(-p, t) for p, t in zip(top[0].tolist(), top[1].tolist())]
        best = sorted(best)[: 2 * c["beams"]]
        cand.append([-p for p, _ in best])
        kept.append([-p for p, t in best if t != s["eos"]][: c["beams"]])
    return [torch.tensor(cand, dtype=torch.float64), None, None, torch.tensor(kept, dtype=torch.float64), None, None]


def exact_pages(c, s):
    table, lens, parents, total, order = beam_state(c)
    k, v = s["k"].double(), s["v"].double()
    held = {order[p] for row in table for p in row}
    if c["what"] == "compact":
        moves = list(zip(sorted(p for p in held if p >= len(held)), sorted(set(range(len(held))) - held)))
    else:
        rows = [[order[p] for p in table[x]] for x in parents]
        holders = {}
        for row in rows:
            for p in row:
                holders[p] = holders.get(p, 0) + 1
        free, moves = iter(sorted(set(range(total)) - set(holders))), []
        for row, x in zip(rows, parents):
            if lens[x] % c["page"] == 0:
                next(free)
            elif holders[row[-1]] > 1:
                holders[row[-1]] -= 1
                moves.append((row[-1], next(free)))
    if moves:
        src, dst = (torch.tensor(m, device="cuda") for m in zip(*moves))
        k[:, dst], v[:, dst] = k[:, src], v[:, src]
    return [None, None, None, k, v] if c["what"] == "compact" else [None, None, None, None, k, v]
