"""The operators of the paged key/value cache, as they are measured.

  append  new rows enter the pages: RMSNorm of q and k, rotary positions on up to three
          axes, one rounding to the cache's type
  attend  rows of one or many sequences attend over their pages: single tokens and chunks,
          causal, with a window, documents, prefixes, a tanh cap, a distance bias, a gate
  weigh   the attention weight that each cached slot received, added up per KV head
  evict   the slots with the largest weights move to a sequence's new pages, in order

`run` computes them in elementary torch operations in 32 bits, or (`own`) through
sensenova_b200.paged. A case is a dict of sizes; lengths, masks and positions follow from
it alone, values from the seed.
"""
import math
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FAR = 2**31 - 1  # a first key that no row reaches: the row sees nothing


# ---- the cases -------------------------------------------------------------------------


def _append(name, seqs, rows, ctx, **kw):
    c = dict(name=name, op="append", seqs=seqs, rows=rows, ctx=ctx, heads=16, kv=4, d=256, page=16, layout="head",
             type="f16", input="f32", rot=64, axes="interleaved", pairs="halves", norm=True)
    return {**c, **kw}


def _attend(name, seqs, rows, ctx, **kw):
    c = dict(name=name, op="attend", seqs=seqs, rows=rows, ctx=ctx, heads=16, kv=4, d=256, page=16, layout="head",
             type="f16", gate=False, cap=0.0, window=0, slopes=False, docs=0, block=0, empty=False)
    return {**c, **kw}


def _weigh(name, seqs, rows, ctx, **kw):
    return {**_attend(name, seqs, rows, ctx), "op": "weigh", "decay": 1.0, **kw}


def _evict(name, seqs, ctx, budget, **kw):
    c = dict(name=name, op="evict", seqs=seqs, rows=1, ctx=ctx, heads=16, kv=4, d=256, page=16, layout="head",
             type="f16", budget=budget, sink=4, recent=64)
    return {**c, **kw}


def listed():
    return [
        # One decode step of eight requests: q, k and v straight from the f32 projection rows of the 9B shape.
        _append("append step of 8", 8, 1, 2048),
        # A prompt with images enters the cache: two chunks, positions on three axes, 16-bit projections.
        _append("append chunk, images", 2, 4096, 6000, input="bf16", type="bf16", page=64, layout="slot", rot=64,
                axes="sections", pairs="halves"),
        # The smallest serving call: one request's next token, gated as the 9B shape's attention is.
        _attend("token, 1 x 517", 1, 1, 517, gate=True),
        # A batch of long requests, lengths up to 32768: the cache is read once, at memory speed.
        _attend("tokens, 16 x 32768", 16, 1, 32768, page=64),
        # Many short requests of a model with heads of 128, a tanh cap on the scores.
        _attend("tokens, 64 x 4096, d128", 64, 1, 4096, heads=32, kv=8, d=128, type="bf16", cap=30.0),
        # A short turn of a conversation: 37 new tokens, an image block seen both ways, and rows of padding.
        _attend("chunk 37 of 1061", 1, 37, 1061, block=24, empty=True, gate=True),
        # A prefill chunk of a long prompt over what is cached already.
        _attend("chunk 2048 of 8192", 1, 2048, 8192, page=64, gate=True),
        # Packed chunks of several requests: documents, a window, a distance bias, heads of 128.
        _attend("chunks, 6 x 1000 of 4000, d128", 6, 1000, 4000, heads=32, kv=8, d=128, type="bf16", page=32,
                layout="slot", window=1500, slopes=True, docs=2000),
        # What a decode step of eight requests looked at.
        _weigh("weigh tokens, 8 x 16384", 8, 1, 16384),
        # What a prefill chunk looked at, before its prompt is thinned out.
        _weigh("weigh chunk 2048 of 8192", 1, 2048, 8192, page=64, decay=0.0),
        # One request over its budget by a little.
        _evict("evict 1100 to 1024", 1, 1100, 1024),
        # Long prompts cut to a quarter.
        _evict("evict 8 x 16384 to 4096", 8, 16384, 4096, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    heads, kv = rng.choice([(16, 4), (4, 1), (32, 8), (12, 4), (8, 8), (20, 4), (32, 2)])
    d = rng.choice([128, 256, 256])
    c = dict(heads=heads, kv=kv, d=d, page=rng.choice([8, 16, 32, 64, 128]), layout=rng.choice(["head", "slot"]),
             type=rng.choice(["f16", "bf16"]))
    op = rng.choice(["append", "attend", "attend", "attend", "weigh", "evict"])
    if op == "append":
        seqs, rows = _log(rng, 1, 16), _log(rng, 1, 2048)
        rows = min(rows, 4096 // seqs)
        g = _append("", seqs, rows, rows + _log(rng, 1, 4096))
        c.update(input=rng.choice(["f32", c["type"]]), rot=rng.choice([32, 64, 128]), norm=rng.random() < 0.7,
                 axes=rng.choice(["one", "sections", "interleaved"]), pairs=rng.choice(["halves", "adjacent"]))
    elif op == "evict":
        ctx = _log(rng, 40, 16384)
        g = _evict("", _log(rng, 1, 8), ctx, max(8, int(ctx * rng.uniform(0.1, 0.95))))
        g.update(sink=rng.randrange(0, 5), recent=min(rng.randrange(0, 64), g["budget"] // 2))
        c["heads"] = 4 * kv
    else:
        if rng.random() < 0.5:
            seqs, rows, ctx = _log(rng, 1, 32), 1, _log(rng, 1, 16384)
        else:
            seqs, rows = _log(rng, 1, 6), _log(rng, 2, 1024)
            ctx = rows + _log(rng, 1, 6000)
            while seqs * rows * ctx * heads * d > 2048 * 8192 * 16 * 256:
                seqs, rows = max(1, seqs // 2), rows if seqs > 1 else rows // 2
        opts = dict(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), window=rng.choice([0, 0, _log(rng, 16, 4096)]),
                    slopes=rng.random() < 0.3, docs=rng.choice([0, 0, _log(rng, 50, 4000)]),
                    block=rng.choice([0, 0, _log(rng, 8, 300)]), empty=rng.random() < 0.2)
        if op == "attend":
            g = _attend("", seqs, rows, ctx, **opts, gate=rng.random() < 0.4)
        else:
            g = _weigh("", seqs, rows, ctx, **opts, decay=rng.choice([0.0, 0.5, 1.0]))
    g.update(c)
    del g["name"]
    return g


def lengths(case):
    """New rows and cached length (those rows included) of each sequence; the first has the case's own."""
    r = random.Random("%d/%d/%d" % (case["seqs"], case["rows"], case["ctx"]))
    rows, lens = [case["rows"]], [case["ctx"]]
    for _ in range(case["seqs"] - 1):
        n = r.randint(max(1, case["rows"] // 2), case["rows"])
        rows.append(n)
        lens.append(max(n, int(case["ctx"] * 2 ** r.uniform(-3, 0))))
    return rows, lens


def bounds(case):
    """For each new row, on the CPU: its sequence, its position, its first key and the end of its keys."""
    rows, lens = lengths(case)
    seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows))
    start = torch.tensor([0] + rows).cumsum(0)
    pos = torch.arange(sum(rows)) - start[seq] + (torch.tensor(lens) - torch.tensor(rows))[seq]
    first, last = torch.zeros_like(pos), torch.zeros_like(pos)
    if case.get("docs"):
        first = pos // case["docs"] * case["docs"]
    if case.get("block"):  # blocks of tokens that see one another whole, as an image's do
        last = (pos // case["block"] + 1) * case["block"]
        last = torch.where((pos // case["block"]) % 2 == 0, last, 0)
    if case.get("empty"):
        first = torch.where(torch.arange(sum(rows)) % 9 == 4, FAR, first)
    lo = first.clone()
    if case.get("window"):
        lo = torch.maximum(lo, pos + 1 - case["window"])
    hi = torch.minimum(torch.maximum(pos + 1, last), torch.tensor(lens)[seq])
    return dict(seq=seq, pos=pos, first=first, last=last, lo=lo, hi=hi, start=start, rows=rows, lens=lens)


def work(case):
    b = bounds(case)
    h, kv, d, n = case["heads"], case["kv"], case["d"], sum(b["rows"])
    if case["op"] == "append":
        size = 4 if case["input"] == "f32" else 2
        new = n * (h + 2 * kv) * d
        return {"bytes": new * (size + 2) + n * (case["rot"] * 4 + 16), "flops": 10.0 * new}
    if case["op"] == "evict":
        kept = sum(min(x, case["budget"]) for x in b["lens"]) * kv
        return {"bytes": 4 * kv * sum(b["lens"]) + kept * (2 * d * 2 * 2 + 12), "flops": 4.0 * kv * sum(b["lens"])}
    pairs = int((b["hi"] - b["lo"].clamp(min=0)).clamp(min=0).sum()) * h
    seen = 0
    for i in range(len(b["rows"])):
        s = (b["seq"] == i) & (b["hi"] > b["lo"])
        if s.any():
            seen += int(b["hi"][s].max() - b["lo"][s].min().clamp(min=0))
    if case["op"] == "weigh":
        return {"bytes": seen * kv * d * 2 + sum(b["lens"]) * kv * 8 + n * h * (d * 2 + 4), "flops": 2.0 * d * pairs}
    return {"bytes": seen * kv * d * 4 + n * h * (d * (6 if case["gate"] else 4) + 4), "flops": 4.0 * d * pairs}


# ---- inputs ----------------------------------------------------------------------------


def _package():
    for p in ("sense-nova-server_b200",):
        if p not in sys.path:
            sys.path.insert(0, p)
    from sensenova_b200 import paged

    return paged


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, type=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").to(type)

    b = bounds(case)
    h, kv, d, page, n = case["heads"], case["kv"], case["d"], case["page"], sum(b["rows"])
    t = TYPES[case["type"]]
    need = [-(-x // page) for x in b["lens"]]
    budget_pages = -(-case.get("budget", 0) // page) if case["op"] == "evict" else 0
    pages = sum(need) + budget_pages * case["seqs"] + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(case["seqs"], max(need), dtype=torch.int32, device="cuda")
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    shape = (pages, kv, page, d) if case["layout"] == "head" else (pages, page, kv, d)

    filled = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for i, x in enumerate(b["lens"]):
        key = torch.arange(x, device="cuda")
        filled[table[i, key // page].long(), key % page] = True

    def pool():
        x = torch.randn(shape, generator=g, device="cuda").to(t)
        x = x if case["layout"] == "head" else x.transpose(1, 2)  # [page, head, slot, d] in either layout
        if case["op"] in ("attend", "weigh"):  # what no token has filled yet holds anything
            x.masked_fill_(~filled[:, None, :, None], math.nan)
        return x

    s = dict(case=case, k=pool(), v=pool(), table=table,
             start=b["start"].to(torch.int32).cuda(), lens=torch.tensor(b["lens"], dtype=torch.int32, device="cuda"),
             seq=b["seq"].cuda(), pos=b["pos"].cuda(), n=n, max_rows=max(b["rows"]), max_len=max(b["lens"]))
    if case["op"] == "append":
        i = TYPES[case["input"]]
        if case["input"] == "f32":  # the engine's projection rows: per head [q | gate], then k, then v
            proj = normal(n, 2 * h * d + 2 * kv * d)
            s["q"] = proj[:, :2 * h * d].view(n, h, 2 * d)[:, :, :d]
            s["new_k"] = proj[:, 2 * h * d:2 * h * d + kv * d].view(n, kv, d)
            s["new_v"] = proj[:, 2 * h * d + kv * d:].view(n, kv, d)
        else:
            s["q"], s["new_k"], s["new_v"] = normal(n, h, d, type=i), normal(n, kv, d, type=i), normal(n, kv, d, type=i)
        s["qn"], s["kn"] = (0.1 * normal(d), 0.1 * normal(d)) if case["norm"] else (None, None)
        pos = b["pos"]
        img = torch.arange(n) // 256 % 2 == 1  # every other 256 rows are an image of 16 x 16
        at = torch.arange(n) % 256
        base = pos - at
        p3 = torch.stack([torch.where(img, base, pos), torch.where(img, base + at // 16, pos),
                          torch.where(img, base + at % 16, pos), torch.zeros_like(pos)], 1)
        s["rpos"] = p3.clamp(min=0).to(torch.int32).cuda()
        m = case["ctx"] + 16
        f = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
        a = torch.arange(m, dtype=torch.float64, device="cuda")[:, None] * 1e7 ** (-2 * f / case["rot"])
        s["rope"] = torch.stack([a.cos(), a.sin()], -1).float().contiguous()
        s["q_out"] = torch.empty(n, h, d, dtype=t, device="cuda")
    elif case["op"] == "evict":
        s["weight"] = torch.rand(pages, kv, page, generator=g, device="cuda") ** 4
        s["weight"] = (s["weight"] * 64).round() / 64 + (s["weight"] > 0.3) * s["weight"]  # many ties among the small
        s["into"] = order[at:at + budget_pages * case["seqs"]].view(case["seqs"], budget_pages).contiguous()
        s["new_lens"] = torch.empty_like(s["lens"])
        s["kept"] = torch.empty(case["seqs"], kv, case["budget"], dtype=torch.int32, device="cuda")
    else:
        s["q"] = normal(n, h, d, type=t) * 1.5
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if case["slopes"] else None
        s["first"] = b["first"].to(torch.int32).cuda() if case["docs"] or case["empty"] else None
        s["last"] = b["last"].to(torch.int32).cuda() if case["block"] else None
        s["lo"], s["hi"] = b["lo"].cuda(), b["hi"].cuda()
        if case["op"] == "attend":
            s["gate"] = normal(n, h, d, type=t) if case["gate"] else None
            s["out"] = torch.empty(n, h, d, dtype=t, device="cuda")
            s["lse"] = torch.empty(n, h, device="cuda")
        else:
            s["weight"] = torch.rand(pages, kv, page, generator=g, device="cuda")
            s["lse"] = _logsum(s)
    if own:
        paged = _package()
        s["cache"] = paged.PagedCache(s["k"], s["v"], s.get("weight"))
        s["batch"] = paged.PagedBatch(s["table"], s["start"], s["lens"], n, s["max_len"])
        if case["op"] == "attend":
            size = s["cache"].attend_workspace(s["batch"], h)
            s["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        if case["op"] == "append":
            s["axes"] = {"one": paged.ONE, "sections": paged.SECTIONS, "interleaved": paged.INTERLEAVED}[case["axes"]]
            s["pairs"] = {"halves": paged.HALVES, "adjacent": paged.ADJACENT}[case["pairs"]]
    return s


def _sections(case):
    """Pairs on the time, height and width axis: about a third each, as (11, 11, 10) of 32."""
    r = case["rot"] // 2
    return (-(-r // 3), -(-(r - 1) // 3), r // 3)


# ---- the plain forms ---------------------------------------------------------------------


def _gather(s, pool):
    """[seqs, kv, length, d] in 32 bits of a pool [page, kv, slot, d]; zero past each length."""
    x = pool[s["table"].long()]  # [seqs, pages, kv, slot, d]
    x = x.transpose(1, 2).reshape(x.shape[0], x.shape[2], -1, x.shape[4])[:, :, :s["max_len"]]
    inside = torch.arange(x.shape[2], device=x.device) < s["lens"][:, None]
    return torch.where(inside[:, None, :, None], x, 0).float()


def _padded(s, rows, fill=0):
    """[seqs, most rows, ...] of a tensor by rows."""
    at = s["start"][:-1, None].long() + torch.arange(s["max_rows"], device=rows.device)
    ok = at < s["start"][1:, None]
    x = rows[torch.where(ok, at, 0)]
    return torch.where(ok.view(*ok.shape, *[1] * (x.dim() - 2)), x, fill)


def _scores(s):
    """[seqs, kv, group, row, key] scores in 32 bits, -inf where the row may not see the key."""
    c = s["case"]
    h, kv, d = c["heads"], c["kv"], c["d"]
    q = _padded(s, s["q"]).float()  # [seqs, row, h, d]
    b, m = q.shape[:2]
    q = q.view(b, m, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, h // kv * m, d)
    x = (q @ _gather(s, s["k"]).transpose(2, 3)).view(b, kv, h // kv, m, -1) / math.sqrt(d)
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    key = torch.arange(x.shape[-1], device=x.device)
    if c["slopes"]:
        gap = (_padded(s, s["pos"])[:, :, None] - key).abs().float()
        x = x - s["slopes"].view(1, kv, -1, 1, 1) * gap[:, None, None]
    seen = (key >= _padded(s, s["lo"], FAR)[:, :, None]) & (key < _padded(s, s["hi"])[:, :, None])
    return x.masked_fill(~seen[:, None, None], -math.inf)


def _by_rows(s, x):
    """[row, head, ...] of [seqs, kv, group, row, ...]."""
    i = torch.arange(s["n"], device=x.device) - s["start"].long()[s["seq"]]
    x = x.permute(0, 3, 1, 2, *range(4, x.dim()))[s["seq"], i]
    return x.reshape(x.shape[0], -1, *x.shape[3:])


def _logsum(s):
    x = _scores(s)
    m = x.amax(-1, keepdim=True)
    l = torch.exp(x - m.masked_fill(m == -math.inf, 0)).sum(-1)
    return _by_rows(s, m.squeeze(-1) + l.log()).contiguous()


def _run_attend(s):
    c = s["case"]
    x = _scores(s)
    b, kv, g, m, n = x.shape
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - top.masked_fill(top == -math.inf, 0))
    l = x.sum(-1, keepdim=True)
    o = (x.view(b, kv, g * m, n) @ _gather(s, s["v"])).view(b, kv, g, m, -1) / l.masked_fill(l == 0, 1)
    o = _by_rows(s, o)
    if c["gate"]:
        o = o * torch.sigmoid(s["gate"].float())
    return {"out": o.to(TYPES[c["type"]]), "lse": _by_rows(s, (top + l.log()).squeeze(-1))}


def _run_weigh(s):
    c = s["case"]
    x = _scores(s)
    lse = _padded(s, s["lse"])  # [seqs, row, h]
    lse = lse.permute(0, 2, 1).reshape(x.shape[0], x.shape[1], x.shape[2], -1, 1)
    add = torch.where(x > -math.inf, torch.exp(x - lse), 0).sum((2, 3))  # [seqs, kv, key]
    key = torch.arange(x.shape[-1], device=x.device)
    rows = s["start"][1:] - s["start"][:-1]
    where = s["table"].long()[:, key // c["page"]], key % c["page"]  # page and slot of each key
    seq, at = torch.nonzero(key < s["lens"][:, None], as_tuple=True)
    page, slot = where[0][seq, at], where[1][at]
    before = s["weight"][page, :, slot] * c["decay"] if c["decay"] else 0
    old = (at < (s["lens"] - rows)[seq])[:, None]
    s["weight"][page, :, slot] = torch.where(old, before, 0) + add[seq, :, at]
    return {"weight": s["weight"]}


def _run_evict(s):
    c = s["case"]
    key = torch.arange(s["max_len"], device="cuda")
    page = s["table"].long()[:, key // c["page"]]
    w = s["weight"][page, :, key % c["page"]].permute(0, 2, 1)  # [seqs, kv, key]
    lens = s["lens"].long()[:, None, None]
    w = torch.where(w.isnan(), -math.inf, w)
    w = torch.where((key < c["sink"]) | (key >= lens - c["recent"]), math.inf, w)
    w = torch.where(key < lens, w, -math.inf)
    best = torch.sort(w, dim=-1, descending=True, stable=True).indices[:, :, :c["budget"]]
    n = lens.clamp(max=c["budget"])
    i = torch.arange(best.shape[2], device="cuda")
    kept = torch.where(i < n, best, FAR).sort(-1).values
    s["kept"].fill_(-1)
    s["kept"][:, :, :kept.shape[2]] = torch.where(i < n, kept, -1).to(torch.int32)
    s["new_lens"].copy_(n[:, 0, 0])
    seq, head, at = torch.nonzero(s["kept"] >= 0, as_tuple=True)
    src = s["kept"].long()[seq, head, at]
    page, slot = s["table"].long()[seq, src // c["page"]], src % c["page"]
    to, new = s["into"].long()[seq, at // c["page"]], at % c["page"]
    for x in (s["k"], s["v"], s["weight"]):
        x[to, head, new] = x[page, head, slot]
    return {"kept": s["kept"], "lens": s["new_lens"], "k": s["k"], "v": s["v"], "weight": s["weight"]}


def _turned(s, x, norm):
    c = s["case"]
    x = x.float()
    if norm is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1 + norm)
    r = c["rot"] // 2
    f = torch.arange(r, device=x.device)
    a, b, _ = _sections(c)
    axis = torch.zeros_like(f)
    if c["axes"] == "sections":
        axis = (f >= a).long() + (f >= a + b).long()
    elif c["axes"] == "interleaved":
        axis = torch.where((f % 3 == 1) & (f < 3 * b), 1, torch.where((f % 3 == 2) & (f < 3 * _sections(c)[2]), 2, 0))
    turn = s["rope"][s["rpos"].long()[:, axis], f]  # [row, pair, (cos, sin)]
    cos, sin = turn[:, None, :, 0], turn[:, None, :, 1]
    y = x.clone()
    p, q = (slice(0, r), slice(r, 2 * r)) if c["pairs"] == "halves" else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
    y[..., p] = x[..., p] * cos - x[..., q] * sin
    y[..., q] = x[..., q] * cos + x[..., p] * sin
    return y


def _run_append(s):
    c = s["case"]
    s["q_out"].copy_(_turned(s, s["q"], s["qn"]))
    page = s["table"].long()[s["seq"], s["pos"] // c["page"]]
    slot = s["pos"] % c["page"]
    s["k"][page, :, slot] = _turned(s, s["new_k"], s["kn"]).to(s["k"].dtype)
    s["v"][page, :, slot] = s["new_v"].to(s["v"].dtype)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def run(s):
    c = s["case"]
    if not own:
        return {"append": _run_append, "attend": _run_attend, "weigh": _run_weigh, "evict": _run_evict}[c["op"]](s)
    cache, batch = s["cache"], s["batch"]
    if c["op"] == "append":
        cache.append(batch, s["q"], s["new_k"], s["new_v"], s["q_out"], s["rpos"], s["rope"], axes=s["axes"],
                     pairs=s["pairs"], sections=_sections(c), q_norm=s["qn"], k_norm=s["kn"], eps=1e-6)
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if c["op"] == "evict":
        cache.evict(batch, c["budget"], s["kept"], s["into"], s["new_lens"], sink=c["sink"], recent=c["recent"])
        return {"kept": s["kept"], "lens": s["new_lens"], "k": s["k"], "v": s["v"], "weight": s["weight"]}
    masks = dict(scale=1 / math.sqrt(c["d"]), cap=c["cap"], window=c["window"], slopes=s["slopes"], first=s["first"],
                 last=s["last"])
    if c["op"] == "attend":
        cache.attend(batch, s["q"], s["out"], s["work"], lse=s["lse"], gate=s["gate"], **masks)
        return {"out": s["out"], "lse": s["lse"]}
    cache.weigh(batch, s["q"], s["lse"], decay=c["decay"], **masks)
    return {"weight": s["weight"]}


# ---- the definitions in 64 bits, one sequence and KV head at a time --------------------------


def _rows_of(s, i):
    return slice(int(s["start"][i]), int(s["start"][i + 1]))


def _keys_of(s, i, pool, head):
    n = int(s["lens"][i])
    at = torch.arange(n, device="cuda")
    return pool[s["table"][i].long()[at // s["case"]["page"]], head, at % s["case"]["page"]].double()


def _exact_scores(s, i, head, g):
    """[row, key] of query head `head * group + g`, and which of them are seen."""
    c = s["case"]
    r = _rows_of(s, i)
    hq = head * (c["heads"] // c["kv"]) + g
    x = s["q"][r, hq].double() @ _keys_of(s, i, s["k"], head).T * c["d"] ** -0.5
    if c["cap"]:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    key = torch.arange(x.shape[1], device="cuda")
    if c["slopes"]:
        x -= float(s["slopes"][hq]) * (key - s["pos"][r, None]).abs()
    return x, (key >= s["lo"][r, None]) & (key < s["hi"][r, None])


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    rows, lens = lengths(case)
    if c["op"] == "append":
        return _exact_append(s)
    if c["op"] == "evict":
        return _exact_evict(s, lens)
    group = c["heads"] // c["kv"]
    if c["op"] == "attend":
        out = torch.zeros(s["n"], c["heads"], c["d"], dtype=torch.float64, device="cuda")
        lse = torch.full((s["n"], c["heads"]), -math.inf, dtype=torch.float64, device="cuda")
        for i in range(len(rows)):
            for head in range(c["kv"]):
                v = _keys_of(s, i, s["v"], head)
                for g in range(group):
                    x, seen = _exact_scores(s, i, head, g)
                    x = torch.where(seen, x, -math.inf)
                    z = torch.logsumexp(x, 1)
                    p = torch.where(seen, torch.exp(x - z[:, None]), 0)
                    out[_rows_of(s, i), head * group + g] = p @ v
                    lse[_rows_of(s, i), head * group + g] = z
        if c["gate"]:
            out /= 1 + torch.exp(-s["gate"].double())
        return {"out": out, "lse": lse}
    w = s["weight"].double()
    for i in range(len(rows)):
        at = torch.arange(lens[i], device="cuda")
        page, slot = s["table"][i].long()[at // c["page"]], at % c["page"]
        for head in range(c["kv"]):
            new = w[page, head, slot] * c["decay"] * (at < lens[i] - rows[i])
            for g in range(group):
                x, seen = _exact_scores(s, i, head, g)
                z = s["lse"][_rows_of(s, i), head * group + g].double()
                new += torch.where(seen, torch.exp(x - z[:, None]), 0).sum(0)
            w[page, head, slot] = new
    return {"weight": w}


def _exact_append(s):
    c = s["case"]
    r = c["rot"] // 2
    a, b, w = _sections(c)
    axis = [0] * r
    for f in range(r):
        if c["axes"] == "sections":
            axis[f] = 0 if f < a else 1 if f < a + b else 2
        elif c["axes"] == "interleaved":
            axis[f] = 1 if f % 3 == 1 and f < 3 * b else 2 if f % 3 == 2 and f < 3 * w else 0
    table = s["rope"].double()

    def turned(x, norm):
        x = x.double()
        if norm is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["d"] + 1e-6) * (1 + norm.double())
        out = x.clone()
        for f in range(r):
            p, q = (f, f + r) if c["pairs"] == "halves" else (2 * f, 2 * f + 1)
            z = torch.view_as_complex(table[s["rpos"][:, axis[f]].long(), f])[:, None]
            y = torch.complex(x[..., p], x[..., q]) * z
            out[..., p], out[..., q] = y.real, y.imag
        return out

    k, v = s["k"].double(), s["v"].double()
    page = s["table"][s["seq"], s["pos"] // c["page"]].long()
    k[page, :, s["pos"] % c["page"]] = turned(s["new_k"], s["kn"])
    v[page, :, s["pos"] % c["page"]] = s["new_v"].double()
    return {"q": turned(s["q"], s["qn"]), "k": k, "v": v}


def _exact_evict(s, lens):
    c = s["case"]
    k, v, w = s["k"].double(), s["v"].double(), s["weight"].double()
    weights = s["weight"].tolist()
    table, into = s["table"].tolist(), s["into"].tolist()
    for i, n in enumerate(lens):
        for head in range(c["kv"]):
            x = [weights[table[i][t // c["page"]]][head][t % c["page"]] for t in range(n)]
            must = [t for t in range(n) if t < c["sink"] or t >= n - c["recent"]]
            free = [t for t in range(n) if c["sink"] <= t < n - c["recent"]]
            free.sort(key=lambda t: (-x[t], t))
            keep = sorted((must + free)[:c["budget"]])
            src = torch.tensor(keep, device="cuda")
            dst = torch.arange(len(keep), device="cuda")
            p0, p1 = s["table"][i].long()[src // c["page"]], s["into"][i].long()[dst // c["page"]]
            for x in (k, v, w):
                x[p1, head, dst % c["page"]] = x[p0, head, src % c["page"]]
    return {"kept": None, "lens": None, "k": k, "v": v, "weight": w}
