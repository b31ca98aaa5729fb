"""The paged-cache operators from their definitions in 64 bits, for the tests, and the
random problems that they are compared on.

Bounds on the errors: u is the unit roundoff of the cache's type (2^-11 f16, 2^-8 bf16). A
score is a product over d elements held in 32 bits, off by at most 16 x 2^-24 of
scale * sum |q||k| (d / 16 steps of one rounding each), and 8 x 2^-24 of its own size for the
scale, the cap, the bias and the change to base 2. The weights of the output sum are rounded
to the cache's type (u each), 32-bit sums over the keys add 2e-5 at these lengths."""
import math
import random

import torch

UNIT = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
TINY = {torch.float16: 2.0**-24, torch.bfloat16: 0.0, torch.float32: 0.0}


class Problem:
    """A cache of random pages (NaN where no token is), a batch over it, rows of q."""

    def __init__(self, lens, rows, heads=4, kv=1, d=256, page=16, layout="head", dtype=torch.float16, seed=0,
                 spare=3, width=0, max_len=None, weight=False, peak=1.5, device="cuda"):
        self.lens, self.rows, self.heads, self.kv, self.d, self.page = list(lens), list(rows), heads, kv, d, page
        self.dtype, self.device, self.group = dtype, device, heads // kv
        g = self.gen = torch.Generator(device=device).manual_seed(seed)
        need = [-(-n // page) for n in self.lens]
        pages = sum(need) + spare
        order = list(range(pages))
        random.Random(seed).shuffle(order)
        table = torch.full((len(need), max(need + [1]) + width), -7, dtype=torch.int32)  # unused entries: no page
        self.pages = []
        for i, n in enumerate(need):
            self.pages.append(order[:n])
            table[i, :n] = torch.tensor(order[:n], dtype=torch.int32)
            order = order[n:]
        self.free = order
        self.table = table.to(device)
        shape = (pages, kv, page, d) if layout == "head" else (pages, page, kv, d)

        def pool():
            x = torch.full(shape, math.nan, dtype=dtype, device=device)
            return x if layout == "head" else x.transpose(1, 2)

        self.k, self.v = pool(), pool()
        self.weight = torch.full((pages, kv, page), math.nan, device=device) if weight else None
        for i, n in enumerate(self.lens):
            pg, sl = self.where(i)
            self.k[pg, :, sl] = self.normal(n, kv, d).to(dtype)
            self.v[pg, :, sl] = self.normal(n, kv, d).to(dtype)
            if weight:
                self.weight[pg, :, sl] = torch.rand(n, kv, generator=g, device=device)
        self.n = sum(self.rows)
        self.start = torch.tensor([0] + self.rows).cumsum(0).to(torch.int32).to(device)
        self.len_t = torch.tensor(self.lens, dtype=torch.int32, device=device)
        self.max_len = max(self.lens) if max_len is None else max_len
        self.q = (self.normal(self.n, heads, d) * peak).to(dtype)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device=self.device)

    def where(self, i):
        """Pages and slots of sequence i's keys."""
        at = torch.arange(self.lens[i])
        pg = torch.tensor(self.pages[i], dtype=torch.long)
        return pg[at // self.page].to(self.device), (at % self.page).to(self.device)

    def keys(self, i, pool):
        pg, sl = self.where(i)
        return pool[pg, :, sl].double()  # [len, kv, d]

    def seq_rows(self, i):
        r0 = sum(self.rows[:i])
        return r0, r0 + self.rows[i]

    def slot(self):
        """Slot of every row."""
        return torch.cat([torch.arange(n - r, n) for n, r in zip(self.lens, self.rows)] + [torch.zeros(0)]).long()

    def batch(self, paged):
        return paged.PagedBatch(self.table, self.start, self.len_t, self.n, self.max_len)

    def cache(self, paged):
        return paged.PagedCache(self.k, self.v, self.weight)


def scores(p, i, q, scale, cap=0.0, window=0, slopes=None, first=None, last=None):
    """Of sequence i: scores [heads, rows, keys], which are seen [rows, keys], and a bound on the error."""
    r0, r1 = p.seq_rows(i)
    dev = p.device
    n = p.lens[i]
    t = torch.arange(n - (r1 - r0), n, device=dev)[:, None]
    key = torch.arange(n, device=dev)[None]
    seen = key <= t
    if last is not None:
        seen = seen | (key < last[r0:r1, None].to(dev))
    if window:
        seen = seen & (key > t - window)
    if first is not None:
        seen = seen & (key >= first[r0:r1, None].to(dev))
    x = q[r0:r1].double().transpose(0, 1)  # [heads, rows, d]
    k = p.keys(i, p.k).transpose(0, 1).repeat_interleave(p.group, 0)  # [heads, keys, d]
    s = x @ k.transpose(1, 2) * scale
    size = x.abs() @ k.abs().transpose(1, 2) * abs(scale)
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        bias = slopes.double()[:, None, None] * (t - key).abs()
        s = s - bias
        size = size + bias.abs()
    return s, seen, 16 * 2.0**-24 * size + 8 * 2.0**-24 * (s.abs() + cap)


def attend(p, q, gate=None, scale=None, v=None, out_dtype=None, **masks):
    """out, lse and the bounds on their errors."""
    scale = p.d**-0.5 if scale is None else scale
    out = torch.zeros(p.n, p.heads, p.d, dtype=torch.float64, device=p.device)
    lse = torch.full((p.n, p.heads), -math.inf, dtype=torch.float64, device=p.device)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    u, uo = UNIT[p.dtype], UNIT[out_dtype or p.dtype]
    for i in range(len(p.lens)):
        r0, r1 = p.seq_rows(i)
        if r1 == r0:
            continue
        s, seen, err = scores(p, i, q, scale, **masks)
        s = torch.where(seen, s, -math.inf)
        err = torch.where(seen, err, 0).amax(-1)  # [heads, rows]
        z = torch.logsumexp(s, -1)
        w = torch.where(seen & (s > -math.inf), torch.exp(s - z[..., None]), 0)
        val = p.keys(i, p.v).transpose(0, 1).repeat_interleave(p.group, 0)
        o = w @ val
        size = w @ val.abs()
        g = 1 if gate is None else torch.sigmoid(gate[r0:r1].double()).transpose(0, 1)
        out[r0:r1] = (o * g).transpose(0, 1)
        tol[r0:r1] = (uo * (o * g).abs() + (u + 2 * err[..., None] + 2e-5) * size * g).transpose(0, 1)
        lse[r0:r1] = z.transpose(0, 1)
        ltol[r0:r1] = (err + 1e-6 * (1 + torch.where(z.isfinite(), z.abs(), 0))).transpose(0, 1)
    return out, lse, tol + TINY[out_dtype or p.dtype], ltol


def weigh(p, q, lse, weight, decay=1.0, scale=None, **masks):
    """The new weights and the bounds on their errors."""
    scale = p.d**-0.5 if scale is None else scale
    w, tol = weight.double().clone(), torch.zeros_like(weight, dtype=torch.float64)
    for i in range(len(p.lens)):
        r0, r1 = p.seq_rows(i)
        pg, sl = p.where(i)
        old = torch.where((torch.arange(p.lens[i], device=p.device) < p.lens[i] - (r1 - r0))[:, None], w[pg, :, sl], 0)
        old = old * decay if decay else torch.zeros_like(old)
        new, err = torch.zeros_like(old), torch.zeros_like(old)
        if r1 > r0 and p.lens[i]:
            s, seen, e = scores(p, i, q, scale, **masks)
            z = lse[r0:r1].double().transpose(0, 1)[..., None]
            a = torch.where(seen, torch.exp(s - z), 0)
            b = a * (e + 4 * 2.0**-24 * (1 + z.abs()).nan_to_num(0, 0, 0))
            new = a.view(p.kv, p.group, *a.shape[1:]).sum((1, 2)).transpose(0, 1)
            err = b.view(p.kv, p.group, *a.shape[1:]).sum((1, 2)).transpose(0, 1)
        w[pg, :, sl] = old + new
        tol[pg, :, sl] = err + 1e-5 * new + 2.0**-23 * (old + new)
    return w, tol


def evict(weights, n, budget, sink, recent):
    """The kept slots of one sequence and head, from a list of weights."""
    if n <= budget:
        return list(range(n))
    must = [t for t in range(n) if t < sink or t >= n - recent]
    value = [-math.inf if math.isnan(x) else x for x in weights[:n]]
    free = sorted(range(sink, n - recent), key=lambda t: (-value[t], t))
    return sorted(must + free[:budget - len(must)])


def turned(x, pos, table, axes, pairs, sections, norm=None, eps=1e-6):
    """RMSNorm and rotary positions of x [rows, heads, d] in 64 bits."""
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (1 + norm.double())
    if table is None:
        return x
    r = table.shape[1]
    out = x.clone()
    for f in range(r):
        axis = 0
        if axes == 1:
            axis = 0 if f < sections[0] else 1 if f < sections[0] + sections[1] else 2
        elif axes == 2:
            axis = 1 if f % 3 == 1 and f < 3 * sections[1] else 2 if f % 3 == 2 and f < 3 * sections[2] else 0
        cs = table[pos[:, axis].long(), f].double()
        a, b = (f, f + r) if pairs == 0 else (2 * f, 2 * f + 1)
        c, s = cs[:, None, 0], cs[:, None, 1]
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
    return out
