"""Three requests served together from one paged cache: their prompts in chunks (one with an
image, whose tokens see one another), their least looked-at slots dropped once they are over
a budget, and then a token each per step, all sequences in one batch.

The model is one gated attention layer of the engine's shape (per head [q | gate], then k and
v; RMSNorm on q and k; M-RoPE on a part of each head) with Q8_0 projections from the seeded
generator, run by snl_mat. Run it on a B200:

    python sense-nova-server_b200/examples/paged_serving.py
"""
from __future__ import annotations

import ctypes as C
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
from sensenova_b200 import ffi, paged  # noqa: E402
from sensenova_b200.config import ModelConfig, small  # noqa: E402


class Projection:
    """A Q8_0 matrix of the seeded generator, applied by snl_mat."""

    def __init__(self, name: str, n: int, k: int, seed: int):
        self.lib, self.n, self.k = ffi.load(), n, k
        self.q = torch.empty(n * k, dtype=torch.uint8, device="cuda")
        self.s = torch.empty(n * k // 32, device="cuda")
        ffi.check(self.lib.snl_synth_quant(seed, name.encode(), ffi.SNL_Q8_0, n, k, self.q.data_ptr(), self.s.data_ptr(), None))

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        y = torch.empty(x.shape[0], self.n, device="cuda")
        step, p = ffi.StepU(x.shape[0], 0, 1, 0), ffi.MatP(self.n, self.k, 0, self.k, 0, self.n, 0, 0)
        ffi.check(self.lib.snl_mat(ffi.SNL_Q8_0, C.byref(step), C.byref(p), x.data_ptr(), self.q.data_ptr(),
                                   self.s.data_ptr(), y.data_ptr(), None))
        return y


class PagedLayer:
    """A gated attention layer over a pool of pages that its sequences share."""

    def __init__(self, cfg: ModelConfig, pages: int, page_size: int = 16, max_pos: int = 4096, seed: int = 1):
        self.cfg, self.page_size = cfg, page_size
        self.proj = Projection("l3.attn", cfg.attn_proj_rows, cfg.hidden, seed)
        self.out = Projection("l3.o", cfg.hidden, cfg.q_dim, seed)
        shape = (pages, cfg.n_kv_heads, page_size, cfg.head_dim)
        self.k, self.v = (torch.empty(shape, dtype=torch.float16, device="cuda") for _ in range(2))
        self.weight = torch.zeros(shape[:3], device="cuda")
        self.cache = paged.PagedCache(self.k, self.v, self.weight)
        self.free = list(range(pages))
        self.tables: list[list[int]] = []
        self.lens: list[int] = []  # slots held: fewer than tokens seen once some were dropped
        self.seen: list[int] = []
        self.rope = torch.empty(max_pos, cfg.rot_dim // 2, 2, device="cuda")
        paged.rope_table(self.rope, cfg.rope_theta)
        self.q_norm, self.k_norm = (torch.zeros(cfg.head_dim, device="cuda") for _ in range(2))

    def add(self) -> int:
        self.tables.append([])
        self.lens.append(0)
        self.seen.append(0)
        return len(self.lens) - 1

    def _table(self, seqs: list[int]) -> torch.Tensor:
        width = max(1, *(len(self.tables[s]) for s in seqs))
        return torch.tensor([self.tables[s] + [0] * (width - len(self.tables[s])) for s in seqs], dtype=torch.int32, device="cuda")

    def _batch(self, seqs: list[int], rows: list[int]) -> paged.PagedBatch:
        start = torch.tensor([0, *rows], dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
        lens = torch.tensor([self.lens[s] for s in seqs], dtype=torch.int32, device="cuda")
        return paged.PagedBatch(self._table(seqs), start, lens, sum(rows), max(self.lens[s] for s in seqs))

    def step(self, seqs: list[int], x: list[torch.Tensor], pos: list[torch.Tensor] | None = None,
             last: list[int | None] | None = None, weigh: bool = False) -> torch.Tensor:
        """The next rows of some sequences: x[i] [rows, hidden] f32. pos[i]: their positions
        [rows, 3] (time, height, width; the token's number unless given); last[i]: the end of a
        block (a prefix, an image) that its rows see whole."""
        cfg, rows = self.cfg, [len(r) for r in x]
        at = []
        for i, s in enumerate(seqs):
            self.lens[s] += rows[i]
            while len(self.tables[s]) * self.page_size < self.lens[s]:
                self.tables[s].append(self.free.pop())
            text = torch.arange(self.seen[s], self.seen[s] + rows[i])[:, None].repeat(1, 3)
            at.append(torch.nn.functional.pad(text if pos is None or pos[i] is None else pos[i], (0, 1)))
            self.seen[s] += rows[i]
        n, q_dim, kv_dim, d = sum(rows), cfg.q_dim, cfg.kv_dim, cfg.head_dim
        h = torch.cat(x)
        proj = self.proj(h * torch.rsqrt(h.square().mean(-1, keepdim=True) + cfg.eps))
        heads = proj[:, :2 * q_dim].view(n, cfg.n_heads, 2, d)  # [q | gate]
        k, v = (proj[:, o:o + kv_dim].view(n, cfg.n_kv_heads, d) for o in (2 * q_dim, 2 * q_dim + kv_dim))
        batch = self._batch(seqs, rows)
        q = torch.empty(n, cfg.n_heads, d, dtype=torch.float16, device="cuda")
        self.cache.append(batch, heads[:, :, 0], k, v, q, torch.cat(at).to(torch.int32).cuda(), self.rope,
                          axes=paged.INTERLEAVED, sections=cfg.mrope_section, q_norm=self.q_norm, k_norm=self.k_norm,
                          eps=cfg.eps)
        out = torch.empty(n, cfg.n_heads, d, device="cuda")
        lse = torch.empty(n, cfg.n_heads, device="cuda")
        work = torch.empty(self.cache.attend_workspace(batch, cfg.n_heads), dtype=torch.uint8, device="cuda")
        ends = None
        if last is not None:
            ends = torch.cat([torch.full((r,), e or 0) for r, e in zip(rows, last)]).to(torch.int32).cuda()
        self.cache.attend(batch, q, out, work, lse=lse, gate=heads[:, :, 1], last=ends)
        if weigh:
            self.cache.weigh(batch, q, lse, last=ends)
        return h + self.out(out.view(n, q_dim))

    def thin(self, seqs: list[int], budget: int, sink: int = 4, recent: int = 32) -> None:
        """Sequences over the budget keep their heaviest slots, in fresh pages; the old ones are
        free again (another sequence may still share them)."""
        batch = self._batch(seqs, [0] * len(seqs))
        width = -(-min(budget, batch.max_len) // self.page_size)
        fresh = [[self.free.pop() for _ in range(width)] for _ in seqs]
        kept = torch.empty(len(seqs), self.cfg.n_kv_heads, budget, dtype=torch.int32, device="cuda")
        lens = torch.empty(len(seqs), dtype=torch.int32, device="cuda")
        self.cache.evict(batch, budget, kept, torch.tensor(fresh, dtype=torch.int32, device="cuda"), lens, sink=sink, recent=recent)
        for s, pages, n in zip(seqs, fresh, lens.tolist()):
            self.free += self.tables[s]
            need = -(-n // self.page_size)
            self.tables[s], self.lens[s] = pages[:need], n
            self.free += pages[need:]


def serve(budget: int = 192, steps: int = 8, seed: int = 0) -> tuple[torch.Tensor, PagedLayer]:
    cfg = small()
    layer = PagedLayer(cfg, pages=128)
    g = torch.Generator(device="cuda").manual_seed(seed)
    prompts = [torch.randn(n, cfg.hidden, generator=g, device="cuda") for n in (300, 45, 129)]
    seqs = [layer.add() for _ in prompts]
    # The second request's tokens 8 to 43 are an image of 6 x 6: one time, rows and columns.
    image = torch.arange(45)[:, None].repeat(1, 3)
    image[8:44] = torch.stack([torch.full((36,), 8), 8 + torch.arange(36) // 6, 8 + torch.arange(36) % 6], 1)
    chunk = 128
    for at in range(0, max(map(len, prompts)), chunk):
        now = [s for s in seqs if at < len(prompts[s])]
        layer.step(now, [prompts[s][at:at + chunk] for s in now], [image if s == 1 else None for s in now],
                   [44 if s == 1 else None for s in now], weigh=True)
        print(f"prompt chunk at {at}: slots {layer.lens}")
    over = [s for s in seqs if layer.lens[s] > budget]
    if over:
        layer.thin(over, budget)
        print(f"thinned to {budget}: slots {layer.lens}, {len(layer.free)} pages free")
    x = torch.stack([p[-1] for p in prompts])
    for i in range(steps):
        x = layer.step(seqs, list(x[:, None]), weigh=True)
    print(f"{steps} tokens each: slots {layer.lens}")
    return x, layer


if __name__ == "__main__":
    out, layer = serve()
    torch.cuda.synchronize()
    err = ffi.load().snl_device_error(1)
    print("last hidden states:", out.square().mean(-1).sqrt().tolist(), "| device error word", err)
