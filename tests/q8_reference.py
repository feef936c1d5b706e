"""The 8-bit paged cache restated token by token in 64 bits, on the CPU: what its tests compare with."""
from __future__ import annotations

import math

import numpy as np
import torch


def page_bytes(dim: int, page: int) -> int:
    return -(-(2 * page * dim + 16 + 2 * dim) // 128) * 128


def quantized(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (int64) and float32 scale of one page's keys or values [heads, page, dim]."""
    x = x.double()
    top = x.abs().amax(dim=(1, 2))
    fine = torch.isfinite(x).flatten(1).all(dim=1)
    some = fine & (top > 0)
    codes = torch.round(127.0 * x / torch.where(some, top, 1.0)[:, None, None])
    codes = torch.where(some[:, None, None], codes, 0.0)
    scale = (torch.where(fine, top, 0.0).numpy() / 127.0).astype(np.float32)
    scale[~fine.numpy()] = np.nan
    return codes.long(), torch.from_numpy(scale)


class Cache:
    """Rows of tokens as they came, and the tensors of a GPU cache that holds them.  Rows own pages `spare` apart in a shuffled order."""

    def __init__(self, batch: int, heads: int, dim: int, page: int, dtype: torch.dtype, blocks: int, seed: int = 0):
        gen = torch.Generator().manual_seed(seed)
        self.batch, self.heads, self.dim, self.page, self.dtype, self.gen = batch, heads, dim, page, dtype, gen
        pages = batch * blocks + 3
        order = torch.randperm(pages, generator=gen)[:batch * blocks]
        self.table = order.view(batch, blocks).int()
        # what lies in pages and rings beforehand must not matter
        self.pages = torch.randint(0, 256, (pages, heads, page_bytes(dim, page)), generator=gen, dtype=torch.uint8)
        self.window = torch.full((batch + 2, 2, heads, page, dim), math.nan, dtype=dtype)
        self.slots = torch.randperm(batch + 2, generator=gen)[:batch]
        self.tokens = [torch.zeros((2, heads, 0, dim), dtype=dtype) for _ in range(batch)]

    def new_tokens(self, count: int, spread: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
        x = torch.randn((2, self.batch, self.heads, count, self.dim), generator=self.gen) * spread
        x = x.to(self.dtype)
        return x[0], x[1]

    def append(self, key: torch.Tensor, value: torch.Tensor, rows=None) -> None:
        for b in range(self.batch) if rows is None else rows:
            before = self.tokens[b].shape[2]
            self.tokens[b] = torch.cat((self.tokens[b], torch.stack((key[b], value[b]))), dim=2)
            total = self.tokens[b].shape[2]
            for block in range(before // self.page, total // self.page):
                self.write_page(int(self.table[b, block]), self.tokens[b][:, :, block * self.page:(block + 1) * self.page])
            for at in range(max(before, total // self.page * self.page), total):
                self.window[self.slots[b], :, :, at % self.page] = self.tokens[b][:, :, at]

    def write_page(self, page_id: int, x: torch.Tensor) -> None:
        size = self.page * self.dim
        for which in range(2):
            codes, scale = quantized(x[which])
            row = self.pages[page_id]
            row[:, which * size:(which + 1) * size] = codes.to(torch.int8).flatten(1).view(torch.uint8)
            row[:, 2 * size + 4 * which:2 * size + 4 * which + 4] = scale[:, None].contiguous().view(torch.uint8)
            if which == 0:
                bounds = torch.stack((codes.amax(1), (-codes).amax(1)), dim=1).to(torch.int8).flatten(1)
                row[:, 2 * size + 16:2 * size + 16 + 2 * self.dim] = bounds.view(torch.uint8)

    @property
    def lengths(self) -> torch.Tensor:
        return torch.tensor([t.shape[2] for t in self.tokens], dtype=torch.long)

    def dense(self, b: int) -> torch.Tensor:
        """Row b as the cache stands for it, [2, heads, n, dim] in 64 bits."""
        x = self.tokens[b].double().clone()
        for block in range(x.shape[2] // self.page):
            part = slice(block * self.page, (block + 1) * self.page)
            for which in range(2):
                codes, scale = quantized(self.tokens[b][which, :, part])
                x[which, :, part] = codes.double() * scale.double()[:, None, None]
        return x

    def known_bytes(self) -> torch.Tensor:
        """Which bytes of a page have a meaning."""
        size = 2 * self.page * self.dim
        known = torch.zeros(self.pages.shape[2], dtype=torch.bool)
        known[:size + 8] = True
        known[size + 16:size + 16 + 2 * self.dim] = True
        return known

    def on(self, device) -> dict:
        return dict(packed_pages=self.pages.to(device), page_table=self.table.to(device), window=self.window.to(device),
                    window_slots=self.slots.to(device))


def attention(query: torch.Tensor, rows: list[torch.Tensor], scaling: float, gate=None, page: int = 0, blocks=None):
    """Output [B, Hq, T, D] in 64 bits and, for the tolerances, the largest sum |q_d k_d| scaling of a seen key and the largest seen |v|."""
    batch, q_heads, tokens, dim = query.shape
    out = torch.zeros(query.shape, dtype=torch.float64)
    reach, most = 0.0, 0.0
    for b, cache in enumerate(rows):
        heads, n = cache.shape[1], cache.shape[2]
        for h in range(q_heads):
            kvh = h // (q_heads // heads)
            for t in range(tokens):
                last = n - tokens + t
                seen = list(range(max(0, last + 1)))
                if blocks is not None:
                    full = n // page * page
                    chosen = [j for j in blocks[b, kvh, t].tolist() if 0 <= j < n // page]
                    seen = [i for j in chosen for i in range(j * page, (j + 1) * page) if i <= last] + [i for i in range(full, n) if i <= last]
                if not seen:
                    continue
                keys, values = cache[0, kvh, seen], cache[1, kvh, seen]
                q = query[b, h, t].double()
                score = keys @ q * scaling
                out[b, h, t] = torch.softmax(score, dim=0) @ values
                bound = (keys.abs() @ q.abs()) * abs(scaling)
                if torch.isfinite(bound).all():
                    reach = max(reach, float(bound.max()))
                if torch.isfinite(values).all():
                    most = max(most, float(values.abs().max()))
    if gate is not None:
        out = out * torch.sigmoid(gate.double())
    return out, reach, most


def attention_bound(out: torch.Tensor, dtype: torch.dtype, dim: int, reach: float, most: float) -> torch.Tensor:
    """How far an output in `dtype` may be from the exact `out`.

    A score is a sum of `dim` products in 32 bits (queries of 16-bit caches are exact, or off by 2^-25 of the largest): off by
    (dim + 3) 2^-24 of the sum of magnitudes, and what a softmax makes of scores that are off by s is off by 2 s of the largest value.  exp2 and
    the sums behind it: 2^-20.  bf16 caches weigh values with weights in fp16, each off by half a step, 2^-11; others with sums of two.  The
    output is rounded to its type, half a step again."""
    weights = 2.0 * (dim + 3) * 2.0 ** -24 * reach + 2.0 ** -20
    if dtype == torch.bfloat16:
        weights += 2.0 ** -11
    return most * weights + torch.finfo(dtype).eps / 2 * out.abs() + torch.finfo(dtype).smallest_normal


def candidates(n: int, tokens: int, t: int, page: int) -> int:
    seen = n - tokens + t + 1
    return 0 if seen <= 0 else min(n // page, -(-seen // page))


def selected(query: torch.Tensor, cache: Cache, count: int, first: int = 1, recent: int = 1) -> torch.Tensor:
    """run_q8_select_blocks from its definition: whole numbers, and float32 products from the left."""
    batch, q_heads, tokens, dim = query.shape
    heads, page = cache.heads, cache.page
    out = np.full((batch, heads, tokens, count), -1, dtype=np.int32)
    size = 2 * page * dim
    for b in range(batch):
        n = cache.tokens[b].shape[2]
        for t in range(tokens):
            there = candidates(n, tokens, t, page)
            for h in range(heads):
                scored = []
                for j in range(there):
                    page_id = int(cache.table[b, j])
                    if not 0 <= page_id < cache.pages.shape[0]:
                        continue
                    row = cache.pages[page_id, h]
                    bounds = row[size + 16:size + 16 + 2 * dim].view(torch.int8).numpy().astype(np.int64)
                    scale = row[size:size + 4].view(torch.float32).numpy()[0]
                    best = -np.inf
                    for g in range(q_heads // heads):
                        q = query[b, h * (q_heads // heads) + g, t].double().numpy()
                        top = np.abs(q).max()
                        if not np.isfinite(top):
                            best = np.inf
                            continue
                        whole = np.rint(q * 32767.0 / (top if top > 0 else 1.0)).astype(np.int64)
                        total = int(np.maximum(whole, 0) @ bounds[:dim] + np.maximum(-whole, 0) @ bounds[dim:])
                        x = np.float32(top) * scale * np.float32(total)
                        best = np.inf if np.isnan(x) else max(best, float(x))
                    forced = j < first or j >= there - recent
                    scored.append((0 if forced else 1, -best, j))
                chosen = sorted(j for _, _, j in sorted(scored)[:count])
                out[b, h, t, :len(chosen)] = chosen
    return torch.from_numpy(out)
