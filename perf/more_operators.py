"""Operators of a KV cache that is held in 8 bits, as cases that can be prepared, run and timed one by one.

Keys and values of a full page (``page`` tokens of one KV head) are int8 codes with one scale for the keys and one for the values
of that page and head; the tokens of a sequence's last, unfinished page stay as they are, in a ring of ``page`` slots.  A page holds,
beside its codes and scales, the largest code and the largest negated code of every key dim, by which a query can tell how large its
product with any key of the page may get.

A case is a dict of plain values; ``kind`` says which calls it makes:

* ``step``    one new token a row is appended (``run_q8_append``), and it attends (``run_q8_paged_attention``)
* ``attend``  attention of the newest tokens of every row over its cache (``run_q8_paged_attention``)
* ``admit``   a chunk of new tokens is appended (``run_q8_append``), and the dense view of the cache that attention of whole chunks
              reads is made (``run_q8_gather``)
* ``select``  for every new token and KV head the pages that it should look at (``run_q8_select_blocks``)
* ``sparse``  that, and attention over those pages and the unfinished one alone (``run_q8_paged_attention`` with ``blocks``)

Sizes follow the benchmark's configurations: 32 query / 8 KV heads, 16 / 4 and 16 / 2, head_dim 64 to 256, pages of 16 and 32
tokens, contexts up to 32768 tokens; for the selection, which is there for long contexts, up to 131072.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ELEM = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed() -> list[dict]:
    return [
        # one chat user: a decode step, nothing but latency
        dict(name="step_one_chat", kind="step", dtype="bf16", batch=1, tokens=1, q_heads=32, kv_heads=8, dim=128, low=4000,
             high=4000, page=16, gate=False, dist="normal"),
        # a decode step of a continuously batched engine: ragged rows
        dict(name="step_ragged", kind="step", dtype="bf16", batch=64, tokens=1, q_heads=16, kv_heads=4, dim=128, low=512,
             high=16384, page=16, gate=False, dist="outlier"),
        # a small fp32 cache, head_dim 64, three query heads to a KV head
        dict(name="step_fp32_pair", kind="step", dtype="fp32", batch=2, tokens=1, q_heads=12, kv_heads=4, dim=64, low=301,
             high=577, page=16, gate=False, dist="normal"),
        # seven drafts of short conversations, gated heads of 256, the cache's default page size
        dict(name="attend_d256_gated", kind="attend", dtype="fp16", batch=16, tokens=8, q_heads=16, kv_heads=2, dim=256, low=400,
             high=4100, page=32, gate=True, dist="normal"),
        # long contexts, one token a sequence: the cache is read once, and that is all
        dict(name="attend_long", kind="attend", dtype="bf16", batch=16, tokens=1, q_heads=32, kv_heads=8, dim=128, low=32768,
             high=32768, page=16, gate=False, dist="normal"),
        # the same with three drafts a sequence
        dict(name="attend_long_drafts", kind="attend", dtype="bf16", batch=16, tokens=4, q_heads=32, kv_heads=8, dim=128,
             low=32768, high=32768, page=16, gate=False, dist="lognormal"),
        # 2048-token chunks of eight prompts behind what is there, and the dense view for their attention
        dict(name="admit_chunks", kind="admit", dtype="bf16", batch=8, tokens=2048, q_heads=16, kv_heads=4, dim=128, low=8192,
             high=8192, page=16, gate=False, dist="outlier"),
        # one prompt of odd length in fp16, heads of 256
        dict(name="admit_prompt", kind="admit", dtype="fp16", batch=1, tokens=3001, q_heads=16, kv_heads=2, dim=256, low=0,
             high=0, page=32, gate=False, dist="normal"),
        # one very long context: which 128 of its 8191 pages
        dict(name="select_one_long", kind="select", dtype="bf16", batch=1, tokens=1, q_heads=32, kv_heads=8, dim=128, low=131070,
             high=131070, page=16, count=128, dist="outlier"),
        # drafts of a ragged batch, four tokens each
        dict(name="select_ragged", kind="select", dtype="bf16", batch=32, tokens=4, q_heads=16, kv_heads=4, dim=128, low=2000,
             high=32768, page=16, count=96, dist="lognormal"),
        # a decode step over the chosen twelfth of one long context
        dict(name="sparse_one_long", kind="sparse", dtype="bf16", batch=1, tokens=1, q_heads=32, kv_heads=8, dim=128, low=49160,
             high=49160, page=16, count=256, gate=False, dist="outlier"),
        # the same of a batch of long contexts
        dict(name="sparse_batch", kind="sparse", dtype="bf16", batch=32, tokens=1, q_heads=32, kv_heads=8, dim=128, low=20000,
             high=32768, page=16, count=128, gate=False, dist="normal"),
    ]


def _log_int(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["step", "attend", "attend", "admit", "select", "sparse"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8]) if dim < 256 else rng.choice([1, 2, 4])
    page = rng.choice([16, 16, 32, 64, 24, 8])
    case = dict(kind=kind, dtype=dtype, dim=dim, kv_heads=kv_heads, page=page, dist=rng.choice(["normal", "outlier", "lognormal"]))
    if kind == "admit":
        batch = _log_int(rng, 1, 32)
        tokens = _log_int(rng, 1, max(1, 16384 * 4 // (batch * kv_heads)))
        high = _log_int(rng, 1, max(1, 65536 * 4 // (batch * kv_heads))) * rng.randint(0, 1)
        high = high // page * page  # a chunk begins a page, so that the same chunk can be appended again
        return dict(case, batch=batch, tokens=tokens, q_heads=kv_heads, low=high, high=high, gate=False)
    group = rng.choice([1, 2, 4, 4, 8, rng.choice([3, 5, 6, 12, 16])])
    tokens = 1 if kind == "step" else rng.choice([1, 1, 2, 3, 4, 5, 8, _log_int(rng, 6, 48)])
    slow = 4 if dtype == "fp32" or page % 16 != 0 else 1
    most = (1 << 19) * 128 // (dim * kv_heads * max(1, tokens * group // 32) * slow)
    batch = _log_int(rng, 1, 64)
    high = _log_int(rng, 3, min(32768 if kind in ("step", "attend") else 131072, max(64, most // batch)))
    case.update(batch=batch, tokens=tokens, q_heads=kv_heads * group, low=max(1, high // rng.randint(1, 8)), high=high)
    if kind in ("select", "sparse"):
        case["tokens"] = min(case["tokens"], 8)
        case["count"] = _log_int(rng, 2, min(300, max(2, (1 << 28) // (batch * kv_heads * case["tokens"] * page * dim))))
    if kind != "select":
        case["gate"] = rng.random() < 0.3
    return case


# ---------------------------------------------------------------------------------------------------------------
# inputs


def _page_bytes(case: dict) -> int:
    """int8 keys [page, dim] | int8 values [page, dim] | float32 scale of the keys, of the values, 8 bytes | int8 [2, dim], the largest
    code and the largest negated code of every key dim | up to a multiple of 128."""
    return (2 * case["page"] * case["dim"] + 16 + 2 * case["dim"] + 127) // 128 * 128


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen: torch.Generator, shape, dtype: torch.dtype) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _lengths(case: dict) -> list[int]:
    """Tokens that the rows have before the call's own (``step``, ``admit``) or with them: spread evenly over [low, high], in a
    fixed shuffled order."""
    n, low, high = case["batch"], case["low"], case["high"]
    if n == 1:
        return [high]
    lengths = [low + (high - low) * i // (n - 1) for i in range(n)]
    random.Random(n).shuffle(lengths)
    return lengths


def _factors(case: dict, gen: torch.Generator):
    """Scale of every channel of keys and values, [2, heads, 1, dim]; None: all one."""
    heads, dim = case["kv_heads"], case["dim"]
    if case["dist"] == "lognormal":
        return torch.exp(0.5 * torch.randn((2, heads, 1, dim), generator=gen, device="cuda"))
    if case["dist"] == "outlier":
        order = torch.rand((2, heads, 1, dim), generator=gen, device="cuda").argsort(dim=-1)
        return torch.where(order < 4, 8.0, 1.0)
    return None


def prepare(case: dict, seed: int):
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    batch, heads, dim, page, tokens = case["batch"], case["kv_heads"], case["dim"], case["page"], case["tokens"]
    factors = _factors(case, gen)
    lengths = _lengths(case)
    appends = case["kind"] in ("step", "admit")
    final = [n + tokens if appends else n for n in lengths]
    blocks = [n // page for n in final]
    total, most = sum(blocks), max(1, max(blocks))
    pool = torch.zeros((total + 5, heads, _page_bytes(case)), dtype=torch.uint8, device="cuda")
    size = page * dim
    signed = pool.view(torch.int8)
    codes = signed[:, :, :2 * size].unflatten(-1, (2, page, dim))
    scales = pool.view(torch.float32)[:, :, size // 2:size // 2 + 2]
    bounds = signed[:, :, 2 * size + 16:2 * size + 16 + 2 * dim].unflatten(-1, (2, dim))
    step = max(1, (1 << 26) // (heads * size))  # pages that are filled at a time
    for at in range(0, total + 5, step):
        n = min(step, total + 5 - at)
        x = torch.randn((n, 2, heads, page, dim), generator=gen, device="cuda")
        if factors is not None:
            x = x * factors
        top = x.abs().amax(dim=(-2, -1)).clamp_min(1e-30)
        x = (x * (127.0 / top[..., None, None])).round().transpose(1, 2)
        codes[at:at + n] = x.to(torch.int8)
        scales[at:at + n] = (top / 127.0).transpose(1, 2)
        bounds[at:at + n, :, 0] = x[:, :, 0].amax(-2).to(torch.int8)
        bounds[at:at + n, :, 1] = (-x[:, :, 0]).amax(-2).to(torch.int8)
    order = torch.rand(total + 5, generator=gen, device="cuda").argsort().to(torch.int32)
    table = torch.full((batch, most), -1, dtype=torch.int32, device="cuda")
    at = 0
    for row, n in enumerate(blocks):
        table[row, :n] = order[at:at + n]
        at += n
    ring = torch.randn((batch + 2, 2, heads, page, dim), generator=gen, device="cuda")
    if factors is not None:
        ring = ring * factors
    state = dict(case=case, packed_pages=pool, codes=codes, scales=scales, bounds=bounds, page_table=table, window=ring.to(dtype),
                 window_slots=torch.randperm(batch + 2, generator=gen, device="cuda")[:batch], longest=max(final),
                 lengths=torch.tensor(final, dtype=torch.long, device="cuda"))
    if appends:
        # projections leave [batch, tokens, heads, dim]; the cache takes the transposed view
        new = torch.randn((2, batch, tokens, heads, dim), generator=gen, device="cuda")
        if factors is not None:
            new = new * factors.transpose(1, 2)[:, None]
        new = new.to(dtype)
        state.update(key=new[0].transpose(1, 2), value=new[1].transpose(1, 2),
                     past_lengths=torch.tensor(lengths, dtype=torch.long, device="cuda"))
    if case["kind"] != "admit":
        shape = (batch, tokens, case["q_heads"], dim)
        state["query"] = _randn(gen, shape, dtype).transpose(1, 2)
        state["gate"] = _randn(gen, shape, dtype).transpose(1, 2) if case.get("gate") else None
    return state


# ---------------------------------------------------------------------------------------------------------------
# one pass: the framework's calls


def _own_run(state):
    import anna_b200

    case, kind = state["case"], state["case"]["kind"]
    cache = dict(packed_pages=state["packed_pages"], page_table=state["page_table"])
    tail = dict(window=state["window"], window_slots=state["window_slots"])
    if kind in ("step", "admit"):
        anna_b200.run_q8_append(key=state["key"], value=state["value"], past_lengths=state["past_lengths"], **cache, **tail)
    if kind == "admit":
        key, value = anna_b200.run_q8_gather(lengths=state["lengths"], max_len=state["longest"], **cache, **tail)
        return dict(key=key, value=value, window=state["window"], scales=state["scales"])
    blocks = None
    if kind in ("select", "sparse"):
        blocks = anna_b200.run_q8_select_blocks(query=state["query"], lengths=state["lengths"], block_size=case["page"],
                                                count=case["count"], **cache)
        if kind == "select":
            return blocks
    out = anna_b200.run_q8_paged_attention(query=state["query"], lengths=state["lengths"], scaling=case["dim"] ** -0.5,
                                           gate=state["gate"], blocks=blocks, **cache, **tail)
    if kind == "step":
        return dict(out=out, window=state["window"], scales=state["scales"])
    return out if blocks is None else dict(blocks=blocks, out=out)


# ---------------------------------------------------------------------------------------------------------------
# one pass: the operators in plain torch


def _plain_append(state):
    """Tokens of the blocks that the call touches, those of the ring in front of the new ones; full blocks are quantized into
    their pages, what is left goes to the ring."""
    case, past = state["case"], state["past_lengths"]
    batch, page, tokens = case["batch"], case["page"], case["tokens"]
    ring = state["window"][state["window_slots"]]  # [B, 2, heads, page, dim]
    count = (tokens + page - 1) // page + 1
    first = past // page
    at = first[:, None] * page + torch.arange(count * page, device="cuda")  # [B, count * page]: positions
    new = torch.stack((state["key"], state["value"]), dim=1)  # [B, 2, heads, T, dim]
    rows = torch.arange(batch, device="cuda")[:, None]
    index = (at - past[:, None]).clamp(0, tokens - 1)
    fresh = new.permute(0, 3, 1, 2, 4)[rows, index]  # [B, count * page, 2, heads, dim]
    old = ring.permute(0, 3, 1, 2, 4)[rows, at % page]
    x = torch.where((at < past[:, None])[..., None, None, None], old, fresh)
    x = x.unflatten(1, (count, page)).permute(0, 1, 4, 3, 2, 5)  # [B, count, heads, 2, page, dim]
    full = (first[:, None] + torch.arange(1, count + 1, device="cuda")) * page <= (past + tokens)[:, None]
    x = x[full].double()
    block = (first[:, None] + torch.arange(count, device="cuda"))[full]
    ids = state["page_table"][rows.expand_as(full)[full], block].long()
    top = x.abs().amax(dim=(-2, -1))  # [n, heads, 2]
    codes = (x * 127.0 / top.clamp_min(1e-300)[..., None, None]).round()
    state["codes"][ids] = codes.to(torch.int8)
    state["scales"][ids] = (top / 127.0).float()
    state["bounds"][ids] = torch.stack((codes[:, :, 0].amax(-2), (-codes[:, :, 0]).amax(-2)), dim=-2).to(torch.int8)
    stays = (at >= past[:, None]) & (at < (past + tokens)[:, None]) & (at >= ((past + tokens) // page * page)[:, None])
    row, column = stays.nonzero(as_tuple=True)
    state["window"][state["window_slots"][row], :, :, at[row, column] % page] = fresh[row, column]


def _cached(state):
    """The whole cache in 32 bits, [B, 2, heads, length, dim]; past a row's length it is the ring again."""
    page, longest, lengths = state["case"]["page"], state["longest"], state["lengths"]
    pages = state["page_table"].long().clamp_min(0)
    x = state["codes"][pages].float() * state["scales"][pages][..., None, None]  # [B, blocks, heads, 2, page, dim]
    x = x.permute(0, 3, 2, 1, 4, 5).flatten(3, 4)
    at = torch.arange(longest, device="cuda")
    packed = (at < (lengths // page * page)[:, None])[:, None, None, :, None]
    ring = state["window"][state["window_slots"]][:, :, :, at % page].float()
    return torch.where(packed, x[:, :, :, at.clamp_max(x.shape[3] - 1)], ring)


def _weighted(scores, hidden):
    scores = scores.masked_fill(hidden, -math.inf)
    weights = (scores - scores.amax(-1, keepdim=True).clamp_min(-1e30)).exp()
    return weights / weights.sum(-1, keepdim=True).clamp_min(1e-30)


def _last_seen(state):
    """Position of every query, [B, T]."""
    return state["lengths"][:, None] - state["case"]["tokens"] + torch.arange(state["case"]["tokens"], device="cuda")


def _finished(state, out):
    if state["gate"] is not None:
        out = out * torch.sigmoid(state["gate"].float())
    return out.to(DTYPES[state["case"]["dtype"]])


def _plain_attend(state):
    case, cache = state["case"], _cached(state)
    query = state["query"].float().unflatten(1, (case["kv_heads"], -1))  # [B, heads, group, T, dim]
    scores = query @ cache[:, 0, :, None].transpose(-1, -2) * case["dim"] ** -0.5
    hidden = (torch.arange(state["longest"], device="cuda") > _last_seen(state)[..., None])[:, None, None]
    return _finished(state, (_weighted(scores, hidden) @ cache[:, 1, :, None]).flatten(1, 2))


def _plain_select(state):
    """Queries rounded to 15 bits and a sign of their head's largest value, so that the sums are whole numbers; scores in 32 bits."""
    case, page = state["case"], state["case"]["page"]
    query = state["query"].double().unflatten(1, (case["kv_heads"], -1))  # [B, heads, group, T, dim]
    top = query.abs().amax(-1, keepdim=True)
    whole = (query * 32767.0 / top.clamp_min(1e-300)).round()
    parts = torch.cat((whole.clamp_min(0), (-whole).clamp_min(0)), dim=-1)
    pages = state["page_table"].long().clamp_min(0)
    bounds = state["bounds"][pages].flatten(-2).permute(0, 2, 3, 1).double()  # [B, heads, 2 * dim, blocks]
    sums = (parts.flatten(2, 3) @ bounds).unflatten(2, (-1, case["tokens"])).float()
    scale = state["scales"][pages][..., 0].transpose(1, 2)[:, :, None, None]
    scores = (top.float() * scale * sums).amax(2)  # [B, heads, T, blocks]
    last = _last_seen(state)
    there = torch.minimum((last + page) // page, (state["lengths"] // page)[:, None]).clamp_min(0)[:, None, :, None]
    at = torch.arange(pages.shape[1], device="cuda")
    scores = scores.masked_fill((at == 0) | (at == there - 1), math.inf).masked_fill(at >= there, -math.inf)
    chosen = torch.sort(scores, dim=-1, descending=True, stable=True)[1][..., :case["count"]]
    none = 1 << 30
    chosen = torch.where(chosen < there, chosen, none).sort(-1)[0]
    chosen = torch.nn.functional.pad(chosen, (0, case["count"] - chosen.shape[-1]), value=none)
    return torch.where(chosen < none, chosen, -1).int()


def _plain_sparse(state, blocks):
    case, page = state["case"], state["case"]["page"]
    batch, heads, tokens = blocks.shape[:3]
    rows = torch.arange(batch, device="cuda")[:, None, None, None]
    ids = state["page_table"][rows, blocks.long().clamp_min(0)].long()
    head = torch.arange(heads, device="cuda")[:, None, None]
    cache = state["codes"][ids, head].float() * state["scales"][ids, head][..., None, None]  # [B, heads, T, count, 2, page, dim]
    cache = cache.transpose(3, 4).flatten(4, 5)  # [B, heads, T, 2, count * page, dim]
    ring = state["window"][state["window_slots"]].float()[:, :, :, None].expand(-1, -1, -1, tokens, -1, -1)
    cache = torch.cat((cache, ring.permute(0, 2, 3, 1, 4, 5)), dim=4)
    slot = torch.arange(page, device="cuda")
    at = blocks.long()[..., None] * page + slot
    at = torch.where(blocks[..., None] >= 0, at, 1 << 40).flatten(3)
    base = state["lengths"] // page * page
    at = torch.cat((at, (base[:, None] + slot)[:, None, None].expand(-1, heads, tokens, -1)), dim=-1)  # [B, heads, T, keys]
    hidden = (at > _last_seen(state)[:, None, :, None])[:, :, None]
    query = state["query"].float().unflatten(1, (heads, -1))  # [B, heads, group, T, dim]
    scores = (query.transpose(2, 3) @ cache[:, :, :, 0].transpose(-1, -2)).transpose(2, 3) * case["dim"] ** -0.5
    out = _weighted(scores, hidden).transpose(2, 3) @ cache[:, :, :, 1]  # [B, heads, T, group, dim]
    return _finished(state, out.transpose(2, 3).flatten(1, 2))


def _plain_run(state):
    kind = state["case"]["kind"]
    if kind in ("step", "admit"):
        _plain_append(state)
    if kind == "admit":
        cache = _cached(state)
        there = (torch.arange(state["longest"], device="cuda") < state["lengths"][:, None])[:, None, :, None]
        key, value = (torch.where(there, cache[:, i], 0.0).to(DTYPES[state["case"]["dtype"]]) for i in range(2))
        return dict(key=key, value=value, window=state["window"], scales=state["scales"])
    if kind == "step":
        return dict(out=_plain_attend(state), window=state["window"], scales=state["scales"])
    if kind == "attend":
        return _plain_attend(state)
    blocks = _plain_select(state)
    return blocks if kind == "select" else dict(blocks=blocks, out=_plain_sparse(state, blocks))


def run(state):
    if own:
        return _own_run(state)
    return _plain_run(state)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without


def work(case: dict) -> dict:
    kind, dim, elem, heads, page, tokens = (case[k] for k in ("kind", "dim", "dtype", "kv_heads", "page", "tokens"))
    elem = ELEM[elem]
    group = case["q_heads"] // heads
    queries = case["batch"] * tokens * case["q_heads"] * dim * elem
    size, flops = 0, 0
    for n in _lengths(case):
        if kind in ("step", "admit"):
            before, n = n, n + tokens
            done, ring = n // page - before // page, n % page
            # new tokens; those of the ring that a page takes; pages that are written; the ring
            size += heads * tokens * 2 * dim * elem + (heads * (before % page) * 2 * dim * elem if done else 0)
            size += heads * (done * (2 * page * dim + 8 + 2 * dim) + min(ring, tokens) * 2 * dim * elem)
        packed = n // page
        if kind == "admit":
            size += heads * (packed * (2 * page * dim + 8) + n % page * 2 * dim * elem + n * 2 * dim * elem)
            continue
        new = min(n, tokens)
        if kind in ("select", "sparse"):
            size += heads * packed * (2 * dim + 4)
            flops += 2 * dim * heads * group * packed * tokens
        if kind == "select":
            size += heads * tokens * case["count"] * 4
        elif kind == "sparse":
            chosen = min(case["count"], packed)  # by every token; all may have chosen the same
            size += heads * (chosen * (2 * page * dim + 8) + n % page * 2 * dim * elem + tokens * case["count"] * 4)
            flops += 4 * dim * case["q_heads"] * new * (chosen * page + n % page)
        else:
            size += heads * (packed * (2 * page * dim + 8) + n % page * 2 * dim * elem)
            flops += 4 * dim * case["q_heads"] * (new * (n - new) + new * (new + 1) // 2)
    if kind != "admit":
        size += queries * (1 if kind == "select" else 2 + bool(case["gate"]))
    return dict(bytes=size, flops=flops)


# ---------------------------------------------------------------------------------------------------------------
# the operators' definitions in 64 bits


def _exact_page(x: torch.Tensor):
    """Codes and scale of one page's keys or values [heads, page, dim]: the nearest whole numbers (of two the even one) to
    127 x / max |x|; the scale, max |x| / 127, is held in 32 bits."""
    top = x.abs().flatten(1).max(dim=1)[0]
    codes = torch.round(127.0 * x / torch.where(top > 0, top, 1.0)[:, None, None])
    return codes, (top / 127.0).float().double()


def _exact_rows(case: dict, state: dict):
    """Every row's cache after the call's own tokens, [2, heads, length, dim]."""
    page = case["page"]
    for b, n in enumerate(state["lengths"].tolist()):
        slot = int(state["window_slots"][b])
        start = n - case["tokens"] if "key" in state else n
        done = start // page  # pages that are there before the call
        ids = state["page_table"][b, :done].long()
        codes = state["codes"][ids].double() * state["scales"][ids].double()[..., None, None]  # [done, heads, 2, page, dim]
        parts = [codes.permute(2, 1, 0, 3, 4).flatten(2, 3)]
        rest = state["window"][slot, :, :, :start % page].double()
        if "key" in state:
            rest = torch.cat((rest, torch.stack((state["key"][b], state["value"][b])).double()), dim=2)
        at, made = 0, []
        while rest.shape[2] - at >= page:
            pair = [_exact_page(x) for x in rest[:, :, at:at + page]]
            parts.append(torch.stack([c * s[:, None, None] for c, s in pair]))
            made.append(torch.stack([s for _, s in pair], dim=-1))
            at += page
        parts.append(rest[:, :, at:])
        yield b, n, torch.cat(parts, dim=2), made, rest[:, :, at:]


def _exact_chosen(case: dict, state: dict, b: int, n: int):
    """Blocks of one row, [heads, T, count]: numbers as the definition rounds them, ties to the lowest index."""
    import numpy as np

    page, count, heads = case["page"], case["count"], case["kv_heads"]
    ids = state["page_table"][b, :n // page].long()
    bounds, scale = state["bounds"][ids].cpu().numpy().astype(np.int64), state["scales"][ids][..., 0].cpu().numpy()
    query = state["query"][b].double().cpu().numpy()  # [q_heads, T, dim]
    group = query.shape[0] // heads
    out = np.full((heads, case["tokens"], count), -1, dtype=np.int32)
    for t in range(case["tokens"]):
        there = min(n // page, max(0, (n - case["tokens"] + t + page) // page))
        if there == 0:
            continue
        for h in range(heads):
            best = np.full(there, -np.inf, dtype=np.float32)
            for g in range(group):
                q = query[h * group + g, t]
                top = np.abs(q).max()
                whole = np.rint(q * 32767.0 / (top if top > 0 else 1.0)).astype(np.int64)
                sums = bounds[:there, h, 0] @ np.maximum(whole, 0) + bounds[:there, h, 1] @ np.maximum(-whole, 0)
                best = np.maximum(best, np.float32(top) * scale[:there, h] * sums.astype(np.float32))
            best[[0, there - 1]] = np.inf
            chosen = np.sort(np.argsort(-best, kind="stable")[:count])
            out[h, t, :len(chosen)] = chosen
    return torch.from_numpy(out).cuda()


def exact(case: dict, seed: int):
    if case["kind"] in ("select", "sparse") and case["batch"] * case["tokens"] * case["q_heads"] * (case["high"] // case["page"]) * case["dim"] > 5e9:
        return None
    state = prepare(case, seed)
    page, tokens, heads = case["page"], case["tokens"], case["kv_heads"]
    if case["kind"] == "select":
        return torch.stack([_exact_chosen(case, state, b, n) for b, n in enumerate(state["lengths"].tolist())])
    window, scales = state["window"].double(), state["scales"].double()
    dense = torch.zeros((2, case["batch"], heads, state["longest"], case["dim"]), dtype=torch.float64, device="cuda") if case["kind"] == "admit" else None
    out = None if case["kind"] == "admit" else torch.zeros(state["query"].shape, dtype=torch.float64, device="cuda")
    chosen = []
    for b, n, cache, made, rest in _exact_rows(case, state):
        if "key" in state:
            first = (n - tokens) // page
            for i, s in enumerate(made):
                scales[state["page_table"][b, first + i].long()] = s
            kept = rest.shape[2]
            fresh = min(kept, tokens)
            window[state["window_slots"][b], :, :, kept - fresh:kept] = rest[:, :, kept - fresh:]
        if dense is not None:
            dense[:, b, :, :n] = cache
            continue
        query = state["query"][b].double().unflatten(0, (heads, -1))  # [heads, group, T, dim]
        at = torch.arange(n, device="cuda")
        last = n - tokens + torch.arange(tokens, device="cuda")
        seen = (at <= last[:, None]).expand(heads, -1, -1)  # [heads, T, n]
        if case["kind"] == "sparse":
            blocks = _exact_chosen(case, state, b, n)
            chosen.append(blocks)
            allowed = torch.zeros((heads, tokens, n // page + 2), dtype=torch.bool, device="cuda")
            allowed.scatter_(2, torch.where(blocks >= 0, blocks, n // page + 1).long(), True)
            allowed[:, :, n // page] = True
            seen = seen & allowed[:, :, at // page]
        score = (query @ cache[0][:, None].transpose(-1, -2)) * case["dim"] ** -0.5
        score = score.masked_fill(~seen[:, None], -math.inf)
        weight = torch.nan_to_num(torch.softmax(score, dim=-1))  # of a query that sees nothing: zeros
        out[b] = (weight @ cache[1][:, None]).flatten(0, 1)
    if dense is not None:
        return dict(key=dense[0], value=dense[1], window=window, scales=scales)
    if state["gate"] is not None:
        out = out / (1.0 + torch.exp(-state["gate"].double()))
    if case["kind"] == "step":
        return dict(out=out, window=window, scales=scales)
    return out if case["kind"] == "attend" else dict(blocks=torch.stack(chosen), out=out)
