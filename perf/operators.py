"""Operators around a serving engine's KV cache that work on several tokens or several sequences at once, as cases that can be
prepared, run and timed one by one.

A case is a dict of plain values; ``kind`` says which call it is:

* ``rotary``        rotary positions with several axes (time, height, width) on queries and keys (``run_multi_axis_rotary``)
* ``rotary_write``  the same, with the rotated keys and the values going straight into un-quantized pages
                    (``run_rotary_paged_kv_write``)
* ``copy``          pages of several pools copied in place, for sequences that fork (``run_page_copy``)
* ``gather``        the live pages of several pools moved to the front of smaller ones (``run_page_gather``)
* ``verify``        attention of the newest tokens of every sequence over a packed TurboQuant cache
                    (``run_tq_paged_multi_decode``)

Sizes follow the benchmark's configurations: 32 query / 8 KV heads, 16 / 4 and 16 / 2, head_dim 64 to 256, pages of 16 and 32
tokens, windows of 128, 2- to 4-bit codes, contexts up to 32768 tokens.
"""
from __future__ import annotations

import json
import math
import random
import struct
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ELEM = {"bf16": 2, "fp16": 2, "fp32": 4}
CODEBOOKS = Path(__file__).resolve().parent.parent / "anna_b200" / "data" / "tq_codebooks.json"


def listed() -> list[dict]:
    return [
        # a decode step of a large batch: one token a row, nothing but latency
        dict(name="rotary_decode", kind="rotary", dtype="bf16", batch=64, tokens=1, q_heads=32, kv_heads=8, dim=128,
             rotary_dim=128, sections="16,24,24", interleaved=False, theta=1e6, span=32768),
        # one long video: odd token count, a quarter of head_dim rotated, axes interleaved, positions far out
        dict(name="rotary_video", kind="rotary", dtype="bf16", batch=1, tokens=16383, q_heads=16, kv_heads=4, dim=256,
             rotary_dim=64, sections="11,11,10", interleaved=True, theta=1e7, span=262144),
        # a decode step of a continuously batched engine: positions from the rows' lengths, keys and values to their pages
        dict(name="rotary_write_decode", kind="rotary_write", dtype="bf16", batch=128, tokens=1, q_heads=16, kv_heads=4,
             dim=128, rotary_dim=128, sections="16,24,24", interleaved=False, theta=1e6, span=16384, page=16, given=False),
        # its prefill side: 2048-token chunks with images
        dict(name="rotary_write_chunks", kind="rotary_write", dtype="bf16", batch=8, tokens=2048, q_heads=32, kv_heads=8,
             dim=128, rotary_dim=128, sections="24,20,20", interleaved=True, theta=5e6, span=8192, page=16, given=True),
        # one prompt forks into eight candidates: the partly filled last page of every layer, seven times
        dict(name="copy_candidates", kind="copy", dtype="bf16", layers=16, pools=2, pages=96, kv_heads=8, rows=16, dim=128,
             copies=7, sources=1),
        # a batch forks before drafts are tried on it: whole window rings
        dict(name="copy_windows", kind="copy", dtype="bf16", layers=4, pools=1, pages=80, kv_heads=8, rows=256, dim=128,
             copies=32, sources=32),
        # a small pool after its long sequences have left
        dict(name="gather_small", kind="gather", dtype="fp16", layers=3, pools=2, pages=301, kv_heads=2, rows=32, dim=256,
             live=131),
        # the packed 4-bit pools of two layers after an evening of churn
        dict(name="gather_packed", kind="gather", dtype="uint8", layers=2, pools=1, pages=40000, kv_heads=8, rows=16,
             dim=152, live=25007),
        # one chat user, three drafted tokens and the next one
        dict(name="verify_one_chat", kind="verify", dtype="bf16", bits=4, batch=1, tokens=4, q_heads=32, kv_heads=8, dim=128,
             low=4000, high=4000, page=16, window=128, gate=False, dist="normal"),
        # a batch of short conversations, seven drafts each, gated heads of 256, the cache's default page size
        dict(name="verify_d256_gated", kind="verify", dtype="fp16", bits=4, batch=16, tokens=8, q_heads=16, kv_heads=2,
             dim=256, low=400, high=4100, page=32, window=128, gate=True, dist="normal"),
        # drafts of a ragged batch over 3-bit codes, channels of very different scale
        dict(name="verify_ragged", kind="verify", dtype="bf16", bits=3, batch=32, tokens=5, q_heads=16, kv_heads=4, dim=128,
             low=512, high=16384, page=16, window=128, gate=False, dist="lognormal"),
        # long contexts: a quarter of one GPU's share of the whole-box decode, four tokens a sequence
        dict(name="verify_long", kind="verify", dtype="bf16", bits=4, batch=16, tokens=4, q_heads=32, kv_heads=8, dim=128,
             low=32768, high=32768, page=16, window=128, gate=False, dist="normal"),
    ]


def _log_int(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["rotary", "rotary_write", "copy", "gather", "verify", "verify", "verify"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8]) if dim < 256 else rng.choice([1, 2, 4])
    case = dict(kind=kind, dtype=dtype, kv_heads=kv_heads, dim=dim)
    if kind in ("rotary", "rotary_write"):
        rotary_dim = rng.choice([dim, dim, dim // 2, dim // 4])
        pairs = rotary_dim // 2
        first = rng.randint(0, pairs)
        second = rng.randint(0, pairs - first)
        chosen = rng.choice([[pairs], [first, pairs - first], [first, second, pairs - first - second]])
        batch = _log_int(rng, 1, 128)
        case.update(batch=batch, tokens=_log_int(rng, 1, max(1, 8192 // batch)), q_heads=kv_heads * rng.choice([1, 3, 4, 8]),
                    rotary_dim=rotary_dim, sections=",".join(map(str, chosen)), interleaved=rng.random() < 0.5,
                    theta=rng.choice([1e4, 1e6, 1e7]), span=_log_int(rng, 100, 1 << 20))
        if kind == "rotary_write":
            case.update(page=rng.choice([16, 16, 32, 24]), given=rng.random() < 0.5, span=min(case["span"], 16384))
        return case
    if kind in ("copy", "gather"):
        case.update(layers=_log_int(rng, 1, 24), pools=rng.choice([1, 2]), rows=rng.choice([8, 16, 32, 128]))
        size = case["layers"] * case["pools"] * kv_heads * case["rows"] * dim * ELEM[dtype]
        case["pages"] = _log_int(rng, 4, max(8, min(20000, (1 << 30) // size)))
        if kind == "gather":
            return dict(case, live=rng.randint(1, case["pages"]))
        copies = rng.randint(1, case["pages"] // 2)
        return dict(case, copies=copies, sources=rng.randint(1, min(copies, case["pages"] - copies)))
    tokens = rng.choice([1, 2, 3, 4, 5, 8, _log_int(rng, 6, 64)])
    group = rng.choice([1, 2, 4, 4, 8, rng.choice([3, 6, 12])])
    most = (1 << 19) // (kv_heads * max(1, tokens * group // 32) * (4 if dtype == "fp32" or dim == 64 else 1))
    batch = _log_int(rng, 1, 64)
    high = _log_int(rng, 3, min(32768, max(64, most // batch)))
    return dict(case, bits=rng.choice([2, 3, 4, 4, 4]), batch=batch, tokens=tokens, q_heads=kv_heads * group,
                low=max(1, high // rng.randint(1, 8)), high=high, page=rng.choice([16, 16, 32, 24]),
                window=rng.choice([128, 128, 64, 5]), gate=rng.random() < 0.3, dist=rng.choice(["normal", "outlier", "lognormal"]))


# ---------------------------------------------------------------------------------------------------------------
# inputs


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen: torch.Generator, shape, dtype: torch.dtype) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _lengths(case: dict) -> list[int]:
    """Context lengths of the rows: spread evenly over [low, high], in a fixed shuffled order."""
    n, low, high = case["batch"], case["low"], case["high"]
    if n == 1:
        return [high]
    lengths = [low + (high - low) * i // (n - 1) for i in range(n)]
    random.Random(n).shuffle(lengths)
    return lengths


def _sections(case: dict) -> tuple[int, ...]:
    return tuple(int(s) for s in case["sections"].split(","))


def _pair_axis(case: dict) -> np.ndarray:
    """Axis that every pair of rotated dims takes its position from."""
    sections, pairs = np.array(_sections(case)), np.arange(case["rotary_dim"] // 2)
    if case["interleaved"]:
        axis = pairs % len(sections)
        return np.where(pairs < len(sections) * sections[axis], axis, 0)
    return np.repeat(np.arange(len(sections)), sections)


def _rotary_inputs(case: dict, seed: int) -> dict:
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    batch, tokens, dim, axes = case["batch"], case["tokens"], case["dim"], len(_sections(case))
    # projections leave [batch, tokens, heads, dim]; attention takes the transposed view
    query = _randn(gen, (batch, tokens, case["q_heads"], dim), dtype).transpose(1, 2)
    key = _randn(gen, (batch, tokens, case["kv_heads"], dim), dtype).transpose(1, 2)
    # time goes on from where the row stands; height and width of a token lie within an image in front of that
    start = torch.randint(0, case["span"], (1, batch, 1), generator=gen, device="cuda")
    patch = torch.randint(0, 64, (axes, batch, tokens), generator=gen, device="cuda")
    positions = start + torch.arange(tokens, device="cuda") // 4 + patch
    state = dict(query=query, key=key, positions=positions, axis=torch.from_numpy(_pair_axis(case)).cuda())
    if case["kind"] == "rotary_write":
        page = case["page"]
        past = torch.randint(0, case["span"], (batch,), generator=gen, device="cuda")
        most = (case["span"] + tokens + page - 1) // page
        used = (tokens + page - 1) // page + 1  # blocks that a row can reach in this pass
        pages = batch * used + 3
        order = torch.rand(pages, generator=gen, device="cuda").argsort().to(torch.int32)[:batch * used].view(batch, used)
        table = torch.full((batch, most + 1), -1, dtype=torch.int32, device="cuda")
        block = (past // page)[:, None] + torch.arange(used, device="cuda")
        inside = block <= most
        rows = torch.arange(batch, device="cuda")[:, None].expand_as(block)
        table[rows[inside], block[inside]] = order[inside]
        shape = (pages, case["kv_heads"], page, dim)
        state.update(value=_randn(gen, (batch, tokens, case["kv_heads"], dim), dtype).transpose(1, 2),
                     key_pages=_randn(gen, shape, dtype), value_pages=_randn(gen, shape, dtype), page_table=table,
                     past_lengths=past, rope_deltas=torch.randint(-200, 1, (batch, 1), generator=gen, device="cuda"))
        if not case["given"]:
            state["positions"] = None
    return state


def _page_inputs(case: dict, seed: int) -> dict:
    gen, rng = _generator(seed), random.Random(seed)
    shape = (case["pages"], case["kv_heads"], case["rows"], case["dim"])
    layers = []
    for _ in range(case["layers"]):
        if case["dtype"] == "uint8":
            pools = [torch.randint(0, 256, shape, generator=gen, device="cuda", dtype=torch.uint8) for _ in range(case["pools"])]
        else:
            pools = [_randn(gen, shape, DTYPES[case["dtype"]]) for _ in range(case["pools"])]
        if case["kind"] == "gather":
            layers.append((pools, rng.sample(range(case["pages"]), case["live"])))
            continue
        ids = rng.sample(range(case["pages"]), case["copies"] + case["sources"])
        sources = ids[case["copies"]:]
        layers.append((pools, [sources[i % len(sources)] for i in range(case["copies"])], ids[:case["copies"]]))
    return dict(layers=layers)


def _signs(dim: int, stream: int) -> np.ndarray:
    """Random signs of the key quantizer's rotations: the top bits of a splitmix64 stream."""
    with np.errstate(over="ignore"):
        x = np.uint64(42) ^ (np.uint64(0xD1B54A32D192ED03) * np.uint64(stream + 1)) ^ (np.uint64(dim) * np.uint64(0x9E3779B97F4A7C15))
        z = x + np.arange(1, dim + 1, dtype=np.uint64) * np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    z = z ^ (z >> np.uint64(31))
    return np.where(z >> np.uint64(63), -1.0, 1.0)


def _codebook(dim: int, index_bits: int) -> dict:
    entry = json.loads(CODEBOOKS.read_text())["tables"][f"d{dim}_m{index_bits}"]
    return {k: [struct.unpack(">f", bytes.fromhex(h))[0] for h in entry[k]] for k in ("centroids", "boundaries")}


def _hadamard(dim: int) -> torch.Tensor:
    at = torch.arange(dim)
    both = (at[:, None] & at)[..., None] >> torch.arange(10) & 1
    return (1.0 - 2.0 * (both.sum(-1) % 2)).cuda()


def _layout(case: dict) -> dict:
    """Bytes of one page of one KV head: offsets of its arrays, each [page tokens, ...]."""
    dim, bits, page, elem = case["dim"], case["bits"], case["page"], ELEM[case["dtype"]]
    key, value, groups = dim * bits // 8, dim // (4 if bits == 2 else 2), dim // 32
    sizes = dict(kcodes=key, knorm=4, krnorm=4, vdata=value, vscale=groups * elem, vzero=groups * elem)
    at, out = 0, {}
    for name, size in sizes.items():
        out[name] = (at, size)
        at += (page * size + 15) // 16 * 16
    return dict(out, bytes=(at + 127) // 128 * 128)


def _fields(x: torch.Tensor, width: int) -> torch.Tensor:
    """[..., n] small numbers -> [..., n * width / 8] bytes, the first number in the lowest bits."""
    per = 8 // width
    shifts = torch.arange(per, device=x.device) * width
    return (x.view(*x.shape[:-1], -1, per).int() << shifts.int()).sum(-1).to(torch.uint8)


def _bytes_of(x: torch.Tensor) -> torch.Tensor:
    return x.contiguous().view(torch.uint8)


def _packed_tokens(case: dict, k: torch.Tensor, v: torch.Tensor, tables: dict) -> dict:
    """Codes of keys and values [..., D]: what a page holds of them, as bytes."""
    dim, bits, dtype = case["dim"], case["bits"], DTYPES[case["dtype"]]
    k, v = k.float(), v.float()
    norm = k.norm(dim=-1, keepdim=True)
    w = (k * tables["signs1"]) @ tables["hadamard"] / norm.clamp_min(1e-20)
    idx = torch.bucketize(w, tables["boundaries"])
    error = w - tables["centroids"][idx]
    sign = ((error * tables["signs2"]) @ tables["hadamard"] >= 0).int()
    rnorm = error.norm(dim=-1, keepdim=True) / math.sqrt(dim)
    if bits == 3:
        codes = torch.cat((_fields(idx, 2), _fields(sign, 1)), dim=-1)
    else:
        codes = _fields(idx + (sign << (bits - 1)), bits)
    groups = v.unflatten(-1, (dim // 32, 32))
    zero = groups.amin(-1).to(dtype)
    scale = ((groups.amax(-1) - zero.float()) / (2 ** bits - 1)).clamp_min(1e-6).to(dtype)
    code = ((groups - zero.float()[..., None]) / scale.float()[..., None]).round().clamp(0, 2 ** bits - 1).flatten(-2)
    return dict(kcodes=codes, knorm=_bytes_of(norm), krnorm=_bytes_of(rnorm), vdata=_fields(code, 2 if bits == 2 else 4),
                vscale=_bytes_of(scale), vzero=_bytes_of(zero))


def _verify_inputs(case: dict, seed: int) -> dict:
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    batch, heads, dim, page, window = case["batch"], case["kv_heads"], case["dim"], case["page"], case["window"]
    factors = None
    if case["dist"] == "lognormal":
        factors = torch.exp(0.5 * torch.randn((2, heads, 1, dim), generator=gen, device="cuda"))
    elif case["dist"] == "outlier":
        order = torch.rand((2, heads, 1, dim), generator=gen, device="cuda").argsort(dim=-1)
        factors = torch.where(order < 4, 8.0, 1.0)
    book = _codebook(dim, case["bits"] - 1)
    tables = {k: torch.tensor(v, dtype=torch.float32, device="cuda") for k, v in book.items()}
    tables.update(signs1=torch.from_numpy(_signs(dim, 0)).float().cuda(), signs2=torch.from_numpy(_signs(dim, 1)).float().cuda(),
                  hadamard=_hadamard(dim))
    lengths = _lengths(case)
    blocks = [(max(0, n - window) + page - 1) // page for n in lengths]
    total, most, layout = sum(blocks), max(1, max(blocks)), _layout(case)
    pages = total + 5
    order = torch.rand(pages, generator=gen, device="cuda").argsort()
    packed = torch.zeros((pages, heads, layout["bytes"]), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 18) // (heads * page))  # pages that are packed at a time
    for at in range(0, total, step):
        ids = order[at:min(total, at + step)]
        pair = []
        for i in range(2):
            x = torch.randn((len(ids), heads, page, dim), generator=gen, device="cuda")
            pair.append((x if factors is None else x * factors[i]).to(dtype))
        for name, data in _packed_tokens(case, *pair, tables).items():
            offset, size = layout[name]
            packed[ids, :, offset:offset + page * size] = data.flatten(-2)
    table = torch.full((batch, most), -1, dtype=torch.int32, device="cuda")
    at = 0
    for row, n in enumerate(blocks):
        table[row, :n] = order[at:at + n]
        at += n
    ring = torch.randn((batch + 2, 2, heads, window, dim), generator=gen, device="cuda")
    if factors is not None:
        ring = ring * factors
    shape = (batch, case["q_heads"], case["tokens"], dim)
    return dict(query=_randn(gen, shape, dtype), gate=_randn(gen, shape, dtype) if case["gate"] else None, packed_pages=packed,
                page_table=table, window=ring.to(dtype), window_slots=torch.randperm(batch + 2, generator=gen, device="cuda")[:batch],
                lengths=torch.tensor(lengths, dtype=torch.long, device="cuda"), tables=tables, longest=max(lengths))


def prepare(case: dict, seed: int):
    kind = case["kind"]
    inputs = _rotary_inputs if kind in ("rotary", "rotary_write") else _verify_inputs if kind == "verify" else _page_inputs
    return dict(case=case, **inputs(case, seed))


# ---------------------------------------------------------------------------------------------------------------
# one pass: the framework's calls


def _own_rotary(state):
    import anna_b200

    case = state["case"]
    how = dict(theta=case["theta"], sections=_sections(case), interleaved=case["interleaved"], rotary_dim=case["rotary_dim"])
    if case["kind"] == "rotary":
        return anna_b200.run_multi_axis_rotary(query=state["query"], key=state["key"], positions=state["positions"], **how)
    query = anna_b200.run_rotary_paged_kv_write(
        query=state["query"], key=state["key"], value=state["value"], key_pages=state["key_pages"],
        value_pages=state["value_pages"], page_table=state["page_table"], past_lengths=state["past_lengths"],
        positions=state["positions"], rope_deltas=None if case["given"] else state["rope_deltas"], **how)
    return query, state["key_pages"], state["value_pages"]


def _own_copy(state):
    import anna_b200

    anna_b200.run_page_copy(copies=[(pool, source, target) for pools, source, target in state["layers"] for pool in pools])
    return [pool for pools, _, _ in state["layers"] for pool in pools]


def _own_gather(state):
    import anna_b200

    return anna_b200.run_page_gather(pools=[(pool, ids) for pools, ids in state["layers"] for pool in pools])


def _own_verify(state):
    import anna_b200

    case = state["case"]
    return anna_b200.run_tq_paged_multi_decode(
        query=state["query"], packed_pages=state["packed_pages"], page_table=state["page_table"], window=state["window"],
        window_slots=state["window_slots"], lengths=state["lengths"], scaling=case["dim"] ** -0.5, bits=case["bits"],
        residual_len=case["window"], block_size=case["page"], value_group_size=32, gate=state["gate"])


# ---------------------------------------------------------------------------------------------------------------
# one pass: elementary operations


def _rotated(case: dict, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    half, width = case["rotary_dim"] // 2, case["rotary_dim"]
    x = x.float()
    first, second = x[..., :half], x[..., half:width]
    return torch.cat((first * cos - second * sin, second * cos + first * sin, x[..., width:]), dim=-1).to(DTYPES[case["dtype"]])


def _plain_rotary(state):
    case = state["case"]
    positions = state["positions"]
    if positions is None:
        steps = torch.arange(case["tokens"], device="cuda")
        positions = (state["past_lengths"][:, None] + state["rope_deltas"] + steps)[None].expand(len(_sections(case)), -1, -1)
    pairs = torch.arange(case["rotary_dim"] // 2, device="cuda", dtype=torch.float64)
    angle = positions[state["axis"]].movedim(0, -1).double() * case["theta"] ** (-2.0 * pairs / case["rotary_dim"])
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    query, key = _rotated(case, state["query"], cos, sin), _rotated(case, state["key"], cos, sin)
    if case["kind"] == "rotary":
        return query, key
    at = state["past_lengths"][:, None] + torch.arange(case["tokens"], device="cuda")
    page = torch.gather(state["page_table"], 1, at // case["page"]).long()
    state["key_pages"][page, :, at % case["page"]] = key.transpose(1, 2)
    state["value_pages"][page, :, at % case["page"]] = state["value"].transpose(1, 2)
    return query, state["key_pages"], state["value_pages"]


def _plain_copy(state):
    for pools, source, target in state["layers"]:
        source, target = torch.tensor(source, device="cuda"), torch.tensor(target, device="cuda")
        for pool in pools:
            pool[target] = pool[source]
    return [pool for pools, _, _ in state["layers"] for pool in pools]


def _plain_gather(state):
    layers = [(pools, torch.tensor(ids, device="cuda")) for pools, ids in state["layers"]]
    return [pool[ids] for pools, ids in layers for pool in pools]


def _unpacked(x: torch.Tensor, width: int) -> torch.Tensor:
    shifts = torch.arange(8 // width, device=x.device, dtype=torch.uint8) * width
    return ((x[..., None] >> shifts) & (2 ** width - 1)).flatten(-2)


def _plain_verify(state):
    case, tables, layout = state["case"], state["tables"], _layout(state["case"])
    dim, bits, page, window, heads = case["dim"], case["bits"], case["page"], case["window"], case["kv_heads"]
    lengths, longest = state["lengths"], state["longest"]
    rows = state["packed_pages"][state["page_table"].clamp_min(0).long()]  # [B, blocks, heads, bytes]

    def tokens(name):
        offset, size = layout[name]
        part = rows[..., offset:offset + page * size].unflatten(-1, (page, size))
        return part.transpose(1, 2).flatten(2, 3)  # [B, heads, tokens, bytes]

    codes = tokens("kcodes")
    if bits == 3:
        index, sign = _unpacked(codes[..., :dim // 4], 2), _unpacked(codes[..., dim // 4:], 1)
    else:
        field = _unpacked(codes, bits)
        index, sign = field & (2 ** (bits - 1) - 1), field >> (bits - 1)
    norm, rnorm = (tokens(name).contiguous().view(torch.float32) for name in ("knorm", "krnorm"))
    turned = (2.0 * sign - 1.0) @ tables["hadamard"] * tables["signs2"] * (rnorm * (math.sqrt(math.pi / 2) / math.sqrt(dim)))
    keys = (tables["centroids"][index.long()] + turned) @ tables["hadamard"] * tables["signs1"] * (norm / dim)
    scale, zero = (tokens(name).contiguous().view(DTYPES[case["dtype"]]).float() for name in ("vscale", "vzero"))
    value = _unpacked(tokens("vdata"), 2 if bits == 2 else 4).unflatten(-1, (dim // 32, 32))
    values = (value * scale[..., None] + zero[..., None]).flatten(-2)

    at = torch.arange(longest, device="cuda")
    packed = (at < (lengths - window)[:, None])[:, None, :, None]  # [B, 1, L, 1]
    ring = state["window"][state["window_slots"]][:, :, :, at % window].float()  # [B, 2, heads, L, D]
    prefix = at.clamp_max(keys.shape[2] - 1)
    keys = torch.where(packed, keys[:, :, prefix], ring[:, 0])
    values = torch.where(packed, values[:, :, prefix], ring[:, 1])
    last = lengths[:, None] - case["tokens"] + torch.arange(case["tokens"], device="cuda")  # newest key that a query sees
    hidden = (at > last[..., None])[:, None, None]
    query = state["query"].float().unflatten(1, (heads, -1))  # [B, heads, group, T, D]
    scores = (query @ keys[:, :, None].transpose(-1, -2) * dim ** -0.5).masked_fill(hidden, -math.inf)
    weights = (scores - scores.amax(-1, keepdim=True).clamp_min(-1e30)).exp()
    out = weights @ values[:, :, None] / weights.sum(-1, keepdim=True).clamp_min(1e-30)
    out = out.flatten(1, 2)
    if state["gate"] is not None:
        out = out * torch.sigmoid(state["gate"].float())
    return out.to(DTYPES[case["dtype"]])


def run(state):
    kind = state["case"]["kind"]
    if own:
        if kind in ("rotary", "rotary_write"):
            return _own_rotary(state)
        return _own_copy(state) if kind == "copy" else _own_gather(state) if kind == "gather" else _own_verify(state)
    if kind in ("rotary", "rotary_write"):
        return _plain_rotary(state)
    return _plain_copy(state) if kind == "copy" else _plain_gather(state) if kind == "gather" else _plain_verify(state)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind in ("copy", "gather"):
        size = case["kv_heads"] * case["rows"] * case["dim"] * ELEM.get(case["dtype"], 1) * case["layers"] * case["pools"]
        if kind == "gather":
            return dict(bytes=2 * size * case["live"], flops=0)
        return dict(bytes=size * (case["copies"] + case["sources"]), flops=0)
    dim, elem = case["dim"], ELEM[case["dtype"]]
    rows = case["batch"] * case["tokens"]
    if kind in ("rotary", "rotary_write"):
        vectors = case["q_heads"] + case["kv_heads"] * (2 if kind == "rotary_write" else 1)
        axes = len(_sections(case)) if case.get("given", True) else 0
        return dict(bytes=rows * (vectors * 2 * dim * elem + 8 * axes), flops=rows * vectors * 3 * case["rotary_dim"])
    total, pairs = rows * case["q_heads"] * dim * elem * (2 + case["gate"]), 0
    token = dim * case["bits"] // 8 + 8 + dim // (4 if case["bits"] == 2 else 2) + 2 * (dim // 32) * elem
    for n in _lengths(case):
        packed = max(0, n - case["window"])
        total += case["kv_heads"] * (packed * token + (n - packed) * 2 * dim * elem)
        new = min(n, case["tokens"])
        pairs += new * (n - new) + new * (new + 1) // 2
    return dict(bytes=total, flops=4 * dim * case["q_heads"] * pairs)


# ---------------------------------------------------------------------------------------------------------------
# the operators' definitions in 64 bits


def _exact_turn(case: dict, x: torch.Tensor, positions: np.ndarray) -> torch.Tensor:
    """Each pair (i, i + rotary_dim / 2) as a complex number, times exp(i * position * theta ** (-2 i / rotary_dim))."""
    half = case["rotary_dim"] // 2
    rate = np.power(case["theta"], -np.arange(half) / half)
    angle = np.stack([positions[a] * rate[i] for i, a in enumerate(_pair_axis(case))], axis=-1)
    turn = torch.from_numpy(np.exp(1j * angle)).cuda()[:, None]
    x = x.double()
    z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
    return torch.cat((z.real, z.imag, x[..., 2 * half:]), dim=-1)


def _exact_rotary(case: dict, state: dict):
    positions = state["positions"]
    if positions is None:
        base = (state["past_lengths"] + state["rope_deltas"][:, 0]).cpu().numpy()
        positions = np.broadcast_to(base[:, None] + np.arange(case["tokens"]), (len(_sections(case)), case["batch"], case["tokens"]))
    else:
        positions = positions.cpu().numpy()
    positions = positions.astype(np.float64)
    query, key = _exact_turn(case, state["query"], positions), _exact_turn(case, state["key"], positions)
    if case["kind"] == "rotary":
        return query, key
    pools = state["key_pages"].double(), state["value_pages"].double()
    table, page = state["page_table"].cpu().numpy(), case["page"]
    for b, past in enumerate(state["past_lengths"].tolist()):
        done = 0
        while done < case["tokens"]:
            block, slot = divmod(past + done, page)
            n = min(page - slot, case["tokens"] - done)
            for pool, x in zip(pools, (key, state["value"])):
                pool[table[b, block], :, slot:slot + n] = x[b, :, done:done + n].double()
            done += n
    return (query, *pools)


def _exact_verify(case: dict, state: dict):
    """Row by row, in the basis of the codes: the queries are rotated, the keys stay as they are."""
    dim, bits, page, window, tokens = case["dim"], case["bits"], case["page"], case["window"], case["tokens"]
    heads, dtype, layout = case["kv_heads"], DTYPES[case["dtype"]], _layout(case)
    t = {k: v.double() for k, v in state["tables"].items()}
    out = torch.zeros(state["query"].shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(state["lengths"].tolist()):
        quantized = max(0, length - window)
        rows = state["packed_pages"][state["page_table"][b, :(quantized + page - 1) // page].long()]

        def part(name):
            at, size = layout[name]
            return rows[:, :, at:at + page * size].unflatten(-1, (page, size)).permute(1, 0, 2, 3).flatten(1, 2)[:, :quantized]

        def field(x, width):
            return torch.stack([(x >> (width * i)) & (2 ** width - 1) for i in range(8 // width)], dim=-1).flatten(-2)

        query = state["query"][b].double().unflatten(0, (heads, -1)).flatten(1, 2)  # [heads, group * T, D]
        first = (query * t["signs1"]) @ t["hadamard"]
        second = (first * t["signs2"]) @ t["hadamard"]
        ring = torch.arange(quantized, length, device="cuda") % window
        recent = state["window"][state["window_slots"][b]][:, :, ring].double()
        scores = [query @ recent[0].transpose(-1, -2)]
        values = [recent[1]]
        if quantized:
            codes = part("kcodes")
            if bits == 3:
                index, sign = field(codes[..., :dim // 4], 2), field(codes[..., dim // 4:], 1)
            else:
                code = field(codes, bits)
                index, sign = code % 2 ** (bits - 1), code // 2 ** (bits - 1)
            norm = part("knorm").contiguous().view(torch.float32)[..., 0].double()[:, None]
            rnorm = part("krnorm").contiguous().view(torch.float32)[..., 0].double()[:, None]
            by_index = first @ t["centroids"][index.long()].transpose(-1, -2)
            by_sign = second @ (2.0 * sign.double() - 1.0).transpose(-1, -2)
            scores.insert(0, norm / dim * (by_index + math.sqrt(math.pi / 2 / dim) * rnorm * by_sign))
            scale = part("vscale").contiguous().view(dtype).double()[..., None]
            zero = part("vzero").contiguous().view(dtype).double()[..., None]
            code = field(part("vdata"), 2 if bits == 2 else 4).double().unflatten(-1, (dim // 32, 32))
            values.insert(0, (code * scale + zero).flatten(-2))
        score = torch.cat(scores, dim=-1).unflatten(1, (-1, tokens)) * dim ** -0.5  # [heads, group, T, length]
        last = length - tokens + torch.arange(tokens, device="cuda")
        score = score.masked_fill(torch.arange(length, device="cuda") > last[:, None], -math.inf)
        seen = last >= 0
        weight = torch.softmax(score[:, :, seen], dim=-1)
        out[b].unflatten(0, (heads, -1))[:, :, seen] = weight @ torch.cat(values, dim=1)[:, None]
    if state["gate"] is not None:
        out = out / (1.0 + torch.exp(-state["gate"].double()))
    return out


def exact(case: dict, seed: int):
    if case["kind"] in ("copy", "gather"):  # nothing is computed
        return None
    state = prepare(case, seed)
    return _exact_verify(case, state) if case["kind"] == "verify" else _exact_rotary(case, state)
