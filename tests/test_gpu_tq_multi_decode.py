"""Attention of several new tokens per sequence over packed pages against a plain implementation in 64 bits.

Tolerances, relative to the visible values that a row averages (``spread``: the weighted sum of |v| over the row's keys):

* fp32: scores are sums of 2 D products in 32 bits, off by at most 2 D * 2^-24 of the sum of their magnitudes, itself at most
  |q| |k| * scaling * sqrt(pi/2) (Cauchy-Schwarz; the signs' part carries the factor); a score that is off by e changes its weight by e.
* 16 bits on CUDA cores: the same, and half a step of the output.
* 16 bits on tensor cores: rotated queries are rounded to 2^-12 of the row's largest value (sqrt(D) times its norm over sqrt(D) at
  most), centroids, residual norms and values to 2^-12 of themselves, probabilities to 2^-12; bf16 caches round zero - 16 * scale,
  2^-12 * 24 scale, and scale <= the group's range / (2^bits - 1).
"""
from __future__ import annotations

import itertools
import math
import threading

import numpy as np
import pytest
import torch

import anna_b200
import oracle
from anna_b200 import _lib, fused_ops
from anna_b200.tq_tables import key_tables

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def hadamard(dim):
    at = np.arange(dim)
    bits = (at[:, None] & at)[..., None] >> np.arange(10) & 1
    return 1.0 - 2.0 * (bits.sum(-1) % 2)


class Case:
    """Random codes in a shuffled pool, a window ring, and the dense keys and values that they stand for, in float64."""

    def __init__(self, *, lengths, tokens, group, kv_heads, dim, bits, page, window, dtype, device, value_group=32, seed=0, holes=False):
        self.__dict__.update(lengths=lengths, tokens=tokens, group=group, kv_heads=kv_heads, dim=dim, bits=bits, page=page,
                             window=window, dtype=DTYPES[dtype], device=device, value_group=value_group)
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        batch, elem = len(lengths), 4 if dtype == "fp32" else 2
        layout = _lib.tq_page_layout(dim, bits, page, fused_ops.dtype_code(self.dtype), value_group)
        self.layout = layout
        quantized = [max(0, n - window) for n in lengths]
        blocks = [(n + page - 1) // page for n in quantized]
        pages = sum(blocks) + 3
        self.packed = torch.randint(0, 256, (pages, kv_heads, layout["chunk_bytes"]), generator=gen, dtype=torch.uint8)
        raw = self.packed.numpy()
        groups = dim // value_group

        def put(offset, values):  # [pages, heads, page, ...] values of a type into the pages' bytes
            data = np.ascontiguousarray(values).view(np.uint8).reshape(pages, kv_heads, -1)
            raw[:, :, offset:offset + data.shape[2]] = data

        norm = rng.uniform(0.5, 2.0, (pages, kv_heads, page)).astype(np.float32) * math.sqrt(dim)
        rnorm = rng.uniform(0.1, 0.4, (pages, kv_heads, page)).astype(np.float32)
        put(layout["off_knorm"], norm)
        put(layout["off_krnorm"], rnorm)
        scale = torch.rand(pages, kv_heads, page, groups, generator=gen).add(0.5).div(2 ** bits).to(self.dtype)
        zero = torch.randn(pages, kv_heads, page, groups, generator=gen).sub(0.5).to(self.dtype)
        put(layout["off_vscale"], scale.view(torch.uint8).numpy())
        put(layout["off_vzero"], zero.view(torch.uint8).numpy())

        def fields(offset, width, count, row_bytes, skip=0):
            rows = raw[:, :, offset:offset + page * row_bytes].reshape(pages, kv_heads, page, row_bytes)[..., skip:]
            bits_of = np.unpackbits(rows, axis=-1, bitorder="little")[..., :count * width].reshape(pages, kv_heads, page, count, width)
            return (bits_of << np.arange(width)).sum(-1)

        if bits == 3:
            index = fields(layout["off_kcodes"], 2, dim, layout["key_bytes"])
            sign = fields(layout["off_kcodes"], 1, dim, layout["key_bytes"], skip=dim // 4)
        else:
            code = fields(layout["off_kcodes"], bits, dim, layout["key_bytes"])
            index, sign = code % 2 ** (bits - 1), code // 2 ** (bits - 1)
        tables = key_tables(head_dim=dim, bits=bits, device="cpu")
        h, s1, s2 = hadamard(dim), tables.signs1.numpy().astype(float), tables.signs2.numpy().astype(float)
        kappa = math.sqrt(math.pi / 2 / dim)
        rotated = tables.centroids.numpy().astype(float)[index] + kappa * rnorm[..., None] * (((2.0 * sign - 1.0) @ h) * s2)
        keys = norm[..., None] / dim * (rotated @ h) * s1
        vcode = fields(layout["off_vdata"], 2 if bits == 2 else 4, dim, layout["value_bytes"])
        wide = lambda x: np.repeat(x.double().numpy(), value_group, axis=-1)  # noqa: E731
        values = vcode * wide(scale) + wide(zero)

        order = rng.permutation(pages)
        table = np.full((batch, max(1, max(blocks)) + 1), -1, np.int32)
        at = 0
        for b, n in enumerate(blocks):
            table[b, :n] = order[at:at + n]
            at += n
        self.hidden = [np.zeros(n, bool) for n in lengths]
        if holes:
            for b, n in enumerate(blocks):
                for j in range(1, n, 3):
                    table[b, j] = pages + 5 if j % 2 else -7
                    self.hidden[b][j * page:min((j + 1) * page, quantized[b])] = True
        self.window_ring = torch.randn(batch + 1, 2, kv_heads, window, dim, generator=gen).to(self.dtype)
        self.slots = torch.from_numpy(rng.permutation(batch + 1)[:batch].copy()).long()
        self.table = torch.from_numpy(table)
        self.dense = []
        for b, n in enumerate(lengths):
            k, v = np.zeros((kv_heads, n, dim)), np.zeros((kv_heads, n, dim))
            for t in range(n):
                if t < quantized[b]:
                    pid = table[b, t // page]
                    if 0 <= pid < pages:
                        k[:, t], v[:, t] = keys[pid, :, t % page], values[pid, :, t % page]
                else:
                    k[:, t], v[:, t] = self.window_ring[self.slots[b], :, :, t % window].double().numpy()
            self.dense.append((k, v))
        self.query = torch.randn(batch, tokens, kv_heads * group, dim, generator=gen).to(self.dtype).transpose(1, 2)
        self.gate = torch.randn(batch, kv_heads * group, tokens, dim, generator=gen).to(self.dtype)
        self.scaling = dim ** -0.5
        self.quantized = quantized

    def run(self, *, gate=False, query=None, lengths=None):
        put = lambda x: x.to(self.device)  # noqa: E731
        return anna_b200.run_tq_paged_multi_decode(
            query=put(self.query) if query is None else query, packed_pages=put(self.packed), page_table=put(self.table),
            window=put(self.window_ring), window_slots=put(self.slots), lengths=put(torch.tensor(self.lengths if lengths is None else lengths)),
            scaling=self.scaling, bits=self.bits, residual_len=self.window, block_size=self.page, value_group_size=self.value_group,
            gate=put(self.gate) if gate else None)

    def expected(self, gate=False):
        """(output, spread) float64 [B, Hq, T, D]; spread: the weighted mean of |v|, times what a relative error of the scores'
        magnitude does to a weight."""
        out, spread, size = (torch.zeros(self.query.shape, dtype=torch.float64) for _ in range(3))
        for b, (k, v) in enumerate(self.dense):
            n = self.lengths[b]
            for h, t in itertools.product(range(self.query.shape[1]), range(self.tokens)):
                kh, end = h // self.group, n - self.tokens + t + 1
                seen = np.arange(n) < end
                seen &= ~self.hidden[b]
                if not seen.any():
                    continue
                q = self.query[b, h, t].double().numpy()
                score = k[kh][seen] @ q * self.scaling
                w = np.exp(score - score.max())
                w /= w.sum()
                out[b, h, t] = torch.from_numpy(w @ v[kh][seen])
                spread[b, h, t] = torch.from_numpy(w @ np.abs(v[kh][seen] - (w @ v[kh][seen])))
                size[b, h, t] = np.linalg.norm(q) * np.linalg.norm(k[kh][seen], axis=-1).max() * abs(self.scaling) * math.sqrt(math.pi / 2)
        weight = 1.0
        if gate:
            weight = torch.sigmoid(self.gate.double())
        return out * weight, spread * weight, size

    def check(self, got, *, gate=False, start=0, rows=None):
        """`got` are the queries from number `start` on; `rows`: a mask of those that count."""
        want, spread, size = (x[:, :, start:] for x in self.expected(gate))
        assert got.shape == want.shape and got.dtype == self.dtype and got.is_contiguous()
        got = got.cpu().double()
        if rows is not None:
            got, want, spread, size = (x[rows.cpu()] for x in (got, want, spread, size))
        assert torch.isfinite(got).all()
        half = torch.finfo(self.dtype).eps / 2
        tensor = self.dtype != torch.float32
        top = max(float(np.abs(v).max(initial=0.0)) for _, v in self.dense)
        # a score off by e: each weight by at most 2 e of itself, so the output by 2 e times the spread
        score = size * (2 * self.dim * 2.0 ** -24)
        value = 2.0 ** -22 * top
        if tensor:
            # Cauchy-Schwarz over the D rounding errors of a rotated query, each at most 2^-12 of the largest of its D values (for
            # a random rotation sqrt(2 ln 2D) times their root mean square): 1 for the centroids' product, 0.4 (the largest
            # residual norm here) times sqrt(pi/2) for the signs'; centroids and residual norms 2^-12 of themselves
            score = score + size * 2.0 ** -12 * (2.0 * math.sqrt(2 * math.log(2 * self.dim)) + 2)
            step = 2.0 ** -12 * (24 * 1.5 / 2 ** self.bits if self.dtype == torch.bfloat16 else 0)
            value = value + (2 * 2.0 ** -12 * top + step)
        limit = 2 * score * spread + value + half * want.abs() * 1.01 + 2e-7
        worst = float(((got - want).abs() / limit).max())
        assert worst <= 1.0, worst
        return worst


SHAPES = [  # kv_heads, group, dim, page, window
    (2, 4, 128, 16, 128), (1, 8, 256, 32, 64), (2, 3, 128, 48, 5), (2, 1, 64, 16, 7), (1, 12, 128, 24, 16), (3, 2, 256, 16, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bits", [2, 3, 4])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("tokens", [1, 2, 5, 17])
def test_against_the_dense_keys_and_values(cuda_device, dtype, bits, shape, tokens):
    kv_heads, group, dim, page, window = shape
    lengths = [window + 3 * page + 7, 1, window, window + 1, 0, 2 * tokens, window + page]  # empty, window alone, a page exactly
    case = Case(lengths=lengths, tokens=tokens, group=group, kv_heads=kv_heads, dim=dim, bits=bits, page=page, window=window,
                dtype=dtype, device=cuda_device, seed=tokens)
    case.check(case.run())
    case.check(case.run(gate=True), gate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,page,bits", [("bf16", 128, 16, 4), ("fp16", 128, 32, 3), ("bf16", 256, 16, 2), ("fp32", 128, 16, 4), ("bf16", 64, 16, 3), ("fp16", 64, 24, 2), ("fp32", 64, 16, 4),
                                                  ("bf16", 64, 16, 4)])
@pytest.mark.parametrize("tokens,group", [(4, 4), (9, 2), (40, 1)])
def test_long_rows_that_several_ctas_share(cuda_device, dtype, dim, page, bits, tokens, group):
    lengths = [3001, 129, 1024, 2047]
    case = Case(lengths=lengths, tokens=tokens, group=group, kv_heads=1, dim=dim, bits=bits, page=page, window=33, dtype=dtype,
                device=cuda_device, seed=5)
    first = case.run()
    case.check(first)
    for _ in range(3):
        assert torch.equal(case.run(), first)  # the merge has an order of its own


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,page", [("bf16", 128, 16), ("fp16", 256, 32), ("fp32", 128, 16)])
@pytest.mark.parametrize("tokens,group", [(3, 4), (6, 4)])
def test_many_rows_of_all_lengths(cuda_device, dtype, dim, page, tokens, group):
    """Shares that hold several streams, end inside one, or hold none; empty rows among them."""
    rng = np.random.default_rng(3)
    lengths = [int(n) for n in rng.integers(0, 400, 70)] + [0, 0, 2500, 1, 16, 0]
    case = Case(lengths=lengths, tokens=tokens, group=group, kv_heads=2, dim=dim, bits=4, page=page, window=20, dtype=dtype,
                device=cuda_device, seed=15)
    first = case.run(gate=True)
    case.check(first, gate=True)
    assert torch.equal(case.run(gate=True), first)


@pytest.mark.gpu
def test_more_rows_than_one_launch_lines_up(cuda_device):
    lengths = [(37 * i) % 23 for i in range(1100)]
    case = Case(lengths=lengths, tokens=2, group=2, kv_heads=1, dim=128, bits=4, page=16, window=4, dtype="bf16", device=cuda_device)
    case.check(case.run(gate=True), gate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,page", [("bf16", 128, 16), ("fp16", 256, 32), ("fp32", 128, 16), ("bf16", 128, 24)])
def test_holes_of_the_block_table_are_keys_that_nobody_sees(cuda_device, dtype, dim, page):
    case = Case(lengths=[900, 500, 20], tokens=3, group=4, kv_heads=2, dim=dim, bits=4, page=page, window=16, dtype=dtype,
                device=cuda_device, holes=True, seed=8)
    case.check(case.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("bits", [2, 3, 4])
@pytest.mark.parametrize("dim,page", [(128, 8), (128, 24), (256, 40), (128, 136), (128, 12), (64, 16), (64, 8), (64, 72)])
@pytest.mark.parametrize("holes", [False, True])
def test_pages_that_end_inside_a_tile(cuda_device, dtype, bits, dim, page, holes):
    case = Case(lengths=[1500, 733, 30, 0, 8 * 33 + 5], tokens=6, group=3, kv_heads=2, dim=dim, bits=bits, page=page, window=9, dtype=dtype,
                device=cuda_device, holes=holes, seed=page)
    got = case.run(gate=True)
    case.check(got, gate=True)
    assert torch.equal(case.run(gate=True), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,page", [("bf16", 128, 16), ("fp32", 128, 16), ("fp16", 256, 32), ("bf16", 128, 24), ("fp16", 256, 8), ("fp16", 64, 16)])
def test_bytes_behind_the_last_token_do_not_count(cuda_device, dtype, dim, page):
    """The last page's free slots, the ring's free slots and the pages of nobody hold NaNs and infinities."""
    case = Case(lengths=[307, 61, 9], tokens=4, group=2, kv_heads=2, dim=dim, bits=4, page=page, window=40, dtype=dtype,
                device=cuda_device, seed=9)
    want = case.run()
    used = set()
    for b, n in enumerate(case.quantized):
        for j in range((n + page - 1) // page):
            used.add((int(case.table[b, j]), min(page, n - j * page)))
    filled = dict(used)
    elem = 4 if dtype == "fp32" else 2
    for pid in range(case.packed.shape[0]):
        for slot in range(filled.get(pid, 0), page):
            for name, width in (("off_knorm", 4), ("off_krnorm", 4), ("off_vscale", dim // 32 * elem), ("off_vzero", dim // 32 * elem)):
                at = case.layout[name] + slot * width
                case.packed[pid, :, at:at + width] = 255  # a NaN in every type
    for b, n in enumerate(case.lengths):
        for p in range(min(n, case.window), case.window):
            case.window_ring[case.slots[b], :, :, p] = math.inf
    assert torch.equal(case.run(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("fp16", 128), ("fp32", 128), ("bf16", 256), ("bf16", 64)])
def test_the_last_queries_alone_see_the_same_keys(cuda_device, dtype, dim):
    tokens, window = 4, 32
    case = Case(lengths=[700, 333, 31], tokens=tokens, group=4, kv_heads=2, dim=dim, bits=4, page=16, window=window, dtype=dtype,
                device=cuda_device, seed=11)
    case.check(case.run())
    for t in range(1, tokens):  # the last queries alone
        case.check(case.run(query=case.query.to(cuda_device)[:, :, t:tokens]), start=t)

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("fp32", 128), ("fp16", 256)])
def test_strides_alignment_and_types_of_query_and_gate(cuda_device, dtype, dim):
    case = Case(lengths=[200, 77], tokens=3, group=2, kv_heads=2, dim=dim, bits=4, page=16, window=16, dtype=dtype, device=cuda_device, seed=2)
    want = case.run()
    q = case.query.to(cuda_device)
    wide = torch.zeros(*q.shape[:3], dim + 8, device=cuda_device, dtype=q.dtype)
    wide[..., :dim] = q
    assert torch.equal(case.run(query=wide[..., :dim]), want)
    flat = torch.zeros(q.numel() + 1, device=cuda_device, dtype=q.dtype)
    odd = flat[1:].view(q.shape)
    odd.copy_(q)
    case.check(case.run(query=odd))
    last = torch.zeros(*q.shape, 2, device=cuda_device, dtype=q.dtype)
    last[..., 0] = q
    assert torch.equal(case.run(query=last[..., 0]), want)
    one = Case(lengths=[99], tokens=2, group=1, kv_heads=1, dim=dim, bits=4, page=16, window=16, dtype=dtype, device=cuda_device, seed=3)
    q1, want1 = one.query.to(cuda_device), one.run()
    assert torch.equal(one.run(query=q1.as_strided(q1.shape, (3, 5, dim, 1))), want1)  # dims of one entry have any stride
    stretched = q[:1, :1].expand(q.shape)
    got = case.run(query=stretched)
    assert torch.equal(got, case.run(query=stretched.contiguous()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("fp16", 256), ("fp32", 64)])
def test_zero_and_negative_scaling_zero_and_huge_queries(cuda_device, dtype, dim):
    case = Case(lengths=[150, 40], tokens=3, group=2, kv_heads=1, dim=dim, bits=4, page=16, window=16, dtype=dtype, device=cuda_device, seed=4)
    for scaling in (0.0, -0.07):
        case.scaling = scaling
        case.check(case.run())
    case.scaling = dim ** -0.5
    case.query[0, 0] = 0
    case.check(case.run())
    case.query[0, 1] *= 0.01
    case.query[1] *= 30  # one key takes nearly everything
    got = case.run().cpu().double()
    want, _, _ = case.expected()
    assert float((got - want)[0].abs().max()) < 2e-2 and torch.isfinite(got).all()


def mask_of(case, newest):
    """The rows that see the newest key of sequence 1 and its second KV head, if `newest`."""
    mask = torch.zeros(case.query.shape[:3], dtype=torch.bool, device=case.device)
    mask[1, case.group:, case.tokens - 1] = newest
    return mask


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("fp16", 256), ("fp32", 128), ("fp16", 64)])
def test_nans_reach_the_rows_that_see_them_and_no_others(cuda_device, dtype, dim):
    case = Case(lengths=[150, 90], tokens=4, group=2, kv_heads=2, dim=dim, bits=4, page=16, window=16, dtype=dtype, device=cuda_device, seed=6)
    case.check(case.run())
    was = case.query[0, 1, 2, 5].clone()
    case.query[0, 1, 2, 5] = math.nan
    got = case.run()
    case.query[0, 1, 2, 5] = was
    bad = torch.isnan(got).any(-1)
    assert bad.nonzero().tolist() == [[0, 1, 2]]
    case.check(got, rows=~bad)
    for what in (0, 1):  # the newest key, then the newest value, of row 1 and its second KV head
        for value in (math.nan, math.inf, -math.inf):
            at = (int(case.slots[1]), what, 1, 89 % 16, 3)
            was = case.window_ring[at].clone()
            case.window_ring[at] = value
            got = case.run()
            case.window_ring[at] = was
            bad = ~torch.isfinite(got).all(-1)
            if what == 1:
                assert bad.nonzero().tolist() == [[1, 2, 3], [1, 3, 3]]
                assert bool((torch.isnan(got[1, 2:, 3, 3]) if math.isnan(value) else got[1, 2:, 3, 3] == value).all())
                assert bool(torch.isfinite(got[1, 2:, 3, 4:]).all())
            assert set(map(tuple, bad.nonzero().tolist())) <= {(1, 2, 3), (1, 3, 3)}  # an infinite key may have no weight
            case.check(got, rows=~bad & ~mask_of(case, what == 0))

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,bits,page", [("bf16", 128, 4, 16), ("fp16", 256, 3, 16), ("fp16", 128, 2, 16), ("fp32", 128, 4, 16),
                                                 ("bf16", 64, 2, 16), ("fp16", 64, 4, 16), ("bf16", 128, 4, 24), ("fp16", 64, 3, 8)])
def test_packed_infinities_behind_a_query(cuda_device, dtype, dim, bits, page):
    """New tokens that have left the window: the scale of one of them is infinite or NaN in one group of dims."""
    window, tokens, length = 2, 9, 70
    case = Case(lengths=[length, 40], tokens=tokens, group=2, kv_heads=2, dim=dim, bits=bits, page=page, window=window, dtype=dtype,
                device=cuda_device, seed=13)
    at = length - 5  # queries 4 .. 8 see it
    elem = 4 if dtype == "fp32" else 2
    for value in (math.inf, math.nan):
        offset = case.layout["off_vzero"] + (at % page * (dim // 32) + 1) * elem
        where = (int(case.table[0, at // page]), 1, slice(offset, offset + elem))
        was = case.packed[where].clone()
        case.packed[where] = torch.tensor([value], dtype=case.dtype).view(torch.uint8)
        got = case.run()
        case.packed[where] = was
        bad = ~torch.isfinite(got)
        assert bad[0, 2:, 4:, 32:64].all() and int(bad.sum()) == 2 * 5 * 32
        assert bool((torch.isnan(got[bad]) if math.isnan(value) else got[bad] == value).all())
        case.check(got, rows=~bad.any(-1))


@pytest.mark.gpu
def test_captured_calls_and_two_graphs_side_by_side(cuda_device):
    cases = [Case(lengths=[2000 + 300 * i, 100], tokens=4, group=4, kv_heads=2, dim=128, bits=4, page=16, window=16, dtype="bf16",
                  device=cuda_device, seed=i) for i in range(2)]
    args = []
    for case in cases:
        put = lambda x: x.to(cuda_device)  # noqa: E731
        args.append(dict(query=put(case.query), packed_pages=put(case.packed), page_table=put(case.table), window=put(case.window_ring),
                         window_slots=put(case.slots), lengths=put(torch.tensor(case.lengths)), scaling=case.scaling, bits=4,
                         residual_len=16, block_size=16, value_group_size=32))
    want = [anna_b200.run_tq_paged_multi_decode(**a) for a in args]
    graphs, outs = [], []
    for a in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(anna_b200.run_tq_paged_multi_decode(**a))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for out, expected in zip(outs, want):
        assert torch.equal(out, expected)


@pytest.mark.gpu
def test_another_stream_and_the_dispatcher(cuda_device):
    case = Case(lengths=[1500], tokens=4, group=4, kv_heads=2, dim=128, bits=4, page=16, window=16, dtype="bf16", device=cuda_device)
    want = case.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = case.run()
    side.synchronize()
    assert torch.equal(got, want)
    put = lambda x: x.to(cuda_device)  # noqa: E731
    got = torch.ops.anna.tq_paged_multi_decode(put(case.query), put(case.packed), put(case.table), put(case.window_ring), put(case.slots),
                                               put(torch.tensor(case.lengths)), case.scaling, 4, 16, 16, 32)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,page", [("bf16", 16), ("fp32", 16), ("fp16", 24)])
def test_threads_that_call_at_once(cuda_device, dtype, page):
    """Two host threads on one stream and two on streams of their own: every call has scratch of its own, and the counters of a stream
    are zero again when the next call on it begins."""
    cases = [Case(lengths=[700 + 200 * i, 130, 0], tokens=1 + 2 * i, group=4, kv_heads=2, dim=128, bits=4, page=page, window=16, dtype=dtype,
                  device=cuda_device, seed=i) for i in range(4)]
    put = lambda x: x.to(cuda_device)  # noqa: E731
    args = [dict(query=put(c.query), packed_pages=put(c.packed), page_table=put(c.table), window=put(c.window_ring), window_slots=put(c.slots),
                 lengths=put(torch.tensor(c.lengths)), scaling=c.scaling, bits=4, residual_len=16, block_size=page, value_group_size=32)
            for c in cases]
    want = [anna_b200.run_tq_paged_multi_decode(**a) for a in args]
    streams = [torch.cuda.current_stream(), torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    wrong = []

    def calls(i):
        with torch.cuda.stream(streams[i]):
            outs = [anna_b200.run_tq_paged_multi_decode(**args[i]) for _ in range(40)]
            streams[i].synchronize()
            wrong.extend(i for out in outs if not torch.equal(out, want[i]))

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(4)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("bf16", 64), ("fp32", 64)])
def test_many_queries_of_a_sequence(cuda_device, dtype, dim):
    case = Case(lengths=[330, 150], tokens=300, group=3, kv_heads=1, dim=dim, bits=4, page=16, window=40, dtype=dtype, device=cuda_device, seed=4)
    case.check(case.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,page", [("bf16", 16), ("bf16", 24), ("fp32", 16)])
def test_lengths_that_the_table_cannot_hold_are_cut(cuda_device, dtype, page):
    """What a table of whole pages and the window hold is all there is: longer lengths read nothing else, negative ones are empty rows."""
    full = 4 * page + 16
    case = Case(lengths=[full, full], tokens=3, group=2, kv_heads=2, dim=128, bits=4, page=page, window=16, dtype=dtype, device=cuda_device, seed=6)
    want = case.run()
    case.check(want)
    case.table = case.table[:, :4].contiguous()  # the fixture's tables have room for more
    got = case.run(lengths=[2 ** 40, full + 1])
    assert torch.equal(got, want)
    got = case.run(lengths=[-5, full])
    assert bool((got[0] == 0).all())
    second = torch.zeros(got.shape[:3], dtype=torch.bool)
    second[1] = True
    case.check(got, rows=second)  # other shares than of two rows, so other roundings


@pytest.mark.gpu
def test_value_groups_and_empty_calls(cuda_device):
    for dim, group in ((128, 8), (128, 16), (128, 64), (128, 2), (256, 4), (256, 256), (64, 64)):
        case = Case(lengths=[90, 3], tokens=2, group=2, kv_heads=1, dim=dim, bits=4, page=16, window=8, dtype="bf16", device=cuda_device,
                    value_group=group)
        case.check(case.run())
    q = torch.zeros(2, 4, 0, 128, device=cuda_device, dtype=torch.bfloat16)
    layout = _lib.tq_page_layout(128, 4, 16, 2, 32)
    got = anna_b200.run_tq_paged_multi_decode(
        query=q, packed_pages=torch.zeros(1, 2, layout["chunk_bytes"], dtype=torch.uint8, device=cuda_device),
        page_table=torch.zeros(2, 0, dtype=torch.int32, device=cuda_device),
        window=torch.zeros(2, 2, 2, 8, 128, device=cuda_device, dtype=torch.bfloat16),
        window_slots=torch.arange(2, device=cuda_device), lengths=torch.zeros(2, dtype=torch.long, device=cuda_device), scaling=1.0, bits=4,
        residual_len=8, block_size=16, value_group_size=32)
    assert got.shape == q.shape


def _host_arguments():
    layout = _lib.tq_page_layout(128, 4, 16, 2, 32)
    return dict(query=torch.zeros(2, 4, 3, 128, dtype=torch.bfloat16), packed_pages=torch.zeros(4, 2, layout["chunk_bytes"], dtype=torch.uint8),
                page_table=torch.zeros(2, 2, dtype=torch.int32), window=torch.zeros(2, 2, 2, 8, 128, dtype=torch.bfloat16),
                window_slots=torch.arange(2), lengths=torch.zeros(2, dtype=torch.long), scaling=1.0, bits=4, residual_len=8, block_size=16,
                value_group_size=32)


def test_calls_that_cannot_be_are_refused():
    good = _host_arguments()
    layout = _lib.tq_page_layout(128, 4, 16, 2, 32)
    for change, match in ((dict(query=good["query"][0]), "query"), (dict(bits=5), "bits"), (dict(packed_pages=good["packed_pages"][..., 1:]), "packed_pages"),
                          (dict(block_size=32), "chunks"), (dict(window=good["window"][:, :, :, :4]), "window"),
                          (dict(page_table=good["page_table"].long()), "page_table"), (dict(lengths=good["lengths"].int()), "lengths"),
                          (dict(window_slots=good["window_slots"][:1]), "window_slots"), (dict(query=good["query"][:, :3]), "multiple"),
                          (dict(gate=good["query"][:, :, :1]), "gate"), (dict(gate=good["query"].float()), "gate"),
                          (dict(packed_pages=torch.zeros(0, 2, layout["chunk_bytes"], dtype=torch.uint8)), "pages"), ({}, "CUDA")):
        with pytest.raises(RuntimeError, match=match):
            anna_b200.run_tq_paged_multi_decode(**{**good, **change})


def test_entry_points_refuse_what_they_cannot_run():
    library, ok = _lib.lib(), 0x10000

    def call(q=ok, pages=ok, table=ok, window=ok, out=ok, scratch=ok, floats=1 << 24, counters=ok, batch=1, heads=4, kv=2, tokens=3,
             dim=128, page=16, window_len=16, bits=4, group=32, num_pages=4, blocks=300, dtype=2):
        return library.anna_tq_paged_multi_decode(q, 1536, 384, 128, pages, table, blocks, window, ok, ok, ok, ok, ok, None, 0, 0, 0, out,
                                                  1536, 384, 128, scratch, floats, counters, batch, heads, kv, tokens, dim, page,
                                                  window_len, bits, group, num_pages, blocks, 0.1, dtype, None)

    for bad, status in ((dict(q=None), 1), (dict(window=None), 1), (dict(out=None), 1), (dict(counters=None), 1), (dict(pages=None), 1),
                        (dict(num_pages=0), 1), (dict(batch=0), 1), (dict(heads=3), 1), (dict(tokens=0), 1), (dict(dtype=7), 1),
                        (dict(bits=5), 2), (dict(group=0), 2), (dict(group=7), 2), (dict(dim=96), 2), (dict(floats=1), 4), (dict(scratch=None), 1),
                        (dict(pages=ok + 8), 1), (dict(window=ok + 8), 1), (dict(scratch=ok + 8), 1),
                        (dict(blocks=1 << 40), 1), (dict(blocks=-1), 1), (dict(page=0), 1), (dict(window_len=0), 1), (dict(tokens=1 << 20), 1),
                        (dict(tokens=60000, blocks=1 << 22), 1)):
        assert call(**bad) == status, bad
        assert "multi_decode" in _lib.last_error() or "head_dim" in _lib.last_error()


def test_plan_needs_no_lengths():
    for batch, (heads, kv_heads), tokens, dim in itertools.product((1, 7, 4096), ((8, 8), (32, 8), (12, 1)), (1, 4, 33), (64, 128, 256)):
        floats, counters = _lib.tq_multi_decode_plan(batch, heads, kv_heads, tokens, dim)
        assert floats == 296 * 2 * 16 * (dim + 2) and counters == batch * kv_heads * -(-tokens * (heads // kv_heads) // 8)
    with pytest.raises(RuntimeError, match="multi_decode_plan"):
        _lib.tq_multi_decode_plan(1, 3, 2, 1, 128)


def test_meta_kernel_gives_the_shape():
    assert anna_b200.maybe_load_gated_delta_library()
    meta = lambda x: x.to("meta") if isinstance(x, torch.Tensor) else x  # noqa: E731
    good = {k: meta(v) for k, v in _host_arguments().items()}
    got = torch.ops.anna.tq_paged_multi_decode(good["query"], good["packed_pages"], good["page_table"], good["window"], good["window_slots"],
                                               good["lengths"], 1.0, 4, 8, 16, 32)
    assert got.shape == good["query"].shape
