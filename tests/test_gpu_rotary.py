"""Rotary positions with several axes against a plain implementation in 64 bits, and the form that writes keys and values to
pages.  Tolerance: cosine and sine are off by at most 2^-24 * pi (their rounded argument) + 2^-23 (the functions) < 3.2e-7, each
output is a product and a fused multiply-add on them (2 * 2^-24 each), so |x1| + |x2| times 6e-7, and the rounding to the output's
type, half a step of the value."""
from __future__ import annotations

import itertools
import math

import numpy as np
import pytest
import torch

import anna_b200
from anna_b200 import _lib, rotary

DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def axes_of(rotary_dim, sections, interleaved):
    pairs = rotary_dim // 2
    if sections is None:
        return [0] * pairs
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    out = [0] * pairs
    for a in range(1, len(sections)):
        for i in range(a, min(pairs, len(sections) * sections[a]), len(sections)):
            out[i] = a
    return out


def turned(x, positions, rotary_dim, *, theta=10000.0, sections=None, interleaved=False, scale=1.0, frequencies=None):
    """(exact result, bound of the error apart from the last rounding), both float64 on the CPU."""
    x, half = x.detach().cpu().double(), rotary_dim // 2
    positions = positions.cpu().double()
    if positions.dim() == 2:
        positions = positions[None].expand(1 if sections is None else len(sections), -1, -1)
    rate = torch.tensor([theta ** (-i / half) for i in range(half)] if frequencies is None else frequencies, dtype=torch.float64)
    angle = positions[axes_of(rotary_dim, sections, interleaved)].movedim(0, -1)[:, None] * rate
    cos, sin = angle.cos() * scale, angle.sin() * scale
    a, b = x[..., :half], x[..., half:rotary_dim]
    out = torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., rotary_dim:]), dim=-1)
    size = 6e-7 * abs(scale) * (a.abs() + b.abs())
    return out, torch.cat((size, size, torch.zeros_like(x[..., rotary_dim:])), dim=-1)


def assert_close(actual, expected, bound):
    half_step = torch.finfo(actual.dtype).eps / 2
    actual = actual.detach().cpu().double()
    limit = bound + half_step * (expected.abs() + bound) + 1e-7 * (actual.dtype == torch.float16)
    assert torch.isfinite(actual).all()
    assert bool(((actual - expected).abs() <= limit + 6e-8).all()), float(((actual - expected).abs() - limit).max())


def states(batch, q_heads, kv_heads, tokens, dim, dtype, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(batch, tokens, q_heads, dim, generator=gen).to(dtype).to(device).transpose(1, 2)
    k = torch.randn(batch, tokens, kv_heads, dim, generator=gen).to(dtype).to(device).transpose(1, 2)
    return q, k


CASES = [  # batch, q_heads, kv_heads, tokens, head_dim, rotary_dim, sections, interleaved
    (2, 4, 2, 7, 128, 128, (16, 24, 24), False),
    (1, 8, 8, 1, 128, 128, (24, 20, 20), True),
    (3, 16, 2, 5, 256, 64, (11, 11, 10), True),
    (1, 1, 1, 33, 64, 64, None, False),
    (2, 3, 1, 9, 64, 32, (5, 11), False),
    (1, 12, 4, 3, 80, 20, (0, 10, 0), False),   # pairs and the rest at odd multiples of 4 bytes
    (1, 2, 1, 4, 6, 2, (1,), True),             # the smallest pair
    (1, 2, 1, 3, 16, 16, None, False),          # one access a head
    (1, 64, 8, 2, 512, 512, (100, 100, 56), False),  # several CTAs a token, more angles than threads
    (2, 5, 5, 3, 34, 34, (17, 0), True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_turned_queries_and_keys(cuda_device, case, dtype):
    batch, q_heads, kv_heads, tokens, dim, width, sections, interleaved = case
    q, k = states(batch, q_heads, kv_heads, tokens, dim, dtype, cuda_device)
    axes = 1 if sections is None else len(sections)
    gen = torch.Generator().manual_seed(1)
    positions = torch.randint(0, 1 << 20, (axes, batch, tokens), generator=gen)
    how = dict(theta=1e6, sections=sections, interleaved=interleaved, rotary_dim=width)
    before = q.clone(), k.clone()
    got = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions.to(cuda_device), **how)
    for x, out in zip((q, k), got):
        assert out.is_contiguous() and out.shape == x.shape and out.dtype == dtype
        assert_close(out, *turned(x, positions, width, theta=1e6, sections=sections, interleaved=interleaved))
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    # in place on views of one fused projection: the same bits
    fused = torch.cat((q.transpose(1, 2), k.transpose(1, 2)), dim=2)
    qi, ki = fused[:, :, :q_heads].transpose(1, 2), fused[:, :, q_heads:].transpose(1, 2)
    again = anna_b200.run_multi_axis_rotary(query=qi, key=ki, positions=positions.to(cuda_device), query_out=qi, key_out=ki, **how)
    assert again[0] is qi and again[1] is ki
    assert torch.equal(qi, got[0]) and torch.equal(ki, got[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(3, 4, 1, 4001, 64, 32, (4, 6, 6), True, 16), (2, 1, 1, 12007, 24, 24, (5, 7), False, 24),
                                  (7, 3, 3, 900, 128, 128, None, False, 8), (1, 9, 2, 3001, 256, 64, (11, 11, 10), True, 32),
                                  (1, 33, 1, 2600, 32, 16, (3, 5), False, 16), (2, 2, 1, 1700, 16, 16, None, False, 16)], ids=str)
def test_many_tokens(cuda_device, case, dtype):
    """Several tokens a CTA, the last of them fewer, rows of the batch inside a CTA."""
    batch, q_heads, kv_heads, tokens, dim, width, sections, interleaved, page = case
    q, k = states(batch, q_heads, kv_heads, tokens, dim, dtype, cuda_device)
    v = states(batch, 1, kv_heads, tokens, dim, dtype, cuda_device, seed=2)[1]
    axes = 1 if sections is None else len(sections)
    positions = torch.randint(0, 1 << 18, (axes, batch, tokens), generator=torch.Generator().manual_seed(1))
    how = dict(theta=1e6, sections=sections, interleaved=interleaved, rotary_dim=width)
    got = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions.to(cuda_device), **how)
    for x, out in zip((q, k), got):
        assert_close(out, *turned(x, positions, width, theta=1e6, sections=sections, interleaved=interleaved))
    past = torch.arange(batch) * 5 + 2
    blocks = (int(past.max()) + tokens + page - 1) // page
    order = torch.randperm(batch * blocks, generator=torch.Generator().manual_seed(3)).view(batch, blocks)
    pools = [torch.zeros(batch * blocks, kv_heads, page, dim, device=cuda_device, dtype=dtype) for _ in range(2)]
    new = torch.zeros(batch, dtype=torch.long, device=cuda_device)
    out = anna_b200.run_rotary_paged_kv_write(query=q, key=k, value=v, key_pages=pools[0], value_pages=pools[1],
                                              page_table=order.int().to(cuda_device), past_lengths=past.to(cuda_device),
                                              positions=positions.to(cuda_device), new_lengths=new, **how)
    assert torch.equal(out, got[0]) and new.tolist() == (past + tokens).tolist()
    want = [torch.zeros_like(pool) for pool in pools]
    at = past[:, None] + torch.arange(tokens)
    pages = order.gather(1, at // page).to(cuda_device)
    for pool, x in zip(want, (got[1], v)):
        pool[pages, :, (at % page).to(cuda_device)] = x.transpose(1, 2)
    assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1])
    qi, ki = q.clone(), k.clone()
    anna_b200.run_multi_axis_rotary(query=qi, key=ki, positions=positions.to(cuda_device), query_out=qi, key_out=ki, **how)
    assert torch.equal(qi, got[0]) and torch.equal(ki, got[1])


@pytest.mark.gpu
def test_far_positions_negative_ones_and_scaling(cuda_device):
    q, k = states(1, 2, 1, 6, 64, torch.float32, cuda_device)
    positions = torch.tensor([[0, 1, -5, 262143, (1 << 31) - 1, -(1 << 31)]])
    frequencies = [math.sqrt(2) ** -i for i in range(32)]
    got = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions.to(cuda_device), inverse_frequencies=frequencies,
                                          attention_scaling=1.25)
    # 2^31 positions times a rate rounded to 64 bits: 2^31 * 2^-52 radian more
    for x, out in zip((q, k), got):
        want, bound = turned(x, positions, 64, frequencies=frequencies, scale=1.25)
        assert_close(out, want, 3 * bound)
    past, deltas = torch.tensor([70000]), torch.tensor([[-200]])
    want = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=(past[:, None] + deltas + torch.arange(6)).to(cuda_device))
    got = anna_b200.run_multi_axis_rotary(query=q, key=k, past_lengths=past.to(cuda_device), rope_deltas=deltas.to(cuda_device))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    exact_zero = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=torch.zeros(1, 6, dtype=torch.long, device=cuda_device))
    assert torch.equal(exact_zero[0], q) and torch.equal(exact_zero[1], k)  # no turn changes no bit


@pytest.mark.gpu
def test_odd_addresses_broadcast_positions_and_empty_calls(cuda_device):
    base = torch.randn(2 * 3 * 5 * 64 + 9, device=cuda_device).to(torch.bfloat16)
    for shift in (1, 2, 4, 7):
        q = base[shift:shift + 2 * 3 * 5 * 64].view(2, 3, 5, 64)
        k = base[shift:shift + 2 * 5 * 64].view(2, 1, 5, 64)
        positions = torch.arange(5, device=cuda_device)[None].expand(2, 5)  # stride 0 over the batch
        out_base = torch.full((q.numel() + 3,), 7.0, device=cuda_device, dtype=torch.bfloat16)
        out = out_base[1:1 + q.numel()].view(q.shape)
        got = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions, query_out=out)
        assert got[0] is out and float(out_base[0]) == 7.0 and bool((out_base[-2:] == 7.0).all())
        assert_close(out, *turned(q, positions, 64))
        assert_close(got[1], *turned(k, positions, 64))
    for shape in ((0, 2, 3, 64), (2, 2, 0, 64)):
        empty = torch.empty(shape, device=cuda_device)
        positions = torch.zeros(shape[0], shape[2], dtype=torch.long, device=cuda_device)
        got = anna_b200.run_multi_axis_rotary(query=empty, key=empty, positions=positions)
        assert got[0].shape == shape and got[1].shape == shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,tokens,page,given", [(3, 1, 16, False), (2, 19, 16, True), (4, 5, 24, False), (1, 40, 8, True)])
def test_keys_and_values_go_to_their_pages(cuda_device, dtype, batch, tokens, page, given):
    q_heads, kv_heads, dim, width, sections = 6, 2, 64, 32, (4, 6, 6)
    q, k = states(batch, q_heads, kv_heads, tokens, dim, dtype, cuda_device)
    v = torch.randn(batch, kv_heads, tokens, dim, device=cuda_device).to(dtype)  # strides of its own
    past = torch.tensor([(7 * b + 3) % 41 for b in range(batch)])
    blocks = (int(past.max()) + tokens + page - 1) // page
    order = torch.randperm(batch * blocks + 2, generator=torch.Generator().manual_seed(3))[:batch * blocks].view(batch, blocks)
    pools = [torch.full((batch * blocks + 2, kv_heads, page, dim), float(i + 2), device=cuda_device, dtype=dtype) for i in range(2)]
    deltas = torch.arange(batch)[:, None] * -2
    positions = torch.randint(0, 5000, (3, batch, tokens), generator=torch.Generator().manual_seed(4))
    new = torch.zeros(batch, dtype=torch.long, device=cuda_device)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    got = anna_b200.run_rotary_paged_kv_write(
        query=q, key=k, value=v, key_pages=pools[0], value_pages=pools[1], page_table=order.int().to(cuda_device),
        past_lengths=past.to(cuda_device), positions=positions.to(cuda_device) if given else None,
        rope_deltas=None if given else deltas.to(cuda_device), rotary_dim=width, sections=sections, new_lengths=new, status=status)
    if not given:
        positions = (past[:, None] + deltas + torch.arange(tokens)).expand(3, batch, tokens)
    assert_close(got, *turned(q, positions, width, sections=sections))
    assert new.tolist() == (past + tokens).tolist() and int(status) == 0
    _, turned_k = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions.to(cuda_device), rotary_dim=width,
                                                  sections=sections)
    want = [torch.full_like(pools[0], 2.0), torch.full_like(pools[1], 3.0)]
    for b, t in itertools.product(range(batch), range(tokens)):
        block, slot = divmod(int(past[b]) + t, page)
        want[0][order[b, block], :, slot] = turned_k[b, :, t]
        want[1][order[b, block], :, slot] = v[b, :, t]
    assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1])  # and nothing else was touched


@pytest.mark.gpu
def test_tokens_without_a_page_are_reported_and_not_written(cuda_device):
    q, k = states(3, 2, 1, 4, 64, torch.bfloat16, cuda_device)
    pools = [torch.zeros(2, 1, 4, 64, device=cuda_device, dtype=torch.bfloat16) for _ in range(2)]
    table = torch.tensor([[0, -1], [1, 9], [-1, -1]], dtype=torch.int32, device=cuda_device)
    past = torch.tensor([2, 3, 100], device=cuda_device)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    got = anna_b200.run_rotary_paged_kv_write(query=q, key=k, value=k, key_pages=pools[0], value_pages=pools[1], page_table=table,
                                              past_lengths=past, status=status)
    assert int(status) == _lib.DEV_BAD_PAGE
    positions = past[:, None] + torch.arange(4, device=cuda_device)
    assert_close(got, *turned(q, positions, 64))
    written = pools[1].abs().sum(-1)[:, 0] > 0
    assert written.tolist() == [[False, False, True, True], [False, False, False, True]]


@pytest.mark.gpu
def test_captured_calls_follow_their_inputs(cuda_device):
    q, k = states(2, 4, 2, 1, 128, torch.bfloat16, cuda_device)
    pools = [torch.zeros(8, 2, 16, 128, device=cuda_device, dtype=torch.bfloat16) for _ in range(2)]
    table = torch.arange(8, dtype=torch.int32, device=cuda_device).view(2, 4)
    past = torch.tensor([5, 20], device=cuda_device)

    def call():
        return anna_b200.run_rotary_paged_kv_write(query=q, key=k, value=k, key_pages=pools[0], value_pages=pools[1],
                                                   page_table=table, past_lengths=past, sections=(16, 24, 24))

    call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call()
    past.add_(7)
    q.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    positions = past[:, None]
    assert_close(out, *turned(q, positions, 128, sections=(16, 24, 24)))
    _, want = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions, sections=(16, 24, 24))
    assert torch.equal(pools[0][0, :, 12], want[0, :, 0]) and torch.equal(pools[0][5, :, 11], want[1, :, 0])


@pytest.mark.gpu
def test_outputs_that_overlap_are_refused(cuda_device):
    whole = torch.randn(1, 4, 9, 64, device=cuda_device)
    q, k = whole[:, :2, :8], whole[:, 2:, :8]
    positions = torch.arange(8, device=cuda_device)[None]
    for bad in (dict(query_out=whole[:, :2, 1:]), dict(query_out=k), dict(query_out=torch.empty(1, 1, 8, 64, device=cuda_device).expand(1, 2, 8, 64)),
                dict(query_out=torch.empty(1, 2, 8, 64)), dict(query_out=torch.empty(1, 2, 8, 128, device=cuda_device)[..., ::2]),
                dict(query_out=torch.empty(1, 2, 8, 64, device=cuda_device).half())):
        with pytest.raises(RuntimeError, match="query_out"):
            anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions, **bad)
    shared = torch.empty(1, 2, 8, 64, device=cuda_device)
    with pytest.raises(RuntimeError, match="overlap"):
        anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions, query_out=shared, key_out=shared)


@pytest.mark.gpu
def test_in_place_on_parts_of_one_projection_and_on_shared_memory(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(0)
    positions = torch.arange(5, device=cuda_device)[None].expand(2, 5)
    tokens = torch.randn(2, 5, 7 * 64, device=cuda_device, generator=gen)  # heads of a token next to each other
    rows = torch.randn(2, 7, 5, 64, device=cuda_device, generator=gen)     # heads of a row next to each other
    by_token = tokens.view(2, 5, 7, 64).transpose(1, 2)
    for q, k in ((by_token[:, :4], by_token[:, 4:6]), (by_token[:, 3:], by_token[:, :2]), (rows[:, :4], rows[:, 4:6]),
                 (rows[:, 3:], rows[:, 1:3])):
        want = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions)
        got = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions, query_out=q, key_out=k)
        assert got[0] is q and got[1] is k and torch.equal(q, want[0]) and torch.equal(k, want[1])
    for q, k in ((rows, rows), (rows[:, :4], rows[:, 3:]), (by_token[:, :4], by_token[:, 3:]), (rows[:, :, :4], rows[:, :, 1:])):
        where = positions[:, :q.shape[2]]
        for outs in (dict(query_out=q), dict(key_out=k), dict(query_out=q, key_out=k)):
            with pytest.raises(RuntimeError, match="in place"):
                anna_b200.run_multi_axis_rotary(query=q, key=k, positions=where, **outs)
    # 2 x 2 rows of 64 dims, 64 and 65 elements apart: two of them share elements
    woven = torch.zeros(256, device=cuda_device).as_strided((1, 2, 2, 64), (256, 65, 64, 1))
    with pytest.raises(RuntimeError, match="query_out"):
        anna_b200.run_multi_axis_rotary(query=woven, key=rows[:1, :1, :2], positions=positions[:1, :2], query_out=woven)


@pytest.mark.gpu
def test_new_lengths_that_are_read_are_refused(cuda_device):
    q, k = torch.randn(3, 2, 1, 64, device=cuda_device), torch.randn(3, 1, 1, 64, device=cuda_device)
    pages = [torch.zeros(4, 1, 8, 64, device=cuda_device) for _ in range(2)]
    table = torch.arange(3, device=cuda_device, dtype=torch.int32)[:, None]
    memory = torch.zeros(9, device=cuda_device, dtype=torch.long)

    def run(**more):
        return anna_b200.run_rotary_paged_kv_write(query=q, key=k, value=k, key_pages=pages[0], value_pages=pages[1], page_table=table,
                                                   **more)

    for more in (dict(past_lengths=memory[:3], new_lengths=memory[:3]), dict(past_lengths=memory[:3], new_lengths=memory[1:4]),
                 dict(past_lengths=memory[:3], new_lengths=memory[4:7], positions=memory[3:6, None]),
                 dict(past_lengths=memory[:3], new_lengths=memory[4:7], rope_deltas=memory[6:])):
        with pytest.raises(RuntimeError, match="new_lengths"):
            run(**more)
    run(past_lengths=memory[:3], new_lengths=memory[3:6], positions=memory[6:, None])
    assert memory.tolist() == [0, 0, 0, 1, 1, 1, 0, 0, 0]


@pytest.mark.gpu
def test_tables_are_kept_and_counted(cuda_device, monkeypatch):
    first = rotary.rotary_tables(64, theta=123.0, device=cuda_device)
    assert rotary.rotary_tables(64, theta=123.0, device=cuda_device) is first
    given = [rotary.rotary_tables(64, sections=s, inverse_frequencies=f, device=cuda_device)
             for s, f in (((20, 12), [0.5] * 32), (torch.tensor([20, 12]), torch.full((32,), 0.5)), ([20, 12], np.full(32, 0.5)))]
    assert given[1] is given[0] and given[2] is given[0]
    for bad in ([0.5] * 31, [math.inf] * 32, [math.nan] * 32):
        with pytest.raises(ValueError, match="inverse_frequencies"):
            rotary.rotary_tables(64, inverse_frequencies=bad, device=cuda_device)
    monkeypatch.setattr(rotary, "_TABLES", {i: first for i in range(4096)})
    with pytest.raises(RuntimeError, match="rotary parameters"):
        rotary.rotary_tables(64, theta=124.0, device=cuda_device)


def test_pairs_to_axes():
    for width, sections, interleaved in ((128, (16, 24, 24), False), (128, (24, 20, 20), True), (64, (11, 11, 10), True),
                                         (64, (32,), True), (8, (0, 0, 4), True), (8, (0, 4), False), (64, None, True)):
        assert rotary.pair_axes(width, sections, interleaved) == axes_of(width, sections, interleaved)
    for bad in ((16, 24, 23), (), (65, -1)):
        with pytest.raises(ValueError, match="sections"):
            rotary.pair_axes(128, bad, False)


def test_calls_that_cannot_be_are_refused():
    q, k = torch.zeros(2, 4, 3, 64), torch.zeros(2, 2, 3, 64)
    positions = torch.zeros(2, 3, dtype=torch.long)
    call = anna_b200.run_multi_axis_rotary
    with pytest.raises(RuntimeError, match="CUDA"):
        call(query=q, key=k, positions=positions)
    with pytest.raises(RuntimeError, match="agree"):
        call(query=q, key=k[:, :, :2], positions=positions)
    with pytest.raises(RuntimeError, match="dtype"):
        call(query=q, key=k.half(), positions=positions)
    for change, match in ((dict(positions=None), "past_lengths"), (dict(positions=None, past_lengths=positions), "past_lengths"),
                          (dict(rope_deltas=positions[:, 0]), "rope_deltas"),
                          (dict(positions=None, past_lengths=positions[:, 0], rope_deltas=positions), "rope_deltas")):
        with pytest.raises(RuntimeError, match=match):
            call(**{**dict(query=q, key=k, positions=positions), **change})
    with pytest.raises(RuntimeError, match="batch, heads"):
        call(query=q[0], key=k, positions=positions)
    with pytest.raises(RuntimeError, match="float16, bfloat16"):
        call(query=q.double(), key=k.double(), positions=positions)
    pages, table = torch.zeros(4, 2, 16, 64), torch.zeros(2, 4, dtype=torch.int32)
    good = dict(query=q, key=k, value=k, key_pages=pages, value_pages=pages, page_table=table, past_lengths=positions[:, 0])
    for change, match in ((dict(value=k[:, :1]), "value"), (dict(value_pages=pages[:2]), "value_pages"),
                          (dict(key_pages=pages[:, :1], value_pages=pages[:, :1]), "kv_heads"), (dict(page_table=table.long()), "page_table"),
                          (dict(past_lengths=table[:, 0]), "past_lengths"), (dict(rope_deltas=positions[:1, 0]), "rope_deltas"),
                          (dict(rope_deltas=positions[:, 0], positions=positions), "rope_deltas"),
                          (dict(key_pages=pages.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous"),
                          (dict(new_lengths=good["past_lengths"]), "new_lengths"), ({}, "CUDA")):
        with pytest.raises(RuntimeError, match=match):
            anna_b200.run_rotary_paged_kv_write(**{**good, **change})


def test_entry_points_refuse_what_they_cannot_run():
    """Made-up addresses: every call is refused before anything is launched."""
    library, ok = _lib.lib(), 0x10000

    def rotary_call(q=ok, out=ok, k=ok, positions=ok, rates=ok, batch=1, heads=2, kv=1, tokens=1, dim=64, width=64, dtype=2):
        return library.anna_multi_axis_rotary(q, 64, 64, 64, out, 64, 64, 64, k, 64, 64, 64, out, 64, 64, 64, positions, 0, 1, 1, None,
                                              None, 0, rates, ok, 1.0, batch, heads, kv, tokens, dim, width, dtype, None)

    for bad in (dict(q=None), dict(out=None), dict(k=None), dict(positions=None), dict(rates=None), dict(batch=0), dict(heads=0),
                dict(tokens=0), dict(width=0), dict(width=63), dict(width=66), dict(dim=8192, width=64), dict(dtype=3), dict(q=ok + 1),
                dict(batch=1 << 16, tokens=1 << 15)):
        assert rotary_call(**bad) == 1, bad
        assert "anna_multi_axis_rotary" in _lib.last_error()
