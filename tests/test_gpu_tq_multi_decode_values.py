"""Attention of several new tokens over packed pages where values or weights are large, small or far apart, against 64 bits.

Limits beside those of test_gpu_tq_multi_decode.py are derived at each test."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch
from test_gpu_tq_multi_decode import Case


def value_parts(case, name, pid, head, slot, group):
    """Where a value group's scale or zero is in the pages' bytes."""
    elem = torch.finfo(case.dtype).bits // 8
    at = case.layout[name] + (slot * (case.dim // case.value_group) + group) * elem
    return pid, head, slice(at, at + elem)


def put_values(case, b, t, head, group, *, scale, zero):
    """Gives a value group of a packed token another scale and zero, in the pages and in the dense values."""
    pid, slot, span = int(case.table[b, t // case.page]), t % case.page, slice(group * case.value_group, (group + 1) * case.value_group)
    was, new = [], []
    for name, value in (("off_vscale", scale), ("off_vzero", zero)):
        where = value_parts(case, name, pid, head, slot, group)
        was.append(float(case.packed[where].clone().view(case.dtype)))
        case.packed[where] = torch.tensor([value], dtype=case.dtype).view(torch.uint8)
        new.append(float(torch.tensor(value, dtype=case.dtype)))
    values = case.dense[b][1][head, t, span]
    codes = np.rint((values - was[1]) / was[0])
    case.dense[b][1][head, t, span] = codes * new[0] + new[1]


def check_each(case, got, floor=2.0 ** -25):
    """As Case.check, but relative to what each query averages in each dim: ``top`` is the largest |v| that the query sees in the dim's
    group of 32.  Probabilities and values are off by 2^-12 of themselves each, so their sum by 2 * 2^-12 of the weighted |v|, at most top.
    ``floor``: half of fp16's smallest step, where values among those of the case may be that small."""
    want, spread, size = case.expected()
    top = torch.zeros_like(want)
    for b, (_, v) in enumerate(case.dense):
        for h in range(want.shape[1]):
            for t in range(case.tokens):
                seen = np.abs(v[h // case.group][:max(0, case.lengths[b] - case.tokens + t + 1)])
                if len(seen):
                    top[b, h, t] = torch.from_numpy(np.repeat(seen.reshape(len(seen), -1, 32).max((0, 2)), 32))
    score = size * (2 * case.dim * 2.0 ** -24 + 2.0 ** -12 * (2.0 * np.sqrt(2 * np.log(2 * case.dim)) + 2))
    half = torch.finfo(case.dtype).eps / 2
    limit = 2 * score * spread + 2 * 2.0 ** -12 * top + floor + half * want.abs() * 1.01
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    assert bool(((got - want).abs() <= limit).all()), float(((got - want).abs() / limit).nan_to_num(0.0).max())


FORMS = [("bf16", 128, 4, 16), ("fp16", 256, 3, 16), ("fp16", 128, 2, 16), ("fp32", 128, 4, 16), ("bf16", 64, 2, 16), ("fp16", 64, 4, 16),
         ("bf16", 128, 4, 24), ("fp16", 64, 3, 8), ("bf16", 256, 2, 32), ("bf16", 128, 4, 12)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,bits,page", FORMS)
@pytest.mark.parametrize("group", [2, 9])
def test_large_values_behind_a_query(cuda_device, dtype, dim, bits, page, group):
    """Finite values near the end of fp16's range, in tokens that some of the queries do not see."""
    window, tokens, length = 2, 9, 70
    case = Case(lengths=[length, 40], tokens=tokens, group=group, kv_heads=2, dim=dim, bits=bits, page=page, window=window, dtype=dtype,
                device=cuda_device, seed=13)
    scale = 66000 / (3 if bits == 2 else 15)
    for t in (length - 5, length - 9, length - 20):
        put_values(case, 0, t, 1, 1, scale=scale, zero=-33000.0)
    put_values(case, 1, 30, 0, 0, scale=-0.9 * scale, zero=30000.0)
    case.check(case.run())
    case.check(case.run(gate=True), gate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,bits,page", [(128, 4, 16), (256, 3, 16), (64, 2, 16), (128, 2, 24), (64, 4, 8)])
@pytest.mark.parametrize("tokens,group", [(9, 2), (4, 4), (12, 6)])
def test_values_beyond_fp16(cuda_device, dim, bits, page, tokens, group):
    """bf16 values up to 1e30, among codes of the same group that are small, before and behind ordinary tokens."""
    case = Case(lengths=[300, 40], tokens=tokens, group=group, kv_heads=2, dim=dim, bits=bits, page=page, window=2, dtype="bf16",
                device=cuda_device, seed=14)
    for t, scale, zero in ((295, 70000.0, -5.0), (293, 9000.0, 0.0), (150, 6000.0, 2.0), (3, 1e5, -1e5)):
        put_values(case, 0, t, 1, 1, scale=scale, zero=zero)
    put_values(case, 1, 20, 0, 0, scale=1e30, zero=-1e30)
    put_values(case, 1, 35, 0, 1, scale=1e20, zero=0.0)
    check_each(case, case.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,kv_heads,group", [(128, 8, 2), (256, 4, 2), (64, 8, 2), (128, 4, 12)])
@pytest.mark.parametrize("sink", [0, 33, -1])
def test_small_weights_beside_one_that_is_large(cuda_device, dtype, dim, kv_heads, group, sink):
    """One key has the weight 2^26 times that of each of the 4111 others, and a value of zero: the output is what the others hold together.
    A stream is one CTA's, whose warp with that key has an eighth of the others.

    Small weights are off by 2^-32 of the large one, 2^-6 of themselves here; the large key's score by what Case.check allows of it (the sum
    of the others is off by as much of itself), all other roundings by 2 * 2^-12 of the output and half a step of it."""
    length, window = 4112, 16
    case = Case(lengths=[length], tokens=2, group=group, kv_heads=kv_heads, dim=dim, bits=4, page=16, window=window, dtype=dtype,
                device=cuda_device, seed=21)
    at = sink % (length - window)
    layout, pages, page, groups = case.layout, case.packed.shape[0], case.page, dim // 32

    def put(name, values, width):
        case.packed[:, :, layout[name]:layout[name] + page * width] = values.contiguous().view(torch.uint8).reshape(pages, kv_heads, -1)

    small = 2.0 ** -20
    key = case.dense[0][0][:, at]  # of each KV head
    old = case.packed[int(case.table[0, at // page]), :, layout["off_knorm"]:layout["off_knorm"] + 4 * page].contiguous().view(torch.float32)
    unit = key / old[:, at % page].double().numpy()[:, None]
    query = torch.from_numpy(unit / np.linalg.norm(unit, axis=1, keepdims=True) * math.sqrt(dim)).to(case.dtype)
    norm = torch.full((pages, kv_heads, page), small)
    score = 26 * math.log(2.0)
    norm[int(case.table[0, at // page]), :, at % page] = torch.from_numpy(score / ((query.double().numpy() * unit).sum(1) * case.scaling)).float()
    put("off_knorm", norm, 4)
    put("off_vscale", torch.zeros(pages, kv_heads, page, groups, dtype=case.dtype), 2 * groups)
    zero = torch.ones(pages, kv_heads, page, groups, dtype=case.dtype)
    zero[int(case.table[0, at // page]), :, at % page] = 0
    put("off_vzero", zero, 2 * groups)
    case.window_ring[:, 0] = 0
    case.window_ring[:, 1] = 1
    batch = 37
    case.query = query[:, None, None].expand(kv_heads, group, 2, dim).reshape(1, -1, 2, dim).repeat(batch, 1, 1, 1)
    case.table, case.slots, case.lengths = case.table.repeat(batch, 1), case.slots.repeat(batch), [length] * batch
    got = case.run().cpu().double()
    others = torch.tensor([length - 2.0, length - 1.0]).double() * math.exp(-score)  # all keys but the large one, and those behind the query
    want = (others / (1 + others))[None, None, :, None].expand(got.shape)
    largest = math.sqrt(math.pi / 2) * score * (2.0 ** -12 * (2.0 * math.sqrt(2 * math.log(2 * dim)) + 2) + 2 * dim * 2.0 ** -24)
    limit = want * (2.0 ** -6 + math.expm1(largest) + 2 * 2.0 ** -12 + torch.finfo(case.dtype).eps / 2 + 1e-3)
    assert float(((got - want).abs() / limit).max()) <= 1.0
