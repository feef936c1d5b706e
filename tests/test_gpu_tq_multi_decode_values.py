"""Attention of several new tokens over packed pages where values or weights are large, small or far apart, against 64 bits.

Limits beside those of test_gpu_tq_multi_decode.py are derived at each test."""
from __future__ import annotations

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
