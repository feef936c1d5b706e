"""Attention of several new tokens over packed pages where values or weights are large, small or far apart, against 64 bits.

Limits beside those of test_gpu_tq_multi_decode.py are derived at each test."""
from __future__ import annotations

import itertools
import math

import numpy as np
import pytest
import torch
from test_gpu_tq_multi_decode import Case, hadamard

import anna_b200
from anna_b200.tq_tables import key_tables


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


def packed_parts(case):
    """(centroid numbers, signs, norms, residual norms) of the codes in a 4-bit case's pages."""
    pages, heads, page, dim, layout = case.packed.shape[0], case.kv_heads, case.page, case.dim, case.layout

    def part(name, size, kind):
        return case.packed[:, :, layout[name]:layout[name] + size].contiguous().view(kind).reshape(pages, heads, page, -1).numpy()

    codes = part("off_kcodes", page * dim // 2, torch.uint8)
    nibbles = np.stack([codes & 15, codes >> 4], -1).reshape(pages, heads, page, dim)
    return nibbles & 7, nibbles >> 3, part("off_knorm", 4 * page, torch.float32)[..., 0], part("off_krnorm", 4 * page, torch.float32)[..., 0]


def rounded(case):
    """The outputs of 64-bit arithmetic in which what the kernel's header names is rounded: the rotated queries to fp16, relative to the
    largest (of fp16 caches those of the residual part alone, the others being sums of two), centroids and residual norms to fp16 at the
    scale where an fp16 cache's centroids lose least, the packed values to fp16, the probabilities of a bf16 cache's packed keys to fp16,
    and the output to its type."""
    half = lambda x: np.asarray(x, np.float16).astype(np.float64)  # noqa: E731
    fp16 = case.dtype == torch.float16
    tables = key_tables(head_dim=case.dim, bits=4, device="cpu")
    centroids, s1, s2 = (x.numpy().astype(float) for x in (tables.centroids, tables.signs1, tables.signs2))
    h, (index, sign, norm, rnorm) = hadamard(case.dim), packed_parts(case)
    scales = 1 + np.arange(512 if fp16 else 1)[:, None] / 512
    at = float(scales[np.argmin(((centroids * scales - half(centroids * scales)) ** 2 / scales ** 2).sum(1))][0])
    out = torch.zeros(case.query.shape, dtype=torch.float64)
    for b, (k, v) in enumerate(case.dense):
        n, lq = case.lengths[b], case.quantized[b]
        where = case.table[b].numpy()[np.arange(lq) // case.page], np.arange(lq) % case.page
        for head, t in itertools.product(range(case.query.shape[1]), range(case.tokens)):
            kvh = head // case.group
            cells = where[0], kvh, where[1]
            query = case.query[b, head, t].double().numpy()
            q1 = h @ (s1 * query)
            q2 = math.sqrt(math.pi / 2 / case.dim) * (h @ (s2 * q1))
            top = max(np.abs(q1).max(), np.abs(q2).max())
            score = (half(centroids * at) / at)[index[cells]] @ (q1 / top if fp16 else half(q1 / top))
            score += half(rnorm[cells] * at) / at * ((2.0 * sign[cells] - 1) @ half(q2 / top))
            score = np.concatenate([score * norm[cells] / case.dim * top, k[kvh][lq:] @ query]) * case.scaling
            score = score[:n - case.tokens + t + 1]
            w = np.exp(score - score.max())
            w_v = w if fp16 else np.concatenate([half(w[:lq] * 128) / 128, w[lq:]])
            out[b, head, t] = torch.from_numpy(w_v @ np.concatenate([half(v[kvh][:lq]), v[kvh][lq:]])[:len(w)] / w.sum())
    return out.to(case.dtype).double()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,group,window,length", [
    ("fp16", 128, 4, 128, 3000), ("fp16", 128, 16, 128, 2000), ("fp16", 256, 32, 64, 1500), ("fp16", 64, 8, 33, 1500), ("fp16", 128, 4, 256, 250),
    ("fp16", 256, 8, 512, 480), ("bf16", 128, 4, 128, 3000), ("bf16", 256, 32, 64, 1500), ("bf16", 128, 4, 256, 250)])
@pytest.mark.parametrize("exact_values", [False, True])
def test_error_of_whole_outputs(cuda_device, dtype, dim, group, window, length, exact_values):
    """Root mean square of the errors: that of 64-bit arithmetic with the roundings which the kernel says it makes, and 3 % for 32-bit
    sums and for chance (thousands of outputs).  With residual norms of zero and values that fp16 holds, little is left but the output's own
    rounding, so that queries or probabilities of a single fp16 would show in an fp16 cache."""
    case = Case(lengths=[length], tokens=4, group=group, kv_heads=2, dim=dim, bits=4, page=16, window=window, dtype=dtype, device=cuda_device, seed=31)
    if exact_values:
        for t in range(case.quantized[0]):
            pid, slot = int(case.table[0, t // 16]), t % 16
            case.packed[pid, :, case.layout["off_krnorm"] + 4 * slot:case.layout["off_krnorm"] + 4 * slot + 4] = 0
            for head, part in itertools.product(range(2), range(dim // 32)):
                put_values(case, 0, t, head, part, scale=0.125, zero=(t * 7 + head + part) % 5 / 8 - 1)
        case.dense[0][0][:, :case.quantized[0]] = keys_of(case)
    want, _, _ = case.expected()
    got = case.run().cpu().double()
    rms = lambda x: float((x - want).square().mean().sqrt() / want.square().mean().sqrt())  # noqa: E731
    print(f"{rms(got):.3e} and {rms(rounded(case)):.3e}")
    assert rms(got) <= 1.03 * rms(rounded(case))


def keys_of(case):
    """De-quantized keys of sequence 0 of a 4-bit case, [KV heads, tokens, D]."""
    tables, (index, sign, norm, rnorm) = key_tables(head_dim=case.dim, bits=4, device="cpu"), packed_parts(case)
    t = np.arange(case.quantized[0])
    index, sign, norm, rnorm = (x[case.table[0].numpy()[t // case.page], :, t % case.page].swapaxes(0, 1) for x in (index, sign, norm, rnorm))
    h, s1, s2 = hadamard(case.dim), tables.signs1.numpy().astype(float), tables.signs2.numpy().astype(float)
    rotated = tables.centroids.numpy().astype(float)[index] + math.sqrt(math.pi / 2 / case.dim) * rnorm[..., None] * (((2.0 * sign - 1.0) @ h) * s2)
    return norm[..., None] / case.dim * (rotated @ h) * s1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,group,page,window,length", [
    ("fp16", 128, 4, 16, 128, 3000), ("fp16", 128, 16, 32, 128, 2000), ("fp16", 256, 8, 16, 64, 1500), ("fp16", 64, 8, 16, 33, 1500),
    ("fp16", 128, 4, 24, 64, 1500), ("fp16", 256, 8, 16, 512, 480), ("bf16", 128, 4, 16, 128, 3000), ("bf16", 256, 6, 32, 64, 1500)])
def test_one_token_is_as_exact_as_one_of_several(cuda_device, dtype, dim, group, page, window, length):
    """The error of a single new token has the bound of test_error_of_whole_outputs, and the same token among others the same answer but for
    what the header's roundings may make of another running maximum: they are at the same places, so the two differ by less than twice that."""
    rms = lambda x, want: float((x - want).square().mean().sqrt() / want.square().mean().sqrt())  # noqa: E731
    case = Case(lengths=[length], tokens=4, group=group, kv_heads=2, dim=dim, bits=4, page=page, window=window, dtype=dtype, device=cuda_device, seed=32)
    several = case.run()[:, :, 3:]
    case.query, case.tokens = case.query[:, :, 3:], 1
    want, _, _ = case.expected()
    got, limit = case.run(), 1.03 * rms(rounded(case), want)
    assert rms(got.cpu().double(), want) <= limit
    assert rms(got.cpu().double(), several.cpu().double()) <= 2 * limit


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 3])
def test_layouts_that_change_nothing(cuda_device, tokens):
    case = Case(lengths=[700, 90], tokens=tokens, group=4, kv_heads=2, dim=128, bits=4, page=16, window=16, dtype="fp16", device=cuda_device, seed=33)
    want = case.run()
    case.slots = torch.stack([case.slots, case.slots], 1)[:, 0]
    case.table = torch.stack([case.table, case.table], 2)[..., 0]
    put = lambda x: x.to(cuda_device) if x.is_contiguous() else torch.stack([x, x], -1).to(cuda_device)[..., 0]  # noqa: E731
    got = anna_b200.run_tq_paged_multi_decode(
        query=put(case.query), packed_pages=put(case.packed), page_table=put(case.table), window=put(case.window_ring), window_slots=put(case.slots),
        lengths=put(torch.tensor([[700, 0], [90, 0]])[:, 0]), scaling=case.scaling, bits=4, residual_len=16, block_size=16, value_group_size=32)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,bits,page", [(128, 4, 16), (256, 3, 16), (64, 2, 16), (128, 2, 24), (64, 4, 8), (128, 4, 12)])
@pytest.mark.parametrize("tokens,group", [(3, 2), (4, 4), (40, 3)])
@pytest.mark.parametrize("power", [-6, -12, -17, -40, -90])
def test_small_values(cuda_device, dim, bits, page, tokens, group, power):
    """bf16 values down to 1e-27, as exact as others."""
    case = Case(lengths=[700, 90, 33], tokens=tokens, group=group, kv_heads=2, dim=dim, bits=bits, page=page, window=9, dtype="bf16",
                device=cuda_device, seed=17)
    pages, groups = case.packed.shape[0], dim // 32
    for name in ("off_vscale", "off_vzero"):
        part = case.packed[:, :, case.layout[name]:case.layout[name] + page * groups * 2]
        scaled = part.contiguous().view(torch.bfloat16).double().mul(2.0 ** power).to(torch.bfloat16)
        part.copy_(scaled.view(torch.uint8).reshape(pages, 2, -1))
    case.window_ring[:, 1] *= 2.0 ** power
    for b in range(3):
        case.dense[b][1][:] *= 2.0 ** power
    check_each(case, case.run(), floor=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,bits,page", [(128, 4, 16), (256, 3, 16), (64, 2, 16), (128, 2, 24)])
@pytest.mark.parametrize("tokens,group", [(3, 2), (12, 6)])
def test_small_and_ordinary_values_together(cuda_device, dim, bits, page, tokens, group):
    """A group of dims with small values beside others, one that is zero at first, and one where an ordinary value comes late."""
    case = Case(lengths=[700, 90], tokens=tokens, group=group, kv_heads=2, dim=dim, bits=bits, page=page, window=9, dtype="bf16",
                device=cuda_device, seed=18)
    for t in range(case.quantized[0]):
        put_values(case, 0, t, 0, 1, scale=2e-7 * (1 + t % 7), zero=1e-6 * (t % 5 - 2))
        late = t in (400, 689)
        put_values(case, 0, t, 1, 0, scale=0.1 if late else 1e-6, zero=0.5 if late else 1e-5)
        put_values(case, 0, t, 1, 1, scale=0.0 if t < 300 else 1e-6, zero=0.0 if t < 300 else 1e-5)
    case.window_ring[case.slots[0], 1, 0, :, 32:64] *= 1e-6
    case.window_ring[case.slots[0], 1, 1, :, :64] *= 1e-6
    for t in range(case.quantized[0], 700):
        case.dense[0][1][:, t] = case.window_ring[case.slots[0], 1, :, t % 9].double().numpy()
    check_each(case, case.run(), floor=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 3])
def test_small_value_groups(cuda_device, tokens):
    for dtype, group in (("fp16", 4), ("bf16", 2), ("fp32", 2), ("fp32", 4), ("bf16", 8)):
        case = Case(lengths=[90, 3], tokens=tokens, group=2, kv_heads=1, dim=128, bits=4, page=16, window=8, dtype=dtype, device=cuda_device,
                    value_group=group)
        case.check(case.run())
