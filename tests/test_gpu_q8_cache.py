"""Kernels of the 8-bit paged cache against a restatement in 64 bits (q8_reference.py)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import anna_b200
from q8_reference import Cache, attention, attention_bound, candidates, quantized, selected

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def filled(device, lengths, heads, dim, page, dtype, *, seed=0, spread=1.0, room=0):
    """A cache whose rows have the lengths, written by the restatement."""
    cache = Cache(len(lengths), heads, dim, page, dtype, max(lengths) // page + 1 + room, seed)
    key, value = cache.new_tokens(max(max(lengths), 1), spread)
    for b, n in enumerate(lengths):
        cache.append(key[:, :, :n], value[:, :, :n], rows=[b])
    return cache, cache.on(device)


def check_same(cache, gpu):
    known = cache.known_bytes()
    used = torch.zeros(cache.pages.shape[0], dtype=torch.bool)
    for b in range(cache.batch):
        used[cache.table[b, :int(cache.lengths[b]) // cache.page].long()] = True
    got, want = gpu["packed_pages"].cpu(), cache.pages
    assert torch.equal(got[used][:, :, known], want[used][:, :, known])
    assert torch.equal(got[~used], want[~used])
    assert torch.equal(gpu["window"].cpu().view(torch.uint8), cache.window.view(torch.uint8))


def check_attention(cache, gpu, query, device, *, gate=None, blocks=None, scaling=None):
    scaling = cache.dim ** -0.5 if scaling is None else scaling
    out = anna_b200.run_q8_paged_attention(query=query.to(device), lengths=cache.lengths.to(device), scaling=scaling,
                                           gate=None if gate is None else gate.to(device),
                                           blocks=None if blocks is None else blocks.to(device), **gpu)
    want, reach, most = attention(query, [cache.dense(b) for b in range(cache.batch)], scaling, gate, cache.page, blocks)
    assert out.dtype == query.dtype and out.shape == query.shape
    got = out.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want)
    off = (got - want).abs()[fine]
    bound = attention_bound(want, query.dtype, cache.dim, reach, most)[fine]
    assert bool((off <= bound).all()), (float((off - bound).max()), float(off.max()))
    return got


# ---------------------------------------------------------------------------------------------------------------
# append


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (256, 32), (128, 24), (64, 1), (256, 8), (64, 130), (128, 64)])
def test_append_writes_the_codes_of_the_definition(cuda_device, dtype, dim, page):
    heads, pasts = 2, [0, 1, page - 1, page, 2 * page + page // 2, 5]
    for tokens in (1, 3, page, 2 * page + 5):
        cache = Cache(len(pasts), heads, dim, page, dtype, (max(pasts) + tokens) // page + 1, seed=tokens)
        key, value = cache.new_tokens(max(pasts) + 1)
        for b, n in enumerate(pasts):
            cache.append(key[:, :, :n], value[:, :, :n], rows=[b])
        gpu = cache.on(cuda_device)
        past = cache.lengths.to(cuda_device)
        key, value = cache.new_tokens(tokens, spread=3.0)
        after = torch.zeros_like(past)
        status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
        anna_b200.run_q8_append(key=key.to(cuda_device), value=value.to(cuda_device), past_lengths=past, new_lengths=after, status=status, **gpu)
        cache.append(key, value)
        check_same(cache, gpu)
        assert after.tolist() == cache.lengths.tolist() and status.item() == 0


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_what_is_stored_does_not_depend_on_the_cuts(cuda_device, dtype):
    cache = Cache(3, 2, 128, 16, dtype, 8)
    gpu = cache.on(cuda_device)
    key, value = cache.new_tokens(101)
    at = 0
    for tokens in (1, 1, 13, 1, 1, 32, 15, 16, 20, 1):
        past = torch.full((3,), at, dtype=torch.long, device=cuda_device)
        anna_b200.run_q8_append(key=key[:, :, at:at + tokens].to(cuda_device), value=value[:, :, at:at + tokens].to(cuda_device),
                                past_lengths=past, **gpu)
        cache.append(key[:, :, at:at + tokens], value[:, :, at:at + tokens])
        at += tokens
        check_same(cache, gpu)
    assert at == 101


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_append_of_ties_tiny_huge_and_zero_pages(cuda_device, dtype):
    """Halves of a code (127 x / m = n + 1/2 exactly), subnormals, the largest finite values, pages of zeros."""
    info = torch.finfo(dtype)
    dim, page = 64, 16
    cache = Cache(1, 6, dim, page, dtype, 2)
    key, value = cache.new_tokens(page)
    ladder = torch.arange(-253, 254, 2).double() / 254.0
    ladder = ladder[torch.arange(page * dim) % len(ladder)].view(page, dim)
    least = info.smallest_normal * info.eps
    for x in (key, value):
        x[0, 0] = (ladder * 127.0).to(dtype)       # halves under m = 127
        x[0, 0, 3, 5] = 127.0
        x[0, 1] = (ladder * 9 * 127.0 / 64).to(dtype)
        x[0, 1, 0, 0] = -9 * 127.0 / 64            # 127 times a number that has no exact reciprocal
        x[0, 2] = (torch.randint(-40, 41, (page, dim), generator=cache.gen).double() * least).to(dtype)
        x[0, 3] = (ladder * info.max).to(dtype)
        x[0, 4] = 0.0
        x[0, 5] = (ladder * info.smallest_normal * 127).to(dtype)
    gpu = cache.on(cuda_device)
    anna_b200.run_q8_append(key=key.to(cuda_device), value=value.to(cuda_device), past_lengths=torch.zeros(1, dtype=torch.long, device=cuda_device), **gpu)
    cache.append(key, value)
    check_same(cache, gpu)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_infinities_and_nans_show_in_the_scale(cuda_device, dtype):
    cache = Cache(1, 4, 128, 16, dtype, 3)
    key, value = cache.new_tokens(32)
    key[0, 0, 3, 17], key[0, 1, 20, 5], value[0, 2, 15, 127], value[0, 3, 16, 0] = math.inf, math.nan, -math.inf, math.nan
    gpu = cache.on(cuda_device)
    anna_b200.run_q8_append(key=key.to(cuda_device), value=value.to(cuda_device), past_lengths=torch.zeros(1, dtype=torch.long, device=cuda_device), **gpu)
    size = 2 * 16 * 128
    scales = gpu["packed_pages"][:, :, size:size + 8].contiguous().view(torch.float32).cpu()[cache.table[0, :2].long()]  # [2, heads, 2]
    want = torch.zeros((2, 4, 2), dtype=torch.bool)
    want[0, 0, 0] = want[1, 1, 0] = want[0, 2, 1] = want[1, 3, 1] = True
    assert torch.equal(torch.isnan(scales), want)
    cache.append(key, value)
    codes = gpu["packed_pages"].cpu()[:, :, :size]
    assert torch.equal(codes, cache.pages[:, :, :size])


def test_append_takes_any_strides(cuda_device):
    cache = Cache(2, 3, 128, 16, BF16, 4)
    gpu = cache.on(cuda_device)
    wide = torch.randn((2, 40, 3, 2, 129), generator=cache.gen).to(BF16)
    past = torch.zeros(2, dtype=torch.long, device=cuda_device)
    on_gpu = wide.to(cuda_device)
    views = [(x[:, :, :, 0, :128].transpose(1, 2), x[:, :, :, 1, 1:].transpose(1, 2)) for x in (wide, on_gpu)]  # rows at odd elements
    anna_b200.run_q8_append(key=views[1][0], value=views[1][1], past_lengths=past, **gpu)
    cache.append(*views[0])
    check_same(cache, gpu)


def test_append_leaves_out_pages_and_rings_that_are_none(cuda_device):
    cache = Cache(3, 1, 64, 16, FP16, 2)
    gpu = cache.on(cuda_device)
    before = {k: v.clone() for k, v in gpu.items()}
    gpu["page_table"][0, 0], gpu["page_table"][1, 0], gpu["window_slots"][2] = -1, cache.pages.shape[0], 5
    key, value = cache.new_tokens(20)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    anna_b200.run_q8_append(key=key.to(cuda_device), value=value.to(cuda_device), past_lengths=torch.zeros(3, dtype=torch.long, device=cuda_device),
                            status=status, **gpu)
    assert status.item() == 1
    cache.append(key, value)
    changed = [int(i) for i in (gpu["packed_pages"] != before["packed_pages"]).flatten(1).any(1).nonzero()]
    assert changed == [int(cache.table[2, 0])]
    rings = gpu["window"].cpu().view(torch.int16) != before["window"].cpu().view(torch.int16)
    assert sorted(int(i) for i in rings.flatten(1).any(1).nonzero()) == sorted(int(s) for s in cache.slots[:2])
    # a block that the table has no column for, and a row of negative length
    past = torch.tensor([32, -1, 31], device=cuda_device)
    status.zero_()
    again = {k: v.clone() for k, v in gpu.items()}
    gpu["window_slots"][2] = int(cache.slots[2])
    anna_b200.run_q8_append(key=key[:, :, :1].to(cuda_device), value=value[:, :, :1].to(cuda_device), past_lengths=past, status=status, **gpu)
    assert status.item() == 0  # the page of row 2 is there
    past = torch.tensor([47, -5, -1], device=cuda_device)
    anna_b200.run_q8_append(key=key[:, :, :1].to(cuda_device), value=value[:, :, :1].to(cuda_device), past_lengths=past, status=status, **gpu)
    assert status.item() == 1
    changed = [int(i) for i in (gpu["packed_pages"] != again["packed_pages"]).flatten(1).any(1).nonzero()]
    assert changed in ([], [int(cache.table[2, 1])])


# ---------------------------------------------------------------------------------------------------------------
# dense view


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 24), (256, 32), (128, 1)])
def test_dense_view(cuda_device, dtype, dim, page):
    lengths = [0, 1, page, 3 * page + page // 2, 77]
    cache, gpu = filled(cuda_device, lengths, 2, dim, page, dtype)
    for max_len in (0, 1, 80, max(lengths)):
        key, value = anna_b200.run_q8_gather(lengths=cache.lengths.to(cuda_device), max_len=max_len, **gpu)
        for b, n in enumerate(lengths):
            want = torch.zeros((2, 2, max_len, dim), dtype=torch.float64)
            n = min(n, max_len)
            want[:, :, :n] = cache.dense(b)[:, :, :n]
            for got, exact in ((key, want[0]), (value, want[1])):
                # a product in 32 bits, rounded to the type
                off = (got[b].cpu().double() - exact).abs()
                assert bool((off <= exact.abs() * (2.0 ** -24 + torch.finfo(dtype).eps / 2)).all())


def test_dense_view_of_missing_pages_is_zero(cuda_device):
    cache, gpu = filled(cuda_device, [40, 40], 2, 64, 16, BF16)
    gpu["page_table"][0, 1], gpu["page_table"][1, 0], gpu["window_slots"][1] = -7, 10 ** 6, -1
    key, value = anna_b200.run_q8_gather(lengths=cache.lengths.to(cuda_device), max_len=48, **gpu)
    for x, which in ((key, 0), (value, 1)):
        x = x.cpu()
        assert not x[0, :, 16:32].any() and not x[1, :, :16].any() and not x[1, :, 32:].any() and not x[0, :, 40:].any()
        assert x[0, :, :16].any() and x[1, :, 16:32].any()
        assert torch.equal(x[0, :, 32:40].double(), cache.dense(0)[which, :, 32:40])


# ---------------------------------------------------------------------------------------------------------------
# attention


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim,page,heads,group,tokens", [
    (128, 16, 2, 4, 1), (128, 16, 1, 8, 4), (64, 16, 2, 3, 1), (64, 32, 2, 1, 7), (256, 32, 1, 8, 1), (256, 16, 2, 5, 6),
    (128, 64, 1, 12, 3), (128, 24, 2, 4, 2), (64, 8, 1, 6, 5), (256, 1, 1, 2, 1), (128, 16, 1, 16, 9), (128, 112, 2, 2, 2)])
def test_attention(cuda_device, dtype, dim, page, heads, group, tokens):
    run_attention(cuda_device, dtype, dim, page, heads, group, tokens)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim,page,heads,group,tokens", [(256, 32, 2, 8, 8), (128, 16, 1, 4, 17), (64, 24, 1, 8, 9), (256, 8, 1, 3, 23), (128, 64, 1, 16, 5),
                                                         (128, 1024, 1, 8, 12), (64, 48, 2, 40, 1)])
def test_attention_of_many_queries(cuda_device, dtype, dim, page, heads, group, tokens):
    run_attention(cuda_device, dtype, dim, page, heads, group, tokens)


def run_attention(cuda_device, dtype, dim, page, heads, group, tokens):
    lengths = [0, 1, page - 1, page, page + 1, 5 * page + page // 2, 333, 16, 15, 17]
    cache, gpu = filled(cuda_device, lengths, heads, dim, page, dtype, seed=dim + page)
    query = torch.randn((len(lengths), heads * group, tokens, dim), generator=cache.gen).to(dtype)
    gate = torch.randn(query.shape, generator=cache.gen).to(dtype) if group % 2 == 0 else None
    check_attention(cache, gpu, query, cuda_device, gate=gate)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim,page,heads,group,tokens", [(128, 16, 2, 4, 1), (64, 16, 2, 3, 3), (256, 32, 1, 8, 2), (128, 24, 2, 12, 2), (128, 64, 1, 20, 1)])
def test_attention_over_named_blocks(cuda_device, dtype, dim, page, heads, group, tokens):
    lengths = [0, 1, page, page + 1, 9 * page + 3, 7 * page, tokens - 1]
    cache, gpu = filled(cuda_device, lengths, heads, dim, page, dtype, seed=3)
    query = torch.randn((len(lengths), heads * group, tokens, dim), generator=cache.gen).to(dtype)
    for width in (1, 4, 13):
        # any order, out of range on either side, twice
        blocks = torch.randint(-2, 11, (len(lengths), heads, tokens, width), generator=cache.gen).int()
        check_attention(cache, gpu, query, cuda_device, blocks=blocks)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_long_rows_are_cut_and_merged(cuda_device, dtype):
    """Rows over many CTAs, of very different lengths, and a batch of more rows than a launch lines up."""
    lengths = [2000, 3, 700, 0, 1200]
    cache, gpu = filled(cuda_device, lengths, 1, 128, 16, dtype)
    query = torch.randn((5, 4, 2, 128), generator=cache.gen).to(dtype)
    first = check_attention(cache, gpu, query, cuda_device)
    for _ in range(3):  # arrival counters are back at zero; the order of arrival changes nothing but roundings of the merge
        again = check_attention(cache, gpu, query, cuda_device)
        assert float((again - first).abs().max()) <= 2.0 ** -6 * float(first.abs().max())
    blocks = torch.arange(125).flip(0).view(1, 1, 1, 125).expand(5, 1, 2, 125).int().contiguous()
    check_attention(cache, gpu, query, cuda_device, blocks=blocks)


def test_many_rows(cuda_device):
    rows = 1100
    gen = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 40, (rows,), generator=gen).tolist()
    cache, gpu = filled(cuda_device, lengths, 1, 64, 16, BF16)
    query = torch.randn((rows, 2, 1, 64), generator=gen).to(BF16)
    check_attention(cache, gpu, query, cuda_device)
    check_attention(cache, gpu, query, cuda_device, blocks=torch.randint(0, 3, (rows, 1, 1, 2), generator=gen).int())


@pytest.mark.parametrize("dtype,page,copies", [(BF16, 16, 1), (FP16, 16, 1), (FP32, 16, 1), (BF16, 24, 1), (FP16, 5, 1), (BF16, 16, 5), (FP16, 24, 5)])
def test_keys_that_a_query_does_not_see_do_not_matter(cuda_device, dtype, page, copies):
    """Infinities and NaN in newer tokens, in rings behind the last token, in pages that are not there or not named.  `copies`: of every head,
    for kernels of many rows."""
    tokens = 3
    lengths = [page * 3 + 1, page * 2, page + 2]
    cache, _ = filled(cuda_device, lengths, 2, 128, page, dtype)
    for b, n in enumerate(lengths):  # the two newest tokens
        x = cache.tokens[b]
        x[0, 0, n - 1, 3], x[1, 0, n - 1, 5], x[1, 1, n - 2, 7], x[0, 1, n - 1, 0] = math.nan, math.inf, math.nan, -math.inf
        for block in range(n // page):
            cache.write_page(int(cache.table[b, block]), x[:, :, block * page:(block + 1) * page])
        for at in range(n // page * page, n):
            cache.window[cache.slots[b], :, :, at % page] = x[:, :, at]
    gpu = cache.on(cuda_device)
    query = torch.randn((3, 8, tokens, 128), generator=cache.gen).to(dtype)
    scaling = 128 ** -0.5
    wide = query.repeat_interleave(copies, dim=1)
    out = anna_b200.run_q8_paged_attention(query=wide.to(cuda_device), lengths=cache.lengths.to(cuda_device), scaling=scaling, **gpu).cpu()
    for i in range(1, copies):
        assert torch.equal(out[:, i::copies].isfinite(), out[:, ::copies].isfinite())
    out = out[:, ::copies]
    rows = [cache.dense(b) for b in range(3)]
    checked = []
    for b, n in enumerate(lengths):
        for t in range(tokens):
            seen = n - tokens + t + 1
            want, reach, most = attention(query[b:b + 1, :, t:t + 1], [torch.nan_to_num(rows[b][:, :, :seen], 0.0, 0.0, 0.0)], scaling)
            bound = attention_bound(want, dtype, 128, reach, most)[0, :, 0]
            for h in range(8):
                if bool(torch.isfinite(rows[b][:, h // 4, :seen]).all()):
                    checked.append((b, t, h))
                    assert bool(((out[b, h, t].double() - want[0, h, 0]).abs() <= bound[h]).all()), (b, t, h)
    # the page before the last token of row 0 has a NaN among the values of its second head
    assert {(0, 0, 0), (0, 1, 3), (2, 0, 0), (2, 0, 7)} <= set(checked) and (0, 0, 4) not in checked
    assert bool(torch.isnan(out[0, :4, 2]).any())  # what sees one shows it


@pytest.mark.parametrize("dtype,page", [(BF16, 16), (FP32, 16), (FP16, 8)])
def test_missing_pages_and_rings_are_left_out(cuda_device, dtype, page):
    lengths = [4 * page + 5, 3 * page, 2 * page + 1]
    cache, gpu = filled(cuda_device, lengths, 1, 64, page, dtype)
    gpu["page_table"][0, 1], gpu["page_table"][0, 3], gpu["page_table"][1, :3], gpu["window_slots"][2] = -1, 10 ** 6, -1, 99
    query = torch.randn((3, 4, 2, 64), generator=cache.gen).to(dtype)
    out = anna_b200.run_q8_paged_attention(query=query.to(cuda_device), lengths=cache.lengths.to(cuda_device), scaling=0.1, **gpu).cpu().double()
    kept = [[0, 2, 4], [], [0, 1]]
    for b, n in enumerate(lengths):
        row = cache.dense(b)
        for t in range(2):
            at = [i for i in range(n - 1 + t) if i // page in kept[b]]
            if not at:
                assert not out[b, :, t].any()
                continue
            want, reach, most = attention(query[b:b + 1, :, t:t + 1], [row[:, :, at]], 0.1)
            assert bool(((out[b, :, t] - want[0, :, 0]).abs() <= attention_bound(want, dtype, 64, reach, most)[0, :, 0]).all())


@pytest.mark.parametrize("dtype,copies", [(BF16, 1), (FP16, 1), (FP32, 1), (BF16, 10), (FP16, 10)])
def test_small_weights_and_pages_of_very_different_scales_count(cuda_device, dtype, copies):
    """One key that takes nearly all weight has no value; what the others add is still exact.  Pages whose scales differ by 2^12."""
    cache = Cache(2, 1, 128, 16, dtype, 40)
    key, value = cache.new_tokens(600)
    query = torch.randn((2, 4, 1, 128), generator=cache.gen).to(dtype)
    direction = query[0].float().mean(dim=(0, 1))
    key[0, 0, 5] = (direction / direction.norm() * 40).to(dtype)
    value[0, 0, :16] = 0.0
    value[1, 0, ::37] *= 4096.0
    cache.append(key, value)
    gpu = cache.on(cuda_device)
    rows = [cache.dense(b) for b in range(2)]
    wide = query.repeat_interleave(copies, dim=1)  # many rows
    out = anna_b200.run_q8_paged_attention(query=wide.to(cuda_device), lengths=cache.lengths.to(cuda_device), scaling=0.09, **gpu).cpu().double()
    out = out[:, ::copies]
    for b in range(2):
        score = torch.einsum("hd,nd->hn", query[b, :, 0].double(), rows[b][0, 0]) * 0.09
        weight = torch.softmax(score, dim=-1)
        want = weight @ rows[b][1, 0]
        reach = float((query[b, :, 0].double().abs() @ rows[b][0, 0].abs().T).max()) * 0.09
        # errors are relative to each weight (fp16 weights: half a step, 2^-11; those below 2^-28 of the largest lose 2^-39 of it)
        share = (2.0 * 131 * 2.0 ** -24 * reach + 2.0 ** -20 + (0 if dtype == FP32 else 2.0 ** -11)) * (weight @ rows[b][1, 0].abs())
        lost = 0.0 if dtype == FP32 else 2.0 ** -39 * weight.max() * rows[b][1, 0].abs().sum(0)
        bound = share + lost + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal
        assert bool(((out[b, :, 0] - want).abs() <= bound).all()), b


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_queries_of_any_magnitude(cuda_device, dtype):
    cache, gpu = filled(cuda_device, [100, 50], 1, 128, 16, dtype)
    info = torch.finfo(dtype)
    for top in (info.max / 4, 1.0, info.smallest_normal * 8):
        query = torch.randn((2, 4, 1, 128), generator=cache.gen).clamp(-3.9, 3.9).double() * (top / 4)
        query = query.to(dtype)
        check_attention(cache, gpu, query, cuda_device, scaling=float(0.3 / top))


def test_strides_of_query_and_gate(cuda_device):
    cache, gpu = filled(cuda_device, [70, 33], 2, 128, 16, BF16)
    wide = torch.randn((2, 3, 8, 2, 130), generator=cache.gen).to(BF16)
    query, gate = wide[:, :, :, 0, 1:129].transpose(1, 2), wide[:, :, :, 1, :128].transpose(1, 2)
    on_gpu = wide.to(cuda_device)
    kwargs = dict(lengths=cache.lengths.to(cuda_device), scaling=0.1, **gpu)
    got = anna_b200.run_q8_paged_attention(query=on_gpu[:, :, :, 0, 1:129].transpose(1, 2), gate=on_gpu[:, :, :, 1, :128].transpose(1, 2), **kwargs)
    plain = anna_b200.run_q8_paged_attention(query=query.contiguous().to(cuda_device), gate=gate.contiguous().to(cuda_device), **kwargs)
    assert torch.equal(got, plain)
    reversed_dims = query.contiguous().to(cuda_device).permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0)
    assert torch.equal(anna_b200.run_q8_paged_attention(query=reversed_dims, gate=gate.contiguous().to(cuda_device), **kwargs), plain)


# ---------------------------------------------------------------------------------------------------------------
# selection


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim,page,heads,group,tokens", [(128, 16, 2, 4, 1), (64, 8, 2, 3, 5), (256, 16, 1, 8, 2), (128, 24, 1, 20, 3), (64, 16, 1, 1, 11)])
def test_selection(cuda_device, dtype, dim, page, heads, group, tokens):
    lengths = [0, 1, page, page + 1, 21 * page + 3, 40 * page, tokens - 1, 13 * page - 1]
    cache, gpu = filled(cuda_device, lengths, heads, dim, page, dtype, seed=5)
    query = torch.randn((len(lengths), heads * group, tokens, dim), generator=cache.gen).to(dtype)
    for count, first, recent in ((2, 1, 1), (7, 1, 1), (7, 0, 0), (9, 3, 5), (64, 2, 2), (1, 0, 1)):
        got = anna_b200.run_q8_select_blocks(query=query.to(cuda_device), packed_pages=gpu["packed_pages"], page_table=gpu["page_table"],
                                             lengths=cache.lengths.to(cuda_device), block_size=page, count=count, first=first, recent=recent)
        assert got.dtype == torch.int32
        assert torch.equal(got.cpu(), selected(query, cache, count, first, recent)), (count, first, recent)


def test_selection_of_equal_scores_takes_the_first(cuda_device):
    cache = Cache(1, 1, 64, 16, BF16, 40)
    key, value = cache.new_tokens(16)
    for i in range(39):
        cache.append(key * (1.0 if i % 3 else 0.5), value)
    gpu = cache.on(cuda_device)
    query = torch.randn((1, 2, 1, 64), generator=cache.gen).to(BF16)
    zero = torch.zeros_like(query)
    for q in (query, zero):
        for count in (2, 5, 20, 30, 38, 39):
            got = anna_b200.run_q8_select_blocks(query=q.to(cuda_device), packed_pages=gpu["packed_pages"], page_table=gpu["page_table"],
                                                 lengths=cache.lengths.to(cuda_device), block_size=16, count=count).cpu()
            assert torch.equal(got, selected(q, cache, count)), count
    assert got.flatten().tolist() == list(range(39))


def test_selection_of_missing_pages_nan_pages_and_nan_queries(cuda_device):
    cache, _ = filled(cuda_device, [400, 400, 400], 1, 64, 16, FP16, seed=2)
    cache.table[0, 3], cache.table[0, 24], cache.table[1, :] = -1, 10 ** 6, -1
    size = 2 * 16 * 64
    cache.pages[int(cache.table[2, 11]), 0, size:size + 4] = torch.tensor([math.nan]).view(torch.uint8)
    gpu = cache.on(cuda_device)
    query = torch.randn((3, 2, 2, 64), generator=cache.gen).to(FP16)
    query[0, 1, 1, 5] = math.nan
    for count in (2, 4, 25, 30):
        got = anna_b200.run_q8_select_blocks(query=query.to(cuda_device), packed_pages=gpu["packed_pages"], page_table=gpu["page_table"],
                                             lengths=cache.lengths.to(cuda_device), block_size=16, count=count).cpu()
        assert torch.equal(got, selected(query, cache, count)), count
    assert not (got[1] >= 0).any() and 11 in got[2, 0, 0].tolist()


def test_selection_bounds_every_key(cuda_device):
    """A page of a key with the largest product is chosen when the bound of no other page reaches that product."""
    cache, gpu = filled(cuda_device, [640], 1, 128, 16, BF16, seed=8)
    query = torch.randn((1, 1, 1, 128), generator=cache.gen).to(BF16)
    size = 2 * 16 * 128
    bound = []
    for j in range(40):
        row = cache.pages[int(cache.table[0, j]), 0]
        codes = row[:16 * 128].view(torch.int8).view(16, 128).double()
        bounds = row[size + 16:size + 16 + 256].view(torch.int8).view(2, 128).double()
        q = query[0, 0, 0].double()
        bound.append(float((q.clamp_min(0) * bounds[0] + (-q).clamp_min(0) * bounds[1]).sum()))
        assert float((codes @ q).max()) <= bound[-1]


@pytest.mark.parametrize("blocks", [12288, 12289, 20001])
def test_selection_of_very_many_pages(cuda_device, blocks):
    """More candidates than shared memory keeps; pages shared between blocks."""
    page, dim, pages = 8, 64, 97
    cache = Cache(1, 1, dim, page, BF16, 1, seed=4)
    gen = cache.gen
    cache.pages = torch.zeros((pages, 1, cache.pages.shape[2]), dtype=torch.uint8)
    for i in range(pages):
        cache.write_page(i, torch.randn((2, 1, page, dim), generator=gen).to(BF16))
    table = torch.randint(0, pages, (1, blocks), generator=gen).int()
    n = blocks * page
    query = torch.randn((1, 1, 1, dim), generator=gen).to(BF16)
    count = 301
    got = anna_b200.run_q8_select_blocks(query=query.to(cuda_device), packed_pages=cache.pages.to(cuda_device), page_table=table.to(cuda_device),
                                         lengths=torch.tensor([n], device=cuda_device), block_size=page, count=count).cpu()
    cache.table = torch.arange(pages).int().view(1, pages)
    cache.tokens = [torch.zeros((2, 1, pages * page, dim))]
    size = 2 * page * dim
    q = query[0, 0, 0].double().numpy()
    whole = np.rint(q * 32767.0 / np.abs(q).max()).astype(np.int64)
    rows = cache.pages[:, 0]
    bounds = rows[:, size + 16:size + 16 + 2 * dim].contiguous().view(torch.int8).numpy().astype(np.int64)
    total = bounds[:, :dim] @ np.maximum(whole, 0) + bounds[:, dim:] @ np.maximum(-whole, 0)
    scale = rows[:, size:size + 4].contiguous().view(torch.float32).numpy()[:, 0]
    score = (np.float32(np.abs(q).max()) * scale * total.astype(np.float32))[table[0].numpy()]
    score[[0, blocks - 1]] = np.inf
    want = np.sort(np.argsort(-score, kind="stable")[:count])
    assert got.flatten().tolist() == want.tolist()


def test_candidates_of_the_restatement():
    assert [candidates(33, 2, t, 16) for t in range(2)] == [2, 2] and candidates(33, 18, 0, 16) == 1 and candidates(3, 5, 0, 16) == 0
    codes, scale = quantized(torch.tensor([[[1.0, -2.0]]]))
    assert codes.flatten().tolist() == [64, -127] and math.isclose(float(scale), 2 / 127, rel_tol=1e-7)


# ---------------------------------------------------------------------------------------------------------------
# together


@pytest.mark.parametrize("dtype,dim,page", [(BF16, 128, 16), (FP16, 256, 32), (FP32, 64, 16)])
def test_a_prompt_forks_and_goes_on(cuda_device, dtype, dim, page):
    """A prompt is appended, attended through the dense view's contents, forked by page copies, and both rows go on with chosen pages."""
    cache = Cache(2, 2, dim, page, dtype, 12)
    gpu = cache.on(cuda_device)
    prompt = 6 * page + 5
    key, value = cache.new_tokens(prompt)
    key[1], value[1] = key[0], value[0]
    past = torch.zeros(2, dtype=torch.long, device=cuda_device)
    one = {k: gpu[k][:1] if k in ("page_table", "window_slots") else gpu[k] for k in gpu}
    anna_b200.run_q8_append(key=key[:1].to(cuda_device), value=value[:1].to(cuda_device), past_lengths=past[:1], **one)
    # row 1 becomes a fork of row 0: its full pages are row 0's, its ring a copy
    gpu["page_table"][1, :6] = gpu["page_table"][0, :6]
    cache.table[1, :6] = cache.table[0, :6]
    anna_b200.run_page_copy(copies=[(gpu["window"], [int(cache.slots[0])], [int(cache.slots[1])])])
    cache.append(key, value)
    lengths = past + prompt
    for step in range(page + 3):
        key, value = cache.new_tokens(1)
        after = torch.empty_like(lengths)
        anna_b200.run_q8_append(key=key.to(cuda_device), value=value.to(cuda_device), past_lengths=lengths, new_lengths=after, **gpu)
        cache.append(key, value)
        lengths = after
        if step % 6:
            continue
        query = torch.randn((2, 8, 1, dim), generator=cache.gen).to(dtype)
        check_attention(cache, gpu, query, cuda_device)
        blocks = anna_b200.run_q8_select_blocks(query=query.to(cuda_device), packed_pages=gpu["packed_pages"], page_table=gpu["page_table"],
                                                lengths=lengths, block_size=page, count=3).cpu()
        assert torch.equal(blocks, selected(query, cache, 3))
        check_attention(cache, gpu, query, cuda_device, blocks=blocks)
    check_same(cache, gpu)


def test_steps_in_a_graph_and_on_another_stream(cuda_device):
    """A captured step (append, selection, attention) that is replayed while lengths go on, beside eager calls on another stream."""
    cache = Cache(2, 2, 128, 16, BF16, 12)
    key, value = cache.new_tokens(50)
    cache.append(key, value)
    gpu = cache.on(cuda_device)
    lengths, after = cache.lengths.to(cuda_device), cache.lengths.to(cuda_device)
    static = [torch.zeros((2, 2, 1, 128), dtype=BF16, device=cuda_device) for _ in range(2)]
    query = torch.randn((2, 8, 1, 128), generator=cache.gen).to(BF16)
    static_query = query.to(cuda_device)

    def step():
        anna_b200.run_q8_append(key=static[0], value=static[1], past_lengths=lengths, new_lengths=after, **gpu)
        blocks = anna_b200.run_q8_select_blocks(query=static_query, packed_pages=gpu["packed_pages"], page_table=gpu["page_table"], lengths=after,
                                                block_size=16, count=2)
        dense = anna_b200.run_q8_paged_attention(query=static_query, lengths=after, scaling=0.09, **gpu)
        sparse = anna_b200.run_q8_paged_attention(query=static_query, lengths=after, scaling=0.09, blocks=blocks, **gpu)
        lengths.copy_(after)
        return blocks, dense, sparse

    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    saved = {k: v.clone() for k, v in gpu.items()}
    start = lengths.clone()
    with torch.cuda.stream(other):
        step()
    torch.cuda.current_stream().wait_stream(other)
    for k in saved:
        gpu[k].copy_(saved[k])
    lengths.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        blocks, dense, sparse = step()
    for k in saved:
        gpu[k].copy_(saved[k])
    lengths.copy_(start)
    for _ in range(20):
        key, value = cache.new_tokens(1)
        static[0].copy_(key)
        static[1].copy_(value)
        graph.replay()
        cache.append(key, value)
        with torch.cuda.stream(other):  # the same kernels on another stream, in scratch of their own
            other.wait_stream(torch.cuda.current_stream())
            eager = anna_b200.run_q8_paged_attention(query=static_query, lengths=after, scaling=0.09, **gpu)
        torch.cuda.current_stream().wait_stream(other)
        rows = [cache.dense(b) for b in range(2)]
        for got, chosen in ((dense, None), (eager, None), (sparse, blocks.cpu())):
            want, reach, most = attention(query, rows, 0.09, None, 16, chosen)
            assert bool(((got.cpu().double() - want).abs() <= attention_bound(want, BF16, 128, reach, most)).all())
        assert torch.equal(blocks.cpu(), selected(query, cache, 2))
    check_same(cache, gpu)
