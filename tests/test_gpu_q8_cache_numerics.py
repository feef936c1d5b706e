"""Attention over the 8-bit paged cache where its numbers come close to the ends of their formats, against a restatement in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import anna_b200
from q8_reference import Cache, attention, quantized
from test_gpu_q8_cache import BF16, FP16, FP32, check_attention, filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,group,tokens", [(16, 1, 1), (24, 3, 2), (32, 12, 2), (5, 2, 1)])
def test_fp32_queries_just_below_a_power_of_two(cuda_device, dim, page, group, tokens):
    """Largest magnitudes of which all 24 bits are set, of either sign."""
    lengths = [3 * page + 2, page, 7 * page + 1]
    cache, gpu = filled(cuda_device, lengths, 2, dim, page, FP32, seed=dim + page)
    for power in (0.5, 1.0, 2.0, 2.0 ** 40):
        top = torch.nextafter(torch.tensor(power), torch.tensor(0.0))
        query = (2.0 * torch.rand((3, 2 * group, tokens, dim), generator=cache.gen) - 1.0) * top
        for entry, sign in ((0, 1.0), (7, -1.0), (dim // 2 + 5, 1.0), (dim - 1, -1.0)):
            query[..., entry] = sign * top
        query[1] = top  # nothing else
        query[2, 0] = -top
        check_attention(cache, gpu, query, cuda_device, scaling=0.3 / power)
        blocks = torch.randint(0, 7, (3, 2, tokens, 3), generator=cache.gen).int()
        check_attention(cache, gpu, query, cuda_device, blocks=blocks, scaling=0.3 / power)


@pytest.mark.parametrize("dim,page,group,tokens", [(64, 16, 1, 1), (128, 16, 4, 1), (128, 24, 2, 2), (256, 32, 8, 2), (128, 16, 8, 4), (128, 5, 2, 1)])
@pytest.mark.parametrize("ring", [0, 3])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_weights_of_16_bit_caches_leave_the_rounding_to_the_output(cuda_device, dtype, dim, page, group, tokens, ring):
    """Values that nearly cancel, so that an output shows what its weights are off by."""
    lengths = [4 * page + ring, page + ring]
    cache = Cache(2, 2, dim, page, dtype, 5, seed=dim + ring)
    key, value = cache.new_tokens(max(lengths), spread=0.05)
    value = torch.where(torch.arange(max(lengths))[:, None] % 2 == 0, 1.0, -1.0) * (1.0 + value.float().abs())
    for b, n in enumerate(lengths):
        cache.append(key[:, :, :n], value[:, :, :n].to(dtype), rows=[b])
    gpu = cache.on(cuda_device)
    query = torch.randn((2, 2 * group, tokens, dim), generator=cache.gen).to(dtype)
    scaling = dim ** -0.5
    out = anna_b200.run_q8_paged_attention(query=query.to(cuda_device), lengths=cache.lengths.to(cuda_device), scaling=scaling, **gpu).cpu().double()
    want, reach, most = attention(query, [cache.dense(b) for b in range(2)], scaling)
    # as for fp32 caches (scores and sums in 32 bits), but a weight is a sum of two fp16, for tokens of the ring of two numbers of the type: off by
    # half a step of the second, 2^-11 of at most 2^-11 of it (bf16: 2^-8 of 2^-8)
    share = 2.0 ** -22 if dtype == FP16 or ring == 0 else 2.0 ** -16
    bound = most * (2.0 * (dim + 3) * 2.0 ** -24 * reach + 2.0 ** -20 + share) + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal
    assert bool(((out - want).abs() <= bound).all()), float(((out - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("page,pages,copies", [(16, 4, 1), (24, 4, 1), (5, 4, 1), (16, 4, 9), (16, 130, 1), (5, 300, 1)])
def test_what_a_query_sees_shows_however_small_its_weight(cuda_device, dtype, page, pages, copies):
    """A NaN among the values of a page or of the ring, and an infinity there, under a key that takes all weight."""
    dim, extra = 64, 3
    n = page * pages + extra
    cache = Cache(4, 1, dim, page, dtype, pages)
    key, value = cache.new_tokens(n, spread=0.1)
    key[:, 0, :, 0] = 0.0
    key[:, 0, n - 1, 0] = 100.0  # a score of 1000
    value[0, 0, 2, 7] = math.nan       # in the first page: all of its values are NaN
    value[1, 0, n - 2, 7] = math.nan   # in the ring
    value[2, 0, n - 2, 9] = -math.inf
    cache.append(key, value)
    gpu = cache.on(cuda_device)
    query = torch.zeros((4, 2 * copies, 1, dim), dtype=dtype)
    query[..., 0] = 10.0
    out = anna_b200.run_q8_paged_attention(query=query.to(cuda_device), lengths=cache.lengths.to(cuda_device), scaling=1.0, **gpu).cpu()
    assert bool(torch.isnan(out[0]).all())
    assert bool(torch.isnan(out[1, ..., 7]).all()) and bool(torch.isfinite(out[1, ..., torch.arange(dim) != 7]).all())
    assert not bool(torch.isfinite(out[2, ..., 9]).any()) and bool(torch.isfinite(out[2, ..., torch.arange(dim) != 9]).all())
    assert torch.equal(out[3], value[3, :, n - 1:].expand(2 * copies, 1, dim))
    # the same tokens behind the queries' own are not seen
    query = torch.cat((query, query), dim=2)
    out = anna_b200.run_q8_paged_attention(query=query.to(cuda_device), lengths=(cache.lengths - 1).to(cuda_device), scaling=1.0, **gpu).cpu()
    assert bool(torch.isfinite(out[1:3, :, 0]).all()) and not bool(torch.isfinite(out[1, :, 1, 7]).any()) and not bool(torch.isfinite(out[2, :, 1, 9]).any())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("ratio", [63.0, 65.0])
@pytest.mark.parametrize("copies", [1, 10])
def test_small_weights_of_pages_with_small_scales(cuda_device, dtype, ratio, copies):
    """A page with much larger values, of which a query sees a key that takes nearly all weight and has no value; what pages with scales just within and just
    past 2^6 of it add, at weights of 2^-20 to 2^-30."""
    page, dim, blocks = 16, 128, 40
    cache = Cache(2, 1, dim, page, dtype, blocks)
    key, value = cache.new_tokens(page * blocks)
    query = torch.zeros((2, 4, 1, dim), dtype=dtype)
    query[..., 0] = 1.0
    scaling = math.log(2.0)
    key *= 0.25
    key[..., 0] = torch.randint(-30, -19, key.shape[:3], generator=cache.gen).to(dtype)  # log2 of a weight
    value[:, :, page:] = 512.0 * value[:, :, page:].clamp(-1.0, 1.0)
    value[:, :, page::page, 0] = 512.0       # the scale is 512 / 127
    value[:, :, :page] *= 0.0
    value[:, :, 1, 0] = 512.0 * ratio        # a large value at a small weight
    key[:, :, :page, 0] = -30.0
    key[:, :, 5, 0] = 0.0
    cache.append(key, value)
    gpu = cache.on(cuda_device)
    rows = [cache.dense(b) for b in range(2)]
    wide = query.repeat_interleave(copies, dim=1)
    out = anna_b200.run_q8_paged_attention(query=wide.to(cuda_device), lengths=cache.lengths.to(cuda_device), scaling=scaling, **gpu).cpu().double()
    for b in range(2):
        score = torch.einsum("hd,nd->hn", query[b, :, 0].double(), rows[b][0, 0]) * scaling
        weight = torch.softmax(score, dim=-1)
        want = (weight @ rows[b][1, 0]).repeat_interleave(copies, dim=0)
        reach = float(score.abs().max())
        share = (2.0 * (dim + 3) * 2.0 ** -24 * reach + 2.0 ** -20 + 2.0 ** -22) * (weight @ rows[b][1, 0].abs())
        # A weight, times the scale of its page in units of at most twice the largest scale, is rounded to a multiple of 2^-24, of which the largest weight has
        # 2^14 or more: it loses 2^-39 of that at most, and is there for a code.
        codes = torch.cat([quantized(cache.tokens[b][1, :, j * page:(j + 1) * page])[0][0] for j in range(blocks)]).double()
        scale = torch.cat([quantized(cache.tokens[b][1, :, j * page:(j + 1) * page])[1] for j in range(blocks)]).double()
        lost = 2.0 ** -39 * weight.amax() * 2.0 * scale.max() * codes.abs().sum(0)
        bound = (share + lost).repeat_interleave(copies, dim=0) + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert bool(((out[b, :, 0] - want).abs() <= bound).all()), (b, float(((out[b, :, 0] - want).abs() / bound).max()))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim,group", [(128, 4), (256, 20), (128, 20), (64, 9), (128, 33), (256, 3)])
def test_outputs_do_not_depend_on_what_calls_before_left_behind(cuda_device, dtype, dim, group):
    """The same call again after others have left pages where its tiles have no rows: as numbers of the type some 2^127, whose products with keys are infinite
    or, with keys of zero, are not.  Scores of a warp's second tile are above those of its first by less than 1 (in powers of two), where the running maximum may
    stay or be raised."""
    page, heads = 128, 40
    lengths = [79, 127, 80]
    cache = Cache(3, heads, dim, page, dtype, 2)
    key, value = cache.new_tokens(127)
    key = torch.where(torch.arange(127)[:, None] < 16, -4.0 - key.float() / 2, 0.0).to(dtype)
    for b, n in enumerate(lengths):
        cache.append(key[:, :, :n], value[:, :, :n], rows=[b])
    gpu = cache.on(cuda_device)
    past = cache.lengths.to(cuda_device)
    query = (1.0 + torch.randn((3, heads * group, 1, dim), generator=cache.gen) / 16).to(dtype).to(cuda_device)
    other = Cache(4, heads, 64, 16, dtype, 40)
    size = 2 * 16 * 64
    pages = torch.tensor([0, 0x7f], dtype=torch.uint8).repeat(other.pages.shape[2] // 2).expand(other.pages.shape).contiguous()
    pages[:, :, size:size + 8] = torch.ones((pages.shape[0], heads, 2)).view(torch.uint8)
    left = dict(other.on(cuda_device), packed_pages=pages.to(cuda_device))
    plain = dict(left, packed_pages=torch.zeros_like(left["packed_pages"]))
    n = torch.full((4,), 640, dtype=torch.long, device=cuda_device)
    results = []
    for tensors in (plain, left, plain, left):
        for other_group in (1, 8):
            noise = torch.randn((4, heads * other_group, 1, 64), generator=cache.gen).to(dtype).to(cuda_device)
            anna_b200.run_q8_paged_attention(query=noise, lengths=n, scaling=0.01, **tensors)
        results.append(anna_b200.run_q8_paged_attention(query=query, lengths=past, scaling=0.5 * math.log(2.0) / (4 * dim), **gpu))
    for got in results[1:]:
        assert int((got != results[0]).sum()) == 0


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("dim,page,group", [(64, 16, 1), (128, 24, 4), (256, 32, 10), (128, 5, 2)])
@pytest.mark.parametrize("power", [-120, -108, 100, 116])
def test_tiny_queries_of_huge_keys_and_huge_ones_of_tiny(cuda_device, dtype, dim, page, group, power):
    """Scores of ordinary size from factors near the ends of the type."""
    lengths = [3 * page + 3, 2 * page]
    cache = Cache(2, 2, dim, page, dtype, 4, seed=dim)
    key, value = cache.new_tokens(max(lengths))
    key = (key.double() * 2.0 ** (-4 - power)).to(dtype)
    for b, n in enumerate(lengths):
        cache.append(key[:, :, :n], value[:, :, :n], rows=[b])
    query = (torch.randn((2, 2 * group, 1, dim), generator=cache.gen).double() * 2.0 ** (power + 4)).to(dtype)
    check_attention(cache, cache.on(cuda_device), query, cuda_device)
