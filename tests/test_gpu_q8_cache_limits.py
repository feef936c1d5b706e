"""The 8-bit paged cache at the ends of what it takes: many rows, heads and pages, a pool past 32 bits, no pool, calls at once."""
from __future__ import annotations

import threading

import pytest
import torch

import anna_b200
from q8_reference import Cache, attention, attention_bound, selected
from test_gpu_q8_cache import BF16, FP16, FP32, check_attention, check_same, filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim,page,group,tokens", [(64, 24, 4, 2), (128, 16, 4, 2), (128, 8, 7, 1), (256, 32, 2, 3), (256, 24, 8, 1), (64, 5, 3, 2)])
def test_attention_of_many_tiles(cuda_device, dtype, dim, page, group, tokens):
    """Enough rows that CTAs share an SM."""
    gen = torch.Generator().manual_seed(dim + page)
    lengths = torch.randint(0, 6 * page, (80,), generator=gen).tolist()
    cache, gpu = filled(cuda_device, lengths, 2, dim, page, dtype, seed=7)
    query = torch.randn((80, 2 * group, tokens, dim), generator=gen).to(dtype)
    check_attention(cache, gpu, query, cuda_device)
    width = 24 if page < 16 else 12
    check_attention(cache, gpu, query, cuda_device, blocks=torch.randint(-1, 7, (80, 2, tokens, width), generator=gen).int())


@pytest.mark.parametrize("dtype,page", [(BF16, 16), (FP16, 8), (FP32, 32), (BF16, 5)])
@pytest.mark.parametrize("pages", [0, 3])
def test_a_table_without_columns(cuda_device, dtype, page, pages):
    """Rows that have not filled a page, no table and no pool yet: all calls go by the ring."""
    lengths = [page - 1, 0, 3]
    cache = Cache(3, 2, 64, page, dtype, 0)
    cache.pages = torch.zeros((pages,) + cache.pages.shape[1:], dtype=torch.uint8)
    cache.table = torch.zeros((3, 0), dtype=torch.int32)
    gpu = cache.on(cuda_device)
    key, value = cache.new_tokens(page)
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        one = dict(gpu, page_table=gpu["page_table"][b:b + 1], window_slots=gpu["window_slots"][b:b + 1])
        anna_b200.run_q8_append(key=key[b:b + 1, :, :n].to(cuda_device), value=value[b:b + 1, :, :n].to(cuda_device),
                                past_lengths=torch.zeros(1, dtype=torch.long, device=cuda_device), **one)
        cache.append(key[:, :, :n], value[:, :, :n], rows=[b])
    check_same(cache, gpu)
    query = torch.randn((3, 8, 2, 64), generator=cache.gen).to(dtype)
    blocks = anna_b200.run_q8_select_blocks(query=query.to(cuda_device), packed_pages=gpu["packed_pages"], page_table=gpu["page_table"],
                                            lengths=cache.lengths.to(cuda_device), block_size=page, count=40).cpu()
    assert bool((blocks == -1).all())
    plain = check_attention(cache, gpu, query, cuda_device)
    assert torch.equal(check_attention(cache, gpu, query, cuda_device, blocks=blocks), plain)
    check_attention(cache, gpu, query, cuda_device, blocks=torch.randint(-2, 9, (3, 2, 2, 5), generator=cache.gen).int())
    dense = anna_b200.run_q8_gather(lengths=cache.lengths.to(cuda_device), max_len=page, **gpu)
    for b, n in enumerate(lengths):
        for which in range(2):
            assert torch.equal(dense[which][b, :, :n].cpu().double(), cache.dense(b)[which]) and not dense[which][b, :, n:].any()


def test_no_tokens_and_no_rows(cuda_device):
    cache, gpu = filled(cuda_device, [20, 3], 2, 64, 16, BF16)
    before = gpu["window"].clone()
    past, after = cache.lengths.to(cuda_device), torch.zeros(2, dtype=torch.long, device=cuda_device)
    none = torch.empty((2, 2, 0, 64), dtype=BF16, device=cuda_device)
    anna_b200.run_q8_append(key=none, value=none, past_lengths=past, new_lengths=after, **gpu)
    assert torch.equal(after, past) and torch.equal(before.view(torch.uint8), gpu["window"].view(torch.uint8))
    query = torch.empty((2, 8, 0, 64), dtype=BF16, device=cuda_device)
    assert anna_b200.run_q8_paged_attention(query=query, lengths=past, scaling=1.0, **gpu).shape == (2, 8, 0, 64)
    empty = dict(gpu, page_table=gpu["page_table"][:0], window_slots=gpu["window_slots"][:0])
    assert anna_b200.run_q8_paged_attention(query=query.new_empty((0, 8, 1, 64)), lengths=past[:0], scaling=1.0, **empty).shape == (0, 8, 1, 64)
    assert anna_b200.run_q8_select_blocks(query=query.new_empty((0, 8, 1, 64)), packed_pages=gpu["packed_pages"], page_table=empty["page_table"],
                                          lengths=past[:0], block_size=16, count=3).shape == (0, 2, 1, 3)
    assert anna_b200.run_q8_gather(lengths=past[:0], max_len=5, **empty)[0].shape == (0, 2, 5, 64)
    assert anna_b200.run_q8_gather(lengths=past, max_len=0, **gpu)[1].shape == (2, 2, 0, 64)


def test_a_pool_past_32_bits(cuda_device):
    """The last pages of a pool of more than 2^32 bytes, written and read."""
    heads, dim, page = 2, 128, 16
    cache = Cache(2, heads, dim, page, BF16, 4, seed=2)
    size = cache.pages.shape[2]
    pages = (2 ** 32 + 2 ** 28) // (heads * size)
    pool = torch.empty((pages, heads, size), dtype=torch.uint8, device=cuda_device)
    gpu = cache.on(cuda_device)
    table = (pages - 1 - torch.arange(8).view(2, 4) * 3).int()
    gpu.update(packed_pages=pool, page_table=table.to(cuda_device))
    key, value = cache.new_tokens(4 * page - 3)
    anna_b200.run_q8_append(key=key.to(cuda_device), value=value.to(cuda_device), past_lengths=torch.zeros(2, dtype=torch.long, device=cuda_device), **gpu)
    cache.append(key, value)
    query = torch.randn((2, 8, 1, dim), generator=cache.gen).to(BF16)
    check_attention(cache, gpu, query, cuda_device)
    blocks = anna_b200.run_q8_select_blocks(query=query.to(cuda_device), packed_pages=pool, page_table=gpu["page_table"],
                                            lengths=cache.lengths.to(cuda_device), block_size=page, count=2).cpu()
    assert torch.equal(blocks, selected(query, cache, 2))
    check_attention(cache, gpu, query, cuda_device, blocks=blocks)
    dense = anna_b200.run_q8_gather(lengths=cache.lengths.to(cuda_device), max_len=3 * page, **gpu)
    for b in range(2):
        for which in range(2):
            assert torch.equal(dense[which][b].cpu(), cache.dense(b)[which, :, :3 * page].to(BF16))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("blocks", [65536, 200001])
def test_very_long_rows(cuda_device, dtype, blocks):
    """A row of millions of tokens, whose table names few pages many times: each counts as often as it is named."""
    dim, page, pages = 64, 16, 31
    cache = Cache(1, 1, dim, page, dtype, pages, seed=6)
    key, value = cache.new_tokens(pages * page)
    cache.append(key, value)
    gpu = cache.on(cuda_device)
    gen = cache.gen
    names = torch.randint(0, pages, (blocks,), generator=gen)
    gpu["page_table"] = gpu["page_table"][:, names.to(cuda_device)].contiguous()
    query = torch.randn((1, 4, 1, dim), generator=gen).to(dtype)
    got = anna_b200.run_q8_paged_attention(query=query.to(cuda_device), lengths=torch.tensor([blocks * page], device=cuda_device), scaling=0.125, **gpu)
    dense = cache.dense(0)
    times = torch.bincount(names, minlength=pages).double().repeat_interleave(page)
    keys, values = dense[0, 0], dense[1, 0]
    q = query[0, :, 0].double()
    score = q @ keys.T * 0.125
    weight = torch.exp(score - score.max()) * times
    want = (weight / weight.sum(1, keepdim=True)) @ values
    reach, most = float((q.abs() @ keys.abs().T).max()) * 0.125, float(values.abs().max())
    # Sums in 32 bits: a CTA has at least 1 / 254 of the row, 800 tiles, as no more partials are merged; were it twice that, in turns of four warps, a
    # warp adds 400 tiles to its sums and 800 weights to its denominator, and the merge 254 partials to both, each off by 2^-24 of the largest
    # value, products of tensor cores by 2^-23: 2 * 400 + 800 + 2 * 254 is under 2^11.
    bound = attention_bound(want, dtype, dim, reach, most) + 2.0 ** -13 * most
    assert bool(((got[0, :, 0].cpu().double() - want).abs() <= bound).all())


def test_selection_of_many_rows_heads_and_groups(cuda_device):
    gen = torch.Generator().manual_seed(3)
    for rows, heads, group, dim, dtype, count in ((1100, 1, 2, 64, BF16, 2), (6, 12, 4, 128, FP16, 5), (3, 9, 1, 64, BF16, 3), (2, 1, 72, 256, BF16, 4),
                                                  (40, 10, 3, 64, FP32, 2)):
        lengths = torch.randint(0, 100, (rows,), generator=gen).tolist()
        cache, gpu = filled(cuda_device, lengths, heads, dim, 8, dtype, seed=rows)
        query = torch.randn((rows, heads * group, 1, dim), generator=gen).to(dtype)
        # a wide table of which little is used: what a CTA takes follows from its columns
        for columns in (0, 3000):
            table = torch.cat((cache.table, torch.full((rows, columns), -1, dtype=torch.int32)), dim=1)
            got = anna_b200.run_q8_select_blocks(query=query.to(cuda_device), packed_pages=gpu["packed_pages"], page_table=table.to(cuda_device),
                                                 lengths=cache.lengths.to(cuda_device), block_size=8, count=count)
            assert torch.equal(got.cpu(), selected(query, cache, count)), (rows, heads, columns)


def test_more_groups_than_the_selection_takes_are_refused(cuda_device):
    cache, gpu = filled(cuda_device, [40], 1, 256, 16, BF16)
    query = torch.zeros((1, 512, 1, 256), dtype=BF16, device=cuda_device)
    with pytest.raises(RuntimeError, match="too many query heads"):
        anna_b200.run_q8_select_blocks(query=query, packed_pages=gpu["packed_pages"], page_table=gpu["page_table"],
                                       lengths=cache.lengths.to(cuda_device), block_size=16, count=2)


def test_one_table_for_all_rows_and_gaps_in_row_numbers(cuda_device):
    """A table that is expanded from one row, slots and lengths with strides."""
    cache, gpu = filled(cuda_device, [16 * 5, 16 * 5], 2, 64, 16, BF16)
    cache.table[1] = cache.table[0]
    cache.tokens[1] = cache.tokens[0]
    gpu["page_table"] = gpu["page_table"][:1].expand(2, -1)
    wide = torch.zeros((2, 2), dtype=torch.long, device=cuda_device)
    wide[:, 0] = cache.slots.to(cuda_device)
    gpu["window_slots"] = wide[:, 0]
    query = torch.randn((2, 4, 1, 64), generator=cache.gen).to(BF16)
    check_attention(cache, gpu, query, cuda_device)
    blocks = anna_b200.run_q8_select_blocks(query=query.to(cuda_device), packed_pages=gpu["packed_pages"], page_table=gpu["page_table"],
                                            lengths=cache.lengths.to(cuda_device), block_size=16, count=3).cpu()
    assert torch.equal(blocks, selected(query, cache, 3))
    key = torch.randn((1, 2, 1, 64), generator=cache.gen).to(BF16)
    anna_b200.run_q8_append(key=key.to(cuda_device).expand(2, 2, 1, 64), value=key.to(cuda_device).expand(2, 2, 1, 64),
                            past_lengths=cache.lengths.to(cuda_device), **gpu)
    cache.append(key.expand(2, 2, 1, 64), key.expand(2, 2, 1, 64))
    check_attention(cache, gpu, query, cuda_device)


def test_lengths_behind_the_largest_are_left_out(cuda_device):
    cache, gpu = filled(cuda_device, [10, 20, 30], 1, 64, 16, BF16)
    before = {k: v.clone() for k, v in gpu.items()}
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    past = torch.tensor([2 ** 30 - 2, 2 ** 40, -5], device=cuda_device)
    after = torch.zeros_like(past)
    fresh = torch.ones((3, 1, 2, 64), dtype=BF16, device=cuda_device)
    anna_b200.run_q8_append(key=fresh, value=fresh, past_lengths=past, new_lengths=after, status=status, **gpu)
    assert int(status) & 1 and torch.equal(after, past + 2)
    assert torch.equal(before["window"].view(torch.uint8), gpu["window"].view(torch.uint8)) and torch.equal(before["packed_pages"], gpu["packed_pages"])


def test_two_graphs_and_two_threads_at_once(cuda_device):
    """Steps of two caches, captured and eager, on streams of their own at the same time."""
    made, graphs = [], []
    for seed in range(2):
        cache, gpu = filled(cuda_device, [700, 90], 2, 128, 16, BF16, seed=seed)
        query = torch.randn((2, 8, 1, 128), generator=cache.gen).to(BF16)
        want, reach, most = attention(query, [cache.dense(b) for b in range(2)], 0.1, None)
        chosen = selected(query, cache, 5)
        made.append((cache, gpu, query.to(cuda_device), cache.lengths.to(cuda_device), want, attention_bound(want, BF16, 128, reach, most), chosen))

    def step(k):
        _, gpu, query, lengths, _, _, _ = made[k]
        blocks = anna_b200.run_q8_select_blocks(query=query, packed_pages=gpu["packed_pages"], page_table=gpu["page_table"], lengths=lengths,
                                                block_size=16, count=5)
        return anna_b200.run_q8_paged_attention(query=query, lengths=lengths, scaling=0.1, **gpu), blocks

    def fine(k, out, blocks):
        return bool(((out.cpu().double() - made[k][4]).abs() <= made[k][5]).all()) and torch.equal(blocks.cpu(), made[k][6])

    streams = [torch.cuda.Stream() for _ in range(2)]
    for k in range(2):
        step(k)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[k]):
            held = step(k)
        graphs.append((graph, held))
    torch.cuda.synchronize()
    for _ in range(50):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k][0].replay()
    torch.cuda.synchronize()
    for k in range(2):
        assert fine(k, *graphs[k][1])

    results, failures = [None, None], []

    def work(k):
        try:
            with torch.cuda.stream(streams[k]):
                for _ in range(50):
                    results[k] = step(k)
            streams[k].synchronize()
        except Exception as error:  # shown below
            failures.append(error)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures
    for k in range(2):
        assert fine(k, *results[k])
