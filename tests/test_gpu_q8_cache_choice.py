"""The choice of pages of the 8-bit cache at every width of the table, among many equal scores, and as a bound on what the pages hold."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import anna_b200
from q8_reference import Cache
from test_gpu_q8_cache import BF16, FP16, FP32

pytestmark = pytest.mark.gpu


def page_scores(cache: Cache, query: torch.Tensor) -> np.ndarray:
    """Score of every page of the pool, float32 [kv_heads, pages], for query [q_heads, dim]."""
    heads, dim, size = cache.heads, cache.dim, 2 * cache.page * cache.dim
    out = np.full((heads, cache.pages.shape[0]), -np.inf, dtype=np.float32)
    for h in range(heads):
        rows = cache.pages[:, h].contiguous()
        bounds = rows[:, size + 16:size + 16 + 2 * dim].contiguous().view(torch.int8).numpy().astype(np.int64)
        scale = rows[:, size:size + 4].contiguous().view(torch.float32).numpy()[:, 0]
        for q in query.view(heads, -1, dim)[h].double().numpy():
            top = np.abs(q).max()
            whole = np.rint(q * 32767.0 / (top if top > 0 else 1.0)).astype(np.int64)
            total = bounds[:, :dim] @ np.maximum(whole, 0) + bounds[:, dim:] @ np.maximum(-whole, 0)
            out[h] = np.maximum(out[h], np.float32(top) * scale * total.astype(np.float32))
    return out


def best(score: np.ndarray, count: int, first: int, recent: int) -> list[int]:
    score = score.copy()
    score[:first] = np.inf
    score[max(0, len(score) - recent):] = np.inf
    chosen = np.sort(np.argsort(-score, kind="stable")[:count]).tolist()
    return chosen + [-1] * (count - len(chosen))


@pytest.mark.parametrize("spread", ["alike", "apart", "equal"])
@pytest.mark.parametrize("columns", [1024, 1025, 2048, 2049, 4096, 4097, 8191, 8192, 8193, 16384, 16385])
def test_choice_at_every_width(cuda_device, columns, spread):
    """Full tables of both sides of every width at which the kernel holds scores another way, and rows that fill them in part.  A few pages are named
    over and over, so that scores are shared by many blocks and counts end among equal ones.  `apart`: scales over many powers of two."""
    pages, heads, page, dim = 61, 2, 8, 64
    cache = Cache(1, heads, dim, page, BF16, 1, seed=columns)
    gen = cache.gen
    cache.pages = torch.zeros((pages, heads, cache.pages.shape[2]), dtype=torch.uint8)
    for i in range(pages):
        factor = {"alike": 1.0 + i / 4096, "apart": 2.0 ** (i % 41 - 20), "equal": 1.0}[spread]
        x = torch.randn((2, heads, page, dim), generator=gen) if spread != "equal" or i == 0 else x
        cache.write_page(i, (x * factor).to(BF16))
    table = torch.randint(0, pages, (3, columns), generator=gen).int()
    lengths = [columns * page, columns * page - 1, columns * page * 5 // 8 + 3]
    query = torch.randn((3, 2 * heads, 1, dim), generator=gen).to(BF16)
    scores = [page_scores(cache, query[b, :, 0]) for b in range(3)]
    for count, first, recent in ((1, 0, 0), (2, 1, 1), (33, 1, 1), (columns // 7, 5, 40), (columns // 2 + 1, 0, 3), (columns - 1, 1, 0), (columns, 1, 1),
                                 (columns + 30, 0, 0)):
        got = anna_b200.run_q8_select_blocks(query=query.to(cuda_device), packed_pages=cache.pages.to(cuda_device), page_table=table.to(cuda_device),
                                             lengths=torch.tensor(lengths, device=cuda_device), block_size=page, count=count, first=first,
                                             recent=recent).cpu()
        for b in range(3):
            for h in range(heads):
                score = scores[b][h][table[b, :lengths[b] // page].numpy()]
                assert got[b, h, 0].tolist() == best(score, count, first, recent), (count, b, h)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 4), (256, 2)])
def test_the_page_of_the_largest_product_is_chosen(cuda_device, dtype, dim, group):
    """Pages as the append writes them: their bounds hold for all of their keys, and a page with a key whose product no other page's bound reaches is the
    first that is chosen."""
    page, blocks = 16, 40
    cache = Cache(1, 1, dim, page, dtype, blocks, seed=dim)
    gpu = cache.on(cuda_device)
    key, value = cache.new_tokens(page * blocks)
    query = torch.randn((1, group, blocks, dim), generator=cache.gen).to(dtype)
    targets = torch.randperm(blocks, generator=cache.gen)[:8].tolist()
    for i, j in enumerate(targets):  # the key that query i looks for
        key[0, 0, j * page + i] = 6.0 * query[0, i % group, i]
    anna_b200.run_q8_append(key=key.to(cuda_device), value=value.to(cuda_device), past_lengths=torch.zeros(1, dtype=torch.long, device=cuda_device), **gpu)
    size = 2 * page * dim
    rows = gpu["packed_pages"].cpu()[cache.table[0].long(), 0]
    codes = rows[:, :page * dim].contiguous().view(torch.int8).view(blocks, page, dim).double()
    scale = rows[:, size:size + 4].contiguous().view(torch.float32).double()  # [blocks, 1]
    bounds = rows[:, size + 16:size + 16 + 2 * dim].contiguous().view(torch.int8).view(blocks, 2, dim).double()
    assert torch.equal(bounds[:, 0], codes.amax(1)) and torch.equal(bounds[:, 1], (-codes).amax(1))
    for i, j in enumerate(targets):
        q = query[0, :, i].double()
        product = torch.einsum("gd,bsd->gbs", q, codes).amax(2) * scale.T
        reach = (q.clamp_min(0) @ bounds[:, 0].T + (-q).clamp_min(0) @ bounds[:, 1].T) * scale.T  # [group, blocks]
        assert bool((product <= reach).all())
        others = reach.amax(0)
        others[j] = -1.0
        # queries in whole numbers are off by half of 1 / 32767 of the largest entry
        assert float(product[:, j].max()) > 1.01 * float(others.max())
        got = anna_b200.run_q8_select_blocks(query=query[:, :, i:i + 1].to(cuda_device), packed_pages=gpu["packed_pages"], page_table=gpu["page_table"],
                                             lengths=torch.tensor([page * blocks], device=cuda_device), block_size=page, count=1, first=0, recent=0)
        assert got.flatten().tolist() == [j]


def test_an_append_writes_the_pages_that_are_there_and_no_others(cuda_device):
    """Rows whose block has no column in the table, that have a negative length, and one that fills its second page."""
    cache = Cache(3, 1, 64, 16, FP16, 2)
    key, value = cache.new_tokens(31)
    cache.append(key, value, rows=[2])
    gpu = cache.on(cuda_device)
    before = {k: v.clone() for k, v in gpu.items()}
    key, value = cache.new_tokens(1)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    anna_b200.run_q8_append(key=key.to(cuda_device), value=value.to(cuda_device), past_lengths=torch.tensor([47, -5, 31], device=cuda_device), status=status,
                            **gpu)
    assert status.item() == 1  # of row 0
    cache.append(key, value, rows=[2])
    page = int(cache.table[2, 1])
    changed = (gpu["packed_pages"] != before["packed_pages"]).flatten(1).any(1).cpu()
    assert changed.nonzero().flatten().tolist() == [page]
    known = cache.known_bytes()
    assert torch.equal(gpu["packed_pages"].cpu()[page][:, known], cache.pages[page][:, known])
    # row 0 closes a page that is none and row 2 one that is: neither leaves a token in its ring; row 1 is left out
    assert torch.equal(gpu["window"].cpu().view(torch.uint8), before["window"].cpu().view(torch.uint8))
