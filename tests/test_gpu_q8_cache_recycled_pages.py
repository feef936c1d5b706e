"""Calls on the 8-bit paged cache that follow one another with nothing between them, over pages that every append writes anew."""
from __future__ import annotations

import pytest
import torch

import anna_b200
from q8_reference import Cache, attention, attention_bound, selected
from test_gpu_q8_cache import BF16, FP16, FP32

pytestmark = pytest.mark.gpu

PAGES, GROUP, COUNT = 6, 4, 2


class Steps:
    """`steps` prompts for the same pages and rings, whose scales go up and down, and what is on the GPU before the first call."""

    def __init__(self, device, dtype, dim, page, steps):
        self.dtype, self.dim, self.page, self.steps = dtype, dim, page, steps
        self.cache = Cache(3, 2, dim, page, dtype, PAGES, seed=dim + page)
        self.gpu = self.cache.on(device)
        n = PAGES * page + page // 2
        made = [self.cache.new_tokens(n, spread=2.0 ** (step * 3 % 7 - 3)) for step in range(steps)]
        self.key, self.value = (torch.stack([pair[i] for pair in made]) for i in range(2))
        self.query = torch.randn((steps, 3, 2 * GROUP, 1, dim), generator=self.cache.gen).to(dtype)
        self.on_gpu = tuple(x.to(device) for x in (self.key, self.value, self.query))
        self.past = torch.zeros(3, dtype=torch.long, device=device)
        self.lengths = torch.full((3,), n, dtype=torch.long, device=device)

    def run(self, step):
        key, value, query = (x[step] for x in self.on_gpu)
        common = dict(query=query, lengths=self.lengths)
        anna_b200.run_q8_append(key=key, value=value, past_lengths=self.past, **self.gpu)
        blocks = anna_b200.run_q8_select_blocks(packed_pages=self.gpu["packed_pages"], page_table=self.gpu["page_table"], block_size=self.page,
                                                count=COUNT, first=0, recent=0, **common)
        dense = anna_b200.run_q8_paged_attention(scaling=0.1, **common, **self.gpu)
        sparse = anna_b200.run_q8_paged_attention(scaling=0.1, blocks=blocks, **common, **self.gpu)
        return blocks, dense, sparse

    def check(self, step, got):
        cache, query = self.cache, self.query[step]
        cache.tokens = [torch.zeros((2, 2, 0, self.dim), dtype=self.dtype) for _ in range(3)]
        cache.append(self.key[step], self.value[step])
        blocks, dense, sparse = (x.cpu() for x in got)
        assert torch.equal(blocks, selected(query, cache, COUNT, 0, 0)), step
        rows = [cache.dense(b) for b in range(3)]
        for out, chosen in ((dense, None), (sparse, blocks)):
            want, reach, most = attention(query, rows, 0.1, None, self.page, chosen)
            assert bool(((out.double() - want).abs() <= attention_bound(want, self.dtype, self.dim, reach, most)).all()), step


@pytest.mark.parametrize("dtype,dim,page", [(BF16, 128, 16), (FP16, 64, 32), (FP32, 128, 16), (BF16, 256, 24), (FP16, 128, 5)])
def test_every_call_sees_the_pages_as_the_append_in_front_of_it_left_them(cuda_device, dtype, dim, page):
    steps = Steps(cuda_device, dtype, dim, page, 24)
    steps.run(0)  # scratch and counters are there
    torch.cuda.synchronize()
    results = [steps.run(step) for step in range(24)]
    torch.cuda.synchronize()
    for step, got in enumerate(results):
        steps.check(step, got)


@pytest.mark.parametrize("dtype,dim,page", [(BF16, 128, 16), (FP32, 64, 8)])
def test_so_do_calls_in_a_graph(cuda_device, dtype, dim, page):
    steps = Steps(cuda_device, dtype, dim, page, 6)
    steps.run(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = [steps.run(step) for step in range(6)]
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    for step, got in enumerate(results):
        steps.check(step, got)
