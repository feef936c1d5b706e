"""Forks and rotary appends at the edges of what a launch holds, and under graph capture."""
from __future__ import annotations

import pytest
import torch
from test_gpu_forks_and_drafts import HEADS, KV_HEADS, ROTARY, append, assert_same, new_cache, states, views


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["none", "turboquant"])
@pytest.mark.parametrize("given", [True, False])
def test_a_captured_rotary_append(cuda_device, mode, given):
    """One replay of a captured append is that append."""
    gen = torch.Generator(device="cuda").manual_seed(41)
    caches = [new_cache(2, mode), new_cache(2, mode)]
    prompt = [states(gen, 2, 37, h) for h in (HEADS, KV_HEADS, KV_HEADS)]
    steps = [[states(gen, 2, 1, h) for h in (HEADS, KV_HEADS, KV_HEADS)] for _ in range(4)]
    positions = [torch.randint(0, 4000, (3, 2, 1), generator=gen, device="cuda") if given else None for _ in steps]
    for cache in caches:
        cache.rope_deltas = torch.tensor([[-3], [5]], device="cuda")
        for layer in range(2):
            cache.update_rotary(*prompt, layer, require_dense_cache=False, **ROTARY)
            for step, at in zip(steps[:2], positions):
                cache.update_rotary(*step, layer, positions=at, require_dense_cache=False, **ROTARY)
    want = [caches[0].update_rotary(*steps[2], layer, positions=positions[2], require_dense_cache=False, **ROTARY)[0] for layer in range(2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [caches[1].update_rotary(*steps[2], layer, positions=positions[2], require_dense_cache=False, **ROTARY)[0] for layer in range(2)]
    for out in got:
        out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert_same(views(caches[1]), views(caches[0]))
    for cache in caches:
        for layer in range(2):
            cache.update_rotary(*steps[3], layer, positions=positions[3], require_dense_cache=False, **ROTARY)
    assert_same(views(caches[1]), views(caches[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["none", "turboquant"])
def test_forks_of_more_pages_than_travel_in_a_launch(cuda_device, mode):
    """1500 forks of a row: 3000 or 6000 copies, whose ids go to the device first."""
    gen = torch.Generator(device="cuda").manual_seed(42)
    cache = new_cache(1, mode, window=8)
    append(cache, states(gen, 1, 37, KV_HEADS), states(gen, 1, 37, KV_HEADS))
    before = views(cache)
    forks = cache.fork_rows([0] * 1500)
    for layer, rows in enumerate(views(forks)):
        k, v = before[layer][0]
        assert all(torch.equal(a, k) and torch.equal(b, v) for a, b in rows)
    forks.release()
    assert_same(views(cache), before)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["none", "turboquant"])
def test_forks_of_more_pools_than_one_launch_takes(cuda_device, mode):
    gen = torch.Generator(device="cuda").manual_seed(43)
    cache = new_cache(2, mode, layers=70, window=8)
    append(cache, states(gen, 2, 21, KV_HEADS), states(gen, 2, 21, KV_HEADS))
    forks = cache.fork_rows([1, 0, 1])
    held, copied = views(cache), views(forks)
    for layer in range(70):
        for i, source in enumerate((1, 0, 1)):
            assert torch.equal(copied[layer][i][0], held[layer][source][0]) and torch.equal(copied[layer][i][1], held[layer][source][1])
    append(forks, states(gen, 3, 1, KV_HEADS), states(gen, 3, 1, KV_HEADS))
    assert_same(views(cache), held)
