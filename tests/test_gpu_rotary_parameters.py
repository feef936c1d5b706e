"""What the parameters of rotary positions may be held in: numbers and tensors of the host or the device, whose values count."""
from __future__ import annotations

import pytest
import torch
from test_gpu_rotary import states, turned

import anna_b200
from anna_b200 import KVCacheConfig, Qwen3DynamicCache, Qwen3PageAllocator, rotary


@pytest.mark.gpu
def test_theta_of_a_tensor_that_changes(cuda_device):
    q, k = states(2, 4, 2, 3, 64, torch.float32, cuda_device)
    positions = torch.randint(0, 500, (2, 3), device=cuda_device)
    theta = torch.tensor(1e4)
    for value in (1e4, 1e6, 5e5):
        theta.fill_(value)
        got = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions, theta=theta)
        want = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions, theta=float(theta))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert rotary.rotary_tables(64, theta=theta, device=q.device) is rotary.rotary_tables(64, theta=5e5, device=q.device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_frequencies_on_the_device(cuda_device, dtype):
    q, k = states(2, 4, 2, 3, 64, torch.float32, cuda_device)
    positions = torch.randint(0, 500, (2, 3), device=cuda_device)
    frequencies = torch.logspace(0, -4, 32, device=cuda_device).to(dtype)
    for _ in range(2):  # the second time with other values
        got = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions, inverse_frequencies=frequencies)
        want = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions, inverse_frequencies=[float(f) for f in frequencies])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        expected, bound = turned(q, positions, 64, frequencies=[float(f) for f in frequencies])
        assert bool(((got[0].cpu().double() - expected.cpu()).abs() <= bound.cpu() + 2.0 ** -24 * expected.cpu().abs()).all())
        frequencies.mul_(0.5)


@pytest.mark.gpu
def test_frequencies_on_the_device_are_refused_under_capture_which_goes_on(cuda_device):
    q, k = states(2, 4, 2, 3, 64, torch.float32, cuda_device)
    positions = torch.randint(0, 500, (2, 3), device=cuda_device)
    frequencies = torch.logspace(0, -4, 32, device=cuda_device)
    values = frequencies.tolist()
    want = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions, inverse_frequencies=values)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="inverse_frequencies in device memory"):
            anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions, inverse_frequencies=frequencies)
        got = anna_b200.run_multi_axis_rotary(query=q, key=k, positions=positions, inverse_frequencies=torch.tensor(values))
    got[0].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_an_append_of_heads_that_are_too_wide_counts_nothing(cuda_device):
    config = KVCacheConfig(num_hidden_layers=1, cache_block_size=4)
    cache = Qwen3DynamicCache(config, allocator=Qwen3PageAllocator(config), batch_size=1)
    q, k = states(1, 2, 1, 3, 4098, torch.bfloat16, cuda_device)
    with pytest.raises(RuntimeError, match="4096"):
        cache.update_rotary(q, k, k, 0, rotary_dim=64)
    assert cache.layer_lengths == [[0]] and cache.page_tables == [[[]]] and cache.allocator.layers[0].used_pages() == 0
