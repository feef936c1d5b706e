"""What the parameters of rotary positions may be held in: numbers and tensors of the host or the device, whose values count."""
from __future__ import annotations

import pytest
import torch
from test_gpu_rotary import states, turned

import anna_b200
from anna_b200 import rotary


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
