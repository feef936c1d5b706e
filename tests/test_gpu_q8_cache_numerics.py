"""Attention over the 8-bit paged cache where its numbers come close to the ends of their formats, against a restatement in 64 bits."""
from __future__ import annotations

import pytest
import torch

from test_gpu_q8_cache import FP32, check_attention, filled

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
