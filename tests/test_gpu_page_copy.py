"""Copies of whole pages within pools and into smaller ones: every byte, and none beside them."""
from __future__ import annotations

import ctypes
import math
import random

import pytest
import torch

import anna_b200
from anna_b200 import _lib


def pool_of(pages, shape, dtype, device, seed=0):
    """Random bytes as a pool of `dtype`."""
    gen = torch.Generator(device=device).manual_seed(seed)
    size = math.prod(shape) * torch.empty(0, dtype=dtype).element_size()
    data = torch.randint(0, 256, (pages, size), generator=gen, device=device, dtype=torch.uint8)
    return data.view(dtype).view(pages, *shape)


def bits(x):
    return x.contiguous().view(torch.uint8)


SHAPES = [  # pages, page shape, dtype
    (9, (2, 16, 128), torch.bfloat16),   # 8 KB: half a unit
    (5, (8, 128, 128), torch.bfloat16),  # 16 units
    (40, (2432,), torch.uint8),          # a unit's last accesses missing
    (7, (3, 5), torch.float32),          # 60 bytes: 4-byte accesses
    (6, (1, 1, 1), torch.uint8),         # one byte
    (5, (16391,), torch.uint8),          # odd, more than a unit
    (4, (2, 3, 50000), torch.float16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("pages,shape,dtype", SHAPES, ids=str)
def test_copies_in_place(cuda_device, pages, shape, dtype):
    rng = random.Random(pages)
    pool = pool_of(pages, shape, dtype, cuda_device)
    want = bits(pool).clone()
    ids = rng.sample(range(pages), pages)
    target, source = ids[:pages // 2], ids[pages // 2:]
    source = [rng.choice(source) for _ in target]  # a page may be copied several times
    for s, t in zip(source, target):
        want[t] = want[s]
    anna_b200.run_page_copy(copies=[(pool, source, target)])
    assert torch.equal(bits(pool), want)


@pytest.mark.gpu
@pytest.mark.parametrize("pages,shape,dtype", SHAPES, ids=str)
@pytest.mark.parametrize("spare", [0, 3])
def test_gathered_pools(cuda_device, pages, shape, dtype, spare):
    rng = random.Random(pages)
    pool = pool_of(pages, shape, dtype, cuda_device)
    before = bits(pool).clone()
    ids = [rng.randrange(pages) for _ in range(pages + 2)]
    new = anna_b200.run_page_gather(pools=[(pool, ids)], spare_pages=spare)[0]
    assert new.shape == (len(ids) + spare, *shape) and new.dtype == dtype
    assert torch.equal(bits(new)[:len(ids)], before[ids]) and torch.equal(bits(pool), before)


@pytest.mark.gpu
@pytest.mark.parametrize("pools,copies", [(3, 4), (33, 5), (40, 30), (200, 3), (2, 3000), (130, 40)])
def test_many_pools_and_pairs_at_once(cuda_device, pools, copies):
    """What travels in the launch, what needs several launches, and what goes through device memory."""
    rng = random.Random(pools)
    lists = []
    for _ in range(3):
        ids = rng.sample(range(2 * copies + 1), 2 * copies)
        lists.append((ids[:copies], ids[copies:]))
    work, want = [], []
    for i in range(pools):
        pool = pool_of(2 * copies + 1, (3 + i % 5, 8), torch.float32, cuda_device, seed=i)
        source, target = lists[i % 3] if i % 4 else ([], [])
        expected = bits(pool).clone()
        if source:
            expected[target] = expected[source]
        work.append((pool, source, target))
        want.append(expected)
    anna_b200.run_page_copy(copies=work)
    for (pool, _, _), expected in zip(work, want):
        assert torch.equal(bits(pool), expected)
    got = anna_b200.run_page_gather(pools=[(pool, source) for pool, source, _ in work])
    for new, (pool, source, _) in zip(got, work):
        assert torch.equal(bits(new), bits(pool)[source])


@pytest.mark.gpu
def test_pools_beyond_four_gigabytes(cuda_device):
    pool = torch.zeros(3000, 1 << 21, dtype=torch.uint8, device=cuda_device)  # 6.3 GB: offsets pass 32 bits
    pool[2999] = torch.arange(1 << 21, device=cuda_device).to(torch.uint8)
    anna_b200.run_page_copy(copies=[(pool, [2999], [2500])])
    assert torch.equal(pool[2500], pool[2999]) and int(pool[2501].max()) == 0 and int(pool[2499].max()) == 0
    new = anna_b200.run_page_gather(pools=[(pool, [0, 2500])])[0]
    assert int(new[0].max()) == 0 and torch.equal(new[1], pool[2999])


@pytest.mark.gpu
def test_pages_at_odd_addresses(cuda_device):
    base = torch.arange(6 * 64 + 5, device=cuda_device).to(torch.uint8)
    for shift in (1, 2, 3, 4):
        pool = base[shift:shift + 6 * 64].view(6, 64)
        want = pool.clone()
        want[[1, 5]] = want[[0, 3]]
        around = base[:shift].clone(), base[shift + 6 * 64:].clone()
        anna_b200.run_page_copy(copies=[(pool, [0, 3], [1, 5])])
        assert torch.equal(pool, want) and torch.equal(base[:shift], around[0]) and torch.equal(base[shift + 6 * 64:], around[1])


@pytest.mark.gpu
def test_captured_copies_run_again(cuda_device):
    for copies in (4, 3000):  # in the launch; through an upload that the graph keeps
        pool = torch.zeros(2 * copies, 64, device=cuda_device)
        source, target = list(range(copies)), list(range(copies, 2 * copies))
        anna_b200.run_page_copy(copies=[(pool, source, target)])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            anna_b200.run_page_copy(copies=[(pool, source, target)])
        for value in (3.0, 5.0):
            pool[:copies] = value
            graph.replay()
            torch.cuda.synchronize()
            assert bool((pool == value).all())


@pytest.mark.gpu
def test_copies_that_depend_on_each_other_are_refused(cuda_device):
    pool, other = torch.zeros(8, 4, device=cuda_device), torch.zeros(8, 4, device=cuda_device)
    call = anna_b200.run_page_copy
    for copies, error in (([(pool, [0, 1], [2, 2])], ValueError), ([(pool, [0, 1], [1, 2])], ValueError), ([(pool, [3], [3])], ValueError),
                          ([(pool, [0], [1]), (pool, [2], [1])], ValueError), ([(pool, [0], [1]), (pool, [1], [2])], ValueError),
                          ([(pool, [0], [8])], IndexError), ([(pool, [-1], [0])], IndexError), ([(pool, [0, 1], [2])], ValueError),
                          ([(pool, [0.5], [2])], ValueError), ([(pool, [[0]], [[2]])], ValueError), ([(pool[:, ::2], [0], [1])], RuntimeError),
                          ([(pool, [0], [1]), (pool[1:], [0], [1])], RuntimeError), ([(pool, [0], [1]), (pool.view(4, 8), [0], [1])], RuntimeError),
                          ([(pool, [0], [1]), (other.cpu(), [0], [1])], RuntimeError),
                          ([(pool, torch.tensor([0], device=cuda_device), [1])], RuntimeError)):
        with pytest.raises(error, match="page_copy"):
            call(copies=copies)
    with pytest.raises(IndexError, match="page_gather"):
        anna_b200.run_page_gather(pools=[(pool, [0, 8])])
    with pytest.raises(ValueError, match="spare_pages"):
        anna_b200.run_page_gather(pools=[(pool, [0])], spare_pages=-1)
    pool[0] = 1.0
    call(copies=[])
    call(copies=[(pool, [], []), (pool, (0, 0), torch.tensor([5, 6])), (other, [0], [1])])
    assert pool[:, 0].tolist() == [1.0, 0.0, 0.0, 0.0, 0.0, 1.0, 1.0, 0.0] and float(other.abs().sum()) == 0.0


def test_host_pools_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        anna_b200.run_page_copy(copies=[(torch.zeros(4, 4), [0], [1])])
    with pytest.raises(RuntimeError, match="CUDA"):
        anna_b200.run_page_gather(pools=[(torch.zeros(4, 4), [0])])


def test_entry_point_refuses_bad_tables():
    library, ok = _lib.lib(), 0x10000
    pairs = (ctypes.c_int32 * 4)(0, 1, 2, 3)

    def call(count=2, first=0, src=ok, size=64, total=2, given=pairs, pages=4, device=None):
        pool = _lib.PagePool(src, ok, size, pages, pages, first, count)
        return library.anna_page_copy(ctypes.addressof(pool), 1, ctypes.addressof(given) if given is not None else None, total, device,
                                      None, None)

    for bad in (dict(count=3), dict(first=1), dict(first=-1), dict(count=-1), dict(src=None), dict(size=-1), dict(pages=-1), dict(given=None),
                dict(total=library.anna_page_copy_max_pairs() + 1), dict(total=-1), dict(device=ok + 4)):
        assert call(**bad) == 1, bad
        assert "anna_page_copy" in _lib.last_error()
    assert call(count=0) == 0 and call(size=0) == 0  # nothing to do: nothing is launched
