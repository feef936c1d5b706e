"""CPU: what the calls on the 8-bit paged cache refuse, and the size of a page."""
from __future__ import annotations

import ctypes

import pytest
import torch

import anna_b200
from anna_b200 import _lib

from q8_reference import page_bytes


@pytest.fixture(scope="module", autouse=True)
def library():
    if not _lib.library_path().exists():
        from anna_b200.build import build

        build()
    return _lib.lib()


def cache(batch=2, heads=2, dim=128, page=16, dtype=torch.bfloat16):
    return dict(packed_pages=torch.zeros((5, heads, page_bytes(dim, page)), dtype=torch.uint8),
                page_table=torch.zeros((batch, 4), dtype=torch.int32), window=torch.zeros((3, 2, heads, page, dim), dtype=dtype),
                window_slots=torch.zeros(batch, dtype=torch.long))


def test_page_bytes():
    for dim in (64, 128, 256):
        for page in (1, 8, 16, 24, 1024):
            assert anna_b200.q8_page_bytes(dim, page) == page_bytes(dim, page)
    for dim, page in ((96, 16), (0, 16), (128, 0), (128, 1025), (128, -1)):
        with pytest.raises(RuntimeError):
            anna_b200.q8_page_bytes(dim, page)


def refused(call, match, **changes):
    with pytest.raises((RuntimeError, ValueError), match=match):
        call(**changes)


def test_append_refuses():
    base = dict(cache(), key=torch.zeros((2, 2, 3, 128), dtype=torch.bfloat16), value=torch.zeros((2, 2, 3, 128), dtype=torch.bfloat16),
                past_lengths=torch.zeros(2, dtype=torch.long))

    def call(**changes):
        anna_b200.run_q8_append(**{**base, **changes})

    refused(call, "must be a CUDA tensor")
    refused(call, "matching", value=base["value"][:, :, :2])
    refused(call, "matching", value=base["value"].half())
    refused(call, "window must be", window=base["window"][:, :1])
    refused(call, "window must be", window=base["window"][:0])
    refused(call, "share the dtype", window=base["window"].half())
    refused(call, "share the dtype", window=base["window"].transpose(3, 4).contiguous().transpose(3, 4))
    refused(call, "kv_heads / head_dim", window=base["window"][:, :, :1].contiguous())
    refused(call, "uint8", packed_pages=base["packed_pages"].view(torch.int8))
    refused(call, "bytes", packed_pages=base["packed_pages"][:, :, :-128].contiguous())
    refused(call, "kv heads", packed_pages=base["packed_pages"][:, :1].contiguous())
    refused(call, "page_table", page_table=base["page_table"].long())
    refused(call, "page_table", page_table=base["page_table"][:1])
    refused(call, "needs pages", packed_pages=base["packed_pages"][:0])
    refused(call, "past_lengths", past_lengths=base["past_lengths"].int())
    refused(call, "window_slots", window_slots=base["window_slots"][:1])
    refused(call, "float16, bfloat16 and float32", key=base["key"].double(), value=base["value"].double(), window=base["window"].double())


def test_attention_refuses():
    base = dict(cache(), query=torch.zeros((2, 8, 1, 128), dtype=torch.bfloat16), lengths=torch.zeros(2, dtype=torch.long), scaling=1.0)

    def call(**changes):
        anna_b200.run_q8_paged_attention(**{**base, **changes})

    refused(call, "must be a CUDA tensor")
    refused(call, "query must be", query=base["query"][0])
    refused(call, "multiple of the kv heads", query=base["query"][:, :7])
    refused(call, "head_dim", query=base["query"][..., :64])
    refused(call, "share the dtype", query=base["query"].half())
    refused(call, "gate must match", gate=base["query"][:, :4])
    refused(call, "lengths", lengths=base["lengths"][:1])
    refused(call, "blocks must be", blocks=torch.zeros((2, 2, 2, 4), dtype=torch.int32))
    refused(call, "blocks must be", blocks=torch.zeros((2, 2, 1, 4), dtype=torch.long))
    refused(call, "room for one", blocks=torch.zeros((2, 2, 1, 0), dtype=torch.int32))
    wide = cache(dim=96)
    refused(call, "64, 128 or 256", **wide, query=torch.zeros((2, 8, 1, 96), dtype=torch.bfloat16))


def test_selection_refuses():
    base = dict(query=torch.zeros((2, 8, 1, 128), dtype=torch.bfloat16), lengths=torch.zeros(2, dtype=torch.long), block_size=16, count=4,
                **{k: v for k, v in cache().items() if not k.startswith("window")})

    def call(**changes):
        anna_b200.run_q8_select_blocks(**{**base, **changes})

    refused(call, "must be a CUDA tensor")
    refused(call, "room for the first", count=1)
    refused(call, "room for the first", count=0, first=0, recent=0)
    refused(call, "room for the first", first=-1)
    refused(call, "bytes", block_size=32)
    refused(call, "must be positive", block_size=0)
    refused(call, "multiple of the kv heads", query=base["query"][:, :7])


def test_gather_refuses():
    base = dict(cache(), lengths=torch.zeros(2, dtype=torch.long), max_len=4)

    def call(**changes):
        anna_b200.run_q8_gather(**{**base, **changes})

    refused(call, "must be a CUDA tensor")
    refused(call, "negative", max_len=-1)
    refused(call, "page_table", page_table=base["page_table"][0])
    refused(call, "lengths", lengths=base["lengths"].int())


def test_entry_points_refuse_before_they_launch(library):
    """Status codes of bad arguments; no GPU is touched."""
    floats, counters = ctypes.c_int64(0), ctypes.c_int(0)

    def plan(*args):
        return library.anna_q8_attention_plan(*args, ctypes.byref(floats), ctypes.byref(counters))

    assert plan(2, 8, 2, 1, 128, 16, 64, 0, 2) == 0 and floats.value > 0
    assert plan(2, 8, 2, 1, 128, 16, 64, 12, 2) == 0
    assert plan(2, 7, 2, 1, 128, 16, 64, 0, 2) == 1
    assert plan(2, 8, 2, 0, 128, 16, 64, 0, 2) == 1
    assert plan(2, 8, 2, 1, 96, 16, 64, 0, 2) == 2
    assert plan(2, 8, 2, 1, 128, 16, 1 << 40, 0, 2) == 1
    assert plan(1, 1 << 20, 1, 1, 128, 16, 64, 0, 2) == 1
    some, other = ctypes.c_void_p(4096), ctypes.c_void_p(8192)

    def append(key=some, new=None, tokens=1, page=16, dim=128, dtype=2, stride=128):
        return library.anna_q8_append(key, stride, stride, stride, some, stride, stride, stride, some, some, 4, some, some, other, new, 2, 2, tokens,
                                      dim, page, 5, 4, 3, dtype, None, None)

    assert append(key=None) == 1 and append(new=other) == 1 and append(tokens=0) == 1 and append(page=0) == 1 and append(dim=80) == 2
    assert append(dtype=7) == 1 and append(key=ctypes.c_void_p(4098)) == 1 and append(stride=129) == 1

    def select(count=4, first=1, recent=1, heads=8):
        return library.anna_q8_select_blocks(some, 128, 128, 128, some, some, 4, some, some, count, first, recent, some, 2, heads, 2, 1, 128, 16, 5, 4,
                                             2, None)

    assert select(count=0) == 1 and select(count=3, first=2, recent=2) == 1 and select(heads=7) == 1 and select(heads=1200) == 2
