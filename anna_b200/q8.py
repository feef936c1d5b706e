"""A paged KV cache in 8 bits: append, attention of the newest tokens, the choice of the pages that a query should look at, and the
dense view.

A full page holds int8 codes with one scale for the keys and one for the values of every KV head; the tokens of a sequence's last,
unfinished page are as they came, in a ring (``include/anna_b200_kv.h`` has the layout).  The tensors of a cache:

* ``packed_pages``  uint8 ``[pages, kv_heads, q8_page_bytes(head_dim, block_size)]``, contiguous; nothing in it has to be initialised
* ``page_table``    int32 ``[batch, max_blocks]``: the page of every full block of a row; other entries are not looked at
* ``window``        ``[slots, 2, kv_heads, block_size, head_dim]`` of the type of keys and values, contiguous
* ``window_slots``  int64 ``[batch]``: the ring of every row, no ring twice in a call that appends

Pages are plain memory: ``run_page_copy`` copies them (and rings) for forks, a full page may be in the tables of several rows.  head_dim is
64, 128 or 256, ``block_size`` at most 1024, types float32, float16 and bfloat16.  Calls work on the current stream, can be captured into a
CUDA graph, and have no gradients.  The reference has no cache of this kind.

Attention works in float32, and where ``block_size`` is a multiple of 8 on tensor cores: codes are exact there, the entries of a query head are whole
numbers of 24 bits, off by 2^-23 of its largest magnitude at most, and a weight is a sum of two fp16 (over tokens of a bf16 ring of two bf16), off by
2^-23 (2^-16) of itself.  That is as good as float32 unless a query's largest entries meet keys that are next to nothing there.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .fused_ops import _require_cuda, dtype_code, launch_module, on_device

_MAX_I32 = 2 ** 31 - 1


def q8_page_bytes(head_dim: int, block_size: int) -> int:
    """Bytes of what a page of ``block_size`` tokens holds of one KV head."""
    bytes_of = ctypes.c_int64(0)
    _lib.check(_lib.lib().anna_q8_page_bytes(int(head_dim), int(block_size), ctypes.byref(bytes_of)), "q8_page_bytes")
    return int(bytes_of.value)


def _check_pages(name: str, packed_pages: torch.Tensor, page_table: torch.Tensor, batch: int, kv_heads: int, head_dim: int,
                 block_size: int) -> None:
    if not 1 <= block_size <= _MAX_I32 or not 1 <= head_dim <= _MAX_I32:
        raise RuntimeError(f"{name}: head_dim and block_size must be positive")
    size = q8_page_bytes(head_dim, block_size)
    if packed_pages.dtype != torch.uint8 or packed_pages.dim() != 3 or not packed_pages.is_contiguous():
        raise RuntimeError(f"{name}: packed_pages must be contiguous uint8 [pages, kv_heads, page_bytes]")
    if int(packed_pages.shape[1]) != kv_heads:
        raise RuntimeError(f"{name}: packed_pages have {int(packed_pages.shape[1])} kv heads, not {kv_heads}")
    if int(packed_pages.shape[2]) != size:
        raise RuntimeError(f"{name}: pages are {int(packed_pages.shape[2])} bytes, head_dim={head_dim} block_size={block_size} needs {size}")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != batch:
        raise RuntimeError(f"{name}: page_table must be int32 [batch, max_blocks]")
    if page_table.shape[1] > 0 and packed_pages.shape[0] == 0:
        raise RuntimeError(f"{name}: a block table needs pages")


def _check_window(name: str, window: torch.Tensor, dtype: torch.dtype) -> None:
    dtype_code(dtype)
    if window.dim() != 5 or window.shape[1] != 2 or window.numel() == 0:
        raise RuntimeError(f"{name}: window must be [slots, 2, kv_heads, block_size, head_dim]")
    if window.dtype != dtype or not window.is_contiguous():
        raise RuntimeError(f"{name}: window must be contiguous and share the dtype of keys, values and queries")


def _check_row_numbers(name: str, batch: int, **tensors: torch.Tensor) -> None:
    for label, tensor in tensors.items():
        if tensor.dtype != torch.long or tensor.shape != (batch,):
            raise RuntimeError(f"{name}: {label} must be int64 [batch]")


def _table(page_table: torch.Tensor) -> torch.Tensor:
    return page_table if page_table.shape[1] <= 1 or page_table.stride(1) == 1 else page_table.contiguous()


def _rows(tensor: torch.Tensor) -> torch.Tensor:
    """In 16-byte pieces, as the kernels load them."""
    pieces = 16 // tensor.element_size()
    fits = tensor.stride(3) == 1 and tensor.data_ptr() % 16 == 0 and all(
        tensor.shape[d] <= 1 or tensor.stride(d) % pieces == 0 for d in range(3))
    return tensor if fits else tensor.clone(memory_format=torch.contiguous_format)


def run_q8_append(*, key: torch.Tensor, value: torch.Tensor, packed_pages: torch.Tensor, page_table: torch.Tensor, window: torch.Tensor,
                  window_slots: torch.Tensor, past_lengths: torch.Tensor, new_lengths: torch.Tensor | None = None,
                  status: torch.Tensor | None = None) -> None:
    """Appends ``key`` and ``value`` ``[B, Hkv, T, D]`` (any strides) to rows of ``past_lengths`` tokens, int64 ``[B]``.  Pages that are
    filled are quantized into the page that ``page_table`` has for their block; what is stored does not depend on how tokens are cut into
    calls.  ``new_lengths`` (int64 ``[B]``, other memory than ``past_lengths``) receives ``past_lengths + T``.  ``status``: int32, bit 0
    is set when a page or ring that is needed is none (its tokens are not written), or a row would be 2^30 tokens or longer."""
    name = "q8_append"
    if launch_module().q8_append(key, value, packed_pages, page_table, window, window_slots, past_lengths, new_lengths, status):
        return
    # not the ordinary call: arguments to be converted or refused
    if key.dim() != 4 or key.shape != value.shape or key.dtype != value.dtype:
        raise RuntimeError(f"{name}: key and value must be matching [batch, kv_heads, tokens, head_dim]")
    batch, kv_heads, tokens, dim = (int(v) for v in key.shape)
    _check_window(name, window, key.dtype)
    if int(window.shape[2]) != kv_heads or int(window.shape[4]) != dim:
        raise RuntimeError(f"{name}: window and keys disagree on kv_heads / head_dim")
    _check_pages(name, packed_pages, page_table, batch, kv_heads, dim, int(window.shape[3]))
    _check_row_numbers(name, batch, window_slots=window_slots, past_lengths=past_lengths)
    device = _require_cuda(name, key=key, value=value, packed_pages=packed_pages, page_table=page_table, window=window,
                           window_slots=window_slots, past_lengths=past_lengths, new_lengths=new_lengths, status=status)
    if new_lengths is not None:
        _check_row_numbers(name, batch, new_lengths=new_lengths)
        if not new_lengths.is_contiguous():
            raise RuntimeError(f"{name}: new_lengths must be contiguous")
        if batch > 0 and new_lengths.data_ptr() == past_lengths.data_ptr():
            raise RuntimeError(f"{name}: new_lengths must be other memory than past_lengths")
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise RuntimeError(f"{name}: status must be int32")
    if key.numel() == 0:
        if new_lengths is not None and batch > 0:
            with on_device(device):
                new_lengths.copy_(past_lengths)
        return
    if not launch_module().q8_append(_rows(key), _rows(value), packed_pages, _table(page_table), window, window_slots.contiguous(),
                                     past_lengths.contiguous(), new_lengths, status):
        raise RuntimeError(f"{name}: arguments that the kernels do not take")


def _check_query(name: str, query: torch.Tensor, kv_heads: int, dim: int) -> None:
    if query.dim() != 4:
        raise RuntimeError(f"{name}: query must be [batch, heads, tokens, head_dim]")
    if int(query.shape[3]) != dim:
        raise RuntimeError(f"{name}: query has head_dim {int(query.shape[3])}, the cache {dim}")
    if kv_heads < 1 or query.shape[1] % kv_heads != 0:
        raise RuntimeError(f"{name}: query heads must be a multiple of the kv heads of the cache")


def _last_dim(tensor: torch.Tensor) -> torch.Tensor:
    return tensor if tensor.stride(-1) == 1 else tensor.contiguous()


def run_q8_paged_attention(*, query: torch.Tensor, packed_pages: torch.Tensor, page_table: torch.Tensor, window: torch.Tensor,
                           window_slots: torch.Tensor, lengths: torch.Tensor, scaling: float, gate: torch.Tensor | None = None,
                           blocks: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the newest T tokens of every row: ``query`` ``[B, Hq, T, D]`` (any strides, ``Hq T`` below 2^20), ``lengths`` int64 ``[B]`` with
    the new tokens among them; query ``t`` sees the keys up to position ``lengths[b] - T + t``, one that sees none gives zeros.  A length is cut at what table
    and ring hold.  ``gate`` (shape and dtype of the query): the output is multiplied by its sigmoid.  An infinity or a NaN that a query sees shows in its
    output, however small its weight.

    ``blocks``, int32 ``[B, Hkv, T, n]`` as ``run_q8_select_blocks`` gives them: of the full pages query ``t`` looks at those of its list
    alone, and at the unfinished page.  A list may be in any order; entries that are no full page of the row are left out, one that is named
    twice counts twice."""
    name = "q8_paged_attention"
    out = launch_module().q8_attention(query, gate, packed_pages, page_table, window, window_slots, lengths, blocks, scaling)
    if out is not None:
        return out
    # not the ordinary call: arguments to be converted or refused
    if query.dim() != 4:
        raise RuntimeError(f"{name}: query must be [batch, heads, tokens, head_dim]")
    _check_window(name, window, query.dtype)
    kv_heads, block_size, dim = (int(v) for v in window.shape[2:])
    _check_query(name, query, kv_heads, dim)
    batch = int(query.shape[0])
    _check_pages(name, packed_pages, page_table, batch, kv_heads, dim, block_size)
    _check_row_numbers(name, batch, window_slots=window_slots, lengths=lengths)
    if gate is not None and (gate.shape != query.shape or gate.dtype != query.dtype):
        raise RuntimeError(f"{name}: gate must match the query in shape and dtype")
    if blocks is not None:
        if blocks.dtype != torch.int32 or blocks.dim() != 4 or tuple(blocks.shape[:3]) != (batch, kv_heads, int(query.shape[2])):
            raise RuntimeError(f"{name}: blocks must be int32 [batch, kv_heads, tokens, n]")
        if blocks.shape[3] == 0:
            raise RuntimeError(f"{name}: blocks must have room for one")
        blocks = blocks.contiguous()
    _require_cuda(name, query=query, packed_pages=packed_pages, page_table=page_table, window=window, window_slots=window_slots,
                  lengths=lengths, gate=gate, blocks=blocks)
    if query.numel() == 0:
        return torch.empty(query.shape, dtype=query.dtype, device=query.device)
    out = launch_module().q8_attention(_last_dim(query), None if gate is None else _last_dim(gate), packed_pages, _table(page_table), window,
                                       window_slots.contiguous(), lengths.contiguous(), blocks, float(scaling))
    if out is None:
        raise RuntimeError(f"{name}: arguments that the kernels do not take")
    return out


def run_q8_select_blocks(*, query: torch.Tensor, packed_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                         block_size: int, count: int, first: int = 1, recent: int = 1) -> torch.Tensor:
    """Which full pages every query should look at: int32 ``[B, Hkv, T, count]``, indices of blocks in ascending order, then -1.  ``query`` and
    ``lengths`` as for ``run_q8_paged_attention``.

    Of the full pages with a token that query ``t`` sees, the ``first`` first and the ``recent`` last ones are always among them, the others are
    those of the best scores; all of them where they are no more than ``count``.  A score bounds the products of the KV head's query heads with the
    page's keys from above: the largest, over those heads, of the sum over dims of the larger of query times largest and query times smallest
    code of the dim, times the page's scale.  Queries count in whole numbers, 32767 for the head's largest magnitude, so that a score is the
    same however it is summed; of equal ones the earlier page is the better, NaN is better than any number."""
    name = "q8_select_blocks"
    block_size, count, first, recent = int(block_size), int(count), int(first), int(recent)
    blocks = launch_module().q8_select(query, packed_pages, page_table, lengths, block_size, count, first, recent)
    if blocks is not None:
        return blocks
    # not the ordinary call: arguments to be converted or refused
    if query.dim() != 4 or packed_pages.dim() != 3:
        raise RuntimeError(f"{name}: query must be [batch, heads, tokens, head_dim], packed_pages [pages, kv_heads, page_bytes]")
    dtype_code(query.dtype)
    kv_heads = int(packed_pages.shape[1])
    _check_query(name, query, kv_heads, int(query.shape[3]))
    batch, _, tokens, dim = (int(v) for v in query.shape)
    _check_pages(name, packed_pages, page_table, batch, kv_heads, dim, block_size)
    _check_row_numbers(name, batch, lengths=lengths)
    if not 1 <= count <= _MAX_I32 or first < 0 or recent < 0 or first + recent > count:
        raise ValueError(f"{name}: count must be positive and have room for the first and recent pages")
    device = _require_cuda(name, query=query, packed_pages=packed_pages, page_table=page_table, lengths=lengths)
    if query.numel() == 0:
        return torch.full((batch, kv_heads, tokens, count), -1, dtype=torch.int32, device=device)
    blocks = launch_module().q8_select(_last_dim(query), packed_pages, _table(page_table), lengths.contiguous(), block_size, count, first, recent)
    if blocks is None:
        raise RuntimeError(f"{name}: arguments that the kernels do not take")
    return blocks


def run_q8_gather(*, packed_pages: torch.Tensor, page_table: torch.Tensor, window: torch.Tensor, window_slots: torch.Tensor,
                  lengths: torch.Tensor, max_len: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Dense keys and values ``[B, Hkv, max_len, D]`` of the first ``lengths`` tokens of every row, zeros behind them and where a page is none:
    what attention of whole chunks (``grouped_query_attention``) reads."""
    name = "q8_gather"
    max_len = int(max_len)
    pair = launch_module().q8_gather(packed_pages, page_table, window, window_slots, lengths, max_len)
    if pair is not None:
        return pair
    # not the ordinary call: arguments to be converted or refused
    if max_len < 0:
        raise ValueError(f"{name}: max_len must not be negative")
    _check_window(name, window, window.dtype)
    kv_heads, block_size, dim = (int(v) for v in window.shape[2:])
    if page_table.dim() != 2:
        raise RuntimeError(f"{name}: page_table must be int32 [batch, max_blocks]")
    batch = int(page_table.shape[0])
    _check_pages(name, packed_pages, page_table, batch, kv_heads, dim, block_size)
    _check_row_numbers(name, batch, window_slots=window_slots, lengths=lengths)
    _require_cuda(name, packed_pages=packed_pages, page_table=page_table, window=window, window_slots=window_slots, lengths=lengths)
    pair = launch_module().q8_gather(packed_pages, _table(page_table), window, window_slots.contiguous(), lengths.contiguous(), max_len)
    if pair is None:
        raise RuntimeError(f"{name}: arguments that the kernels do not take")
    return pair
