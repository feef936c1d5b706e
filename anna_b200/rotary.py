"""Rotary positions with several axes (time, height and width of images and video) on queries and keys, and the same fused with
the write of keys and values into un-quantized pages.

Stands in for the rotary part of ``Qwen3Attention._forward_attention`` (``src/anna/model/ops.py:1900-1914``): pair ``i`` of a
head is its dims ``(i, i + rotary_dim / 2)``, which a token turns by ``positions[axis(i)] * theta ** (-2 i / rotary_dim)``; the
dims behind ``rotary_dim`` stay as they are.  ``sections`` says how many pairs belong to each axis, one section after the other
or, with ``interleaved``, in turns: pair ``i`` belongs to axis ``a = i % n`` while ``i < n * sections[a]``, else to the first.
The angles are formed and reduced to one turn in 64 bits, which leaves nothing to see in 32 for positions up to 2^28; at 2^31 they are off
by 5e-7 of a radian at most.
"""
from __future__ import annotations

import math
import threading
from collections.abc import Sequence
from dataclasses import dataclass

import torch

from . import _lib
from .fused_ops import _require_cuda, dtype_code, launch_module, on_device, ptr, stream_ptr


@dataclass(frozen=True)
class RotaryTables:
    axis_count: int
    rates: torch.Tensor  # float64 [rotary_dim / 2], turns per position
    axes: torch.Tensor   # int32 [rotary_dim / 2]


_TABLES: dict[tuple, RotaryTables] = {}
_LOCK = threading.Lock()


def pair_axes(rotary_dim: int, sections: Sequence[int] | None, interleaved: bool) -> list[int]:
    """Axis of every pair of rotated dims."""
    pairs = rotary_dim // 2
    if sections is None:
        return [0] * pairs
    sections = [int(s) for s in sections]
    if not sections or min(sections) < 0 or sum(sections) != pairs:
        raise ValueError(f"sections {tuple(sections)} must be counts of pairs that add up to rotary_dim / 2 = {pairs}")
    if interleaved:
        count = len(sections)
        return [i % count if i < count * sections[i % count] else 0 for i in range(pairs)]
    return [axis for axis, size in enumerate(sections) for _ in range(size)]


def rotary_tables(rotary_dim: int, *, theta: float = 10000.0, sections: Sequence[int] | None = None, interleaved: bool = False,
                  inverse_frequencies: Sequence[float] | None = None, device: torch.device) -> RotaryTables:
    """Rates and axes of the pairs on the device, made once for each set of parameters.  ``inverse_frequencies`` (radians per
    position, one for each pair) stands in for the powers of ``theta``; a tensor in device memory is read back on every call."""
    if inverse_frequencies is not None:  # values, whatever holds them
        if isinstance(inverse_frequencies, torch.Tensor):
            if inverse_frequencies.is_cuda:
                with on_device(inverse_frequencies.device):
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("inverse_frequencies in device memory cannot be read under graph capture: pass their values "
                                           "(a list, or a tensor of the host)")
            inverse_frequencies = inverse_frequencies.tolist()
        inverse_frequencies = tuple(float(f) for f in inverse_frequencies)
    sections = None if sections is None else tuple(int(s) for s in sections)
    theta = float(theta)
    key = (rotary_dim, theta, sections, bool(interleaved), inverse_frequencies, device)
    found = _TABLES.get(key)
    if found is not None:
        return found
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    pairs = rotary_dim // 2
    axes = pair_axes(rotary_dim, sections, interleaved)
    if inverse_frequencies is None:
        if not theta > 0 or not math.isfinite(theta):
            raise ValueError(f"theta must be positive, got {theta}")
        frequencies = [theta ** (-i / pairs) for i in range(pairs)]
    else:
        frequencies = list(inverse_frequencies)
        if len(frequencies) != pairs or not all(map(math.isfinite, frequencies)):
            raise ValueError(f"inverse_frequencies must hold rotary_dim / 2 = {pairs} finite values")
    with on_device(device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first call with new rotary parameters uploads their tables: make it outside graph capture")
    with _LOCK:
        found = _TABLES.get(key)
        if found is not None:  # another thread's
            return found
        # Graphs and other streams may read tables at any time, so none is given back.
        if len(_TABLES) >= 4096:
            raise RuntimeError("more than 4096 sets of rotary parameters: their tables stay on the device, so they are for parameters of "
                               "models, not for some that change from call to call")
        tables = RotaryTables(axis_count=1 if sections is None else len(sections),
                              rates=torch.tensor([f / (2.0 * math.pi) for f in frequencies], dtype=torch.float64, device=device),
                              axes=torch.tensor(axes, dtype=torch.int32, device=device))
        _TABLES[key] = tables
    return tables


def _check_rows(name: str, query: torch.Tensor, key: torch.Tensor) -> None:
    if query.dim() != 4 or key.dim() != 4:
        raise RuntimeError(f"{name}: query and key must be [batch, heads, tokens, head_dim]")
    if query.shape[0] != key.shape[0] or query.shape[2] != key.shape[2] or query.shape[3] != key.shape[3]:
        raise RuntimeError(f"{name}: query and key must agree in batch, tokens and head_dim")
    if query.dtype != key.dtype:
        raise RuntimeError(f"{name}: query and key must share the dtype")
    dtype_code(query.dtype)


def _check_positions(name: str, positions: torch.Tensor, axes: int, batch: int, tokens: int) -> tuple[int, int, int]:
    """Element strides per axis, batch and token."""
    if positions.dtype != torch.long:
        raise RuntimeError(f"{name}: positions must be int64")
    if tuple(positions.shape) == (batch, tokens) and positions.dim() == 2:
        return 0, positions.stride(0), positions.stride(1)
    if tuple(positions.shape) != (axes, batch, tokens):
        raise RuntimeError(f"{name}: positions must be [{axes}, {batch}, {tokens}] (axes, batch, tokens) or [{batch}, {tokens}], "
                           f"got {list(positions.shape)}")
    return positions.stride(0), positions.stride(1), positions.stride(2)


def _extent(tensor: torch.Tensor) -> tuple[int, int]:
    last = sum((size - 1) * stride for size, stride in zip(tensor.shape, tensor.stride()))
    return tensor.data_ptr(), tensor.data_ptr() + (last + 1) * tensor.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    (begin, end), (other_begin, other_end) = _extent(a), _extent(b)
    return begin < other_end and other_begin < end


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether ``[B, H, T, D]`` tensors of the same B and T share no element: they lie apart, or they are parts of one fused
    projection, next to each other in every row or in every token."""
    if not _overlap(a, b):
        return True
    offset, rest = divmod(b.data_ptr() - a.data_ptr(), a.element_size())
    if rest:
        return False
    for outer in ((0,), (0, 2)):
        if any(a.shape[d] > 1 and a.stride(d) != b.stride(d) for d in outer):
            continue
        steps = sorted((a.stride(d), a.shape[d]) for d in outer if a.shape[d] > 1)
        if not steps or steps[0][0] <= 0 or any(step < before * size for (before, size), (step, _) in zip(steps, steps[1:])):
            continue
        window = steps[0][0]  # elements of one row or token, a's and b's parts among them
        span_a, span_b = (1 + sum((x.shape[d] - 1) * x.stride(d) for d in range(4) if d not in outer) for x in (a, b))
        if (offset >= span_a and offset + span_b <= window) or (-offset >= span_b and -offset + span_a <= window):
            return True
    return False


def _output(name: str, label: str, given: torch.Tensor | None, source: torch.Tensor, others: list[torch.Tensor]) -> torch.Tensor:
    """The tensor that receives the turned ``source``: a new one, or the caller's (the source itself for in place)."""
    if given is None:
        return torch.empty(source.shape, dtype=source.dtype, device=source.device)
    if given.shape != source.shape or given.dtype != source.dtype or given.device != source.device:
        raise RuntimeError(f"{name}: {label} must match its input in shape, dtype and device")
    if given.stride(3) != 1 or any(size > 1 and stride <= 0 for size, stride in zip(given.shape, given.stride())):
        raise RuntimeError(f"{name}: {label} needs a contiguous last dim and memory of its own for every element")
    reach = 0  # of the dims with smaller strides
    for stride, size in sorted((stride, size) for size, stride in zip(given.shape, given.stride()) if size > 1):
        if stride <= reach:
            raise RuntimeError(f"{name}: {label} needs memory of its own for every element")
        reach += (size - 1) * stride
    if given.data_ptr() == source.data_ptr() and given.stride() == source.stride():  # in place
        if not all(_apart(given, other) for other in others):
            raise RuntimeError(f"{name}: {label} is written in place and overlaps another input")
        return given
    if any(_overlap(given, other) for other in (source, *others)):
        raise RuntimeError(f"{name}: {label} must be its input itself or lie outside the memory of the inputs")
    return given


def _rows(tensor: torch.Tensor) -> torch.Tensor:
    return tensor if tensor.stride(3) == 1 else tensor.contiguous()


def _check_row_starts(name: str, batch: int, positions, past_lengths, rope_deltas) -> None:
    """Positions, or what they are derived from: lengths before the call and offsets of text behind images."""
    if past_lengths is not None and (past_lengths.dtype != torch.long or tuple(past_lengths.shape) != (batch,)):
        raise RuntimeError(f"{name}: past_lengths must be int64 [batch]")
    if rope_deltas is not None:
        if positions is not None:
            raise RuntimeError(f"{name}: rope_deltas belong to positions=None")
        if rope_deltas.dtype != torch.long or tuple(rope_deltas.shape) not in ((batch,), (batch, 1)):
            raise RuntimeError(f"{name}: rope_deltas must be int64 [batch] or [batch, 1]")


def check_rotary_arguments(name: str, query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor | None,
                           rope_deltas: torch.Tensor | None, *, theta: float = 10000.0, sections: Sequence[int] | None = None,
                           interleaved: bool = False, rotary_dim: int | None = None,
                           inverse_frequencies: Sequence[float] | None = None, attention_scaling: float = 1.0) -> None:
    """Refuses what ``run_multi_axis_rotary`` and ``run_rotary_paged_kv_write`` would, and makes the tables: for callers that count
    tokens before they launch."""
    _check_rows(name, query, key)
    batch, _, tokens, dim = (int(v) for v in query.shape)
    if positions is not None or rope_deltas is not None:
        _check_row_starts(name, batch, positions, None, rope_deltas)
    device = _require_cuda(name, query=query, key=key, positions=positions, rope_deltas=rope_deltas)
    width = dim if rotary_dim is None else int(rotary_dim)
    if width > dim:
        raise RuntimeError(f"{name}: rotary_dim {width} is larger than head_dim {dim}")
    if dim > 4096:
        raise RuntimeError(f"{name}: head_dim {dim} is larger than 4096")
    float(attention_scaling)
    tables = rotary_tables(width, theta=theta, sections=sections, interleaved=interleaved, inverse_frequencies=inverse_frequencies,
                           device=device)
    if positions is not None:
        _check_positions(name, positions, tables.axis_count, batch, tokens)
    if (query.shape[1] == 0) != (key.shape[1] == 0):
        raise RuntimeError(f"{name}: query and key need at least one head each")


def run_multi_axis_rotary(*, query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor | None = None,
                          past_lengths: torch.Tensor | None = None, rope_deltas: torch.Tensor | None = None, theta: float = 10000.0,
                          sections: Sequence[int] | None = None, interleaved: bool = False, rotary_dim: int | None = None,
                          inverse_frequencies: Sequence[float] | None = None, attention_scaling: float = 1.0,
                          query_out: torch.Tensor | None = None,
                          key_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Turned ``[B, Hq, T, D]`` queries and ``[B, Hkv, T, D]`` keys (any strides; new contiguous tensors unless ``query_out`` /
    ``key_out`` are given, which may be the inputs themselves).

    ``positions``: int64 ``[axes, B, T]``, or ``[B, T]`` for the same on every axis; None: ``past_lengths[b] + t + rope_deltas[b]``
    on every axis (``past_lengths`` int64 ``[B]``, ``rope_deltas`` int64 ``[B]`` or ``[B, 1]``, None: 0).  ``sections`` (pairs per axis; None: one
    axis), ``interleaved``, ``theta`` and ``inverse_frequencies``: see the module.  ``attention_scaling`` multiplies cosine and
    sine.  The first call with new parameters makes their tables and cannot be captured into a graph."""
    name = "multi_axis_rotary"
    if query_out is None and key_out is None and query.is_cuda and (rotary_dim or 0) <= query.shape[-1]:
        width = query.shape[-1] if rotary_dim is None else rotary_dim
        tables = rotary_tables(width, theta=theta, sections=sections, interleaved=interleaved,
                               inverse_frequencies=inverse_frequencies, device=query.device)
        turned = launch_module().rotary(query, key, positions, past_lengths, rope_deltas, tables.rates, tables.axes, tables.axis_count, width, attention_scaling)
        if turned is not None:
            return turned
    # not the ordinary call: arguments to be checked or converted
    _check_rows(name, query, key)
    if positions is None and past_lengths is None:
        raise RuntimeError(f"{name}: positions or past_lengths must be given")
    _check_row_starts(name, int(query.shape[0]), positions, past_lengths, rope_deltas)
    device = _require_cuda(name, query=query, key=key, positions=positions, past_lengths=past_lengths, rope_deltas=rope_deltas)
    batch, heads, tokens, dim = (int(v) for v in query.shape)
    width = dim if rotary_dim is None else int(rotary_dim)
    if width > dim:
        raise RuntimeError(f"{name}: rotary_dim {width} is larger than head_dim {dim}")
    tables = rotary_tables(width, theta=theta, sections=sections, interleaved=interleaved,
                           inverse_frequencies=inverse_frequencies, device=device)
    strides = (0, 0, 0) if positions is None else _check_positions(name, positions, tables.axis_count, batch, tokens)
    past_lengths = None if past_lengths is None else past_lengths.contiguous()
    query_to = _output(name, "query_out", query_out, query, [key])
    key_to = _output(name, "key_out", key_out, key, [query])
    if query_out is not None and key_out is not None:
        in_place = query_to.data_ptr() == query.data_ptr() and key_to.data_ptr() == key.data_ptr()
        if not in_place and _overlap(query_to, key_to):
            raise RuntimeError(f"{name}: query_out and key_out must not overlap")
    if query.numel() == 0 or key.numel() == 0:
        if query.numel() or key.numel():
            raise RuntimeError(f"{name}: query and key need at least one head each")
        return query_to, key_to
    query, key = _rows(query), _rows(key)
    with on_device(device):
        _lib.check(_lib.lib().anna_multi_axis_rotary(
            ptr(query), *query.stride()[:3], ptr(query_to), *query_to.stride()[:3], ptr(key), *key.stride()[:3], ptr(key_to),
            *key_to.stride()[:3], ptr(positions), *strides, ptr(past_lengths), ptr(rope_deltas),
            0 if rope_deltas is None else rope_deltas.stride(0), ptr(tables.rates), ptr(tables.axes), float(attention_scaling), batch,
            heads, int(key.shape[1]), tokens, dim, width, dtype_code(query.dtype), stream_ptr(device)), name)
    return query_to, key_to


def run_rotary_paged_kv_write(*, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor,
                              value_pages: torch.Tensor, page_table: torch.Tensor, past_lengths: torch.Tensor,
                              positions: torch.Tensor | None = None, rope_deltas: torch.Tensor | None = None,
                              theta: float = 10000.0, sections: Sequence[int] | None = None, interleaved: bool = False,
                              rotary_dim: int | None = None, inverse_frequencies: Sequence[float] | None = None,
                              attention_scaling: float = 1.0, new_lengths: torch.Tensor | None = None,
                              status: torch.Tensor | None = None) -> torch.Tensor:
    """Turned queries ``[B, Hq, T, D]``; the turned keys and the values of ``[B, Hkv, T, D]`` go to their pages
    ``[P, Hkv, S, D]`` at positions ``past_lengths[b] + t``, all in one launch.

    ``positions`` and ``rope_deltas``: as for ``run_multi_axis_rotary``.  ``new_lengths``
    (int64 ``[B]``) receives ``past_lengths + T``; a token whose page id is invalid is not written and reported in ``status``
    (int32 ``[1]``).  The page pools must be contiguous."""
    name = "rotary_paged_kv_write"
    if query.is_cuda and (rotary_dim or 0) <= query.shape[-1]:
        width = query.shape[-1] if rotary_dim is None else rotary_dim
        tables = rotary_tables(width, theta=theta, sections=sections, interleaved=interleaved,
                               inverse_frequencies=inverse_frequencies, device=query.device)
        turned = launch_module().rotary_write(query, key, value, key_pages, value_pages, page_table, past_lengths, positions, rope_deltas,
                                              new_lengths, status, tables.rates, tables.axes, tables.axis_count, width,
                                              attention_scaling)
        if turned is not None:
            return turned
    # not the ordinary call: arguments to be checked or converted
    _check_rows(name, query, key)
    if value.shape != key.shape or value.dtype != key.dtype:
        raise RuntimeError(f"{name}: key and value must share shape and dtype")
    if key_pages.dim() != 4 or key_pages.shape != value_pages.shape:
        raise RuntimeError(f"{name}: key_pages and value_pages must be matching [pages, kv_heads, block_size, head_dim]")
    if key_pages.shape[1] != key.shape[1] or key_pages.shape[3] != key.shape[3]:
        raise RuntimeError(f"{name}: pages and keys disagree on kv_heads / head_dim")
    if not (key_pages.dtype == value_pages.dtype == key.dtype):
        raise RuntimeError(f"{name}: pages and keys must share the dtype")
    if not key_pages.is_contiguous() or not value_pages.is_contiguous():
        raise RuntimeError(f"{name}: page pools must be contiguous")
    batch, heads, tokens, dim = (int(v) for v in query.shape)
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != batch:
        raise RuntimeError(f"{name}: page_table must be int32 [batch, max_blocks]")
    _check_row_starts(name, batch, positions, past_lengths, rope_deltas)
    if new_lengths is not None:
        if new_lengths.dtype != torch.long or tuple(new_lengths.shape) != (batch,) or not new_lengths.is_contiguous():
            raise RuntimeError(f"{name}: new_lengths must be contiguous int64 [batch]")
        read = [x for x in (past_lengths, positions, rope_deltas) if x is not None and x.numel() > 0]
        if batch > 0 and any(_overlap(new_lengths, x) for x in read):
            raise RuntimeError(f"{name}: new_lengths must lie outside the memory of past_lengths, positions and rope_deltas")
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1):
        raise RuntimeError(f"{name}: status must be int32 [1]")
    device = _require_cuda(name, query=query, key=key, value=value, key_pages=key_pages, value_pages=value_pages,
                           page_table=page_table, past_lengths=past_lengths, positions=positions, rope_deltas=rope_deltas,
                           new_lengths=new_lengths, status=status)
    width = dim if rotary_dim is None else int(rotary_dim)
    if width > dim:
        raise RuntimeError(f"{name}: rotary_dim {width} is larger than head_dim {dim}")
    tables = rotary_tables(width, theta=theta, sections=sections, interleaved=interleaved,
                           inverse_frequencies=inverse_frequencies, device=device)
    strides = (0, 0, 0) if positions is None else _check_positions(name, positions, tables.axis_count, batch, tokens)
    out = torch.empty(query.shape, dtype=query.dtype, device=device)
    if query.numel() == 0 or key.numel() == 0:
        if query.numel() or key.numel():
            raise RuntimeError(f"{name}: query and key need at least one head each")
        if new_lengths is not None:
            new_lengths.copy_(past_lengths)
        return out
    if key_pages.shape[0] == 0 or page_table.shape[1] == 0:
        raise RuntimeError(f"{name}: there are no pages to write to")
    query, key, value = _rows(query), _rows(key), _rows(value)
    page_table = page_table if page_table.stride(1) == 1 else page_table.contiguous()
    past_lengths = past_lengths.contiguous()
    with on_device(device):
        _lib.check(_lib.lib().anna_rotary_paged_kv_write(
            ptr(query), *query.stride()[:3], ptr(out), *out.stride()[:3], ptr(key), *key.stride()[:3], ptr(value),
            *value.stride()[:3], ptr(key_pages), ptr(value_pages), ptr(page_table), page_table.stride(0), ptr(past_lengths),
            ptr(new_lengths), ptr(positions), *strides, ptr(rope_deltas), 0 if rope_deltas is None else rope_deltas.stride(0),
            ptr(tables.rates), ptr(tables.axes), float(attention_scaling), batch, heads, int(key.shape[1]), tokens, dim, width,
            int(key_pages.shape[2]), int(key_pages.shape[0]), int(page_table.shape[1]), dtype_code(query.dtype), ptr(status),
            stream_ptr(device)), name)
    return out
