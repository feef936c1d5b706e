"""Copies of whole pages: in place between pages of pools (forks of sequences), and of a pool's live pages into a smaller one
(compaction).  Any number of pools goes in one launch.

The reference copies page by page and layer by layer when a cache is cloned (``src/anna/model/ops.py:1323-1381``) and never
shrinks a pool that still has pages in use (``ops.py:186-196``).
"""
from __future__ import annotations

import ctypes
from collections.abc import Sequence

import numpy as np
import torch

from . import _lib
from .fused_ops import MetadataUploader, launch_module, on_device, stream_ptr


def _ids(name: str, values) -> np.ndarray:
    """Page ids as int64; refuses what is no flat sequence of whole numbers."""
    if isinstance(values, torch.Tensor):
        if values.device.type != "cpu":
            raise RuntimeError(f"{name}: page ids are host values (a list of ints)")
        values = values.numpy()
    ids = np.asarray(values)
    if ids.ndim != 1 or (ids.size and ids.dtype.kind not in "iu"):
        raise ValueError(f"{name}: page ids must be a flat sequence of ints")
    return ids.astype(np.int64)


def _check_range(name: str, ids: np.ndarray, pages: int, what: str) -> None:
    if ids.size and (int(ids.min()) < 0 or int(ids.max()) >= pages):
        raise IndexError(f"{name}: {what} page ids must be in [0, {pages})")


def _check_pool(name: str, pool: torch.Tensor, device: torch.device | None) -> torch.device:
    if pool.device.type != "cuda":
        raise RuntimeError(f"{name}: pools must be CUDA tensors (there is no CPU implementation of this op)")
    if device is not None and pool.device != device:
        raise RuntimeError(f"{name}: all pools must be on the same device")
    if pool.dim() < 2 or not pool.is_contiguous():
        raise RuntimeError(f"{name}: a pool must be a contiguous [pages, ...] tensor")
    if pool.shape[0] >= 2 ** 31:
        raise RuntimeError(f"{name}: too many pages")
    return pool.device


def _page_bytes(pool: torch.Tensor) -> int:
    return pool.numel() // pool.shape[0] * pool.element_size() if pool.shape[0] else 0


class _Pairs:
    """(source, target) ids of a call, those of pools that name the same lists once."""

    def __init__(self) -> None:
        self.parts: list[np.ndarray] = []
        self.total = 0

    def add(self, source: np.ndarray, target: np.ndarray) -> int:
        first = self.total
        part = np.empty((source.size, 2), dtype=np.int32)
        part[:, 0], part[:, 1] = source, target
        self.parts.append(part)
        self.total += source.size
        return first


def _launch(name: str, device: torch.device, entries: list[tuple], pairs: _Pairs) -> None:
    """entries: (source address, target address, bytes of a page, source pages, target pages, first pair, count)."""
    if pairs.total == 0:
        return
    pools = (_lib.PagePool * len(entries))(*entries)
    flat = np.concatenate(pairs.parts)
    library = _lib.lib()
    with on_device(device):
        on_gpu = None
        if pairs.total > library.anna_page_copy_max_pairs():
            on_gpu = MetadataUploader.for_device(device).upload_i32(flat.reshape(-1))
        _lib.check(library.anna_page_copy(ctypes.addressof(pools), len(entries), flat.ctypes.data, pairs.total,
                                          None if on_gpu is None else on_gpu.data_ptr(), None, stream_ptr(device)), name)


def run_page_copy(*, copies: Sequence[tuple[torch.Tensor, Sequence[int], Sequence[int]]]) -> None:
    """For every ``(pool, source, target)``: page ``source[i]`` of the contiguous ``[pages, ...]`` pool is copied to page
    ``target[i]``, in place.  A source may have several targets; no page may be a target twice, or a target and a source (the
    copies of a call have no order)."""
    name = "page_copy"
    copies = list(copies)
    if launch_module().page_copy(copies):
        return
    # not the ordinary call: arguments to be converted or refused, or a pool that is named twice
    device = None
    pairs, entries = _Pairs(), []
    known: dict[tuple[int, int], tuple[np.ndarray, np.ndarray, int]] = {}
    of_pool: dict[int, tuple[int, list[np.ndarray], list[np.ndarray]]] = {}
    for pool, source, target in copies:
        device = _check_pool(name, pool, device)
        hit = known.get((id(source), id(target)))
        if hit is None:
            src, dst = _ids(name, source), _ids(name, target)
            if src.size != dst.size:
                raise ValueError(f"{name}: {src.size} source pages for {dst.size} target pages")
            hit = known[(id(source), id(target))] = (src, dst, pairs.add(src, dst))
        src, dst, first = hit
        pages, size = int(pool.shape[0]), _page_bytes(pool)
        _check_range(name, src, pages, "source")
        _check_range(name, dst, pages, "target")
        base = pool.data_ptr()
        if src.size and size:
            if base in of_pool and of_pool[base][0] != size:
                raise RuntimeError(f"{name}: pools must not overlap")
            _, sources, targets = of_pool.setdefault(base, (size, [], []))
            sources.append(src)
            targets.append(dst)
            entries.append((base, base, size, pages, pages, first, src.size))
    checked: set[tuple[int, ...]] = set()
    for base, (_, sources, targets) in of_pool.items():
        which = tuple(id(a) for a in sources + targets)
        if which in checked:  # the same lists for another pool
            continue
        checked.add(which)
        written = np.concatenate(targets) if len(targets) > 1 else targets[0]
        read = np.concatenate(sources) if len(sources) > 1 else sources[0]
        distinct = np.unique(written)
        if distinct.size != written.size:
            raise ValueError(f"{name}: a page is named as target twice")
        if np.isin(read, distinct).any():
            raise ValueError(f"{name}: a page is source and target of one call")
    spans = sorted({(base, base + size * pages) for base, _, size, pages, _, _, _ in entries})
    if any(end > begin for (_, end), (begin, _) in zip(spans, spans[1:])):
        raise RuntimeError(f"{name}: pools must not overlap")
    if device is not None:
        _launch(name, device, entries, pairs)


def run_page_gather(*, pools: Sequence[tuple[torch.Tensor, Sequence[int]]], spare_pages: int = 0) -> list[torch.Tensor]:
    """For every ``(pool, page ids)`` a new pool ``[len(ids) + spare_pages, ...]`` that begins with those pages in that order;
    what the spare pages hold is undefined.  Ids may repeat."""
    name = "page_gather"
    if spare_pages < 0:
        raise ValueError(f"{name}: spare_pages must not be negative")
    pools = list(pools)
    new_pools = launch_module().page_gather(pools, spare_pages)
    if new_pools is not None:
        return new_pools
    device = None
    pairs, entries, out = _Pairs(), [], []
    known: dict[int, tuple[np.ndarray, int]] = {}
    for pool, ids in pools:
        device = _check_pool(name, pool, device)
        hit = known.get(id(ids))
        if hit is None:
            src = _ids(name, ids)
            hit = known[id(ids)] = (src, pairs.add(src, np.arange(src.size, dtype=np.int64)))
        src, first = hit
        pages, size = int(pool.shape[0]), _page_bytes(pool)
        _check_range(name, src, pages, "source")
        new = torch.empty((src.size + spare_pages, *pool.shape[1:]), dtype=pool.dtype, device=device)
        out.append(new)
        if src.size and size:
            entries.append((pool.data_ptr(), new.data_ptr(), size, pages, src.size + spare_pages, first, src.size))
    if device is not None:
        _launch(name, device, entries, pairs)
    return out
