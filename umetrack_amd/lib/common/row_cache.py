"""Rows of state caches: copy, fork, free and compact (csrc/row_cache.hip).

One row is one hand track's state.  The temporal memory of a ``UmeTrackModel`` is such a cache (temporal.py:41-42; the
reference only ever grows it, temporal.py:102-125), the state of ``gated_filter.gated_step`` is another.  ``buffers`` lists
what moves together: tensors [rows, ...] on one GPU, contiguous, of any dtype, and / or a model, which stands for its temporal
rows (at least as many rows have to be reserved).  Tracks that end are freed, hypotheses are forked, and ``compact_rows``
closes the cache up so that ``head_sequence`` and lock-step batches run on rows 0..n-1.

Row numbers and ``live`` (bool [rows], True = in use) stay on the GPU and nothing synchronises.  Bad row numbers do nothing
and OR a bit into ``status`` (int32[1] on the GPU): UMT_STATUS_BAD_ROW (32), UMT_STATUS_NO_FREE_ROW (64).
"""
import ctypes
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd.graph import increment_version

from ... import _native as nat


def _collect(buffers, rows: Optional[int]):
    """-> (umt_row_buffer array, its length, rows, device, tensors).  `rows` None: what the first tensor has, else the model."""
    if isinstance(buffers, torch.Tensor) or not isinstance(buffers, (list, tuple)):
        buffers = [buffers]
    entries, dev, models, tensors, name = [], None, [], [], "row cache"
    for b in buffers:
        if isinstance(b, torch.Tensor):
            have, size = b.shape[0] if b.dim() else 0, b.nbytes
            if b.dim() < 1 or not b.is_cuda or not b.is_contiguous() or have and not size:
                raise ValueError(f"{name}: a buffer is a contiguous GPU tensor [rows, ...], got {tuple(b.shape)} on {b.device}")
            if b.requires_grad and torch.is_grad_enabled():
                raise nat.UmtError(f"{name}: a buffer that requires gradients cannot be moved in place")
            if nat.dual_level():
                nat.no_tangents(name, b)
            rows = have if rows is None else rows
            if have != rows:
                raise ValueError(f"{name}: a buffer has {have} rows and not {rows}")
            d = b.device
            entries.append((b.data_ptr(), size // rows if rows else 1))
            tensors.append(b)
        elif hasattr(b, "memory_buffers"):
            d = b.device
            if d is None:
                raise nat.UmtError(f"{name}: the model is on no GPU yet")
            models.append((b, len(entries)))
            entries += [None, None]
        else:
            raise TypeError(f"{name}: a buffer is a tensor or a model, got {type(b).__name__}")
        if dev is not None and d != dev:
            raise ValueError(f"{name}: buffers on {dev} and {d}")
        dev = d
    if not entries or len(entries) > nat.ROW_BUFFERS_MAX:
        raise ValueError(f"{name}: 1 to {nat.ROW_BUFFERS_MAX} buffers (a model counts as two), got {len(entries)}")
    if not tensors:                                        # those are on a GPU
        nat.require_gpu(dev)
    for m, at in models:
        arr, have = m.memory_buffers()
        rows = have if rows is None else rows
        if have < rows:
            raise ValueError(f"{name}: the model has {have} memory rows reserved and not {rows}")
        entries[at:at + 2] = [(arr[0].data, arr[0].row_bytes), (arr[1].data, arr[1].row_bytes)]
    if rows >= 1 << 31:                                                        # the library takes them as ints
        raise ValueError(f"{name}: {rows} rows")
    arr = (nat.RowBuffer * len(entries))(*entries)
    return arr, len(entries), rows, dev, tensors


def _ids(name: str, t, dev) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int64 or t.dim() != 1 or t.device != dev:
        raise ValueError(f"{name}: expected a one-dimensional int64 tensor on {dev}")
    if t.shape[0] >= 1 << 31:
        raise ValueError(f"{name}: {t.shape[0]} row numbers")
    return t.contiguous()


def _live(t) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.bool or t.dim() != 1 or not t.is_cuda or not t.is_contiguous():
        raise ValueError("live: expected a contiguous bool tensor (rows,) on a GPU")
    return t


def _status(t, dev):
    if t is not None and (t.dtype != torch.int32 or t.numel() != 1 or t.device != dev):
        raise ValueError(f"status: expected int32[1] on {dev}")
    return None if t is None else t.data_ptr()


def _work(nbytes: int, dev):
    if nbytes < 0:
        nat.check(1, "workspace size")
    ws = torch.empty(max(16, nbytes), dtype=torch.uint8, device=dev)
    return ws, ctypes.c_void_p(ws.data_ptr()), ws.numel()


def copy_rows(buffers: Sequence, src: torch.Tensor, dst: torch.Tensor, status: Optional[torch.Tensor] = None) -> None:
    """Row dst[i] becomes what row src[i] was before the call (so permutations and swaps are fine); of several writes to one
    row the highest i counts."""
    arr, n_buf, rows, dev, tensors = _collect(buffers, None)
    src, dst = _ids("src", src, dev), _ids("dst", dst, dev)
    if src.shape != dst.shape:
        raise ValueError(f"copy_rows: {src.shape[0]} sources and {dst.shape[0]} targets")
    n, st = src.shape[0], _status(status, dev)
    if n == 0:
        return
    L = nat.lib()
    with nat.on_device(dev):
        ws, p, size = _work(L.umt_rows_copy_workspace_bytes(arr, n_buf, rows, n), dev)
        nat.check(L.umt_rows_copy(arr, n_buf, rows, src.data_ptr(), dst.data_ptr(), n, st, p, size, nat.raw_stream(dev)), "umt_rows_copy")
    increment_version(tensors)                             # a backward pass that has saved one of them raises


def fork_rows(buffers: Sequence, live: torch.Tensor, src: torch.Tensor, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """For each of ``src``, in order, the lowest free row becomes a live copy of it.  Returns the new row numbers (int64);
    -1 where src[i] is not a live row or no free row was left."""
    live = _live(live)
    arr, n_buf, rows, dev, tensors = _collect(buffers, live.shape[0])
    if live.device != dev:
        raise ValueError(f"live: expected a contiguous bool tensor ({rows},) on {dev}")
    src = _ids("src", src, dev)
    n, st = src.shape[0], _status(status, dev)
    ids = torch.empty(n, dtype=torch.int64, device=dev)
    if n == 0:
        return ids
    L = nat.lib()
    with nat.on_device(dev):
        ws, p, size = _work(L.umt_rows_fork_workspace_bytes(rows, n), dev)
        nat.check(L.umt_rows_fork(arr, n_buf, rows, live.data_ptr(), src.data_ptr(), n, ids.data_ptr(), st, p, size,
                                  nat.raw_stream(dev)), "umt_rows_fork")
    increment_version(tensors + [live])
    return ids


def free_rows(live: torch.Tensor, rows: torch.Tensor, status: Optional[torch.Tensor] = None) -> None:
    """live[rows] = False.  The content stays until a fork or a step overwrites it: start a new track with
    use_memory=False."""
    live = _live(live)
    if live.shape[0] >= 1 << 31:
        raise ValueError(f"live: {live.shape[0]} rows")
    dev = live.device
    rows = _ids("rows", rows, dev)
    st = _status(status, dev)
    if rows.shape[0] == 0:
        return
    with nat.on_device(dev):
        nat.check(nat.lib().umt_rows_free(live.data_ptr(), live.shape[0], rows.data_ptr(), rows.shape[0], st, nat.raw_stream(dev)),
                  "umt_rows_free")
    increment_version(live)


def compact_rows(buffers: Sequence, live: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Moves the last live rows into the free rows before them, so that rows 0..count-1 are the live ones (``live`` is
    updated).  Only rows that have to move do; the others keep their numbers.  Returns (now, count): now[r] (int64 [rows]) is
    the row that holds what row r held, -1 for a free one; count is int64[1]."""
    live = _live(live)
    arr, n_buf, rows, dev, tensors = _collect(buffers, live.shape[0])
    if live.device != dev:
        raise ValueError(f"live: expected a contiguous bool tensor ({rows},) on {dev}")
    now = torch.empty(rows, dtype=torch.int64, device=dev)
    count = torch.empty(1, dtype=torch.int64, device=dev)
    L = nat.lib()
    with nat.on_device(dev):
        ws, p, size = _work(L.umt_rows_compact_workspace_bytes(rows), dev)
        nat.check(L.umt_rows_compact(arr, n_buf, rows, live.data_ptr(), now.data_ptr(), count.data_ptr(), p, size,
                                     nat.raw_stream(dev)), "umt_rows_compact")
    increment_version(tensors + [live])
    return now, count
