"""Gated linear recurrence over tracked sequences: smoothing of landmarks (or of any feature) along a recording.

    h[t] = a[t] * h[t-1] + (1 - a[t]) * x[t],      a = sigmoid(gate)

The reference reports MPJPA, the mean acceleration of the keypoints (load_eval.py:84-86), and leaves the tracked keypoints
as the frames gave them.  ``gated_scan`` filters whole recordings in one call (csrc/gated_scan.hip) and is differentiable,
so a filter's constants can be learned from labelled recordings; ``gated_step`` does the same one frame at a time over a
cache of rows, the way ``UmeTrackModel.temporal_step`` advances the temporal memory.  There is no CPU implementation.
"""
import functools
import math
from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from ... import _native as nat

_DTYPES = {torch.float32: nat.VALUES_F32, torch.bfloat16: nat.VALUES_BF16}


def _split(name: str, x: torch.Tensor, gate: torch.Tensor, lead: int) -> Tuple[int, int]:
    """(groups, share) of features x.shape[lead:] under gates gate.shape[lead:]: the gate's dimensions are the first of the
    feature's, up to dimensions of size 1 behind them; the features behind share a gate."""
    return _split_shapes(name, x.shape, gate.shape, lead)


@functools.lru_cache(maxsize=256)                          # a tracker asks for the same two shapes every frame
def _split_shapes(name: str, x_shape, gate_shape, lead: int) -> Tuple[int, int]:
    xs, gs = tuple(x_shape), tuple(gate_shape)
    feat, g = xs[lead:], gs[lead:]
    if xs[:lead] != gs[:lead]:
        raise ValueError(f"{name}: x is {xs} and gate {gs}: the first {lead} dimensions differ")
    while g and (len(g) > len(feat) or g[-1] == 1 != feat[len(g) - 1]):
        if g[-1] != 1:
            break
        g = g[:-1]
    if g != feat[:len(g)]:
        raise ValueError(f"{name}: gates {gs[lead:]} are no leading dimensions of the features {feat}")
    groups, share = math.prod(g), math.prod(feat[len(g):])
    if max(xs[:lead]) >= 1 << 31 or max(groups, share) >= 1 << 31:             # the library takes them as ints
        raise ValueError(f"{name}: x is {xs}")
    return groups, share


def _check_values(name: str, x, gate, *others) -> torch.device:
    """The device of x and gate; `others`: what else may carry derivatives."""
    if not (isinstance(x, torch.Tensor) and isinstance(gate, torch.Tensor)):
        raise TypeError(f"{name}: x and gate are tensors")
    if nat.dual_level():
        nat.no_tangents(name, x, gate, *others)
    if x.dtype not in _DTYPES or gate.dtype != x.dtype:
        raise TypeError(f"{name}: x and gate are both float32 or both bfloat16, got {x.dtype} and {gate.dtype}")
    dev = x.device
    if not x.is_cuda:
        nat.require_gpu()
    if not x.is_cuda or gate.device != dev:
        raise ValueError(f"{name}: x is on {x.device} and gate on {gate.device}: both have to be on one GPU")
    return dev


def _rows_of(t: torch.Tensor, n: int) -> torch.Tensor:
    """[T, R, ...] as [T, R, n] whose last axis is contiguous; the first two keep their strides (0 included) where they can."""
    if t.is_contiguous():
        return t                                           # only the address and the first two strides are read
    if n == 1:
        return t.reshape(t.shape[0], t.shape[1], 1)
    want = 1
    for size, stride in zip(reversed(t.shape[2:]), reversed(t.stride()[2:])):
        if size != 1 and stride != want:
            return t.contiguous()
        want *= size
    return t


def _mask(name: str, m, shape, dev) -> Optional[torch.Tensor]:
    if m is None:
        return None
    if not isinstance(m, torch.Tensor) or m.dtype not in (torch.bool, torch.uint8) or m.shape != shape or m.device != dev:
        raise ValueError(f"{name}: expected a bool tensor {tuple(shape)} on {dev}")
    return m


def _state(name: str, s, shape, dev) -> Optional[torch.Tensor]:
    if s is None:
        return None
    if not isinstance(s, torch.Tensor) or s.dtype != torch.float32 or s.shape != shape or s.device != dev:
        raise ValueError(f"{name}: expected a float32 tensor {tuple(shape)} on {dev}")
    return s.contiguous()


def _like(x: torch.Tensor, feat=None) -> torch.Tensor:
    """An uninitialised tensor of x's first two dimensions and `feat` (None: x's) in x's memory order (rows or time outermost)."""
    if feat is None:
        feat = x.shape[2:]
        if x.is_contiguous():
            return torch.empty_like(x)
    T, R = x.shape[:2]
    if x.stride(1) > x.stride(0) and T > 1 and R > 1:
        return torch.empty((R, T) + tuple(feat), dtype=x.dtype, device=x.device).transpose(0, 1)
    return torch.empty((T, R) + tuple(feat), dtype=x.dtype, device=x.device)


def _raw(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _shape(x, gate, use, valid, groups, share, out) -> nat.GatedShape:
    T, R = x.shape[:2]
    xs, gs, os = x.stride(), gate.stride(), out.stride()
    us, vs = (0, 0) if use is None else use.stride(), (0, 0) if valid is None else valid.stride()
    return nat.GatedShape(_DTYPES[x.dtype], T, R, groups, share, xs[0], xs[1], gs[0], gs[1], os[0], os[1], us[0], us[1], vs[0], vs[1])


def _workspace(nbytes: int, dev):
    if nbytes < 0:
        nat.check(1, "workspace size")
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _scan(x, gate, h0, use, valid, groups: int, share: int, keep: bool):
    """-> (h, h_last, kept).  Arguments are checked by the caller."""
    dev = x.device
    T, R = x.shape[:2]
    n = groups * share
    xs, gs = _rows_of(x, n), _rows_of(gate, groups)
    h = _like(x)
    last = torch.empty(x.shape[1:], dtype=torch.float32, device=dev) if h0 is None else torch.empty_like(h0)
    kept = torch.empty((-(-T // nat.GATED_KEEP), R * n), dtype=torch.float32, device=dev) if keep else None
    if R * n:
        shape = _shape(xs, gs, use, valid, groups, share, h)
        L = nat.lib()
        with nat.on_device(dev):
            ws = _workspace(L.umt_gated_scan_workspace_bytes(shape), dev)
            nat.check(L.umt_gated_scan(shape, xs.data_ptr(), gs.data_ptr(), _raw(use), _raw(valid), _raw(h0), h.data_ptr(), last.data_ptr(),
                                       _raw(kept), _raw(ws), 0 if ws is None else ws.numel(), nat.raw_stream(dev)), "umt_gated_scan")
    return h, last, kept


def _backward(x, gate, kept, dh, dh_last, use, valid, groups: int, share: int, need):
    """-> (dx, dgate, dh0), None where not needed.  Arguments are checked by the caller."""
    dev = x.device
    R, n = x.shape[1], groups * share
    xs, gs, ds = _rows_of(x, n), _rows_of(gate, groups), _rows_of(dh, n)
    dx = _like(x) if need[0] else None
    dgate = None if not need[1] else torch.empty_like(gate) if gate.is_contiguous() and x.is_contiguous() else _like(x, gate.shape[2:])
    if dgate is not None and not n:
        dgate.zero_()                                      # gates of no features
    dh0 = torch.empty(x.shape[1:], dtype=torch.float32, device=dev) if need[2] else None
    if R * n and any(need):
        shape = _shape(xs, gs, use, valid, groups, share, xs if dx is None else dx)
        shape.dh_t, shape.dh_row = ds.stride()[:2]
        if dgate is not None:
            shape.dgate_t, shape.dgate_row = dgate.stride()[:2]
        L = nat.lib()
        with nat.on_device(dev):
            ws = _workspace(L.umt_gated_scan_backward_workspace_bytes(shape), dev)
            nat.check(L.umt_gated_scan_backward(shape, xs.data_ptr(), gs.data_ptr(), _raw(use), _raw(valid), kept.data_ptr(), ds.data_ptr(),
                                                _raw(dh_last), _raw(dx), _raw(dgate), _raw(dh0), _raw(ws), 0 if ws is None else ws.numel(),
                                                nat.raw_stream(dev)), "umt_gated_scan_backward")
    return dx, dgate, dh0


def gated_scan_backward(x: torch.Tensor, gate: torch.Tensor, kept: torch.Tensor, dh: torch.Tensor,
                        dh_last: Optional[torch.Tensor] = None, use_memory: Optional[torch.Tensor] = None,
                        valid: Optional[torch.Tensor] = None, need: Tuple[bool, bool, bool] = (True, True, True)):
    """(dx, dgate, dh0) of ``gated_scan(..., keep=True)`` for the gradients dh (of h, x's dtype) and dh_last (of h_last,
    float32): what autograd calls, and what a program calls that captures its backward pass into a HIP graph, where
    autograd's own bookkeeping of leaves does not belong.  ``need`` leaves out gradients that nobody asked for (None)."""
    dev = _check_values("gated_scan_backward", x, gate, kept, dh, dh_last)
    if x.dim() < 2:
        raise ValueError(f"gated_scan_backward: x is [T, R, ...], got {tuple(x.shape)}")
    groups, share = _split("gated_scan_backward", x, gate, 2)
    T, R = x.shape[:2]
    use, ok = _mask("use_memory", use_memory, (T, R), dev), _mask("valid", valid, (T, R), dev)
    if not isinstance(dh, torch.Tensor) or dh.shape != x.shape or dh.dtype != x.dtype or dh.device != dev:
        raise ValueError(f"gated_scan_backward: dh is {x.dtype} {tuple(x.shape)} on {dev}")
    kept = _state("kept", kept, (-(-T // nat.GATED_KEEP), R * groups * share), dev)
    if kept is None:
        raise ValueError("gated_scan_backward: kept is what gated_scan(..., keep=True) returned")
    dh_last = _state("dh_last", dh_last, x.shape[1:], dev)
    with torch.no_grad():
        return _backward(x, gate, kept, dh, dh_last, use, ok, groups, share, need)


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, use, valid, groups, share):
        h, last, kept = _scan(x, gate, h0, use, valid, groups, share, keep=True)
        ctx.save_for_backward(x, gate, kept, use, valid)
        ctx.set_materialize_grads(False)
        ctx.split = groups, share
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dh_last):
        if dh is None and dh_last is None:
            return None, None, None, None, None, None, None
        if nat.dual_level():
            nat.no_tangents("gated_scan's backward pass", dh, dh_last)
        x, gate, kept, use, valid = ctx.saved_tensors
        if dh is None:
            dh = torch.zeros((), dtype=x.dtype, device=x.device).expand(x.shape)
        if dh_last is not None:
            dh_last = dh_last.contiguous()
        return _backward(x, gate, kept, dh, dh_last, use, valid, *ctx.split, ctx.needs_input_grad) + (None, None, None, None)


def gated_scan(x: torch.Tensor, gate: torch.Tensor, h0: Optional[torch.Tensor] = None,
               use_memory: Optional[torch.Tensor] = None, valid: Optional[torch.Tensor] = None, keep: bool = False):
    """x [T, R, ...features] (float32 or bfloat16, time-major as ``UmeTrackModel.head_sequence``; any strides of the first two
    dimensions, so ``keypoints.transpose(0, 1)`` of a [R, T, ...] array is taken as it lies), gate [T, R, ...leading feature
    dimensions] in x's dtype: the logit of the memory's weight, shared by the features behind its dimensions ([T, R] one per
    row, [T, R, 21] one per landmark, ...; expanded tensors are read as they are).

    h0 [R, ...features] float32 is the state before the first step (None: zero).  use_memory [T, R] bool: False drops the
    memory in that frame (h = x).  valid [T, R] bool: False skips the frame (h stays; x and gate may hold anything there, NaN
    included).  Both False: h = 0.

    Returns (h [T, R, ...] in x's dtype and memory order, h_last [R, ...] float32, the state after the last step), and the
    states a backward pass starts from as a third value with ``keep``, for ``gated_scan_backward``; autograd records nothing
    then.  Without ``keep`` differentiable with respect to x, gate and h0, once and in reverse mode; tensors with forward-mode
    tangents are refused."""
    dev = _check_values("gated_scan", x, gate, h0)
    if x.dim() < 2:
        raise ValueError(f"gated_scan: x is [T, R, ...features], got {tuple(x.shape)}")
    groups, share = _split("gated_scan", x, gate, 2)
    h0 = _state("h0", h0, x.shape[1:], dev)
    use, ok = _mask("use_memory", use_memory, x.shape[:2], dev), _mask("valid", valid, x.shape[:2], dev)
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (h0 is not None and h0.requires_grad)):
        if not keep:
            return _GatedScan.apply(x, gate, h0, use, ok, groups, share)
        with torch.no_grad():
            return _scan(x, gate, h0, use, ok, groups, share, True)
    h, last, kept = _scan(x, gate, h0, use, ok, groups, share, keep)
    return (h, last, kept) if keep else (h, last)


def gated_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, memory_idx: Optional[torch.Tensor] = None,
               use_memory: Optional[torch.Tensor] = None, valid: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One frame: sample b of x [B, ...features], gate [B, ...] advances row memory_idx[b] (int64; None: row b) of ``state``
    [rows, ...features] float32 in place; returns its new value in x's dtype.  Masks [B] as ``gated_scan``'s.  Duplicates in
    memory_idx all read the previous row and the highest b writes it; an index outside the cache runs without memory, writes
    none and ORs UMT_STATUS_BAD_MEMORY_IDX into ``status`` (int32[1] on the device).  Not differentiable."""
    dev = _check_values("gated_step", x, gate, state, out)
    if x.dim() < 1 or not isinstance(state, torch.Tensor):
        raise ValueError("gated_step: x is [B, ...features] and state a tensor")
    groups, share = _split("gated_step", x, gate, 1)
    B, feat = x.shape[0], x.shape[1:]
    if state.dtype != torch.float32 or state.dim() < 1 or state.shape[1:] != feat or state.device != dev or not state.is_contiguous():
        raise ValueError(f"gated_step: state is a contiguous float32 tensor [rows, {', '.join(map(str, feat))}] on {dev}")
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or state.requires_grad or out is not None and out.requires_grad):
        raise nat.UmtError("gated_step is not differentiable: use gated_scan, or call it under torch.no_grad()")
    rows = state.shape[0]
    if rows >= 1 << 31:
        raise ValueError(f"gated_step: state is {tuple(state.shape)}")
    if memory_idx is not None:
        if not isinstance(memory_idx, torch.Tensor) or memory_idx.dtype != torch.int64 or memory_idx.shape != (B,) or memory_idx.device != dev:
            raise ValueError(f"gated_step: memory_idx is an int64 tensor ({B},) on {dev}")
        memory_idx = memory_idx.contiguous()
    elif B > rows:
        raise ValueError(f"gated_step: {B} samples and {rows} rows without memory_idx")
    use, ok = _mask("use_memory", use_memory, (B,), dev), _mask("valid", valid, (B,), dev)
    use, ok = None if use is None else use.contiguous(), None if ok is None else ok.contiguous()
    x, gate = x.contiguous(), gate.contiguous()
    written = (state,) if out is None else (state, out)
    if out is None:
        out = torch.empty_like(x)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"gated_step: out is a contiguous {x.dtype} tensor {tuple(x.shape)} on {dev}")
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1 or status.device != dev):
        raise ValueError(f"gated_step: status is int32[1] on {dev}")
    if out.numel() == 0:
        return out
    L = nat.lib()
    with nat.on_device(dev):
        ws = _workspace(L.umt_gated_step_workspace_bytes(B, rows) if memory_idx is not None else 0, dev)
        nat.check(L.umt_gated_step(_DTYPES[x.dtype], x.data_ptr(), gate.data_ptr(), _raw(memory_idx), _raw(use), _raw(ok), B, groups, share,
                                   state.data_ptr(), rows, out.data_ptr(), _raw(status), _raw(ws), 0 if ws is None else ws.numel(),
                                   nat.raw_stream(dev)), "umt_gated_step")
    increment_version(written)                             # a backward pass that has saved one of them raises
    return out
