"""Gated linear recurrence over tracked sequences: smoothing of landmarks (or of any feature) along a recording.

    h[t] = a[t] * h[t-1] + (1 - a[t]) * x[t],      a = sigmoid(gate)

The reference reports MPJPA, the mean acceleration of the keypoints (load_eval.py:84-86), and leaves the tracked keypoints
as the frames gave them.  ``gated_scan`` filters whole recordings in one call (csrc/gated_scan.hip) and is differentiable,
so a filter's constants can be learned from labelled recordings; ``gated_step`` does the same one frame at a time over a
cache of rows, the way ``UmeTrackModel.temporal_step`` advances the temporal memory.  There is no CPU implementation.
"""
import math
from typing import Optional, Tuple

import torch

from ... import _native as nat

_DTYPES = {torch.float32: nat.VALUES_F32, torch.bfloat16: nat.VALUES_BF16}


def _split(name: str, x: torch.Tensor, gate: torch.Tensor, lead: int) -> Tuple[int, int]:
    """(groups, share) of features x.shape[lead:] under gates gate.shape[lead:]: the gate's dimensions are the first of the
    feature's, up to dimensions of size 1 behind them; the features behind share a gate."""
    feat, g = tuple(x.shape[lead:]), tuple(gate.shape[lead:])
    if tuple(x.shape[:lead]) != tuple(gate.shape[:lead]):
        raise ValueError(f"{name}: x is {tuple(x.shape)} and gate {tuple(gate.shape)}: the first {lead} dimensions differ")
    while g and (len(g) > len(feat) or g[-1] == 1 != feat[len(g) - 1]):
        if g[-1] != 1:
            break
        g = g[:-1]
    if g != feat[:len(g)]:
        raise ValueError(f"{name}: gates {tuple(gate.shape[lead:])} are no leading dimensions of the features {feat}")
    return math.prod(g), math.prod(feat[len(g):])


def _check_values(name: str, x, gate) -> torch.device:
    if not (isinstance(x, torch.Tensor) and isinstance(gate, torch.Tensor)):
        raise TypeError(f"{name}: x and gate are tensors")
    if x.dtype not in _DTYPES or gate.dtype != x.dtype:
        raise TypeError(f"{name}: x and gate are both float32 or both bfloat16, got {x.dtype} and {gate.dtype}")
    dev = nat.require_gpu(x.device if x.is_cuda else None)
    if x.device != dev or gate.device != dev:
        raise ValueError(f"{name}: x is on {x.device} and gate on {gate.device}: both have to be on one GPU")
    return dev


def _rows_of(t: torch.Tensor, n: int) -> torch.Tensor:
    """[T, R, ...] as [T, R, n] whose last axis is contiguous; the first two keep their strides (0 included) where they can."""
    v = t
    if n == 1:
        v = t.reshape(t.shape[0], t.shape[1], 1)
    elif t.dim() != 3 or t.stride(2) != 1:
        inner, want = t.shape[2:], 1
        dense = True
        for size, stride in zip(reversed(inner), reversed(t.stride()[2:])):
            if size != 1 and stride != want:
                dense = False
            want *= size
        v = t.as_strided((t.shape[0], t.shape[1], n), (t.stride(0), t.stride(1), 1)) if dense \
            else t.contiguous().view(t.shape[0], t.shape[1], n)
    return v


def _mask(name: str, m, shape, dev) -> Optional[torch.Tensor]:
    if m is None:
        return None
    if not isinstance(m, torch.Tensor) or m.dtype not in (torch.bool, torch.uint8) or tuple(m.shape) != tuple(shape) or m.device != dev:
        raise ValueError(f"{name}: expected a bool tensor {tuple(shape)} on {dev}")
    return m


def _state(name: str, s, shape, dev) -> Optional[torch.Tensor]:
    if s is None:
        return None
    if not isinstance(s, torch.Tensor) or s.dtype != torch.float32 or tuple(s.shape) != tuple(shape) or s.device != dev:
        raise ValueError(f"{name}: expected a float32 tensor {tuple(shape)} on {dev}")
    return s.contiguous()


def _like(x: torch.Tensor, feat) -> torch.Tensor:
    """An uninitialised tensor of x's first two dimensions and `feat` in x's memory order (rows outermost or time outermost)."""
    T, R = x.shape[:2]
    if x.stride(1) > x.stride(0) and T > 1 and R > 1:
        return torch.empty((R, T) + tuple(feat), dtype=x.dtype, device=x.device).transpose(0, 1)
    return torch.empty((T, R) + tuple(feat), dtype=x.dtype, device=x.device)


def _raw(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _shape(x, gate, use, valid, groups, share, out) -> nat.GatedShape:
    s = nat.GatedShape(_DTYPES[x.dtype], x.shape[0], x.shape[1], groups, share, x.stride(0), x.stride(1), gate.stride(0),
                       gate.stride(1), out.stride(0), out.stride(1))
    if use is not None:
        s.use_t, s.use_row = use.stride()
    if valid is not None:
        s.valid_t, s.valid_row = valid.stride()
    return s


def _workspace(nbytes: int, dev):
    if nbytes < 0:
        nat.check(1, "workspace size")
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _scan(x, gate, h0, use, valid, keep: bool):
    """-> (h, h_last, kept).  Shapes are checked by the callers."""
    dev = x.device
    groups, share = _split("gated_scan", x, gate, 2)
    feat = tuple(x.shape[2:])
    xs, gs = _rows_of(x, groups * share), _rows_of(gate, groups)
    h = _like(x, feat)
    last = torch.empty((x.shape[1],) + feat, dtype=torch.float32, device=dev)
    T, R = x.shape[:2]
    kept = torch.empty((-(-T // nat.GATED_KEEP), R * groups * share), dtype=torch.float32, device=dev) if keep else None
    if h.numel() or last.numel():
        shape = _shape(xs, gs, use, valid, groups, share, h)
        L = nat.lib()
        with torch.cuda.device(dev):
            ws = _workspace(L.umt_gated_scan_workspace_bytes(shape), dev)
            nat.check(L.umt_gated_scan(shape, _raw(xs), _raw(gs), _raw(use), _raw(valid), _raw(h0), _raw(h), _raw(last), _raw(kept),
                                       _raw(ws), 0 if ws is None else ws.numel(), nat.stream_ptr(dev)), "umt_gated_scan")
    return h, last, kept


def gated_scan_backward(x: torch.Tensor, gate: torch.Tensor, kept: torch.Tensor, dh: torch.Tensor,
                        dh_last: Optional[torch.Tensor] = None, use_memory: Optional[torch.Tensor] = None,
                        valid: Optional[torch.Tensor] = None, need: Tuple[bool, bool, bool] = (True, True, True)):
    """(dx, dgate, dh0) of ``gated_scan(..., keep=True)`` for the gradients dh (of h, x's dtype) and dh_last (of h_last,
    float32): what autograd calls, and what a program calls that captures its backward pass into a HIP graph, where
    autograd's own bookkeeping of leaves does not belong.  ``need`` leaves out gradients that nobody asked for (None)."""
    dev = _check_values("gated_scan_backward", x, gate)
    if x.dim() < 2:
        raise ValueError(f"gated_scan_backward: x is [T, R, ...], got {tuple(x.shape)}")
    groups, share = _split("gated_scan_backward", x, gate, 2)
    T, R = x.shape[:2]
    feat, n = tuple(x.shape[2:]), groups * share
    use, ok = _mask("use_memory", use_memory, (T, R), dev), _mask("valid", valid, (T, R), dev)
    if tuple(dh.shape) != tuple(x.shape) or dh.dtype != x.dtype or dh.device != dev:
        raise ValueError(f"gated_scan_backward: dh is {x.dtype} {tuple(x.shape)} on {dev}")
    kept = _state("kept", kept, (-(-T // nat.GATED_KEEP), R * n), dev)
    if kept is None:
        raise ValueError("gated_scan_backward: kept is what gated_scan(..., keep=True) returned")
    dh_last = _state("dh_last", dh_last, (R,) + feat, dev)
    xs, gs, ds = _rows_of(x, n), _rows_of(gate, groups), _rows_of(dh, n)
    dx = _like(x, feat) if need[0] else None
    dgate = _like(x, tuple(gate.shape[2:])) if need[1] else None
    dh0 = torch.empty((R,) + feat, dtype=torch.float32, device=dev) if need[2] else None
    if R * n and any(need):
        shape = _shape(xs, gs, use, ok, groups, share, dx if dx is not None else xs)
        shape.dh_t, shape.dh_row = ds.stride(0), ds.stride(1)
        if dgate is not None:
            shape.dgate_t, shape.dgate_row = dgate.stride(0), dgate.stride(1)
        L = nat.lib()
        with torch.cuda.device(dev):
            ws = _workspace(L.umt_gated_scan_backward_workspace_bytes(shape), dev)
            nat.check(L.umt_gated_scan_backward(shape, _raw(xs), _raw(gs), _raw(use), _raw(ok), _raw(kept), _raw(ds), _raw(dh_last),
                                                _raw(dx), _raw(dgate), _raw(dh0), _raw(ws), 0 if ws is None else ws.numel(),
                                                nat.stream_ptr(dev)), "umt_gated_scan_backward")
    return dx, dgate, dh0


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, use, valid):
        h, last, kept = _scan(x, gate, h0, use, valid, keep=True)
        ctx.save_for_backward(x, gate, kept, use, valid)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dh_last):
        x, gate, kept, use, valid = ctx.saved_tensors
        if dh is None and dh_last is None:
            return None, None, None, None, None
        if dh is None:
            dh = torch.zeros((), dtype=x.dtype, device=x.device).expand(x.shape)
        return gated_scan_backward(x, gate, kept, dh, dh_last, use, valid, ctx.needs_input_grad[:3]) + (None, None)


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
    states a backward pass starts from as a third value with ``keep``.  Differentiable with respect to x, gate and h0."""
    dev = _check_values("gated_scan", x, gate)
    if x.dim() < 2:
        raise ValueError(f"gated_scan: x is [T, R, ...features], got {tuple(x.shape)}")
    _split("gated_scan", x, gate, 2)
    T, R = x.shape[:2]
    h0 = _state("h0", h0, (R,) + tuple(x.shape[2:]), dev)
    use, ok = _mask("use_memory", use_memory, (T, R), dev), _mask("valid", valid, (T, R), dev)
    if not keep and torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (h0 is not None and h0.requires_grad)):
        return _GatedScan.apply(x, gate, h0, use, ok)
    with torch.no_grad():
        h, last, kept = _scan(x, gate, h0, use, ok, keep)
    return (h, last, kept) if keep else (h, last)


def gated_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, memory_idx: Optional[torch.Tensor] = None,
               use_memory: Optional[torch.Tensor] = None, valid: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One frame: sample b of x [B, ...features], gate [B, ...] advances row memory_idx[b] (int64; None: row b) of ``state``
    [rows, ...features] float32 in place; returns its new value in x's dtype.  Masks [B] as ``gated_scan``'s.  Duplicates in
    memory_idx all read the previous row and the highest b writes it; an index outside the cache runs without memory, writes
    none and ORs UMT_STATUS_BAD_MEMORY_IDX into ``status`` (int32[1] on the device).  Not differentiable."""
    dev = _check_values("gated_step", x, gate)
    if x.dim() < 1 or not isinstance(state, torch.Tensor):
        raise ValueError("gated_step: x is [B, ...features] and state a tensor")
    groups, share = _split("gated_step", x, gate, 1)
    B, feat = x.shape[0], tuple(x.shape[1:])
    if state.dtype != torch.float32 or state.dim() < 1 or tuple(state.shape[1:]) != feat or state.device != dev or not state.is_contiguous():
        raise ValueError(f"gated_step: state is a contiguous float32 tensor [rows, {', '.join(map(str, feat))}] on {dev}")
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or state.requires_grad):
        raise nat.UmtError("gated_step is not differentiable: use gated_scan, or call it under torch.no_grad()")
    rows = state.shape[0]
    if memory_idx is not None:
        if memory_idx.dtype != torch.int64 or tuple(memory_idx.shape) != (B,) or memory_idx.device != dev:
            raise ValueError(f"gated_step: memory_idx is an int64 tensor ({B},) on {dev}")
        memory_idx = memory_idx.contiguous()
    elif B > rows:
        raise ValueError(f"gated_step: {B} samples and {rows} rows without memory_idx")
    use, ok = _mask("use_memory", use_memory, (B,), dev), _mask("valid", valid, (B,), dev)
    use, ok = None if use is None else use.contiguous(), None if ok is None else ok.contiguous()
    if out is None:
        out = torch.empty((B,) + feat, dtype=x.dtype, device=dev)
    elif tuple(out.shape) != (B,) + feat or out.dtype != x.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"gated_step: out is a contiguous {x.dtype} tensor {(B,) + feat} on {dev}")
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1 or status.device != dev):
        raise ValueError(f"gated_step: status is int32[1] on {dev}")
    if out.numel() == 0:
        return out
    x, gate = x.contiguous(), gate.contiguous()
    L = nat.lib()
    with torch.cuda.device(dev):
        ws = _workspace(L.umt_gated_step_workspace_bytes(B, rows) if memory_idx is not None else 0, dev)
        nat.check(L.umt_gated_step(_DTYPES[x.dtype], _raw(x), _raw(gate), _raw(memory_idx), _raw(use), _raw(ok), B, groups, share,
                                   _raw(state), rows, _raw(out), _raw(status), _raw(ws), 0 if ws is None else ws.numel(),
                                   nat.stream_ptr(dev)), "umt_gated_step")
    return out
