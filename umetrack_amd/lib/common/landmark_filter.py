"""Smoothing of tracked landmarks with the gated recurrence (gated_filter.py).

The reference scores jitter (MPJPA, load_eval.py:29-37, 84-86) and does nothing about it.  ``LandmarkFilter`` mixes every
tracked landmark with its filtered predecessor; the memory's weight is the sigmoid of a logit per landmark that may grow
with the landmark's predicted uncertainty (RegressorOutput.landmark_uncertainty_sigmas).  It runs over whole recordings
(``forward``), one frame at a time behind the tracker (``step``; HandTrackerOpts.landmark_filter), and its 42 constants can be
fitted to recordings with labels (``fit_landmark_filter``).
"""
import math
from typing import Iterable, Optional, Tuple

import torch

from . import gated_filter as gf
from .hand import NUM_LANDMARKS_PER_HAND


def memory_after_gaps(valid: torch.Tensor, before: Optional[torch.Tensor] = None) -> torch.Tensor:
    """use_memory [T, R] of the tracker's rule for valid [T, R]: a hand's memory counts in a frame when the hand was tracked
    in the one before (tracker.py:233-236, 278-285); `before` [R] says so for the frame ahead of the first (None: no hand was)."""
    use = torch.zeros_like(valid)
    use[1:] = valid[:-1]
    if before is not None:
        use[:1] = before
    return use


class LandmarkFilter(torch.nn.Module):
    """logit(memory weight) = bias[landmark] + slope[landmark] * log(sigma[landmark]).  ``memory`` in [0, 1) is the initial
    weight of every landmark; with slope 0 (the start) the sigmas are not needed."""

    def __init__(self, memory: float = 0.5):
        super().__init__()
        if not 0.0 <= memory < 1.0:
            raise ValueError(f"memory is a weight in [0, 1), got {memory}")
        logit = math.log(memory / (1 - memory)) if memory > 0 else -100.0          # sigmoid(-100) < 2^-126: the input itself
        self.bias = torch.nn.Parameter(torch.full((NUM_LANDMARKS_PER_HAND,), logit))
        self.slope = torch.nn.Parameter(torch.zeros(NUM_LANDMARKS_PER_HAND))

    def gate(self, lead: Tuple[int, ...], sigmas: Optional[torch.Tensor]) -> torch.Tensor:
        """Logits [*lead, 21]; without sigmas one stretched row of 21, which the kernels read as it lies."""
        if sigmas is None:
            return self.bias.expand(*lead, NUM_LANDMARKS_PER_HAND)
        if tuple(sigmas.shape) != tuple(lead) + (NUM_LANDMARKS_PER_HAND,):
            raise ValueError(f"sigmas: expected {tuple(lead) + (NUM_LANDMARKS_PER_HAND,)}, got {tuple(sigmas.shape)}")
        return torch.addcmul(self.bias, self.slope, torch.log(sigmas))

    def forward(self, landmarks: torch.Tensor, valid: Optional[torch.Tensor] = None, sigmas: Optional[torch.Tensor] = None,
                h0: Optional[torch.Tensor] = None, use_memory: Optional[torch.Tensor] = None,
                valid_before: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """landmarks [T, R, 21, 3] float32 (any order of the first two dimensions, e.g. a result file's [2, T, 21, 3]
        transposed), valid [T, R] bool: what landmarks and sigmas hold in untracked frames does not matter.  sigmas [T, R, 21]
        > 0.  use_memory defaults to the tracker's rule for `valid`.  Returns (filtered landmarks, state after the last frame
        [R, 21, 3]).

        By that rule the first untracked frame of a gap still holds the last filtered landmarks; from the second one on the
        memory is gone and the landmarks (and the state, where the recording ends there) are 0, as the result files have them.
        use_memory = memory_after_gaps(valid) | ~valid holds the last ones through the whole gap; tracked frames are the same.

        A recording filtered in pieces: h0 is the state that the piece before returned, valid_before [R] its last frame's
        `valid`, so that a hand that was not tracked there starts afresh.  Both can be left out where every hand was tracked in
        every frame (valid None); with `valid`, h0 needs valid_before, or use_memory [T, R] in the place of the rule."""
        lead = tuple(landmarks.shape[:2])
        if valid_before is not None:
            if h0 is None or use_memory is not None:
                raise ValueError("valid_before goes with h0 and without use_memory")
            if tuple(valid_before.shape) != lead[1:] or valid_before.dtype != torch.bool:
                raise ValueError(f"valid_before: expected a bool tensor {lead[1:]}")
        elif h0 is not None and valid is not None and use_memory is None:
            raise ValueError("h0 with valid: valid_before [R] has to say which hands were tracked in the frame before (or use_memory, "
                             "in which frames memory counts)")
        if use_memory is None:
            rule = valid if valid is not None else torch.ones(lead, dtype=torch.bool, device=landmarks.device)
            use_memory = memory_after_gaps(rule, torch.ones_like(rule[:1]) if h0 is not None and valid_before is None else valid_before)
        if valid is not None and sigmas is not None:       # a gate's gradient is 0 there, and 0 times the log of anything need not be
            sigmas = torch.where(valid[..., None], sigmas, torch.ones((), device=sigmas.device))
        return gf.gated_scan(landmarks, self.gate(lead, sigmas), h0=h0, use_memory=use_memory, valid=valid)

    @torch.no_grad()
    def step(self, landmarks: torch.Tensor, state: torch.Tensor, use_memory: torch.Tensor, memory_idx: Optional[torch.Tensor] = None,
             sigmas: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One frame of landmarks [B, 21, 3]; row memory_idx[b] of state [rows, 21, 3] advances (gated_filter.gated_step)."""
        return gf.gated_step(landmarks, self.gate((landmarks.shape[0],), sigmas), state, memory_idx=memory_idx, use_memory=use_memory, out=out)


def filter_loss(filtered: torch.Tensor, gt: torch.Tensor, valid: torch.Tensor, jitter: float) -> torch.Tensor:
    """Mean squared landmark error of the valid frames plus `jitter` times the mean squared difference of the second
    differences (load_eval.py:30) of filtered and labelled landmarks, where three frames in a row are valid.  [T, R, 21, 3]."""
    d = torch.where(valid[..., None, None], filtered - gt, torch.zeros((), device=gt.device))
    loss = d.square().sum() / valid.sum().clamp(min=1)
    if jitter and d.shape[0] > 2:
        three = (valid[:-2] & valid[1:-1] & valid[2:])
        a = torch.where(three[..., None, None], d[:-2] + d[2:] - 2 * d[1:-1], torch.zeros((), device=gt.device))
        loss = loss + jitter * a.square().sum() / three.sum().clamp(min=1)
    return loss


def fit_landmark_filter(filt: LandmarkFilter, recordings: Iterable, jitter: float = 1.0, steps: int = 100, lr: float = 0.05) -> LandmarkFilter:
    """Gradient descent (Adam) on filter_loss over `recordings`: tuples (landmarks, gt, valid[, sigmas]) in forward's layout on
    the filter's device."""
    data = [tuple(r) + (None,) * (4 - len(tuple(r))) for r in recordings]
    opt = torch.optim.Adam(filt.parameters(), lr=lr)
    for _ in range(steps):
        opt.zero_grad()
        for lm, gt, valid, sigmas in data:
            # labels under skipped frames may hold anything: filter_loss leaves them out, and a zero times NaN would not
            gt = torch.where(valid[..., None, None], gt, torch.zeros((), device=gt.device))
            filter_loss(filt(lm, valid, sigmas)[0], gt, valid, jitter).backward()
        opt.step()
    return filt
