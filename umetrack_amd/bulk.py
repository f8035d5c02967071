"""Bulk scheduling of recordings: backbone in bulk, temporal memory in lock-step.

The reference walks a recording frame by frame (run_eval_known_skeleton.py:68-86) although only the
tiny temporal module (0.87 MMAC per hand, temporal.py:93-139) depends on the previous frame: crop
cameras come from ground truth, so warp, backbone and view fusion of every frame are independent
(SURVEY.md section 3.1).  ``BulkSequenceRunner`` therefore

  1. runs warp -> backbone -> fusion over all frames of all recordings in large chunks, and
  2. steps the temporal memory + regressor once per time index over all (recording, hand) pairs
     in lock-step, memory row = 2*recording + hand.

Samples are ordered [recording][hand][t] (umetrack_amd.synthetic).  Results equal what the
frame-by-frame calls produce, because every output pixel is accumulated in the same order whatever
the batch size.
"""
from typing import Optional

import torch

from . import _native as nat
from .lib.common.landmark_filter import LandmarkFilter
from .lib.models.regressor import RegressorOutput
from .lib.models.umetrack_model import InputSkeletonData, UmeTrackModel
from .lib.tracker import warp as gpu_warp


class BulkSequenceRunner:
    def __init__(self, model: UmeTrackModel, n_rec: int, T: int, chunk_samples: int = 4096):
        self.model, self.n_rec, self.T = model, n_rec, T
        self.S = n_rec * 2 * T
        # chunks hold whole (recording, hand) rows so that a chunk is a [rows, T] block
        self.chunk = max(T, min(chunk_samples, self.S) // T * T)
        dev = model.device
        self.dev = dev
        R = n_rec * 2
        # phase-1 output in time-major order [T, rows, 72, 6, 6]: a lock-step is one contiguous slice
        self.fused_t = torch.empty(T, R, 72, 6, 6, dtype=torch.float32, device=dev)
        self.crops = torch.empty(2 * self.chunk, 96, 96, dtype=torch.float32, device=dev)
        self.memory_idx = torch.arange(R, device=dev)
        self.sample_range = (torch.arange(self.chunk, device=dev)[:, None] * 2
                             + torch.tensor([0, 2], device=dev)).contiguous()
        self._temporal = torch.empty(R, 72, 6, 6, dtype=torch.float32, device=dev)

    @property
    def fused(self) -> torch.Tensor:
        """Fused features in sample order [S,72,6,6] (a copy; the runner keeps them time-major)."""
        return self.fused_t.transpose(0, 1).reshape(self.S, 72, 6, 6)

    def features(self, images, src_off, src_pitch, src_cams, dst_cams, K, E, warp_mode=gpu_warp.MODE_CV2):
        """Phase 1: fused per-sample features (all samples 2-view), stored time-major."""
        cs, T = self.chunk, self.T
        for s0 in range(0, self.S, cs):
            s1 = min(s0 + cs, self.S)
            n = s1 - s0
            c0, c1 = 2 * s0, 2 * s1
            crops = self.crops[:2 * n]
            gpu_warp.warp_crops(images, src_off[c0:c1], src_pitch[c0:c1], src_cams[c0:c1], dst_cams[c0:c1],
                                mode=warp_mode, out=crops)
            feats = self.model.backbone(crops)
            fused = self.model.fuse_views(feats, K[c0:c1], E[c0:c1], self.sample_range[:n])
            self.fused_t[:, s0 // T:s1 // T] = fused.view(n // T, T, 72, 6, 6).transpose(0, 1)
        return self.fused_t

    def run(self, E, hand_idx, skel: InputSkeletonData, valid: Optional[torch.Tensor] = None,
            stepwise: bool = False) -> RegressorOutput:
        """Phase 2: T lock-step temporal + regressor steps.  ``valid`` [n_rec*2, T] marks tracked
        hand-frames; a hand uses its memory when it was tracked in the previous frame
        (tracker.py:233-236, 278-285).  Rows of untracked hand-frames are computed but meaningless."""
        m, T, R = self.model, self.T, self.n_rec * 2
        m.reset_memory()
        dev = self.dev
        # time-major views of the per-sample inputs, built once: no gathers inside the loop
        cam0_t = E[0::2].view(R, T, 4, 4).transpose(0, 1).contiguous()
        hand_rows = hand_idx.view(R, T)[:, 0].contiguous()
        valid_t = valid.t().contiguous() if valid is not None else torch.ones(T, R, dtype=torch.bool, device=dev)
        if not stepwise:
            # one launch for all T steps (csrc/head_seq.hip): a workgroup per memory row keeps the row's state and
            # activations in LDS; bit-identical to the stepwise loop below, which stays as the check
            use_t = torch.cat([torch.zeros(1, R, dtype=torch.bool, device=dev), valid_t[:-1]], 0).contiguous()
            out = m.head_sequence(nat.HEAD_KNOWN_SKELETON, self.fused_t, cam0_t, use_t, hand_rows.repeat(T, 1), skel)
            return RegressorOutput(out.joint_angles.transpose(0, 1).reshape(self.S, 22),
                                   out.wrist_xfs.transpose(0, 1).reshape(self.S, 4, 4), None,
                                   out.landmark_uncertainty_sigmas.transpose(0, 1).reshape(self.S, 21))
        ja_t = torch.empty(T, R, 22, device=dev)
        wx_t = torch.empty(T, R, 4, 4, device=dev)
        sg_t = torch.empty(T, R, 21, device=dev)
        prev_ok = torch.zeros(R, dtype=torch.bool, device=dev)
        for t in range(T):
            temporal = m.temporal_step(self.fused_t[t], cam0_t[t], self.memory_idx, prev_ok, required_rows=R,
                                       out=self._temporal)
            m.regress_decode(nat.HEAD_KNOWN_SKELETON, temporal, cam0_t[t], hand_rows, skel,
                             out=RegressorOutput(ja_t[t], wx_t[t], None, sg_t[t]), want_raw=False)
            prev_ok = valid_t[t]
        return RegressorOutput(ja_t.transpose(0, 1).reshape(self.S, 22), wx_t.transpose(0, 1).reshape(self.S, 4, 4), None,
                               sg_t.transpose(0, 1).reshape(self.S, 21))

    def smooth_landmarks(self, landmarks: torch.Tensor, filt: LandmarkFilter, out: Optional[RegressorOutput] = None,
                         valid: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Landmarks [S,21,3] of ``run``'s poses (skin_landmarks) smoothed along every (recording, hand) row in one call; same
        order and shape.  ``out``: run's outputs, whose sigmas the filter may weigh by; ``valid`` as ``run``'s: untracked
        hand-frames hold the last landmarks once and are 0 from a gap's second frame on (LandmarkFilter.forward)."""
        T, R = self.T, self.n_rec * 2
        sig = None if out is None else out.landmark_uncertainty_sigmas.view(R, T, 21).transpose(0, 1)
        h, _ = filt(landmarks.view(R, T, 21, 3).transpose(0, 1), None if valid is None else valid.t(), sig)
        return h.transpose(0, 1).reshape(self.S, 21, 3)
