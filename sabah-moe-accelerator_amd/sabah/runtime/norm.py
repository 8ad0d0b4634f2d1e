"""
Sabah / runtime / norm

The norms around a block: after it, with the block's gate and the scale of its
branch on the residual stream, and before the next block (MoEExecutor.block_norm,
block_norm_backward).
"""
from __future__ import annotations

import ctypes

import torch

from . import rt
from .lora import TYPES

MAX_WIDTH = 8192


class BlockNorm:
    """The weights `w_after` and `w_before` [width] f32 (ones at first; None for a norm that the block does not
    have), eps, and the branch's scale:
        out = x + scale * sigmoid(gate) * n(y; w_after),  h = n(out; w_before),
        n(v; w) = v / sqrt(mean(v^2) + eps) * w
    Without `after`, y is added as it is.  The tensors are the norm's own: change their values, not the tensors."""

    def __init__(self, width: int, after: bool = True, before: bool = True, eps: float = 1e-6, scale: float = 1.0,
                 device: str = "cuda:0"):
        if not 0 < width <= MAX_WIDTH:
            raise ValueError("norm of width %d, expected 1 to %d" % (width, MAX_WIDTH))
        self.width, self.eps, self.scale, self.device = width, float(eps), float(scale), torch.device(device)
        self.w_after = torch.ones(width, dtype=torch.float32, device=device) if after else None
        self.w_before = torch.ones(width, dtype=torch.float32, device=device) if before else None
        self.index = next((w.get_device() for w in (self.w_after, self.w_before) if w is not None), None)   # None: any
        self._descs, self._space = {}, {}

    def ref(self, dtype: torch.dtype, after: bool = True):
        """The C descriptor for activations of a type; after: whether the call has a y."""
        key = dtype, after, self.eps, self.scale
        d = self._descs.get(key)
        if d is None:
            if dtype not in TYPES:
                raise ValueError("block_norm: activations are float32, float16 or bfloat16, not %s" % dtype)
            if len(self._descs) > 64:
                self._descs.clear()
            d = self._descs[key] = ctypes.byref(rt.NormDesc(
                self.w_after.data_ptr() if after and self.w_after is not None else None,
                self.w_before.data_ptr() if self.w_before is not None else None, TYPES[dtype], self.width, self.eps, self.scale))
        return d

    def space(self, lib, tokens: int) -> int:
        """sabah_block_norm_workspace of a call, asked once for each size."""
        n = self._space.get(tokens)
        if n is None:
            if len(self._space) > 4096:
                self._space.clear()
            n = self._space[tokens] = lib.sabah_block_norm_workspace(self.width, tokens)
        return n
