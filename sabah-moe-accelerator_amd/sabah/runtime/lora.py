"""
Sabah / runtime / lora

Low-rank adapters of a projection, resident beside the expert bank.  Many
requests run at once on one frozen bank, each with its own fine-tune: a pair
A [rank, k], B [rows, rank] and a scale per adapter, or a pair per (adapter,
expert) where the experts' own matrices are adapted (MUL_MAT_ID).  The bank
holds them in the checkpoints' layout, so a pair is loaded by a copy.

MoEExecutor.lora_apply adds them to a projection's output, lora_backward gives
their gradients.
"""
from __future__ import annotations

import ctypes

import torch

from . import rt

# ggml type codes of the adapters' storage types
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
MAX_RANK = 128


class LoraBank:
    """n_adapters adapters of up to `rank` for a projection k -> rows: `a`
    [n_adapters, n_experts, rank, k] and `b` [n_adapters, n_experts, rows, rank] in one
    type, `scale` [n_adapters] f32 and `ranks` [n_adapters] int32 (an
    adapter's own rank; what lies past it is not read into the result).  The
    tensors are the bank's own: change their values, not the tensors."""

    def __init__(self, n_adapters: int, rank: int, k: int, rows: int, n_experts: int = 1,
                 dtype: torch.dtype = torch.bfloat16, device: str = "cuda:0"):
        if dtype not in TYPES:
            raise ValueError("adapters are float32, float16 or bfloat16, not %s" % dtype)
        if min(n_adapters, rank, k, rows, n_experts) <= 0 or rank > MAX_RANK:
            raise ValueError("adapter bank of %d adapters, %d experts, rank %d (at most %d), %d -> %d"
                             % (n_adapters, n_experts, rank, MAX_RANK, k, rows))
        self.n_adapters, self.n_experts, self.rank, self.k, self.rows = n_adapters, n_experts, rank, k, rows
        self.dtype, self.device = dtype, torch.device(device)
        self.a = torch.zeros(n_adapters, n_experts, rank, k, dtype=dtype, device=device)
        self.b = torch.zeros(n_adapters, n_experts, rows, rank, dtype=dtype, device=device)
        self.scale = torch.ones(n_adapters, dtype=torch.float32, device=device)
        self.ranks = torch.full((n_adapters,), rank, dtype=torch.int32, device=device)
        self.desc = rt.LoraDesc(self.a.data_ptr(), self.b.data_ptr(), self.scale.data_ptr(), self.ranks.data_ptr(),
                                TYPES[dtype], n_adapters, n_experts, rank, k, rows)
        self.ref = ctypes.byref(self.desc)
        self.index = self.a.get_device()
        self._space = {}

    def space(self, lib, slots: int, tokens: int, backward: int = 0) -> int:
        """sabah_lora_workspace of a call, asked once for each size."""
        key = (slots, tokens, backward)
        n = self._space.get(key)
        if n is None:
            if len(self._space) > 4096:
                self._space.clear()
            n = self._space[key] = lib.sabah_lora_workspace(self.ref, slots, tokens, backward)
        return n

    def load(self, adapter: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """One adapter: a [r, k] and b [rows, r], or [n_experts, r, k] and [n_experts, rows, r],
        with r up to the bank's rank."""
        if not 0 <= adapter < self.n_adapters:
            raise IndexError("adapter %d outside [0, %d)" % (adapter, self.n_adapters))
        if a.dim() == 2 and b.dim() == 2:
            a, b = a[None], b[None]
        r = a.shape[1] if a.dim() == 3 else -1
        if a.shape != (self.n_experts, r, self.k) or b.shape != (self.n_experts, self.rows, r) or r > self.rank:
            raise ValueError("adapter of shapes %s and %s in a bank of %d experts, rank %d, %d -> %d"
                             % (tuple(a.shape), tuple(b.shape), self.n_experts, self.rank, self.k, self.rows))
        self.a[adapter].zero_()
        self.b[adapter].zero_()
        self.a[adapter, :, :r].copy_(a)
        self.b[adapter, :, :, :r].copy_(b)
        self.scale[adapter] = scale
        self.ranks[adapter] = r
