"""
Sabah / runtime / experts

Experts kept in a float type, beside the quantised bank: what is trained, or served
as it was trained.  MoEExecutor.group_rows groups the (token, slot) rows by expert, once for all products
over the same ids; expert_mul and expert_mul_backward are one projection's products.
"""
from __future__ import annotations

import ctypes

import torch

from . import rt
from .lora import TYPES


class FloatExperts:
    """One projection's matrices `w` [n_experts, rows, k] in float32, float16 or bfloat16 (zeros at first).  The tensor is
    the object's own: change its values, not the tensor."""

    def __init__(self, n_experts: int, k: int, rows: int, dtype: torch.dtype = torch.bfloat16, device: str = "cuda:0"):
        if dtype not in TYPES:
            raise ValueError("experts are float32, float16 or bfloat16, not %s" % dtype)
        if min(n_experts, k, rows) <= 0:
            raise ValueError("%d experts, %d -> %d" % (n_experts, k, rows))
        self.n_experts, self.k, self.rows, self.dtype, self.device = n_experts, k, rows, dtype, torch.device(device)
        self.w = torch.zeros(n_experts, rows, k, dtype=dtype, device=device)
        self.index = self.w.get_device()
        self.desc = rt.ExpertDesc(self.w.data_ptr(), TYPES[dtype], n_experts, k, rows)
        self.ref = ctypes.byref(self.desc)


class RowGroups:
    """The rows of n_tokens tokens with n_ids slots each, grouped by expert (MoEExecutor.group_rows writes it).  Products
    read it until they have run; a captured graph keeps it."""

    def __init__(self, n_tokens: int, n_ids: int, n_experts: int, device: str = "cuda:0"):
        self.bytes = rt.lib().sabah_expert_groups_bytes(n_ids, n_tokens, n_experts)
        if not self.bytes:
            rt.check(-1, "expert groups")
        self.n_tokens, self.n_ids, self.n_experts = n_tokens, n_ids, n_experts
        self.buffer = torch.zeros(self.bytes, dtype=torch.uint8, device=device)
        self.index = self.buffer.get_device()
