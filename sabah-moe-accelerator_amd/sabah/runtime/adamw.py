"""
Sabah / runtime / adamw

AdamW over many tensors at once: adapters (LoraBank.a, .b), experts (FloatExperts.w),
norms' weights, a router's matrix, with the gradients that the executor's backward calls write.
"""
from __future__ import annotations

import ctypes

import torch

from . import rt
from .lora import TYPES

BLOCK = 256                                     # values that share a scale where moments have 8 bits


class AdamW:
    """One step a call over all `params` from `grads` (tensors of the same numbers of values; both contiguous, in
    float32, float16 or bfloat16, kept by reference: write new gradients into the same tensors):
        g = c * grad;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
        p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
    lr: a number, or a float32 tensor [1] on the device, read by the step itself (a captured one follows it).  `lr` and
    `max_norm` may be set between steps, lr from a number to a tensor too, a max_norm only where there was one.
    weight_decay: a number, or one for each tensor.  bits: 32 or 8, of the moments; 8 are codes with a scale for each
    256 values (sabah_adamw_desc in include/sabah_rt.h), a quarter of the memory.  A step stores the nearest codes, which
    lose what is less than half a step of them: with a beta2 of 0.999 v comes out too large, 1.1 times after 2,000 steps of even
    noise, 1.4 times after 5,000 (and growing), 45 times where a block's gradients but one become a tenth, and steps too
    small by its root.  unbiased: one of the two codes around a value, in proportion to where it lies between, chosen by the
    step's number and the value's place: right in the mean, with a noise of about 9 % of a large v; for runs of more than some
    hundred steps.  master: tensors of 16 bits have a
    float32 copy, which is what steps read and change (new values go into the copy too); without it small steps are lost in the tensor's rounding.  max_norm: the
    gradients are scaled down to that norm; a step whose norm is infinite or NaN changes nothing (`grad_norm`
    [1] says it: it is infinite or NaN after such steps alone, and at most f32's largest number after others); None: neither.

    `step_count` [1] int64, `m`, `v` (and `m_scale`, `v_scale`, `master`) are the state, on the device.  In the flat ones each tensor
    begins at a multiple of 256: tensor i at `starts[i]`."""

    def __init__(self, params, grads, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01, bits: int = 32,
                 master: bool = False, max_norm: float | None = None, unbiased: bool = False):
        self.params, self.grads = list(params), list(grads)
        n = len(self.params)
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [float(weight_decay)] * n
        if not n or len(self.grads) != n or len(decay) != n:
            raise ValueError("adamw: %d tensors, %d gradients, %d decays" % (n, len(self.grads), len(decay)))
        if bits not in (8, 32):
            raise ValueError("adamw: moments of %r bits, expected 32 or 8" % (bits,))
        if unbiased and bits != 8:
            raise ValueError("adamw: unbiased codes are of 8 bits, not of %d" % bits)
        self.device, self.index = self.params[0].device, self.params[0].get_device()
        for p, g in zip(self.params, self.grads):
            if (p.dtype not in TYPES or g.dtype not in TYPES or p.numel() != g.numel() or not p.is_contiguous()
                    or not g.is_contiguous() or p.get_device() != self.index or g.get_device() != self.index):
                raise ValueError("adamw: tensor %s %s with gradient %s %s, expected contiguous float ones on %s"
                                 % (tuple(p.shape), p.dtype, tuple(g.shape), g.dtype, self.device))
        if self.index >= 0:
            rt.init(self.index)
        self.bits, self.unbiased, self.max_norm, self.lr = bits, unbiased, max_norm, lr
        self._rate()
        self.starts, self.n_values = [], 0
        for p in self.params:
            self.starts.append(self.n_values)
            self.n_values += -(-p.numel() // BLOCK) * BLOCK
        dev, blocks = self.device, self.n_values // BLOCK
        self.master = None
        if master and any(p.dtype != torch.float32 for p in self.params):
            self.master = torch.zeros(self.n_values, dtype=torch.float32, device=dev)
            for p, at in zip(self.params, self.starts):
                self.master[at:at + p.numel()].copy_(p.detach().reshape(-1))
        self.m = torch.zeros(self.n_values, dtype=torch.float32 if bits == 32 else torch.int8, device=dev)
        self.v = torch.zeros(self.n_values, dtype=torch.float32 if bits == 32 else torch.uint8, device=dev)
        self.m_scale = torch.zeros(blocks, dtype=torch.float32, device=dev) if bits == 8 else None
        self.v_scale = torch.zeros(blocks, dtype=torch.float32, device=dev) if bits == 8 else None
        self.step_count = torch.zeros(1, dtype=torch.int64, device=dev)
        self.grad_norm = torch.zeros(1, dtype=torch.float32, device=dev) if max_norm is not None else None
        lib = rt.lib()
        ts = (rt.AdamWTensor * n)()
        for i, (p, g) in enumerate(zip(self.params, self.grads)):
            own = self.master is not None and p.dtype != torch.float32 and p.numel()
            ts[i] = rt.AdamWTensor(p.data_ptr(), g.data_ptr(), self.master.data_ptr() + 4 * self.starts[i] if own else None,
                                   decay[i], p.numel(), TYPES[p.dtype], TYPES[g.dtype])
        values = ctypes.c_longlong()
        size = lib.sabah_adamw_table_bytes(ts, n, ctypes.byref(values))
        if not size:
            rt.check(-1, "adamw")
        host = torch.empty(size, dtype=torch.uint8)
        rt.check(lib.sabah_adamw_table(ts, n, host.data_ptr(), size), "adamw")
        self.table = host.to(dev)
        self.workspace = torch.empty(lib.sabah_adamw_workspace(), dtype=torch.uint8, device=dev)
        self.desc = rt.AdamWDesc(self.table.data_ptr(), size, n, bits | (rt.ADAMW_UNBIASED if unbiased else 0),
                                 self.m.data_ptr(), self.v.data_ptr(), self.m_scale.data_ptr() if bits == 8 else None,
                                 self.v_scale.data_ptr() if bits == 8 else None, self._rate()[0], betas[0], betas[1], eps, 1.0,
                                 max_norm or 0.0, self._rate()[1], self.step_count.data_ptr(),
                                 self.grad_norm.data_ptr() if max_norm is not None else None, self.workspace.data_ptr(),
                                 self.workspace.numel())
        self.ref = ctypes.byref(self.desc)

    def _on_gpu(self) -> None:
        if self.index < 0:
            raise ValueError("adamw: the tensors are on %s, not on a GPU" % self.device)

    def _rate(self):
        """(lr, d_lr) of the C descriptor."""
        lr = self.lr
        if not isinstance(lr, torch.Tensor):
            return float(lr), None
        if lr.dtype != torch.float32 or lr.numel() != 1 or lr.get_device() != self.index:
            raise ValueError("adamw: lr is %s %s, expected float32 [1] on %s" % (tuple(lr.shape), lr.dtype, self.device))
        return 0.0, lr.data_ptr()

    def step(self, grad_scale: float = 1.0) -> None:
        """One step on torch's current stream.  grad_scale: what the gradients are multiplied by first (one over a loss scale)."""
        self._on_gpu()
        if (self.max_norm is None) != (self.grad_norm is None):
            raise ValueError("adamw: max_norm %r, the steps were made %s one" % (self.max_norm, "with" if self.max_norm is None else "without"))
        d = self.desc
        d.lr, d.d_lr = self._rate()
        d.max_norm = self.max_norm or 0.0
        d.grad_scale = grad_scale
        rc = rt.lib().sabah_adamw_step(self.ref, torch._C._cuda_getCurrentRawStream(self.index))
        if rc:
            rt.check(rc, "adamw step")

    def moments(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(m, v) as flat f32 values: the state itself with 32 bits, with 8 bits what the codes stand for."""
        if self.bits == 32:
            return self.m, self.v
        self._on_gpu()
        m = torch.empty(self.n_values, dtype=torch.float32, device=self.device)
        v = torch.empty(self.n_values, dtype=torch.float32, device=self.device)
        rt.check(rt.lib().sabah_adamw_moments_read(
            self.m.data_ptr(), self.v.data_ptr(), self.m_scale.data_ptr(), self.v_scale.data_ptr(), self.n_values,
            m.data_ptr(), v.data_ptr(), torch._C._cuda_getCurrentRawStream(self.index)), "adamw moments")
        return m, v

    def load_moments(self, m: torch.Tensor, v: torch.Tensor, step: int) -> None:
        """Flat f32 moments in the layout of moments() (zeros between the tensors) and the number of steps made: a checkpoint's."""
        if step < 0:
            raise ValueError("adamw: %d steps made" % step)
        for t in (m, v):
            if t.dtype != torch.float32 or t.shape != (self.n_values,) or not t.is_contiguous() or t.get_device() != self.index:
                raise ValueError("adamw: moments %s %s, expected contiguous f32 [%d] on %s"
                                 % (tuple(t.shape), t.dtype, self.n_values, self.device))
        if self.bits == 32:
            self.m.copy_(m)
            self.v.copy_(v)
        else:
            self._on_gpu()
            rt.check(rt.lib().sabah_adamw_moments_write(
                m.data_ptr(), v.data_ptr(), self.n_values, self.m.data_ptr(), self.v.data_ptr(), self.m_scale.data_ptr(),
                self.v_scale.data_ptr(), torch._C._cuda_getCurrentRawStream(self.index)), "adamw moments")
        self.step_count.fill_(step)
