"""
Sabah / runtime / executor

Executes routed-MoE work on the HBM-resident bank.

The contract this file keeps (the reference's, executor.py:1-16):

    given router output (expert ids, routing weights), the arithmetic performed
    is exactly

        y = sum_k  w_k * W_down[e_k]^T ( silu(W_gate[e_k]^T x) * W_up[e_k]^T x )

    over the ids the router produced, using those experts' real quantized
    weights - with the activations quantised to q8 as ggml's CPU path does.

Every method calls the HIP runtime through the C ABI; there is no host-side
arithmetic and no fallback.  Work is enqueued on torch's current stream
(except `run_block`, which keeps the reference's library-stream signature).
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import rt
from .bank import ROLES, DenseExpert, ExpertBank
from .lora import LoraBank


# A small call is bound by what Python does before the launch, so the hot
# methods read each tensor's strides once and pass plain integers where the
# binding declares pointers.  Measured on an eager Q4_K gate node, one token (kernel 5 us):
# 9.7 us a call before, 7.2 after; the router at 8 tokens 8.9, 7.6.
def _stream(device) -> int:
    """The handle of torch's current stream on the device (no Stream object made)."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if device.index is None else device.index)


def _vp(t: torch.Tensor) -> int:
    return t.data_ptr()


class RouterBalance:
    """What MoEExecutor.balance computes, kept for the gradient: `counts` [n_groups, n_experts] int32,
    `mean_p` [n_groups, n_experts], `losses` [2] (balance loss, z loss) and `n_valid`
    [n_groups + 2] int32 (valid tokens of each group, of all, groups with any)."""

    def __init__(self, n_experts: int, n_groups: int = 1, device: str = "cuda:0"):
        self.n_experts, self.n_groups = n_experts, n_groups
        self.counts = torch.empty(n_groups, n_experts, dtype=torch.int32, device=device)
        self.mean_p = torch.empty(n_groups, n_experts, dtype=torch.float32, device=device)
        self.losses = torch.empty(2, dtype=torch.float32, device=device)
        self.n_valid = torch.empty(n_groups + 2, dtype=torch.int32, device=device)


class MoEExecutor:
    def __init__(self, bank: ExpertBank, max_used: int = 16, max_tokens: int = 512,
                 shared: DenseExpert | None = None):
        rt.init(bank.device.index or 0)
        self.bank = bank
        self.shared = shared
        self.device = bank.device
        self._index = bank.storage.get_device()
        self.d_model = bank.d_model
        self.ff = bank.d_ff
        self.max_used = max_used
        dev = self.device
        self.d_x = torch.zeros(self.d_model, dtype=torch.float32, device=dev)
        self.d_out = torch.zeros(self.d_model, dtype=torch.float32, device=dev)
        self.d_h = torch.zeros(max_used * self.ff, dtype=torch.float32, device=dev)
        self.d_w = torch.zeros(max_used, dtype=torch.float32, device=dev)
        self.d_ptr = torch.zeros(3 * max_used, dtype=torch.int64, device=dev)

    # ---- reference-shaped block API (executor.py:42-98) --------------------
    def upload_x(self, x: np.ndarray) -> None:
        x = np.ascontiguousarray(x, dtype=np.float32)
        if x.size != self.d_model:
            raise ValueError("x has %d elements, expected %d" % (x.size, self.d_model))
        self.d_x.copy_(torch.from_numpy(x))
        torch.cuda.current_stream(self.device).synchronize()

    def download_out(self) -> np.ndarray:
        self.sync()
        return self.d_out.cpu().numpy()

    def zero_out(self) -> None:
        self.d_out.zero_()
        torch.cuda.current_stream(self.device).synchronize()

    def run_block(self, block: int, ids, weights, accumulate: bool = False) -> None:
        """One MoE block for one token through sabah_moe_block (pointer table + weights on the device)."""
        ids = [int(i) for i in ids]
        w = np.ascontiguousarray(weights, dtype=np.float32)
        n = len(ids)
        if n != w.size:
            raise ValueError("%d ids but %d weights" % (n, w.size))
        if n > self.max_used:
            raise ValueError("n_used %d exceeds executor capacity %d" % (n, self.max_used))
        flat = np.array([self.bank.expert_ptr(block, r, e) for r in ROLES for e in ids], dtype=np.int64)
        self.d_ptr[:3 * n].copy_(torch.from_numpy(flat))
        self.d_w[:n].copy_(torch.from_numpy(w))
        torch.cuda.current_stream(self.device).synchronize()     # the block runs on the library stream
        q = {r: self.bank.layer_qtype(block, r) for r in ROLES}
        rt.check(rt.lib().sabah_moe_block(_vp(self.d_x), _vp(self.d_out), _vp(self.d_h), _vp(self.d_ptr),
                                          _vp(self.d_w), self.d_model, self.ff, n,
                                          q["gate"], q["up"], q["down"], 1 if accumulate else 0), "moe_block")

    def sync(self) -> None:
        rt.check(rt.lib().sabah_sync_compute(), "sync library stream")
        torch.cuda.current_stream(self.device).synchronize()

    # ---- the drop-in operator ----------------------------------------------
    def mul_mat_id(self, layer: int, role: str, x: torch.Tensor, ids: torch.Tensor,
                   out: torch.Tensor | None = None, source: int | None = None, lora: LoraBank | None = None,
                   adapters: torch.Tensor | None = None) -> torch.Tensor:
        """ggml MUL_MAT_ID through sabah_rt_mul_mat_id_v2 on (layer, role).

        x [n_tokens, x_rows, k] f32 (x_rows = 1 or n_ids), ids [n_tokens, n_ids] i32
        -> [n_tokens, n_ids, rows] f32.  `source` overrides the src0 address
        (e.g. a registered caller-side key).  With `lora` and `adapters` [n_tokens] i32
        each token's adapter is added (lora_apply): a pair per expert, or one
        pair for all when the adapter bank has one expert."""
        b = self.bank
        T, n_ids = ids.shape
        rows, k, qt = b.rows[role], b.cols[role], b.layer_qtype(layer, role)
        if lora is not None and (adapters is None or lora.n_experts not in (1, b.n_experts)
                                 or (lora.k, lora.rows) != (k, rows)):
            raise ValueError("adapters of %d experts, %d -> %d, beside a bank of %d, %d -> %d"
                             % (lora.n_experts, lora.k, lora.rows, b.n_experts, k, rows))
        if out is None:
            out = torch.empty((T, n_ids, rows), dtype=torch.float32, device=self.device)
        src = b.base_ptr(layer, role) if source is None else source
        row_bytes = rt.row_bytes(qt, k)
        xs, ns, os = x.stride(), ids.stride(), out.stride()
        ids_ptr = ids.data_ptr()
        rc = rt.lib().sabah_rt_mul_mat_id_v2(
            src, rows * row_bytes, row_bytes,
            x.data_ptr(), xs[1] * 4, x.shape[1], xs[0] * 4,
            ids_ptr, ns[1] * 4, ns[0] * 4, n_ids, T,
            out.data_ptr(), os[1] * 4, os[0] * 4,
            rows, k, b.n_experts, qt, _stream(self.device), ids_ptr)
        if rc:
            rt.check(rc, "MUL_MAT_ID")
        if lora is not None:
            self.lora_apply(lora, x, adapters, out, ids=ids if lora.n_experts > 1 else None, out=out)
        return out

    # ---- adapters beside a projection --------------------------------------------
    # These calls too wait for what Python does before the launch: shapes and strides are read once, and devices
    # compared as numbers.
    def _lora_rows(self, lora: LoraBank, x: torch.Tensor, adapters: torch.Tensor, ids: torch.Tensor | None,
                   y: torch.Tensor | None):
        """The checks that the two calls share; (tokens, slots, C arguments of x, adapters and ids).
        y: a tensor with the output's shape [T, rows] or [T, n_ids, rows], if there is one."""
        shape, xs, dev = x.shape, x.stride(), self._index
        if len(shape) == 3:
            xr, xi = shape[1], xs[1] * 4
        elif len(shape) == 2:
            xr, xi = 1, 0
        else:
            raise ValueError("adapters: x %s, expected [T, %d] or [T, x_rows, %d]" % (tuple(shape), lora.k, lora.k))
        T, k = shape[0], lora.k
        if ids is not None:
            ns = ids.stride()
            if ids.dtype is not torch.int32 or len(ns) != 2 or ids.shape[0] != T or ids.get_device() != dev:
                raise ValueError("adapters: ids %s %s for %d tokens" % (tuple(ids.shape), ids.dtype, T))
            slots = ids.shape[1]
            ids_args = ids.data_ptr(), ns[1] * 4, ns[0] * 4
        else:
            slots = y.shape[1] if y is not None and len(y.shape) == 3 else 1
            if lora.n_experts != 1:
                raise ValueError("adapters of %d experts need ids" % lora.n_experts)
            ids_args = None, 0, 0
        if (x.dtype is not torch.float32 or shape[-1] != k or (xs[-1] != 1 and T) or (xr != 1 and xr != slots)
                or adapters.dtype is not torch.int32 or adapters.shape != (T,)
                or not adapters.is_contiguous()):
            raise ValueError("adapters: x %s %s for %d values, adapters %s %s"
                             % (tuple(shape), x.dtype, k, tuple(adapters.shape), adapters.dtype))
        if x.get_device() != dev or adapters.get_device() != dev or lora.index != dev:
            raise ValueError("adapters: the tensors are not on %s" % self.device)
        return T, slots, (x.data_ptr(), xi, xr, xs[0] * 4, adapters.data_ptr(), *ids_args, slots, T)

    def _lora_y(self, what: str, y: torch.Tensor, T: int, slots: int, width: int):
        """(address, slot stride, token stride) of rows [T, width] or [T, slots, width] f32."""
        shape, s = y.shape, y.stride()
        three = len(shape) == 3
        if (y.dtype is not torch.float32 or shape != ((T, slots, width) if three or slots != 1 else (T, width))
                or (s[-1] != 1 and T) or y.get_device() != self._index):
            raise ValueError("adapters: %s is %s %s, expected f32 [%d, %d, %d] with contiguous rows on %s"
                             % (what, tuple(shape), y.dtype, T, slots, width, self.device))
        return (y.data_ptr(), s[1] * 4, s[0] * 4) if three else (y.data_ptr(), 0, s[0] * 4)

    def lora_apply(self, lora: LoraBank, x: torch.Tensor, adapters: torch.Tensor, base: torch.Tensor | None = None,
                   ids: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """base + scale * B (A x) with each token's adapter (sabah_lora_apply): x [T, k] or
        [T, x_rows, k] f32, adapters [T] i32 (-1: none), ids [T, n_ids] i32 where the
        bank has a pair per expert, base [T, rows] or [T, n_ids, rows] f32 (None: zeros).
        `out` may be `base` itself."""
        T, slots, rows = self._lora_rows(lora, x, adapters, ids, base if base is not None else out)
        if out is None:
            out = (torch.empty_like(base) if base is not None else
                   torch.empty((T, lora.rows) if x.dim() == 2 and ids is None else (T, slots, lora.rows),
                               dtype=torch.float32, device=self.device))
        y = self._lora_y("out", out, T, slots, lora.rows)
        b = y if base is out else self._lora_y("base", base, T, slots, lora.rows) if base is not None else (None, 0, 0)
        lib = rt.lib()
        ws, n = None, lora.space(lib, slots, T)
        if n:
            ws = torch.empty(n, dtype=torch.uint8, device=self.device)
        rc = lib.sabah_lora_apply(lora.ref, *rows, *b, *y, ws.data_ptr() if n else None, n, _stream(self.device))
        if rc:
            rt.check(rc, "lora_apply")
        return out

    def lora_backward(self, lora: LoraBank, x: torch.Tensor, adapters: torch.Tensor, dy: torch.Tensor,
                      ids: torch.Tensor | None = None, dx: torch.Tensor | None = None,
                      da: torch.Tensor | None = None, db: torch.Tensor | None = None, add_dx: bool = False,
                      add_dw: bool = False, need_dx: bool = True, need_dw: bool = True):
        """The gradients (dx, da, db) of lora_apply for dy, the gradient of its result
        (sabah_lora_backward): dx [T, k] or [T, n_ids, k], da and db f32 in the shapes of lora.a
        and lora.b, written, or with add_dx / add_dw added to the tensors given; None for
        what need_dx / need_dw leave out."""
        T, slots, rows = self._lora_rows(lora, x, adapters, ids, dy)
        if (add_dx and dx is None) or (add_dw and (da is None or db is None)):
            raise ValueError("lora_backward: add_dx needs dx, add_dw needs da and db")
        if dx is None and need_dx:
            dx = torch.empty((T, lora.k) if dy.dim() == 2 else (T, slots, lora.k), dtype=torch.float32,
                             device=self.device)
        if need_dw:
            da = torch.empty(lora.a.shape, dtype=torch.float32, device=self.device) if da is None else da
            db = torch.empty(lora.b.shape, dtype=torch.float32, device=self.device) if db is None else db
            for g, w in ((da, lora.a), (db, lora.b)):
                if g.shape != w.shape or g.dtype != torch.float32 or not g.is_contiguous() or g.get_device() != self._index:
                    raise ValueError("lora_backward: a weight gradient is %s %s, expected contiguous f32 %s"
                                     % (tuple(g.shape), g.dtype, tuple(w.shape)))
        d = self._lora_y("dx", dx, T, slots, lora.k) if need_dx else (None, 0, 0)
        n = lora.space(rt.lib(), slots, T, 1)
        ws = torch.empty(n, dtype=torch.uint8, device=self.device) if n else None
        rc = rt.lib().sabah_lora_backward(lora.ref, *rows, *self._lora_y("dy", dy, T, slots, lora.rows), *d,
                                          int(add_dx), da.data_ptr() if need_dw else None,
                                          db.data_ptr() if need_dw else None, int(add_dw),
                                          ws.data_ptr() if n else None, n, _stream(self.device))
        if rc:
            rt.check(rc, "lora_backward")
        return dx if need_dx else None, da if need_dw else None, db if need_dw else None

    # ---- fused layer / chain --------------------------------------------------
    def run_layer(self, layer: int, x: torch.Tensor, ids: torch.Tensor, w: torch.Tensor,
                  out: torch.Tensor | None = None, resid: torch.Tensor | None = None) -> torch.Tensor:
        """One MoE layer for x [T, d_model] with ids/w [T, k]; adds the shared expert if the
        executor has one and `resid` if given."""
        if out is None:
            out = torch.empty_like(x)
        desc = self.bank.layer_desc(layer, self.shared)
        T, k = ids.shape
        rt.check(rt.lib().sabah_moe_layer(ctypes.byref(desc), _vp(x), _vp(ids), _vp(w), k, T, _vp(out),
                                          _vp(resid) if resid is not None else None, _stream(self.device)),
                 "moe_layer")
        return out

    def route(self, logits: torch.Tensor, n_used: int | None = None, norm_w: bool = True,
              w_scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
        """Router gating on the device (sabah_moe_route): ids [T, n_used] int32 and
        weights [T, n_used] f32 from router logits [T, n_experts] f32."""
        k = self.max_used if n_used is None else n_used
        T, E = logits.shape
        ids = torch.empty((T, k), dtype=torch.int32, device=logits.device)
        w = torch.empty((T, k), dtype=torch.float32, device=logits.device)
        rt.check(rt.lib().sabah_moe_route(_vp(logits), T, E, k, int(norm_w), ctypes.c_float(w_scale), _vp(ids),
                                          _vp(w), _stream(self.device)), "moe_route")
        return ids, w

    def _router_rows(self, logits: torch.Tensor, ids: torch.Tensor, mask: torch.Tensor | None, n_groups: int):
        dev = self._index
        if (logits.dim() != 2 or ids.dim() != 2 or logits.dtype is not torch.float32
                or (logits.stride(1) != 1 and logits.shape[0]) or logits.get_device() != dev or ids.dtype is not torch.int32
                or ids.shape[0] != logits.shape[0] or not ids.is_contiguous() or ids.get_device() != dev):
            raise ValueError("router: logits %s %s, ids %s %s" % (tuple(logits.shape), logits.dtype, tuple(ids.shape),
                                                                 ids.dtype))
        T, E = logits.shape
        if mask is not None and (mask.dtype not in (torch.bool, torch.uint8) or mask.numel() != T
                                 or not mask.is_contiguous() or mask.get_device() != dev):
            raise ValueError("router: mask %s %s for %d tokens" % (tuple(mask.shape), mask.dtype, T))
        return T, E, ids.shape[1]

    def balance(self, logits: torch.Tensor, ids: torch.Tensor, mask: torch.Tensor | None = None, n_groups: int = 1,
                out: RouterBalance | None = None) -> RouterBalance:
        """The router's balance loss, z loss, mean probabilities and per-expert counts
        (sabah_moe_balance) from logits [T, n_experts] f32 and route()'s ids [T, n_used]
        over the tokens where mask [T] (bool or uint8) holds, in n_groups groups of equal length
        (`out` brings its own number)."""
        T, E, k = self._router_rows(logits, ids, mask, n_groups)
        if out is None:
            out = RouterBalance(E, n_groups, device=self.device)
        n_groups = out.n_groups
        if out.n_experts != E or out.counts.get_device() != self._index:
            raise ValueError("balance: %d experts on %s, out has %d on %s"
                             % (E, self.device, out.n_experts, out.counts.device))
        lib = rt.lib()
        n = lib.sabah_moe_balance_workspace(T, E, n_groups)
        if not n:
            rt.check(-1, "moe_balance")
        ws = torch.empty(n, dtype=torch.uint8, device=self.device)
        rc = lib.sabah_moe_balance(logits.data_ptr(), logits.stride(0) * 4 if T > 1 else E * 4, ids.data_ptr(),
                                   mask.data_ptr() if mask is not None else None, T, E, k, n_groups,
                                   out.counts.data_ptr(), out.mean_p.data_ptr(), out.losses.data_ptr(),
                                   out.n_valid.data_ptr(), ws.data_ptr(), n, _stream(self.device))
        if rc:
            rt.check(rc, "moe_balance")
        return out

    def route_backward(self, logits: torch.Tensor, ids: torch.Tensor, dw: torch.Tensor | None = None,
                       balance: RouterBalance | None = None, c_balance: float = 0.0, c_z: float = 0.0,
                       mask: torch.Tensor | None = None, norm_w: bool = True, w_scale: float = 1.0,
                       out: torch.Tensor | None = None) -> torch.Tensor:
        """The logits' gradient [T, n_experts] (sabah_moe_route_backward): through
        route()'s weights, dw [T, n_used] f32 (None: nothing), and of c_balance * losses[0] +
        c_z * losses[1] of `balance`, which balance() computed with the same mask."""
        n_groups = balance.n_groups if balance is not None else 1
        T, E, k = self._router_rows(logits, ids, mask, n_groups)
        if balance is not None and (balance.n_experts != E or balance.counts.get_device() != self._index):
            raise ValueError("route_backward: %d experts on %s, balance has %d on %s"
                             % (E, self.device, balance.n_experts, balance.counts.device))
        if dw is not None and (dw.dtype is not torch.float32 or dw.shape != ids.shape or not dw.is_contiguous()
                               or dw.get_device() != self._index):
            raise ValueError("route_backward: dw %s %s, ids %s" % (tuple(dw.shape), dw.dtype, tuple(ids.shape)))
        if out is None:
            out = torch.empty((T, E), dtype=torch.float32, device=self.device)
        elif (out.dtype is not torch.float32 or out.shape != logits.shape or out.stride(1) != 1
              or out.get_device() != self._index):
            raise ValueError("route_backward: out %s %s" % (tuple(out.shape), out.dtype))
        rc = rt.lib().sabah_moe_route_backward(
            logits.data_ptr(), logits.stride(0) * 4 if T > 1 else E * 4, ids.data_ptr(),
            mask.data_ptr() if mask is not None else None, T, E, k, int(norm_w), w_scale, dw.data_ptr() if dw is not None else None,
            balance.counts.data_ptr() if balance is not None else None,
            balance.n_valid.data_ptr() if balance is not None else None, n_groups, c_balance, c_z,
            out.data_ptr(), out.stride(0) * 4 if T > 1 else E * 4, _stream(self.device))
        if rc:
            rt.check(rc, "moe_route_backward")
        return out

    def run_prefill_layer(self, layer: int, x: torch.Tensor, ids: torch.Tensor, w: torch.Tensor,
                          out: torch.Tensor | None = None, resid: torch.Tensor | None = None) -> torch.Tensor:
        """run_layer computed group-major (sabah_moe_prefill_layer): the (token, slot)
        pairs grouped by expert on the device, each expert's rows read once."""
        if out is None:
            out = torch.empty_like(x)
        desc = self.bank.layer_desc(layer, self.shared)
        T, k = ids.shape
        rt.check(rt.lib().sabah_moe_prefill_layer(ctypes.byref(desc), _vp(x), _vp(ids), _vp(w), k, T, _vp(out),
                                                  _vp(resid) if resid is not None else None,
                                                  _stream(self.device)), "moe_prefill_layer")
        return out

    def layer_descs(self) -> ctypes.Array:
        arr = (rt.MoeLayerDesc * self.bank.n_layers)()
        for l in range(self.bank.n_layers):
            arr[l] = self.bank.layer_desc(l, self.shared)
        return arr

    def run_chain(self, x: torch.Tensor, ids: torch.Tensor, w: torch.Tensor, descs=None) -> torch.Tensor:
        """x <- x + layer_l(x) for every layer, in place; ids/w [n_layers, T, k]."""
        L, T, k = ids.shape
        descs = self.layer_descs() if descs is None else descs
        rt.check(rt.lib().sabah_moe_chain(descs, L, _vp(x), _vp(ids), _vp(w), k, T, _stream(self.device)),
                 "moe_chain")
        return x


class ChainGraph:
    """The decode chain (every layer's gate/up and down kernels) captured once
    as a HIP graph over static x / ids / weights buffers.  replay() copies one
    step's inputs in and replays the graph: the host submits one graph per
    step instead of two kernels per layer.  An eager call before the capture
    sizes the library scratch, so nothing is allocated inside it.  The graph
    keeps the scratch it was captured with: a later, larger call grows the
    library scratch by allocating new buffers and retires the old ones without
    freeing them (they live until sabah_rt_shutdown), so replays stay valid.
    Replays and eager calls must not overlap on different streams: both use
    the same scratch while no call has outgrown it."""

    def __init__(self, ex: MoEExecutor, n_tokens: int, k: int, descs=None):
        dev = ex.device
        self.ex = ex
        self.descs = ex.layer_descs() if descs is None else descs
        L = len(self.descs)                   # a chain may apply a layer more than once
        self.x = torch.zeros(n_tokens, ex.d_model, dtype=torch.float32, device=dev)
        self.ids = torch.zeros(L, n_tokens, k, dtype=torch.int32, device=dev)
        self.w = torch.zeros(L, n_tokens, k, dtype=torch.float32, device=dev)
        ex.run_chain(self.x, self.ids, self.w, self.descs)       # eager: sizes the library scratch
        torch.cuda.synchronize(dev)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            ex.run_chain(self.x, self.ids, self.w, self.descs)
        torch.cuda.synchronize(dev)

    def replay(self, x: torch.Tensor, ids: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
        """x [n_tokens, d_model], ids / w [n_layers, n_tokens, k]; returns the
        static output buffer (valid in stream order)."""
        self.x.copy_(x)
        self.ids.copy_(ids)
        self.w.copy_(w)
        self.graph.replay()
        return self.x

    def replay_static(self) -> torch.Tensor:
        """Replay on the inputs already in place: the graph's launches only."""
        self.graph.replay()
        return self.x
