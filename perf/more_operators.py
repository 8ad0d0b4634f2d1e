"""Performance cases of the operators that train a block's own weights beside the frozen bank: the norms
around the block, the experts' products in float types, and the step of their optimiser.

  norm          x' = x + scale * sigmoid(gate) * n(y), h = n(x'), n(v) = v / sqrt(mean(v^2) + eps) * w: the norm
                after a block with its gate and residual scale, and the norm before the next one
                (MoEExecutor.block_norm)
  norm_grad     the gradients of x, y, the gate's logits and both norms' weights (MoEExecutor.block_norm_backward)
  experts       y[t][i] = W[ids[t][i]] x[t][i]: the (token, slot) rows grouped by expert, then one product a
                group, of ragged sizes (MoEExecutor.group_rows, then MoEExecutor.expert_mul)
  experts_grad  the gradients of x and W for dy, with the groups that the forward pass has made
                (MoEExecutor.expert_mul_backward)
  adamw         an AdamW step over many tensors at once, moments in 32 or in 8 bits, with the gradients' norm
                clipped (AdamW.step, and AdamW.moments, which reads the moments back)

Sizes are those of runtime/workloads.py and the tests (2048 / 768, 2560 / 640, top-10 of 512, top-8 of 128), or
generic ones around them.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ESIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
SCALE = 0.5                                     # of the block's branch on the residual stream
LR, BETA1, BETA2, ADAM_EPS, DECAY, MAX_NORM, STEP = 1e-3, 0.9, 0.999, 1e-8, 0.01, 1.0, 100
BLOCK = 256                                     # values that share a scale where moments have 8 bits


def _norm(kind, tokens, width, dtype, after="norm", gate=True, before=True):
    """after: "norm" (y is normed), "plain" (y is added as it is) or "none" (no y)."""
    return {"kind": kind, "tokens": tokens, "width": width, "dtype": dtype, "after": after, "gate": gate, "before": before}


def _experts(kind, tokens, experts, slots, k, rows, dtype, each=False, padded=False):
    """each: x has a row per slot; padded: the last tokens have no expert (-1)."""
    return {"kind": kind, "tokens": tokens, "experts": experts, "slots": slots, "k": k, "rows": rows, "dtype": dtype,
            "each": each, "padded": padded}


def _adamw(count, a, b, dtype, bits, clip=True):
    """count tensors, of a and b values in turn; 16-bit ones have a 32-bit master copy."""
    return {"kind": "adamw", "count": count, "a": a, "b": b, "dtype": dtype, "bits": bits, "clip": clip}


def listed():
    cases = {
        # one token decodes: the residual stream between two blocks
        "norm_decode_t1": _norm("norm", 1, 2048, "f32"),
        # a prompt batch at the shipped model's width, without gates
        "norm_prompt_t4001": _norm("norm", 4001, 2560, "bf16", gate=False),
        # a small training batch of a narrow model, y added as it is
        "norm_grad_t333": _norm("norm_grad", 333, 640, "f16", after="plain"),
        # a training batch
        "norm_grad_t16384": _norm("norm_grad", 16384, 2048, "bf16"),
        # one token decodes on experts kept in bf16: the gate rows, top-10 of 512
        "experts_decode_t1": _experts("experts", 1, 512, 10, 2048, 768, "bf16"),
        # drafted tokens of many requests verified together: the down rows, top-8 of 128
        "experts_verify_t47": _experts("experts", 47, 128, 8, 768, 2048, "f16", each=True),
        # a padded training batch, the gate rows, top-8 of 128
        "experts_t8191": _experts("experts", 8191, 128, 8, 2048, 768, "bf16", padded=True),
        # a small batch on few experts in f32
        "experts_grad_t300": _experts("experts_grad", 300, 8, 2, 2560, 640, "f32"),
        # a training batch, the down rows, top-8 of 128
        "experts_grad_t4096": _experts("experts_grad", 4096, 128, 8, 768, 2048, "bf16", each=True),
        # the adapters of 48 layers: 96 small tensors in f32
        "adamw_adapters": _adamw(96, 16 * 2048, 16 * 768, "f32", 32),
        # gate, up and down of 64 experts in bf16 with master copies, moments in 8 bits
        "adamw_experts_bits8": _adamw(3, 64 * 2048 * 768, 64 * 2048 * 768, "bf16", 8),
        # the same of 128 experts in f32, moments in 32 bits
        "adamw_experts": _adamw(3, 128 * 2048 * 768, 128 * 2048 * 768, "f32", 32, clip=False),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = [work(c) for c in listed()]
    most = {q: max(w[q] for w in top) for q in ("bytes", "flops")}
    while True:
        kind = rng.choices(["norm", "norm_grad", "experts", "experts_grad", "adamw"], [2, 2, 4, 4, 3])[0]
        dtype = rng.choice(["f32", "f16", "bf16"])
        if kind.startswith("norm"):
            width = rng.choice([512, 640, 768, 1024, 2048, 2560, rng.randint(1, 8192), rng.randint(1, 8192)])
            after = rng.choice(["norm", "norm", "plain", "none"])
            case = _norm(kind, _log_int(rng, 1, 16384), width, dtype, after, after != "none" and rng.random() < 0.5,
                         after == "none" or rng.random() < 0.8)
        elif kind.startswith("experts"):
            experts, slots = rng.choice([(8, 2), (60, 6), (64, 6), (128, 8), (512, 10)])
            k, rows = rng.choice([(2048, 768), (768, 2048), (2560, 640), (640, 2560), (1024, 2048),
                                  (rng.randint(16, 2560), rng.randint(16, 2560))])
            case = _experts(kind, _log_int(rng, 1 if kind == "experts" else 16, 8192), experts, slots, k, rows, dtype,
                            rng.random() < 0.5, rng.random() < 0.3)
            if dtype == "f32" and work(case)["flops"] > 2e10:
                continue
        else:
            bits = rng.choice([8, 32])
            case = _adamw(_log_int(rng, 1, 400), _log_int(rng, 1, 1 << 24), _log_int(rng, 1, 1 << 24), dtype, bits,
                          rng.random() < 0.6)
            if sum(_sizes(case)) > 1 << 28:
                continue
        w = work(case)
        if all(w[q] <= most[q] for q in most):
            return case


def _sizes(case):
    return [case["b"] if i % 2 else case["a"] for i in range(case["count"])]


def work(case):
    es = ESIZE[case["dtype"]]
    if case["kind"].startswith("norm"):
        T, d = case["tokens"], case["width"]
        weights = (case["after"] == "norm") + case["before"]
        if case["kind"] == "norm":
            rows = 1 + 2 * (case["after"] != "none") + case["before"]   # x, y, x' and h
        else:
            rows = 4 if case["before"] else 1                           # the gradients of x' and h, x', that of x
            rows += (case["after"] != "none") + (case["after"] == "norm" or case["gate"])   # that of y, y
            weights *= 2
        return {"bytes": T * d * rows * es + 4 * d * weights + 4 * T * case["gate"], "flops": 8 * T * d * (weights + 1)}
    if case["kind"].startswith("experts"):
        T, K, E, k, rows = (case[q] for q in ("tokens", "slots", "experts", "k", "rows"))
        R = T * K
        used = E * (1.0 - (1.0 - K / E) ** T) * k * rows
        x = (R if case["each"] else T) * k
        if case["kind"] == "experts":
            return {"bytes": int(es * (used + x + R * rows) + 4 * R), "flops": 2 * R * k * rows}
        return {"bytes": int(es * (used + x + R * rows + R * k) + 4 * E * k * rows), "flops": 4 * R * k * rows}
    n = sum(_sizes(case))
    moments = 16 if case["bits"] == 32 else 4 + 8                       # read and written; 8 bits: and read back as values
    each = 4 + moments + (8 if es == 4 else 10)                         # the gradient; the weights and their master copies
    return {"bytes": n * each, "flops": 16 * n}


# ---- inputs ---------------------------------------------------------------
def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 6007 + 29)
    dt = DTYPES[case["dtype"]]
    st = dict(case=case)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=DEVICE, dtype=dtype)
    if case["kind"].startswith("norm"):
        T, d = case["tokens"], case["width"]
        st["x"] = (normal(T, d) * 2).to(dt)                             # backward: x', as the forward pass left it
        st["y"] = normal(T, d).to(dt) if case["after"] != "none" else None
        st["gate"] = normal(T) if case["gate"] else None
        st["w_after"] = 1 + 0.2 * normal(d) if case["after"] == "norm" else None
        st["w_before"] = 1 + 0.2 * normal(d) if case["before"] else None
        if case["kind"] == "norm_grad":
            st["dout"] = (normal(T, d) * 0.01).to(dt)
            st["dh"] = (normal(T, d) * 0.01).to(dt) if case["before"] else None
    elif case["kind"].startswith("experts"):
        T, K, E, k, rows = (case[q] for q in ("tokens", "slots", "experts", "k", "rows"))
        logits = normal(T, E) + 0.3 * normal(E)
        st["ids"] = logits.topk(K, dim=1).indices.to(torch.int32)
        if case["padded"]:
            st["ids"][T - T // 16:] = -1
        st["x"] = normal(T, K if case["each"] else 1, k, dtype=dt)
        st["w"] = normal(E, rows, k, dtype=dt) * 0.02
        if case["kind"] == "experts_grad":
            st["dy"] = normal(T, K, rows, dtype=dt) * 0.01
    else:
        sizes = _sizes(case)
        st["at"], n = [], 0                                             # each tensor starts at a block's start
        for s in sizes:
            st["at"].append((n, n + s))
            n += -(-s // BLOCK) * BLOCK
        inside = torch.zeros(n, device=DEVICE)
        for lo, hi in st["at"]:
            inside[lo:hi] = 1
        master = normal(n) * 0.02 * inside
        st["p"] = master.to(dt)
        st["master"] = master if dt != torch.float32 else None
        st["g"] = normal(n) * 1e-3 * inside
        if case["bits"] == 32:
            st["m"] = normal(n) * 1e-4 * inside
            st["v"] = normal(n).square() * 1e-6 * inside
        else:
            def codes(least, most):
                c = torch.randint(least, most + 1, (n // BLOCK, BLOCK), generator=gen, device=DEVICE, dtype=torch.int16)
                c[:, 0] = most                                          # a block's largest value is its scale
                return c * inside.reshape(-1, BLOCK).to(torch.int16)
            st["m_code"], st["v_code"] = codes(-127, 127).to(torch.int8), codes(1, 255).to(torch.uint8)
            st["m_scale"] = torch.exp(normal(n // BLOCK, 1)) * 1e-4
            st["v_scale"] = torch.exp(normal(n // BLOCK, 1)) * 1e-6
        st["t"] = STEP
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        _prepare_own(st)
    elif case["kind"].startswith("experts"):
        # rows of the longest group: the capacity that a padded product needs
        ids = st["ids"].reshape(-1)
        st["capacity"] = int(torch.bincount(ids[ids >= 0].long(), minlength=case["experts"]).max())
    elif case["kind"] == "adamw":
        decay = [1 - LR * (0.0 if i % 2 else DECAY) for i in range(case["count"])]
        blocks = torch.tensor([-(-(hi - lo) // BLOCK) for lo, hi in st["at"]], device=DEVICE)
        st["decay"] = torch.tensor(decay, device=DEVICE).repeat_interleave(blocks)[:, None]
    return st


# ---- the framework's calls ---------------------------------------------------
def _prepare_own(st):
    root = os.path.abspath("sabah-moe-accelerator_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from sabah.runtime.adamw import AdamW
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    from sabah.runtime.experts import FloatExperts, RowGroups
    from sabah.runtime.norm import BlockNorm
    case = st["case"]
    ex = st["ex"] = MoEExecutor(ExpertBank(1, 8, 256, 256, {"gate": 21, "up": 21, "down": 21}, device=DEVICE))
    if case["kind"].startswith("norm"):
        st["norm"] = BlockNorm(case["width"], after=case["after"] == "norm", before=case["before"], eps=EPS, scale=SCALE,
                               device=DEVICE)
        if case["after"] == "norm":
            st["norm"].w_after.copy_(st["w_after"])
        if case["before"]:
            st["norm"].w_before.copy_(st["w_before"])
    elif case["kind"].startswith("experts"):
        T, K, E, k, rows = (case[q] for q in ("tokens", "slots", "experts", "k", "rows"))
        st["experts"] = FloatExperts(E, k, rows, dtype=st["w"].dtype, device=DEVICE)
        st["experts"].w.copy_(st.pop("w"))
        st["groups"] = RowGroups(T, K, E, device=DEVICE)
        if case["kind"] == "experts":
            st["y"] = torch.empty(T, K, rows, dtype=st["x"].dtype, device=DEVICE)
        else:
            ex.group_rows(st["ids"], out=st["groups"])                  # the forward pass's
            st["dx"] = torch.empty(T, K, k, dtype=st["x"].dtype, device=DEVICE)
            st["dw"] = torch.empty(E, rows, k, device=DEVICE)
    else:
        opt = st["opt"] = AdamW([st["p"][lo:hi] for lo, hi in st["at"]], [st["g"][lo:hi] for lo, hi in st["at"]],
                                lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
                                weight_decay=[0.0 if i % 2 else DECAY for i in range(case["count"])], bits=case["bits"],
                                master=st["master"] is not None, max_norm=MAX_NORM if case["clip"] else None)
        if case["bits"] == 32:
            opt.load_moments(st.pop("m"), st.pop("v"), STEP)
        else:
            m = (_signed(st.pop("m_code").double()) * st.pop("m_scale")).float()
            v = (_unsigned(st.pop("v_code").double()) * st.pop("v_scale")).float()
            opt.load_moments(m.reshape(-1), v.reshape(-1), STEP)
        if st["master"] is not None:
            opt.master.copy_(st.pop("master"))


def _run_own(st):
    case, ex = st["case"], st.get("ex")
    if case["kind"] == "norm":
        return ex.block_norm(st["norm"], st["x"], st["y"], st["gate"])
    if case["kind"] == "norm_grad":
        return tuple(ex.block_norm_backward(st["norm"], st["x"], st["y"], st["gate"], dout=st["dout"], dh=st["dh"]))
    if case["kind"] == "experts":
        groups = ex.group_rows(st["ids"], out=st["groups"])
        return ex.expert_mul(st["experts"], st["x"], groups, out=st["y"])
    if case["kind"] == "experts_grad":
        return ex.expert_mul_backward(st["experts"], st["x"], st["groups"], st["dy"], dx=st["dx"], dw=st["dw"])
    opt = st["opt"]
    opt.step()
    return st["p"], opt.master, opt.moments(), opt.grad_norm if case["clip"] else None


# ---- the plain forms ------------------------------------------------------------
def run(st):
    if own:
        return _run_own(st)
    kind = st["case"]["kind"]
    if kind.startswith("norm"):
        return _plain_norm(st) if kind == "norm" else _plain_norm_grad(st)
    return _plain_adamw(st) if kind == "adamw" else _plain_experts(st, kind == "experts_grad")


def _inverse_rms(v):
    return 1.0 / torch.sqrt((v * v).mean(dim=1, keepdim=True) + EPS)


def _plain_norm(st):
    x, y, dt = st["x"].float(), st["y"], st["x"].dtype
    out = None
    if y is not None:
        y = y.float()
        if st["w_after"] is not None:
            y = y * _inverse_rms(y) * st["w_after"]
        if st["gate"] is not None:
            y = y * (1.0 / (1.0 + torch.exp(-st["gate"])))[:, None]
        out = (x + SCALE * y).to(dt)
        x = out.float()                                                 # the next block's norm is of what is kept
    h = (x * _inverse_rms(x) * st["w_before"]).to(dt) if st["w_before"] is not None else None
    return out, h


def _plain_norm_back(v, dn, w):
    """The gradients of v and w through n(v; w)."""
    r = _inverse_rms(v)
    unit, d = v * r, dn * w
    return r * (d - unit * (d * unit).mean(dim=1, keepdim=True)), (dn * unit).sum(dim=0)


def _plain_norm_grad(st):
    x, dt = st["x"].float(), st["x"].dtype
    d = st["dout"].float()
    dy = dgate = dw_after = dw_before = None
    if st["w_before"] is not None:
        part, dw_before = _plain_norm_back(x, st["dh"].float(), st["w_before"])
        d = d + part
    if st["y"] is not None:
        y = st["y"].float()
        n = y * _inverse_rms(y) * st["w_after"] if st["w_after"] is not None else y
        dn = SCALE * d
        if st["gate"] is not None:
            g = 1.0 / (1.0 + torch.exp(-st["gate"]))
            dgate = g * (1.0 - g) * (dn * n).sum(dim=1)
            dn = dn * g[:, None]
        dy = dn
        if st["w_after"] is not None:
            dy, dw_after = _plain_norm_back(y, dn, st["w_after"])
        dy = dy.to(dt)
    return d.to(dt), dy, dgate, dw_after, dw_before


def _plain_experts(st, grad):
    case = st["case"]
    T, K, E, k, rows = (case[q] for q in ("tokens", "slots", "experts", "k", "rows"))
    R, dt = T * K, st["x"].dtype
    e = st["ids"].reshape(-1).long()
    some = e >= 0
    x = st["x"].float().expand(T, K, k).reshape(R, k)
    if R <= E and not grad:                                             # a matrix for each row
        w = st["w"].index_select(0, e.clamp(min=0)).float()
        y = torch.bmm(w, x[:, :, None])[:, :, 0] * some[:, None]
        return y.reshape(T, K, rows).to(dt)
    # rows at their places in a batch of `capacity` rows for each expert; the last place is of rows without one
    C = st["capacity"]
    key = torch.where(some, e, E)
    order = torch.argsort(key, stable=True)
    counts = (key[:, None] == torch.arange(E + 1, device=key.device)).sum(dim=0)
    start = torch.cumsum(counts, dim=0) - counts
    rank = torch.empty_like(order)
    rank[order] = torch.arange(R, device=key.device) - start[key[order]]
    place = torch.where(some, key * C + rank, E * C)
    xs = torch.zeros(E * C + 1, k, device=key.device)
    xs[place] = x
    xs = xs[:E * C].reshape(E, C, k)
    w = st["w"].float()
    if not grad:
        ys = torch.bmm(xs, w.transpose(1, 2)).reshape(E * C, rows)
        y = ys[place.clamp(max=E * C - 1)] * some[:, None]
        return y.reshape(T, K, rows).to(dt)
    dys = torch.zeros(E * C + 1, rows, device=key.device)
    dys[place] = st["dy"].float().reshape(R, rows)
    dys = dys[:E * C].reshape(E, C, rows)
    dxs = torch.bmm(dys, w).reshape(E * C, k)
    dx = dxs[place.clamp(max=E * C - 1)] * some[:, None]
    xs = xs * (torch.arange(C, device=key.device)[:, None] < counts[:E, None, None])
    return dx.reshape(T, K, k).to(dt), torch.bmm(dys.transpose(1, 2), xs)


def _signed(code, most=127.0):
    """What codes of m stand for, in shares of their block's scale: even steps of the square root."""
    q = code / most
    return q * q.abs()


def _unsigned(code, most=255.0):
    """The same of v: even steps of the fourth root."""
    q = code / most
    q = q * q
    return q * q


def _plain_adamw(st):
    case = st["case"]
    st["t"] += 1
    # codes of 8 bits are found in 64: next to a border between two of them an error of 32 bits is a whole step
    wide = torch.float32 if case["bits"] == 32 else torch.float64
    norm, c = None, 1.0
    if case["clip"]:
        total = torch.sqrt(st["g"].double().square().sum())
        norm = total.float().reshape(1)
        c = (MAX_NORM / (total + 1e-6)).clamp(max=1.0).to(wide)
    g = st["g"].reshape(-1, BLOCK).to(wide) * c
    if case["bits"] == 32:
        m, v = st["m"].reshape(-1, BLOCK), st["v"].reshape(-1, BLOCK)
    else:
        m, v = _signed(st["m_code"].to(wide)) * st["m_scale"], _unsigned(st["v_code"].to(wide)) * st["v_scale"]
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    rate, root = LR / (1 - BETA1 ** st["t"]), 1 / math.sqrt(1 - BETA2 ** st["t"])
    p = (st["p"] if st["master"] is None else st["master"]).reshape(-1, BLOCK)
    p.copy_(p * st["decay"] - m / (torch.sqrt(v) * root + ADAM_EPS) * rate)
    if st["master"] is not None:
        st["p"].copy_(st["master"])
    if case["bits"] == 32:
        st["m"].copy_(m.reshape(-1))
        st["v"].copy_(v.reshape(-1))
        return st["p"], st["master"], (st["m"], st["v"]), norm
    # a block's scale is its largest value, in 32 bits
    st["m_scale"], st["v_scale"] = m.abs().amax(dim=1, keepdim=True).float(), v.amax(dim=1, keepdim=True).float()
    at = torch.sqrt(m.abs() / st["m_scale"].to(wide).clamp(min=1e-45)) * 127.0
    m_code = (torch.round(at) * torch.sign(m)).clamp(min=-127.0, max=127.0)
    at = torch.round(torch.sqrt(torch.sqrt(v / st["v_scale"].to(wide).clamp(min=1e-45))) * 255.0)
    v_code = torch.where(v > 0, at.clamp(min=1.0), at).clamp(max=255.0)  # no v above 0 becomes 0
    st["m_code"], st["v_code"] = m_code.to(torch.int8), v_code.to(torch.uint8)
    m, v = _signed(m_code) * st["m_scale"], _unsigned(v_code) * st["v_scale"]
    return st["p"], st["master"], (m.reshape(-1).float(), v.reshape(-1).float()), norm


# ---- the definitions in 64 bits -------------------------------------------------
def exact(case, seed):
    st = _inputs(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(st)
    if case["kind"] == "norm_grad":
        return _exact_norm_grad(st)
    if case["kind"].startswith("experts"):
        return _exact_experts(st, case["kind"] == "experts_grad")
    return _exact_adamw(st)


def _exact_norm(st):
    x, out = st["x"].double(), None
    if st["y"] is not None:
        b = st["y"].double()
        if st["w_after"] is not None:
            b = b * torch.rsqrt(b.square().mean(1, keepdim=True) + EPS) * st["w_after"].double()
        if st["gate"] is not None:
            b = torch.sigmoid(st["gate"].double())[:, None] * b
        out = x + SCALE * b
        x = out.to(st["x"].dtype).double()
    h = None
    if st["w_before"] is not None:
        h = st["w_before"].double() * x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
    return out, h


def _exact_norm_grad(st):
    """By the chain rule through u = v r, r = (mean v^2 + eps)^(-1/2), dr/dv = -r^3 v / d."""
    def through(v, w, dn):
        width = v.shape[1]
        r = (v.square().sum(1) / width + EPS).pow(-0.5)[:, None]
        dv = dn * w * r - v * r.pow(3) * (dn * w * v).sum(1, keepdim=True) / width
        return dv, (dn * v * r).sum(0)
    x, d = st["x"].double(), st["dout"].double()
    dy = dgate = dw_after = dw_before = None
    if st["w_before"] is not None:
        dv, dw_before = through(x, st["w_before"].double(), st["dh"].double())
        d = d + dv
    if st["y"] is not None:
        y, s = st["y"].double(), torch.full((x.shape[0], 1), SCALE, device=x.device, dtype=torch.float64)
        if st["gate"] is not None:
            g = torch.sigmoid(st["gate"].double())[:, None]
            w = st["w_after"].double() if st["w_after"] is not None else None
            n = y if w is None else y * (y.square().mean(1, keepdim=True) + EPS).pow(-0.5) * w
            dgate = (s * g * (1 - g) * n * d).sum(1)
            s = s * g
        if st["w_after"] is not None:
            dy, dw_after = through(y, st["w_after"].double(), s * d)
        else:
            dy = s * d
    return d, dy, dgate, dw_after, dw_before


def _exact_experts(st, grad):
    case = st["case"]
    T, K, E, k, rows = (case[q] for q in ("tokens", "slots", "experts", "k", "rows"))
    e = st["ids"].reshape(-1)
    x = st["x"].expand(T, K, k).reshape(T * K, k)
    y = torch.zeros(T * K, k if grad else rows, dtype=torch.float64, device=x.device)
    if grad:
        dw = torch.zeros(E, rows, k, dtype=torch.float64, device=x.device)
        dy = st["dy"].reshape(T * K, rows)
    for n in torch.unique(e[e >= 0]).tolist():
        at = torch.nonzero(e == n)[:, 0]
        w = st["w"][n].double()
        if grad:
            d = dy[at].double()
            y[at] = d @ w
            dw[n] = d.t() @ x[at].double()
        else:
            y[at] = x[at].double() @ w.t()
    y = y.reshape(T, K, -1)
    return (y, dw) if grad else y


def _exact_adamw(st):
    case, t = st["case"], STEP + 1
    g = st["g"].double().reshape(-1, BLOCK)
    norm, c = None, 1.0
    if case["clip"]:
        norm = g.square().sum().sqrt().reshape(1)
        c = min(1.0, MAX_NORM / (float(norm) + 1e-6))
    g = c * g
    if case["bits"] == 32:
        m, v = st["m"].double().reshape(-1, BLOCK), st["v"].double().reshape(-1, BLOCK)
    else:
        m = st["m_code"].double()
        m = torch.sign(m) * (m / 127).square() * st["m_scale"].double()
        v = (st["v_code"].double() / 255).pow(4) * st["v_scale"].double()
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g.square(), v, BETA2)
    p = st["p"] if st["master"] is None else st["master"]
    p = p.double().reshape(-1, BLOCK)
    blocks = torch.tensor([-(-(hi - lo) // BLOCK) for lo, hi in st["at"]], device=p.device)
    decay = torch.tensor([0.0 if i % 2 else DECAY for i in range(case["count"])], device=p.device, dtype=torch.float64)
    p = p - LR * decay.repeat_interleave(blocks)[:, None] * p
    p = p - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS)
    if case["bits"] == 8:
        ms, vs = m.abs().amax(1, keepdim=True).float().double(), v.amax(1, keepdim=True).float().double()
        tiny = torch.finfo(torch.float64).tiny
        m = torch.sign(m) * (torch.round(127 * (m.abs() / ms.clamp(min=tiny)).sqrt()) / 127).square() * ms
        code = torch.round(255 * (v / vs.clamp(min=tiny)).pow(0.25))
        v = (torch.where(v > 0, code.clamp(min=1), code) / 255).pow(4) * vs
    p = p.reshape(-1)
    return p, None if st["master"] is None else p, (m.reshape(-1), v.reshape(-1)), norm
