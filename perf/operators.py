"""Performance cases of the operators that adapt a frozen expert bank: low-rank
adapters of many requests beside a shared projection, and the router's balance
loss, per-expert counts and gradient.

  adapters       y = base + scale_a B_a (A_a x), each token with the adapter a of
                 its request (-1: none), beside a dense projection or beside MUL_MAT_ID's
                 (token, slot) rows, where each expert has its own pair (A, B)
                 (MoEExecutor.lora_apply)
  adapters_grad  the gradients of x, A and B (MoEExecutor.lora_backward)
  balance        balance loss, z loss, mean probabilities and counts, and the losses'
                 gradient (MoEExecutor.balance, then MoEExecutor.route_backward)
  router_grad    the logits' gradient from the weights', the balance loss's and the
                 z loss's, where a training step goes backward (MoEExecutor.route_backward)

Projection sizes are those of runtime/workloads.py and the tests (2048 / 768,
2560 / 640, a shared expert of 512), or generic ones around them.
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


def _lora(kind, tokens, k, rows, rank, adapters, dtype, spread, experts=1, slots=1):
    return {"kind": kind, "tokens": tokens, "k": k, "rows": rows, "rank": rank, "adapters": adapters, "dtype": dtype,
            "spread": spread, "experts": experts, "slots": slots}


def _router(kind, tokens, experts, slots, groups=1, padded=False, norm_w=True, dw=True):
    return {"kind": kind, "tokens": tokens, "experts": experts, "slots": slots, "groups": groups, "padded": padded,
            "norm_w": norm_w, "dw": dw}


def listed():
    cases = {
        # one request decodes: one token through a square projection, one of 8 adapters
        "adapters_decode_t1": _lora("adapters", 1, 2048, 2048, 16, 8, "bf16", "each"),
        # 32 requests decode together, each with its own of 64 adapters (some with none): a shared expert's gate
        "adapters_decode_t32": _lora("adapters", 32, 2048, 512, 16, 64, "bf16", "each"),
        # drafted tokens of 30 requests verified together, an odd rank, the down projection
        "adapters_verify_t250": _lora("adapters", 250, 768, 2048, 12, 30, "f16", "mixed"),
        # adapters of the experts themselves: the gate rows of MUL_MAT_ID, top-8 of 128, four requests' prompts
        "adapters_experts_t512": _lora("adapters", 512, 2048, 768, 8, 4, "bf16", "segments", experts=128, slots=8),
        # a prompt batch of ragged requests, high rank, the shipped model's sizes
        "adapters_prompt_t1999": _lora("adapters", 1999, 2560, 640, 64, 8, "f16", "segments"),
        # the largest: a long prompt batch of 16 requests
        "adapters_prompt_t16384": _lora("adapters", 16384, 2048, 2048, 32, 16, "bf16", "segments"),
        # a small training batch, adapters kept in f32
        "adapters_grad_t512": _lora("adapters_grad", 512, 2048, 768, 16, 4, "f32", "segments"),
        # a large training batch of eight fine-tunes
        "adapters_grad_t8192": _lora("adapters_grad", 8192, 2048, 2048, 64, 8, "bf16", "segments"),
        # the router's losses and their gradient over one prompt-sized batch, top-10 of 512
        "balance_t512_e512": _router("balance", 512, 512, 10),
        # eight padded sequences, each balanced on its own, top-8 of 128
        "balance_t16384_e128": _router("balance", 16384, 128, 8, groups=8, padded=True),
        # gradient of a small batch without the weights' normalisation, an odd number of experts
        "router_grad_t300_e60": _router("router_grad", 300, 60, 6, norm_w=False),
        # gradient of a training batch of padded sequences, top-10 of 512
        "router_grad_t16384_e512": _router("router_grad", 16384, 512, 10, groups=8, padded=True),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = [work(c) for c in listed()]
    most = {q: max(w[q] for w in top) for q in ("bytes", "flops")}
    while True:
        kind = rng.choices(["adapters", "adapters_grad", "balance", "router_grad"], [5, 3, 2, 2])[0]
        if kind.startswith("adapters"):
            k, rows = rng.choice([(2048, 768), (768, 2048), (2048, 512), (2560, 640), (640, 2560), (2048, 2048),
                                  (rng.randint(33, 2560), rng.randint(33, 2560))])
            case = _lora(kind, _log_int(rng, 1 if kind == "adapters" else 16, 16384), k, rows, _log_int(rng, 4, 128),
                         _log_int(rng, 1, 64), rng.choice(["f32", "f16", "bf16"]), rng.choice(["each", "segments", "mixed"]))
            if rng.random() < 0.25:
                case["experts"], case["slots"] = rng.choice([(8, 2), (64, 6), (128, 8)])
                case["tokens"] = min(case["tokens"], 1024)
            if case["adapters"] * case["experts"] * case["rank"] > 8192:
                continue
        else:
            experts, slots = rng.choice([(8, 2), (60, 6), (64, 6), (128, 8), (256, 8), (512, 10)])
            groups = rng.choice([1, 1, 2, 8])
            case = _router(kind, groups * _log_int(rng, 1, 16384 // groups), experts, slots, groups,
                           rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.8)
        w = work(case)
        if all(w[q] <= most[q] for q in most):
            return case


def work(case):
    T, K = case["tokens"], case["slots"]
    if case["kind"] == "balance":
        E, G = case["experts"], case["groups"]
        return {"bytes": 8 * T * E + 4 * T * K + T + 8 * G * E, "flops": 14 * T * E}
    if case["kind"] == "router_grad":
        E, G = case["experts"], case["groups"]
        return {"bytes": 8 * T * E + 8 * T * K + T + 4 * G * E, "flops": 12 * T * E}
    R, k, rows, r = T * K, case["k"], case["rows"], case["rank"]
    keys = case["adapters"] * case["experts"]
    used = keys * (1.0 - (1.0 - 1.0 / keys) ** R)                       # pairs (A, B) that some row reads
    weights = int(used * r * (k + rows) * ESIZE[case["dtype"]])
    if case["kind"] == "adapters":
        return {"bytes": 4 * T * k + 8 * R * rows + weights, "flops": 2 * R * r * (k + rows)}
    return {"bytes": 8 * R * k + 4 * R * rows + weights + 4 * keys * r * (k + rows), "flops": 2 * R * r * (3 * k + 2 * rows)}


# ---- inputs ---------------------------------------------------------------
def _adapter_of_tokens(case, gen):
    """int32 [tokens]: the adapter of each token's request, about one request in sixteen without."""
    T, n = case["tokens"], case["adapters"]

    def pick(m):
        a = torch.randint(0, n, (m,), generator=gen, device=DEVICE)
        none = torch.rand(m, generator=gen, device=DEVICE) < 1 / 16
        return torch.where(none, -1, a) if m > 1 else a
    if case["spread"] == "segments":                                    # ragged requests one after the other
        m = max(1, min(T, n))
        cuts = torch.sort(torch.randint(0, T + 1, (m - 1,), generator=gen, device=DEVICE)).values
        return pick(m)[torch.bucketize(torch.arange(T, device=DEVICE), cuts, right=True)].to(torch.int32)
    return pick(T).to(torch.int32)                                      # each token its own, in any order


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 17)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)
    st = dict(case=case)
    T, K, E = case["tokens"], case["slots"], case["experts"]
    if case["kind"].startswith("adapters"):
        k, rows, r, n = case["k"], case["rows"], case["rank"], case["adapters"]
        dt = DTYPES[case["dtype"]]
        st["x"] = normal(T, 1 if case["kind"] == "adapters" else K, k)
        st["adapters"] = _adapter_of_tokens(case, gen)
        st["ids"] = None
        if E > 1:
            st["ids"] = torch.rand(T, E, generator=gen, device=DEVICE).topk(K, dim=1).indices.to(torch.int32)
        st["a"] = (normal(n, E, r, k) / math.sqrt(k)).to(dt)
        st["b"] = (normal(n, E, rows, r) * 0.02).to(dt)
        st["scale"] = (2.0 * torch.rand(n, generator=gen, device=DEVICE) + 0.25)
        if case["kind"] == "adapters":
            st["base"] = normal(T, K, rows)
            st["out"] = torch.empty(T, K, rows, device=DEVICE)
        else:
            st["dy"] = normal(T, K, rows) * 0.01
            st["dx"] = torch.empty(T, K, k, device=DEVICE)
    else:
        G = case["groups"]
        popularity = normal(E) * 0.7
        st["logits"] = normal(T, E) * 1.3 + popularity
        st["ids"] = st["logits"].topk(K, dim=1).indices.to(torch.int32)
        st["mask"] = None
        if case["padded"]:
            S = T // G
            lengths = torch.randint(1, S + 1, (G, 1), generator=gen, device=DEVICE)
            st["mask"] = (torch.arange(S, device=DEVICE) < lengths).reshape(T)
        if case["kind"] == "router_grad":
            st["dw"] = normal(T, K) * 0.01 if case["dw"] else None
            valid = torch.ones(T, device=DEVICE, dtype=torch.bool) if st["mask"] is None else st["mask"]
            st["counts"], st["n_valid"] = _counts(st["ids"], valid, E, G)
        else:
            st["dw"] = None
        st["dlogits"] = torch.empty(T, E, device=DEVICE)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        _prepare_own(st)
    return st


def _counts(ids, valid, E, G):
    """counts [G, E] of the valid tokens' ids; valid tokens of each group, of all, and groups with any."""
    T, K = ids.shape
    group = torch.arange(T, device=ids.device) // (T // G)
    at = (group[:, None] * E + ids).reshape(-1)
    one = valid[:, None].expand(T, K).reshape(-1).to(torch.int32)
    counts = torch.zeros(G * E, dtype=torch.int32, device=ids.device).index_add_(0, at, one).reshape(G, E)
    n = torch.zeros(G, dtype=torch.int32, device=ids.device).index_add_(0, group, valid.to(torch.int32))
    return counts, torch.cat([n, n.sum(dtype=torch.int32)[None], (n > 0).sum(dtype=torch.int32)[None]])


C_BALANCE, C_Z = 0.01, 0.001                                            # the losses' weights in a training loss


# ---- the framework's calls ---------------------------------------------------
def _prepare_own(st):
    root = os.path.abspath("sabah-moe-accelerator_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor, RouterBalance
    from sabah.runtime.lora import LoraBank
    case = st["case"]
    st["ex"] = MoEExecutor(ExpertBank(1, 8, 256, 256, {"gate": 21, "up": 21, "down": 21}, device=DEVICE))
    if case["kind"].startswith("adapters"):
        n, E, r, k = st["a"].shape
        lora = st["lora"] = LoraBank(n, r, k, case["rows"], n_experts=E, dtype=st["a"].dtype, device=DEVICE)
        lora.a.copy_(st["a"])
        lora.b.copy_(st["b"])
        lora.scale.copy_(st["scale"])
        if case["kind"] == "adapters_grad":
            st["da"] = torch.empty(lora.a.shape, device=DEVICE)
            st["db"] = torch.empty(lora.b.shape, device=DEVICE)
    else:
        st["balance"] = RouterBalance(case["experts"], case["groups"], device=DEVICE)
        if case["kind"] == "router_grad":
            st["balance"].counts.copy_(st["counts"])
            st["balance"].n_valid.copy_(st["n_valid"])


def _run_own(st):
    case, ex = st["case"], st["ex"]
    if case["kind"] == "adapters":
        return ex.lora_apply(st["lora"], st["x"], st["adapters"], st["base"], ids=st["ids"], out=st["out"])
    if case["kind"] == "adapters_grad":
        return ex.lora_backward(st["lora"], st["x"], st["adapters"], st["dy"], ids=st["ids"], dx=st["dx"], da=st["da"],
                                db=st["db"])
    if case["kind"] == "balance":
        b = ex.balance(st["logits"], st["ids"], mask=st["mask"], out=st["balance"])
        d = ex.route_backward(st["logits"], st["ids"], None, b, C_BALANCE, C_Z, mask=st["mask"], out=st["dlogits"])
        return b.losses, b.mean_p, b.counts, b.n_valid, d
    return ex.route_backward(st["logits"], st["ids"], st["dw"], st["balance"], C_BALANCE, C_Z, mask=st["mask"],
                             norm_w=case["norm_w"], out=st["dlogits"])


# ---- the plain forms ------------------------------------------------------------
def _key_mask(st, n, E, r):
    """[T, K, n * E * r]: 1 where a column belongs to the row's (adapter, expert)."""
    key = st["adapters"].long()[:, None]
    if st["ids"] is not None:
        key = torch.where(key >= 0, key * E + st["ids"], -1)
    else:
        key = key.expand(-1, st["case"]["slots"])
    return (key[:, :, None] == torch.arange(n * E * r, device=DEVICE) // r).float()


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    if case["kind"].startswith("adapters"):
        n, E, r, k = st["a"].shape
        rows, T, K = case["rows"], case["tokens"], case["slots"]
        a = st["a"].float().reshape(n * E * r, k)
        b = st["b"].float() * st["scale"][:, None, None, None]
        b = b.permute(0, 1, 3, 2).reshape(n * E * r, rows)
        mask = _key_mask(st, n, E, r)
        s = torch.matmul(st["x"], a.t()) * mask                         # x has one row per token, or one per slot
        if case["kind"] == "adapters":
            return st["base"] + torch.matmul(s, b)
        u = torch.matmul(st["dy"], b.t()) * mask
        dx = torch.matmul(u, a)
        da = torch.matmul(u.reshape(T * K, -1).t(), st["x"].reshape(T * K, k)).reshape(n, E, r, k)
        db = torch.matmul(s.reshape(T * K, -1).t(), st["dy"].reshape(T * K, rows)).reshape(n, E, r, rows)
        return dx, da, (db * st["scale"][:, None, None, None]).transpose(2, 3).contiguous()
    logits, ids, E, G = st["logits"], st["ids"].long(), case["experts"], case["groups"]
    T, K = ids.shape
    valid = torch.ones(T, device=DEVICE, dtype=torch.bool) if st["mask"] is None else st["mask"]
    m = logits.max(dim=1, keepdim=True).values
    e = torch.exp(logits - m)
    s = e.sum(dim=1, keepdim=True)
    p = e / s
    lse = (m + torch.log(s))[:, 0]
    counts, n_valid = _counts(ids, valid, E, G) if case["kind"] == "balance" else (st["counts"], st["n_valid"])
    n_g, n, filled = n_valid[:G, None].float(), n_valid[G].float(), n_valid[G + 1].float()
    f = counts.float() / torch.clamp(n_g * K, min=1)
    if case["kind"] == "balance":
        mean_p = (p * valid[:, None]).reshape(G, T // G, E).sum(dim=1) / torch.clamp(n_g, min=1)
        losses = torch.stack([E * (f * mean_p).sum() / filled, (lse * lse * valid).sum() / n])
    f = f.repeat_interleave(T // G, dim=0)
    weight = C_BALANCE * E / (torch.clamp(n_g, min=1) * filled)
    d = p * (f - (f * p).sum(dim=1, keepdim=True)) * weight.repeat_interleave(T // G, dim=0)
    d = d + p * (2 * C_Z / n * lse)[:, None]
    if st["dw"] is not None:
        q = p.gather(1, ids)
        if case["norm_w"]:
            q = q / q.sum(dim=1, keepdim=True)
            d = d.scatter_add(1, ids, q * (st["dw"] - (q * st["dw"]).sum(dim=1, keepdim=True)))
        else:
            d = d.scatter_add(1, ids, q * st["dw"]) - p * (q * st["dw"]).sum(dim=1, keepdim=True)
    d = d * valid[:, None]
    return (losses, mean_p, counts, n_valid, d) if case["kind"] == "balance" else d


# ---- the definitions in 64 bits -------------------------------------------------
def exact(case, seed):
    st = _inputs(case, seed)
    if case["kind"].startswith("adapters"):
        return _exact_adapters(st)
    return _exact_router(st)


def _exact_adapters(st):
    case = st["case"]
    T, K, E = case["tokens"], case["slots"], case["experts"]
    grad = case["kind"] == "adapters_grad"
    x = st["x"].double().expand(T, K, -1).reshape(T * K, -1)
    who = st["adapters"].long()[:, None].expand(T, K).reshape(-1)
    which = torch.zeros_like(who) if st["ids"] is None else st["ids"].long().reshape(-1)
    if grad:
        dy = st["dy"].double().reshape(T * K, -1)
        dx = torch.zeros_like(x)
        da, db = torch.zeros_like(st["a"], dtype=torch.float64), torch.zeros_like(st["b"], dtype=torch.float64)
    else:
        y = st["base"].double().reshape(T * K, -1).clone()
    for key in torch.unique(torch.where(who >= 0, who * E + which, -1)).tolist():
        if key < 0:
            continue
        n, e = divmod(key, E)
        at = torch.nonzero((who == n) & (which == e))[:, 0]
        A, B, c = st["a"][n, e].double(), st["b"][n, e].double(), st["scale"][n].double()
        s = x[at] @ A.t().contiguous()
        if not grad:
            y[at] += c * (s @ B.t().contiguous())
            continue
        u = c * (dy[at] @ B)
        dx[at] = u @ A
        da[n, e] = u.t().contiguous() @ x[at]
        db[n, e] = c * (dy[at].t().contiguous() @ s)
    if grad:
        return dx.reshape(T, K, -1), da, db
    return y.reshape(T, K, -1)


def _exact_router(st):
    case = st["case"]
    T, E, K, G = case["tokens"], case["experts"], case["slots"], case["groups"]
    S = T // G
    logits, ids = st["logits"].double(), st["ids"].long()
    valid = torch.ones(T, device=DEVICE, dtype=torch.float64) if st["mask"] is None else st["mask"].double()
    lse = torch.logsumexp(logits, dim=1)
    p = torch.exp(logits - lse[:, None])
    chosen = torch.zeros(T, E, device=DEVICE, dtype=torch.float64)
    for j in range(K):
        chosen[torch.arange(T, device=DEVICE), ids[:, j]] += valid
    n_g = valid.reshape(G, S).sum(dim=1)
    some = n_g > 0
    n, filled = n_g.sum(), some.sum()
    counts = chosen.reshape(G, S, E).sum(dim=1)
    safe = torch.where(some, n_g, 1.0)[:, None]
    f = counts / (safe * K)
    if case["kind"] == "balance":
        mean_p = (p * valid[:, None]).reshape(G, S, E).sum(dim=1) / safe
        losses = torch.stack([E * (f * mean_p).sum() / filled, (valid * lse.square()).sum() / n])
        n_valid = torch.cat([n_g, n[None], filled[None].double()])
    # by the chain rule over p: d = p o (g - <g, p>), g the loss's derivative by p
    g = (C_BALANCE * E / (safe * filled) * f).repeat_interleave(S, dim=0)
    out = p * (g - (g * p).sum(dim=1, keepdim=True)) + 2 * C_Z / n * lse[:, None] * p
    if st["dw"] is not None:
        dw = st["dw"].double()
        picked = torch.gather(logits, 1, ids)
        if case["norm_w"]:
            q = torch.softmax(picked, dim=1)
            part = q * (dw - (q * dw).sum(dim=1, keepdim=True))
            rows = torch.arange(T, device=DEVICE)
            for j in range(K):
                out[rows, ids[:, j]] += part[:, j]
        else:
            h = torch.zeros_like(p)
            for j in range(K):
                h[torch.arange(T, device=DEVICE), ids[:, j]] += dw[:, j]
            out += p * (h - (h * p).sum(dim=1, keepdim=True))
    out = out * valid[:, None]
    if case["kind"] == "balance":
        return losses, mean_p, counts.to(torch.int32), n_valid.to(torch.int32), out
    return out
