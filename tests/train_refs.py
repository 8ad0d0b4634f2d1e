"""Plain forms in 64 bits of a block's norms, the experts' products and AdamW, with the error bounds that
follow from 32-bit sums.  u: half a step of f32 next to 1; a value rounded to a type is off by half a step of it."""
import math

import torch

U = 2.0 ** -24


def half_step(v, dtype):
    """What one rounding of v to dtype may change (16 bits; f32's is in the bounds of the sums)."""
    if dtype == torch.float32:
        return torch.zeros_like(v)
    info = torch.finfo(dtype)
    return v.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def close(got, want, tol, what=""):
    got, want, tol = got.detach().double().cpu(), want.detach().double().cpu(), tol.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), [(got[tuple(i)].item(), want[tuple(i)].item(), tol[tuple(i)].item())
                                                 for i in bad.nonzero()[:4].tolist()])


# ---- norms.  A row's sum of squares is of positive terms: each of its (at most 16 in a lane, 6 across lanes, 16 waves)
# additions and the product is off by u of the sum, so it by 39 u; its root's inverse by half of that, 3 more roundings and
# 2 of the products behind it: 25 u of the result, 32 with exp and the sigmoid's.  Sums of signed terms are off by 40 u
# of the sum of their sizes.
def norm(x, y, gate, wa, wb, eps, scale):
    """(out, branch size): before rounding."""
    x = x.double()
    if y is None:
        return x, torch.zeros_like(x)
    b = y.double()
    if wa is not None:
        b = b / torch.sqrt(b.square().mean(1, keepdim=True) + eps) * wa.double()
    b = b * scale
    if gate is not None:
        b = b * torch.sigmoid(gate.double())[:, None]
    return x + b, b.abs()


def norm_h(out, wb, eps):
    out = out.double()
    return out / torch.sqrt(out.square().mean(1, keepdim=True) + eps) * wb.double()


def norm_back(out, y, gate, wa, wb, dout, dh, eps, scale):
    """{name: (value, bound)}, bounds before the last rounding."""
    out = out.double()
    D = out.shape[1]
    d = dout.double() if dout is not None else torch.zeros_like(out)
    size, res = d.abs(), {}
    if wb is not None:
        g = dh.double()
        r = 1 / torch.sqrt(out.square().mean(1, keepdim=True) + eps)
        u, gw = out * r, g * wb.double()
        d = d + r * (gw - u * (gw * u).sum(1, keepdim=True) / D)
        size = size + r * (gw.abs() + u.abs() * (gw * u).abs().sum(1, keepdim=True) / D)
        res["dw_before"] = (g * u).sum(0), (64 + 32) * U * (g * u).abs().sum(0)
        res["dx"] = d, 80 * U * size
    if y is not None:
        y, s = y.double(), torch.full_like(out[:, :1], scale)
        sg = torch.sigmoid(gate.double())[:, None] if gate is not None else None
        if gate is not None:
            s = s * sg
        n, r = y, None
        if wa is not None:
            r = 1 / torch.sqrt(y.square().mean(1, keepdim=True) + eps)
            n = y * r * wa.double()
        if gate is not None:
            res["dgate"] = ((1 - sg) * s * (d * n).sum(1, keepdim=True))[:, 0], \
                (200 * U * (1 - sg) * s.abs() * (size * n.abs()).sum(1, keepdim=True))[:, 0]
        if wa is not None:
            u, dn = y * r, s * d * wa.double()
            big = s.abs() * size * wa.double().abs()
            res["dy"] = r * (dn - u * (dn * u).sum(1, keepdim=True) / D), \
                200 * U * r * (big + u.abs() * (big * u.abs()).sum(1, keepdim=True) / D)
            res["dw_after"] = (s * d * u).sum(0), (64 + 200) * U * (s.abs() * size * u.abs()).sum(0)
        else:
            res["dy"] = s * d, 120 * U * s.abs() * size
    return res


# ---- experts -----------------------------------------------------------------
def expert_mul(w, x, ids):
    """y [T, K, rows] in 64 bits and its bound: each of the sum's k additions is off by at most a step (2 u) of the terms'
    sizes.  NaN for a bad id, zeros for -1."""
    T, K = ids.shape
    E, rows, k = w.shape
    x = x.double().reshape(T, -1, k).expand(T, K, k)
    y, size = torch.zeros(T, K, rows, dtype=torch.float64), torch.zeros(T, K, rows, dtype=torch.float64)
    for e in range(E):
        at = ids == e
        if at.any():
            y[at] = x[at] @ w[e].double().t()
            size[at] = x[at].abs() @ w[e].double().abs().t()
    y[(ids < -1) | (ids >= E)] = math.nan
    return y, 2 * U * (k + 4) * size


def expert_back(w, x, ids, dy):
    """((dx, bound), (dw, bound))."""
    T, K = ids.shape
    E, rows, k = w.shape
    x, dy = x.double().reshape(T, -1, k).expand(T, K, k), dy.double()
    dx, sx = torch.zeros(T, K, k, dtype=torch.float64), torch.zeros(T, K, k, dtype=torch.float64)
    dw, sw = torch.zeros(E, rows, k, dtype=torch.float64), torch.zeros(E, rows, k, dtype=torch.float64)
    n = 0
    for e in range(E):
        at = ids == e
        if at.any():
            n = max(n, int(at.sum()))
            dx[at], sx[at] = dy[at] @ w[e].double(), dy[at].abs() @ w[e].double().abs()
            dw[e], sw[e] = dy[at].t() @ x[at], dy[at].abs().t() @ x[at].abs()
    dx[(ids < -1) | (ids >= E)] = math.nan
    return (dx, 2 * U * (rows + 4) * sx), (dw, 2 * U * (n + 4) * sw)


# ---- AdamW -------------------------------------------------------------------
def m_value(code):
    q = code.double() / 127
    return q * q.abs()


def v_value(code):
    return (code.double() / 255).pow(4)


def m_code(m, scale):
    """(code, distance of the root from the nearest border) of values against their blocks' scales."""
    at = (m.double().abs() / scale.double().clamp(min=1e-300)).sqrt() * 127
    return torch.round(at).clamp(max=127) * torch.sign(m.double()), (at - torch.floor(at) - 0.5).abs()


def v_code(v, scale):
    at = (v.double() / scale.double().clamp(min=1e-300)).pow(0.25) * 255
    code = torch.round(at).clamp(max=255)
    return torch.where(v > 0, code.clamp(min=1), code), (at - torch.floor(at) - 0.5).abs()


def adamw(p, g, m, v, t, lr, betas, eps, decay, c):
    b1, b2 = betas
    g = g.double() * c
    m = b1 * m.double() + (1 - b1) * g
    v = b2 * v.double() + (1 - b2) * g * g
    step = lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps)
    return p.double() * (1 - lr * decay) - step, m, v, step
