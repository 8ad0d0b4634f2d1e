"""Plain 64-bit forms of the operators that adapt a frozen bank, with a bound on
what f32 sums may be off by.  Every bound counts roundings: a sum of n products
rounded once each is off by at most n u sum |terms|, u = 2^-24 (half of
torch.finfo(float32).eps, relative), whatever the order of its terms."""
import numpy as np

U = 2.0 ** -24


def lora_forward(x, adapters, ids, a, b, scale, ranks, base):
    """x [T, x_rows, k], adapters [T], ids [T, n] or None, a [N, E, r, k], b [N, E, rows, r], base [T, n, rows]:
    (y, bound), float64."""
    T, n = base.shape[:2]
    y, bound = base.copy(), 2 * U * np.abs(base)
    for t in range(T):
        ad = adapters[t]
        if ad < 0:
            bound[t] = 0
            continue
        for i in range(n):
            e = 0 if ids is None else ids[t, i]
            rk = min(max(ranks[ad], 0), a.shape[2])
            A, B, c, xr = a[ad, e, :rk], b[ad, e, :, :rk], scale[ad], x[t, i % x.shape[1]]
            y[t, i] += c * (B @ (A @ xr))
            mag = abs(c) * (np.abs(B) @ (np.abs(A) @ np.abs(xr)))
            # k products into s, rank products into the row, the pieces of split operands, scale, base
            bound[t, i] += U * ((x.shape[2] + rk + 8) * mag + 2 * np.abs(y[t, i]))
    return y, bound


def lora_backward(x, adapters, ids, a, b, scale, ranks, dy):
    """((dx, da, db), bounds), float64; dx [T, n, k]."""
    T, n, rows = dy.shape
    k = x.shape[2]
    dx, da, db = np.zeros((T, n, k)), np.zeros(a.shape), np.zeros(b.shape)
    bx, ba, bb = np.zeros_like(dx), np.zeros_like(da), np.zeros_like(db)
    R = T * n
    for t in range(T):
        ad = adapters[t]
        if ad < 0:
            continue
        rk = min(max(ranks[ad], 0), a.shape[2])
        for i in range(n):
            e = 0 if ids is None else ids[t, i]
            A, B, c, xr, g = a[ad, e, :rk], b[ad, e, :, :rk], scale[ad], x[t, i % x.shape[1]], dy[t, i]
            s, u = A @ xr, c * (B.T @ g)
            sm, um = np.abs(A) @ np.abs(xr), abs(c) * (np.abs(B.T) @ np.abs(g))
            dx[t, i] = A.T @ u
            bx[t, i] = U * (rows + rk + 8) * (np.abs(A.T) @ um) + U * np.abs(dx[t, i])
            da[ad, e, :rk] += np.outer(u, xr)
            ba[ad, e, :rk] += U * (rows + R + 8) * np.outer(um, np.abs(xr))
            db[ad, e, :, :rk] += c * np.outer(g, s)
            bb[ad, e, :, :rk] += U * (k + R + 8) * abs(c) * np.outer(np.abs(g), sm)
    return (dx, da, db), (bx, ba, bb)


def router_losses(logits, ids, mask, groups):
    """counts, mean_p, losses, n_valid, valid and the bounds of mean_p and losses, float64."""
    T, E = logits.shape
    k = ids.shape[1]
    S = T // groups if groups else 0
    valid = np.ones(T, bool) if mask is None else mask.astype(bool).copy()
    valid &= ~np.all(np.isneginf(logits), axis=1)
    counts = np.zeros((groups, E), np.int64)
    psum, n_g, z, zb, spread = np.zeros((groups, E)), np.zeros(groups, np.int64), 0.0, 0.0, 0.0
    for t in range(T):
        if not valid[t]:
            continue
        g = t // S
        m = logits[t].max()
        ex = np.exp(logits[t] - m)
        lse = m + np.log(ex.sum())
        psum[g] += ex / ex.sum()
        n_g[g] += 1
        for e in ids[t]:
            counts[g, e] += 1
        z += lse * lse
        zb += 2 * abs(lse) * U * (abs(lse) + abs(m) + E + 8)
        spread = max(spread, m - logits[t][np.isfinite(logits[t])].min())
    some = n_g > 0
    safe = np.where(some, n_g, 1)[:, None]
    mean_p = psum / safe
    # the argument of exp, exp, the sum of E terms, the reciprocal, the sum over the tokens
    rel = U * (spread + E + T + 12)
    loss = (E * (counts / (safe * k) * mean_p).sum() / some.sum()) if some.any() else 0.0
    zl = z / n_g.sum() if some.any() else 0.0
    zbound = (zb / n_g.sum() + U * (T + 4) * zl) if some.any() else 0.0
    n_valid = np.concatenate([n_g, [n_g.sum()], [some.sum()]])
    return counts, mean_p, np.array([loss, zl]), n_valid, valid, rel * mean_p, np.array([rel * loss, zbound])


def router_gradient(logits, ids, valid, groups, dw, norm_w, w_scale, c_balance, c_z):
    """(dlogits, bound), float64, valid as router_losses gives it."""
    T, E = logits.shape
    k = ids.shape[1]
    S = T // groups
    counts = np.zeros((groups, E))
    n_g = valid.reshape(groups, S).sum(axis=1)
    for t in range(T):
        if valid[t]:
            np.add.at(counts[t // S], ids[t], 1)
    filled, n = max((n_g > 0).sum(), 1), max(n_g.sum(), 1)
    d, bound = np.zeros((T, E)), np.zeros((T, E))
    for t in range(T):
        if not valid[t]:
            continue
        g = t // S
        m = logits[t].max()
        ex = np.exp(logits[t] - m)
        p = ex / ex.sum()
        lse = m + np.log(ex.sum())
        finite = logits[t][np.isfinite(logits[t])]
        rel = U * (2 * (m - finite.min()) + 2 * E + 2 * k + 24)
        f = counts[g] / (n_g[g] * k)
        cb = c_balance * E / (n_g[g] * filled)
        d[t] = p * (cb * (f - f @ p) + 2 * c_z * lse / n)
        mag = p * (abs(cb) * (f + f @ p) + 2 * abs(c_z) * (abs(lse) + abs(m) + 1) / n)
        if dw is not None:
            q = p[ids[t]]
            if norm_w:
                sel = np.exp(logits[t, ids[t]] - logits[t, ids[t]].max()) if np.isfinite(logits[t, ids[t]]).any() else 0 * q
                q = sel / sel.sum() if np.sum(sel) > 0 else sel
                np.add.at(d[t], ids[t], w_scale * q * (dw[t] - q @ dw[t]))
                np.add.at(mag, ids[t], w_scale * q * (np.abs(dw[t]) + q @ np.abs(dw[t])))
            else:
                h = np.zeros(E)
                np.add.at(h, ids[t], dw[t])
                d[t] += w_scale * p * (h - q @ dw[t])
                np.add.at(mag, ids[t], w_scale * q * np.abs(dw[t]))
                mag += w_scale * p * (q @ np.abs(dw[t]))
        # p below 2^-126 may be held with fewer bits or as zero: each p is off by at most that, and the
        # gradient by that times what multiplies p (or q)
        tiny = 2.0 ** -126 * (abs(cb) * (f + f @ p).max() + 2 * abs(c_z * lse) / n + 1
                              + (0 if dw is None else w_scale * 2 * np.abs(dw[t]).sum()))
        bound[t] = rel * mag + tiny
    return d, bound
