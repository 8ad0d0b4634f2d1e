"""The router's losses, counts and gradient (needs an MI355X), against the 64-bit
forms of adapt_refs.py within their counted roundings."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import adapt_refs as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def ex(hip_rt):
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    return MoEExecutor(ExpertBank(1, 8, 256, 256, {"gate": 21, "up": 21, "down": 21}, device="cuda:0"))


def T(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def batch(seed, n, E, k, groups=1, masked=0.0, spread=1.5):
    g = np.random.default_rng(seed)
    logits = (g.standard_normal((n, E)) * spread + g.standard_normal(E)).astype(np.float32)
    mask = g.random(n) >= masked if masked else None
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :k].astype(np.int32)
    return logits, ids, mask, g.standard_normal((n, k)).astype(np.float32)


def close(got, want, bound, what):
    got = got.double().cpu().numpy().reshape(np.shape(want))
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g of its bound" % (
        what, bad.sum(), bad.size, np.nanmax(np.abs(got - want) / np.maximum(bound, 1e-300)))


def check(ex, logits, ids, mask, dw, groups, norm_w=True, w_scale=1.0, c=(0.7, 0.3)):
    counts, mean_p, losses, n_valid, valid, pb, lb = ref.router_losses(logits.astype(np.float64), ids, mask, groups)
    d_l, d_i, d_m, d_w = T(logits), T(ids), None if mask is None else T(mask), None if dw is None else T(dw)
    b = ex.balance(d_l, d_i, mask=d_m, n_groups=groups)
    torch.cuda.synchronize()
    assert np.array_equal(b.counts.cpu().numpy(), counts) and np.array_equal(b.n_valid.cpu().numpy(), n_valid)
    close(b.mean_p, mean_p, pb, "mean_p")
    close(b.losses, losses, lb, "losses")
    want, bound = ref.router_gradient(logits.astype(np.float64), ids, valid, groups,
                                      None if dw is None else dw.astype(np.float64), norm_w, w_scale, *c)
    got = ex.route_backward(d_l, d_i, d_w, b, *c, mask=d_m, norm_w=norm_w, w_scale=w_scale,
                            out=torch.full_like(d_l, float("nan")))
    close(got, want, bound, "dlogits")
    return b, got


@pytest.mark.parametrize("n,E,k,groups,masked", [
    (1, 1, 1, 1, 0), (1, 8, 2, 1, 0), (3, 60, 6, 1, 0), (64, 64, 64, 1, 0), (65, 65, 3, 1, 0.3), (250, 128, 8, 1, 0),
    (512, 512, 10, 1, 0.1), (77, 513, 10, 7, 0.5), (96, 300, 5, 8, 0.3), (40, 1000, 16, 2, 0.2), (12, 2048, 8, 1, 0),
    (10, 4096, 64, 5, 0.2), (2500, 16, 4, 1, 0.5), (1200, 8, 2, 300, 0.6)])
@pytest.mark.parametrize("norm_w", [True, False])
def test_losses_counts_and_gradient(ex, n, E, k, groups, masked, norm_w):
    logits, ids, mask, dw = batch(n + E, n, E, k, groups, masked)
    check(ex, logits, ids, mask, dw, groups, norm_w, 1.0 if norm_w else 2.5)


@pytest.mark.parametrize("c,with_dw", [((0.0, 0.0), True), ((0.5, 0.0), False), ((0.0, 0.5), False), ((0.0, 0.0), False)])
def test_each_part_of_the_gradient_alone(ex, c, with_dw):
    logits, ids, mask, dw = batch(5, 90, 128, 8, 3, 0.2)
    check(ex, logits, ids, mask, dw if with_dw else None, 3, c=c)
    got = ex.route_backward(T(logits), T(ids), T(dw))
    want, bound = ref.router_gradient(logits.astype(np.float64), ids, np.ones(90, bool), 1, dw.astype(np.float64), True,
                                      1.0, 0, 0)
    close(got, want, bound, "without losses")


@pytest.mark.parametrize("E,k", [(24, 4), (512, 10), (700, 8)])
def test_masked_experts_rows_and_groups(ex, E, k):
    """Minus infinities and the type's lowest value in places, rows of nothing but minus
    infinities, NaN in masked tokens' rows, a group with no token left."""
    logits, ids, _, dw = batch(E, 60, E, k)
    logits[1, ::2] = -np.inf
    logits[2, 1::3] = np.finfo(np.float32).min
    logits[3, 1:] = -np.inf                                             # one expert left: p = 1 there
    logits[4, :] = -np.inf
    logits[5, :] = np.finfo(np.float32).min                             # all equal: p = 1 / E, no infinities; lse^2 overflows
    logits[6] *= 30
    mask = np.ones(60, bool)
    mask[5] = False
    mask[7] = False
    mask[20:30] = False
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :k].astype(np.int32)
    poisoned = logits.copy()
    poisoned[7] = np.nan
    poisoned[20:30] = np.inf
    bad_ids, bad_dw = ids.copy(), dw.copy()
    bad_ids[20:30] = 9999
    bad_dw[7] = np.nan
    logits[2] = poisoned[2]
    counts, mean_p, losses, n_valid, valid, pb, lb = ref.router_losses(
        np.where(mask[:, None], logits, 0).astype(np.float64), ids, mask, 6)
    assert not valid[4] and n_valid[2] == 0
    b = ex.balance(T(poisoned), T(bad_ids), mask=T(mask), n_groups=6)
    torch.cuda.synchronize()
    assert np.array_equal(b.counts.cpu().numpy(), counts) and np.array_equal(b.n_valid.cpu().numpy(), n_valid)
    # row 2's spread of 3e38 passes through exp as an exact 0
    finite = np.where(np.isfinite(logits) & (logits > -1e30), logits, np.nan)
    finite = finite[~np.isnan(finite).all(axis=1)]
    rel = ref.U * (np.nanmax(np.nanmax(finite, 1) - np.nanmin(finite, 1)) + E + 60 + 12)
    close(b.mean_p, mean_p, rel * mean_p, "mean_p")
    close(b.losses, losses, rel * losses * 4, "losses")
    safe = np.where(mask[:, None], np.maximum(logits, -1e5), 0).astype(np.float64)
    safe[np.isneginf(logits) & mask[:, None]] = -np.inf
    want, bound = ref.router_gradient(safe, ids, valid, 6, np.where(mask[:, None], dw, 0).astype(np.float64), True, 1.0,
                                      0.7, 0.3)
    got = ex.route_backward(T(poisoned), T(bad_ids), T(bad_dw), b, 0.7, 0.3, mask=T(mask))
    close(got, want, bound, "dlogits")
    assert not got[torch.from_numpy(~valid).to(DEV)].any()
    from sabah.runtime import rt
    rt.check(rt.lib().sabah_rt_check_errors(), "masked tokens' ids are not read")


def test_a_batch_without_valid_tokens_and_an_empty_one(ex):
    logits, ids, _, dw = batch(1, 12, 16, 2)
    b, got = check(ex, logits, ids, np.zeros(12, bool), dw, 3)
    assert not b.losses.any() and not b.mean_p.any() and not b.counts.any() and not got.any()
    e = ex.balance(T(logits)[:0], T(ids)[:0], n_groups=2)
    assert not e.losses.any() and not e.mean_p.any() and not e.counts.any() and not e.n_valid.any()
    assert ex.route_backward(T(logits)[:0], T(ids)[:0], T(dw)[:0], e, 0.5, 0.5).shape == (0, 16)


def test_an_expert_named_twice_gets_both_parts(ex):
    logits, ids, _, dw = batch(2, 30, 40, 6)
    ids[:, 3] = ids[:, 0]
    ids[5] = ids[5, 0]
    check(ex, logits, ids, None, dw, 1, True)
    check(ex, logits, ids, None, dw, 1, False)


def test_nan_logits_are_passed_on(ex):
    logits, ids, _, dw = batch(3, 20, 96, 4)
    logits[4, 7] = np.nan
    logits[5, :] = np.nan
    b = ex.balance(T(logits), T(ids))
    got = ex.route_backward(T(logits), T(ids), T(dw))
    assert b.losses.isnan().all() and b.mean_p.isnan().all() and b.n_valid.tolist() == [20, 20, 1]
    assert got[5].isnan().all() and got[[0, 1, 2, 3] + list(range(6, 20))].isfinite().all()


@pytest.mark.parametrize("E", [48, 512, 3000])
def test_an_id_out_of_range_fails_the_next_call(ex, hip_rt, E):
    logits, ids, _, dw = batch(E, 9, E, 4)
    want = ex.balance(T(logits), T(ids)).counts.clone()
    bad = ids.copy()
    bad[2, 1], bad[6, 3] = E, -1
    b = ex.balance(T(logits), T(bad))
    torch.cuda.synchronize()
    for t, j in ((2, 1), (6, 3)):
        want[0, ids[t, j]] -= 1
    assert torch.equal(b.counts, want)
    with pytest.raises(hip_rt.SabahRuntimeError, match="expert id"):
        ex.balance(T(logits), T(ids))
    got = ex.route_backward(T(logits), T(bad), T(dw))
    torch.cuda.synchronize()
    rows = got.isnan().all(dim=1)
    assert rows.nonzero()[:, 0].tolist() == [2, 6] and got[~rows].isfinite().all()
    with pytest.raises(hip_rt.SabahRuntimeError, match="expert id"):
        hip_rt.check(hip_rt.lib().sabah_rt_check_errors(), "sticky")


def test_strided_logits_and_rows_behind(ex):
    logits, ids, _, dw = batch(8, 33, 70, 5)
    wide, out = torch.zeros(33, 75, device=DEV), torch.full((35, 77), 7.0, device=DEV)
    wide[:, 3:73] = T(logits)
    b = ex.balance(wide[:, 3:73], T(ids))
    got = ex.route_backward(wide[:, 3:73], T(ids), T(dw), b, 0.7, 0.3, out=out[:33, 5:75])
    same, want = check(ex, logits, ids, None, dw, 1)
    assert torch.equal(got, want) and torch.equal(b.losses, same.losses) and torch.equal(b.mean_p, same.mean_p)
    out[:33, 5:75] = 7.0
    assert bool((out == 7.0).all())


def test_gradient_against_differences(ex):
    """Along random directions, with the counts and ids held: central differences of the
    64-bit loss (its third derivatives times h^2 are below the bound) against the kernel's gradient."""
    logits, ids, mask, dw = batch(6, 48, 64, 6, 2, 0.25)
    b = ex.balance(T(logits), T(ids), mask=T(mask), n_groups=2)
    got = ex.route_backward(T(logits), T(ids), T(dw), b, 0.7, 0.3, mask=T(mask)).double().cpu().numpy()

    def loss(l):
        total = ref.router_losses(l, ids, mask, 2)[2] @ np.array([0.7, 0.3])
        for t in np.flatnonzero(mask):
            s = np.exp(l[t, ids[t]] - l[t, ids[t]].max())
            total += (s / s.sum()) @ dw[t].astype(np.float64)
        return total
    g = np.random.default_rng(0)
    for _ in range(8):
        way = g.standard_normal(logits.shape)
        h = 1e-4
        l = logits.astype(np.float64)
        slope = (loss(l + h * way) - loss(l - h * way)) / (2 * h)
        size = np.abs(got * way).sum()
        # differences: |way|^3 h^2 / 6 of each token's terms; 64-bit cancellation; the gradient's own roundings
        assert abs((got * way).sum() - slope) <= 200 * h * h * np.abs(dw).sum() + 1e-11 / h + 400 * ref.U * size


@pytest.mark.parametrize("n,E,groups", [(40, 64, 1), (900, 512, 3)])
def test_captured_calls_replay(ex, n, E, groups):
    logits, ids, mask, dw = batch(n, n, E, 8, groups, 0.2)
    from sabah.runtime.executor import RouterBalance
    d_l, d_i, d_m, d_w = T(logits), T(ids), T(mask), T(dw)
    b, out = RouterBalance(E, groups), torch.empty_like(d_l)

    def step():
        ex.balance(d_l, d_i, mask=d_m, out=b)
        return ex.route_backward(d_l, d_i, d_w, b, 0.7, 0.3, mask=d_m, out=out)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = torch.Generator(device=DEV).manual_seed(n)
    for rep in range(4):
        d_l.copy_(torch.randn(n, E, generator=g, device=DEV))
        d_m.copy_(torch.rand(n, generator=g, device=DEV) > 0.3)
        step()
        want = [t.clone() for t in (b.counts, b.mean_p, b.losses, b.n_valid, out)]
        for t in (b.counts, b.mean_p, b.losses, b.n_valid, out):
            t.fill_(-5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((b.counts, b.mean_p, b.losses, b.n_valid, out), want)), rep
        (d_l * 2).sum().item()


def test_refusals_of_the_executor(ex, hip_rt):
    logits, ids, mask, dw = (None if a is None else T(a) for a in batch(4, 12, 16, 2, 1, 0.2))
    b = ex.balance(logits, ids)
    for call in (lambda: ex.balance(logits.double(), ids), lambda: ex.balance(logits, ids.long()),
                 lambda: ex.balance(logits, ids[:5]), lambda: ex.balance(logits.cpu(), ids),
                 lambda: ex.balance(logits.t().contiguous().t(), ids), lambda: ex.balance(logits, ids, mask=mask[:5]),
                 lambda: ex.balance(logits[:, :8].contiguous(), ids, out=b),
                 lambda: ex.route_backward(logits, ids, dw[:, :1]), lambda: ex.route_backward(logits, ids, dw.half()),
                 lambda: ex.route_backward(logits[:, :8].contiguous(), ids, dw, b),
                 lambda: ex.route_backward(logits, ids, dw, out=torch.empty(12, 15, device=DEV))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ex.balance(logits, ids, n_groups=5), lambda: ex.route_backward(logits, ids, dw, c_balance=1.0),
                 lambda: ex.route_backward(logits, ids, dw, w_scale=0.0)):
        with pytest.raises(hip_rt.SabahRuntimeError):
            call()


def test_route_then_its_gradient(ex):
    """The gradient goes with route()'s own weights: sum_j dw_j w_j falls as it says along -dlogits."""
    logits, _, _, dw = batch(9, 64, 128, 8)
    d_l, d_w = T(logits), T(dw)
    for norm_w, scale in ((True, 1.0), (False, 2.0)):
        ids, w = ex.route(d_l, 8, norm_w, scale)
        got = ex.route_backward(d_l, ids, d_w, norm_w=norm_w, w_scale=scale)
        l64 = d_l.double()
        p = torch.softmax(l64, dim=1).gather(1, ids.long())
        ref_w = scale * (p / p.sum(dim=1, keepdim=True) if norm_w else p)
        assert torch.allclose(w.double(), ref_w, rtol=1e-5, atol=0)
        want, bound = ref.router_gradient(logits.astype(np.float64), ids.cpu().numpy(), np.ones(64, bool), 1,
                                          dw.astype(np.float64), norm_w, scale, 0, 0)
        close(got, want, bound, "dlogits")
