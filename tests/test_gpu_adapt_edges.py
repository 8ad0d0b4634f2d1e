"""Adapters and the router's losses where types and sizes end: wide ranges within a row, infinite
weights, rows of infinities, high ranks, long batches (needs an MI355X).  Against the
64-bit forms of adapt_refs.py within their counted roundings."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import adapt_refs as ref
from test_gpu_balance import T as to_dev, batch
from test_gpu_lora import BF16, DEV, F16, F32, Case, close, hip_ok

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])


@pytest.fixture(scope="module")
def ex(hip_rt):
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    return MoEExecutor(ExpertBank(1, 8, 256, 256, {"gate": 21, "up": 21, "down": 21}, device="cuda:0"))


def all_close(got, want, bound):
    for g, w, b, what in zip(got, want, bound, ("dx", "da", "db")):
        close(g, w, b, what)


@pytest.mark.parametrize("E,k", [(60, 6), (512, 10), (700, 8)])
@pytest.mark.parametrize("norm_w", [True, False])
def test_the_routes_own_ids_of_a_row_without_experts_raise_nothing(ex, E, k, norm_w):
    """route() has no expert for a row of minus infinities and says -1.  Such a token counts as masked: its
    gradient is zeros, and the next call goes through."""
    logits, _, _, dw = batch(E, 21, E, k)
    logits[3], logits[20] = -np.inf, -np.inf
    d_l = to_dev(logits)
    ids, _ = ex.route(d_l, k, norm_w)
    b = ex.balance(d_l, ids, n_groups=3)
    got = ex.route_backward(d_l, ids, to_dev(dw), b, 0.7, 0.3, norm_w=norm_w)
    torch.cuda.synchronize()
    hip_ok()
    host = ids.cpu().numpy()
    _, _, _, n_valid, valid, _, _ = ref.router_losses(logits.astype(np.float64), host, None, 3)
    assert not valid[3] and not valid[20] and np.array_equal(b.n_valid.cpu().numpy(), n_valid)
    want, bound = ref.router_gradient(logits.astype(np.float64), host, valid, 3, dw.astype(np.float64), norm_w, 1.0, 0.7, 0.3)
    close(got, want, bound, "dlogits")
    assert not got[3].any() and not got[20].any()


@pytest.mark.parametrize("E", [24, 512, 700])
def test_an_infinite_logit_has_an_infinite_log_sum(ex, E):
    """lse of a row with an infinity is infinite, of one with a NaN a NaN; neither has probabilities."""
    logits, ids, _, dw = batch(E, 12, E, 4)
    logits[5, 7] = np.inf
    b = ex.balance(to_dev(logits), to_dev(ids))
    assert b.losses[1].item() == float("inf") and b.losses[0].isnan() and b.mean_p.isnan().all()
    got = ex.route_backward(to_dev(logits), to_dev(ids), to_dev(dw), b, 0.0, 0.3)
    assert got[5].isnan().all()
    logits[6, 3] = np.nan
    assert ex.balance(to_dev(logits), to_dev(ids)).losses.isnan().all()
    logits[6] = np.inf
    assert ex.balance(to_dev(logits), to_dev(ids)).losses[1].item() == float("inf")


@TYPES
@pytest.mark.parametrize("T,rank", [(5, 8), (40, 24), (200, 40), (600, 64), (600, 100), (4500, 20)])
@pytest.mark.parametrize("size", [3e5, 1e8, 1e12])
def test_a_large_value_that_no_weight_meets(ex, T, rank, size, dtype):
    """One value of some rows is up to 1e12 times the others and its weights are zeros, or it makes an s
    (u) that large whose weights are zeros: what the others give is right to f32 all the same, and
    rows without such values keep their bits."""
    c = Case(T + rank, T, 100, 44, rank, 2, dtype, adapters=[t % 2 for t in range(T)])
    clean = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base)
    c.lora.a[:, :, :, 5] = 0
    c.lora.a[:, :, 2, 70] = 100.0
    c.lora.a[:, :, :2, 70] = 0
    c.lora.a[:, :, 3:, 70] = 0
    c.lora.b[:, :, :, 2] = 0
    clean = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base)
    wide = np.arange(T) % 3 == 0
    c.x[wide, :, 5] = size
    c.x[wide, :, 70] = size / 100
    c.d_x.copy_(torch.from_numpy(c.x))
    want, bound = c.forward()
    got = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base)
    close(got, want, bound, "forward")
    same = torch.from_numpy(~wide).to(DEV)
    assert torch.equal(got[same], clean[same])
    # the same backward: dy's value 3 meets zeros of B but at rank 1, whose row of A is zeros
    c.lora.b[:, :, 3, :] = 0
    c.lora.b[:, :, 3, 1] = 1.0
    c.lora.b[:, :, 9, :] = 0
    c.lora.a[:, :, 1, :] = 0
    clean = ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy)[0]
    c.dy[wide, :, 3] = size
    c.dy[wide, :, 9] = -size
    c.d_dy.copy_(torch.from_numpy(c.dy))
    want, bound = c.backward()
    got = ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy)
    all_close(got, want, bound)
    assert torch.equal(got[0][same], clean[same])


def by_sums(w, v):
    """w [.., n, m] and v [.., m]: the sums over m in the definition's arithmetic, infinities and NaN included."""
    with np.errstate(invalid="ignore", over="ignore"):
        return (w * v[..., None, :]).sum(axis=-1)


def same_places(got, want, what):
    """Where the definition gives an infinity or a NaN, the call gives the same."""
    got = got.double().cpu().numpy().reshape(want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    at = np.isinf(want)
    assert np.array_equal(np.isinf(got), at) and np.array_equal(got[at], want[at]), what


@TYPES
@pytest.mark.parametrize("T,rank", [(1, 6), (6, 6), (150, 20), (600, 40), (600, 128), (4500, 16)])
@pytest.mark.parametrize("where", ["a", "b", "both"])
def test_infinite_weights_give_what_the_sums_give(ex, T, rank, where, dtype):
    """Infinities in one adapter's A or B, beside values of few bits, of many, and zeros; rows of the other
    adapter keep their bits."""
    c = Case(T + rank, T, 70, 72, rank, 2, dtype, adapters=[t % 2 for t in range(T)])
    c.x[:, 0, 5] = np.array([1.0, -0.5, 0.3, -1.7, 0.0, 3.0])[np.arange(T) // 2 % 6]
    c.dy[:, 0, 7] = np.array([1.0, -0.5, 0.3, -1.7, 2.0, 0.0])[np.arange(T) // 2 % 6]
    c.d_x.copy_(torch.from_numpy(c.x))
    c.d_dy.copy_(torch.from_numpy(c.dy))
    clean = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base), *ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy)
    inf = float("inf")
    if where != "b":
        c.lora.a[0, 0, 2, 5] = inf
    if where != "a":
        c.lora.b[0, 0, 7, 3], c.lora.b[0, 0, 70, 1] = -inf, inf
    a, b, scale, _ = c.weights()
    A, B, s = a[c.ad, 0], b[c.ad, 0], scale[c.ad][:, None]
    with np.errstate(invalid="ignore"):
        y = by_sums(B, s * by_sums(A, c.x[:, 0].astype(np.float64))) + c.base[:, 0]
        dx = by_sums(A.transpose(0, 2, 1), s * by_sums(B.transpose(0, 2, 1), c.dy[:, 0].astype(np.float64)))
    out = c.d_base.clone()
    got = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base), *ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy)
    same_places(got[0], y, "forward")
    same_places(got[1], dx, "dx")
    ex.lora_apply(c.lora, c.d_x, c.d_ad, out, out=out)
    same_places(out, y, "in place")
    c.lora.a[0], c.lora.b[0] = c.lora.a[0].nan_to_num(0, 0, 0), c.lora.b[0].nan_to_num(0, 0, 0)
    want, bound = c.forward()
    finite = np.isfinite(y)
    assert np.all((np.abs(got[0].double().cpu().numpy()[:, 0] - want[:, 0]) <= bound[:, 0])[finite])
    want, bound = c.backward()
    finite = np.isfinite(dx)
    assert np.all((np.abs(got[1].double().cpu().numpy().reshape(T, -1) - want[0][:, 0]) <= bound[0][:, 0])[finite])
    if T > 1:
        assert torch.equal(got[0][1::2], clean[0][1::2]) and torch.equal(got[1][1::2], clean[1][1::2])
        assert torch.equal(got[2][1], clean[2][1]) and torch.equal(got[3][1], clean[3][1])


@TYPES
@pytest.mark.parametrize("T,rank", [(6, 16), (150, 40), (600, 113), (1300, 16), (4500, 24)])
def test_rows_of_nan_and_infinity_of_every_type(ex, T, rank, dtype):
    """A NaN, infinities of both signs and a row with both touch no other row, forward and backward; what
    they give is what the sums give."""
    c = Case(T + rank, T, 70, 40, rank, 2, dtype, adapters=[t % 2 for t in range(T)])
    clean = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base), ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy)[0]
    inf = np.inf
    c.x[1, 0, 5], c.x[2, 0, 69], c.x[4, 0, 1] = np.nan, inf, -inf
    c.x[5, 0, 3], c.x[5, 0, 66] = inf, np.nan
    c.dy[0, 0, 5], c.dy[2, 0, 39], c.dy[4, 0, 1] = np.nan, -inf, inf
    a, b, scale, _ = c.weights()
    A, B, s = a[c.ad, 0], b[c.ad, 0], scale[c.ad][:, None]
    with np.errstate(invalid="ignore"):
        y = by_sums(B, s * by_sums(A, c.x[:, 0].astype(np.float64))) + c.base[:, 0]
        dx = by_sums(A.transpose(0, 2, 1), s * by_sums(B.transpose(0, 2, 1), c.dy[:, 0].astype(np.float64)))
    x, dy = torch.from_numpy(c.x).to(DEV), torch.from_numpy(c.dy).to(DEV)
    got = ex.lora_apply(c.lora, x, c.d_ad, c.d_base), ex.lora_backward(c.lora, x, c.d_ad, dy, need_dw=False)[0]
    same_places(got[0], y, "forward")
    same_places(got[1], dx, "dx")
    rest = torch.ones(T, dtype=torch.bool, device=DEV)
    rest[[1, 2, 4, 5]] = False
    assert torch.equal(got[0][rest], clean[0][rest])
    rest = torch.ones(T, dtype=torch.bool, device=DEV)
    rest[[0, 2, 4]] = False
    assert torch.equal(got[1][rest], clean[1][rest])


@pytest.mark.parametrize("T,k,rows,rank", [(63, 72, 40, 113), (300, 40, 36, 113), (2100, 36, 24, 113), (200, 100, 36, 64),
                                           (256, 40, 130, 128), (90, 65, 70, 33), (2049, 20, 12, 128)])
def test_high_ranks_kept_in_f32(ex, T, k, rows, rank):
    c = Case(T + rank, T, k, rows, rank, 3, F32, adapters="runs")
    want, bound = c.forward()
    close(ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base), want, bound, "forward")
    all_close(ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy), *c.backward())
    hip_ok()


@TYPES
@pytest.mark.parametrize("T,rank", [(3, 24), (200, 40), (600, 24), (600, 128), (4500, 24)])
def test_values_past_an_adapters_own_rank_count_nowhere(ex, T, rank, dtype):
    """NaN and infinities past the own ranks of half of the adapters, in calls of every size."""
    c = Case(T, T, 68, 36, rank, 4, dtype, adapters="each", ranks=[rank, 7, 0, 300])
    for n, r in ((1, 7), (2, 0)):
        c.lora.a[n, :, r:] = float("nan")
        c.lora.b[n, :, :, r:] = float("inf")
    a, b, scale, ranks = c.weights()
    a, b = np.nan_to_num(a, nan=0, posinf=0), np.nan_to_num(b, nan=0, posinf=0)
    want, bound = ref.lora_forward(c.x.astype(np.float64), c.ad, None, a, b, scale, ranks, c.base.astype(np.float64))
    close(ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base), want, bound, "forward")
    all_close(ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy),
              *ref.lora_backward(c.x.astype(np.float64), c.ad, None, a, b, scale, ranks, c.dy.astype(np.float64)))


def test_a_bank_on_the_current_device_without_a_number(hip_rt):
    """device="cuda" names the device that its tensors call cuda:0."""
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    ex = MoEExecutor(ExpertBank(1, 8, 256, 256, {"gate": 21, "up": 21, "down": 21}, device="cuda"))
    c = Case(4, 30, 64, 48, 8, 2, BF16)
    da, db = torch.zeros(c.lora.a.shape, device=DEV), torch.zeros(c.lora.b.shape, device=DEV)
    all_close(ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy, da=da, db=db, add_dw=True), *c.backward())
    assert da.any() and db.any()


@pytest.mark.parametrize("n,E,groups", [(1 << 24, 8, 1), (1 << 21, 516, 1), (1 << 22, 40, 64)])
def test_the_means_of_long_batches(ex, n, E, groups):
    """The same row in every token: each rounding of a long sum goes the same way.  Its mean is p and the
    z loss lse^2, within the roundings of p and lse, runs of 64 terms, the sides' and the result's."""
    row = torch.linspace(-1.0, 1.3, E, device=DEV)
    logits = row.expand(n, E).contiguous()
    ids = torch.arange(2, dtype=torch.int32, device=DEV).expand(n, 2).contiguous()
    b = ex.balance(logits, ids, n_groups=groups)
    l64 = row.double()
    p, lse = torch.softmax(l64, 0), torch.logsumexp(l64, 0)
    # exp's argument and exp, the sum of E terms, the reciprocal and product; 64 terms; four sides; the result
    rel = ref.U * (2.3 + E + 12 + 64 + 4 + 4)
    assert ((b.mean_p.double() - p).abs() <= rel * p).all()
    want = lse * lse
    assert abs(b.losses[1].double() - want) <= ref.U * (2 * (abs(lse) * 2 + E + 8) * abs(lse) + 76 * want)
    assert (b.counts[:, :2] == n // groups).all() and not b.counts[:, 2:].any()


def test_the_gradient_of_as_many_tokens_as_a_call_takes(ex):
    """2^24 tokens of 513 experts: all but a few at both ends and between are masked."""
    n, E, k = 1 << 24, 513, 4
    at = [0, 1, 4095, (1 << 20) - 1, 1 << 20, (1 << 23) + 5, n - 2, n - 1]
    logits, ids, _, dw = batch(1, len(at), E, k)
    d_l = torch.empty(n, E, device=DEV)
    d_i, d_w = torch.zeros(n, k, dtype=torch.int32, device=DEV), torch.zeros(n, k, device=DEV)
    mask = torch.zeros(n, dtype=torch.bool, device=DEV)
    d_l[at], d_i[at], d_w[at], mask[at] = to_dev(logits), to_dev(ids), to_dev(dw), True
    out = torch.full((n, E), 5.0, device=DEV)
    got = ex.route_backward(d_l, d_i, d_w, mask=mask, out=out)
    want, bound = ref.router_gradient(logits.astype(np.float64), ids, np.ones(len(at), bool), 1, dw.astype(np.float64),
                                      True, 1.0, 0, 0)
    close(got[at], want, bound, "dlogits")
    got[at] = 0
    assert not any(bool(part.any()) for part in got.split(1 << 21))


@pytest.mark.parametrize("T", [1, 5, 300])
def test_in_place_through_views_of_other_shapes(ex, T):
    """The same rows as [T, rows] and as [T, 1, rows], or one token with any token stride."""
    c = Case(T, T, 64, 48, 8, 2, BF16, adapters="each")
    want = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base)
    rows = c.d_base.clone()
    assert ex.lora_apply(c.lora, c.d_x, c.d_ad, rows[:, 0], out=rows) is rows
    assert torch.equal(rows, want)
    one = c.d_base[:1].clone()
    ex.lora_apply(c.lora, c.d_x[:1], c.d_ad[:1], one.as_strided((1, 1, 48), (4096, 48, 1)), out=one)
    assert torch.equal(one, want[:1])


@pytest.mark.parametrize("T", [4, 90, 2600])
def test_accumulated_gradients_touch_only_pairs_with_rows(ex, T):
    """With add_dw, pairs that no row uses and what lies past an adapter's own rank keep their bits (a zero its
    sign), so that calls at the same time may add to different adapters of one gradient."""
    c = Case(T, T, 72, 40, 20, 5, BF16, adapters=[(0, 3, -1, 3)[t % 4] for t in range(T)], ranks=[20, 20, 20, 7, 20])
    _, a, b = ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy, need_dx=False)
    da, db = torch.full_like(a, -0.0), torch.full_like(b, -0.0)
    ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy, da=da, db=db, add_dw=True, need_dx=False)
    assert torch.equal(da, a) and torch.equal(db, b)
    for n in (1, 2, 4):
        assert da[n].signbit().all() and db[n].signbit().all()
    assert da[3, 0, 7:].signbit().all() and db[3, 0, :, 7:].signbit().all()
