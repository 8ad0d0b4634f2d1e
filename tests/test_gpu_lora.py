"""Low-rank adapters of many requests and their gradients, through the
executor and the C ABI (needs an MI355X), against the 64-bit forms of
adapt_refs.py within their counted roundings."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import adapt_refs as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ex(hip_rt):
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    return MoEExecutor(ExpertBank(1, 8, 256, 256, {"gate": 21, "up": 21, "down": 21}, device="cuda:0"))


class Case:
    """A batch in host and device memory; adapters: "each" token its own, "runs" of one request after another,
    or a list."""

    def __init__(self, seed, T, k, rows, rank, n, dtype=BF16, E=1, slots=1, x_rows=1, adapters="each", ranks=None):
        from sabah.runtime.lora import LoraBank
        g = np.random.default_rng(seed)
        self.lora = LoraBank(n, rank, k, rows, n_experts=E, dtype=dtype, device="cuda:0")
        self.lora.a.copy_(torch.from_numpy(g.standard_normal((n, E, rank, k)) / np.sqrt(k)))
        self.lora.b.copy_(torch.from_numpy(g.standard_normal((n, E, rows, rank)) * 0.1))
        self.lora.scale.copy_(torch.from_numpy(g.uniform(-2, 2, n)))
        if ranks is not None:
            self.lora.ranks.copy_(torch.tensor(ranks, dtype=torch.int32))
        if adapters == "each":
            ad = g.integers(-1, n, T)
        elif adapters == "runs":
            ad = np.sort(g.integers(-1, n, T))
            ad = ad[np.argsort(g.permutation(n + 1)[ad + 1], kind="stable")]
        else:
            ad = np.array(adapters)
        self.ad = ad.astype(np.int32)
        self.ids = None if E == 1 else np.stack([g.permutation(E)[:slots] for _ in range(T)]).astype(np.int32)
        self.x = g.standard_normal((T, x_rows, k)).astype(np.float32)
        self.base = g.standard_normal((T, slots, rows)).astype(np.float32)
        self.dy = g.standard_normal((T, slots, rows)).astype(np.float32)
        self.d_x, self.d_ad, self.d_base, self.d_dy = (torch.from_numpy(v).to(DEV) for v in
                                                       (self.x, self.ad, self.base, self.dy))
        self.d_ids = None if self.ids is None else torch.from_numpy(self.ids).to(DEV)

    def weights(self):
        L = self.lora
        return (L.a.double().cpu().numpy(), L.b.double().cpu().numpy(), L.scale.double().cpu().numpy(),
                L.ranks.cpu().numpy())

    def forward(self):
        return ref.lora_forward(self.x.astype(np.float64), self.ad, self.ids, *self.weights(),
                                self.base.astype(np.float64))

    def backward(self):
        return ref.lora_backward(self.x.astype(np.float64), self.ad, self.ids, *self.weights(),
                                 self.dy.astype(np.float64))


def close(got, want, bound, what):
    got = got.double().cpu().numpy().reshape(want.shape)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g of its bound" % (
        what, bad.sum(), bad.size, np.nanmax(np.abs(got - want) / np.maximum(bound, 1e-300)))


SHAPES = [
    # T, k, rows, rank, n, dtype, E, slots, x_rows, adapters
    (1, 2048, 2048, 16, 8, BF16, 1, 1, 1, [3]),
    (1, 33, 35, 5, 2, F16, 1, 1, 1, [1]),
    (2, 1, 1, 1, 1, F32, 1, 1, 1, [0, -1]),
    (31, 256, 130, 16, 40, BF16, 1, 1, 1, "each"),
    (32, 768, 512, 12, 64, F16, 1, 1, 1, "each"),
    (65, 100, 77, 17, 3, BF16, 1, 1, 1, "runs"),
    (70, 160, 96, 31, 2, F32, 1, 1, 1, "each"),
    (129, 320, 64, 64, 1, F16, 1, 1, 1, [0] * 129),
    (200, 257, 129, 33, 5, BF16, 1, 1, 1, "runs"),
    (300, 64, 200, 128, 4, BF16, 1, 1, 1, "runs"),
    (40, 64, 48, 127, 3, F16, 1, 1, 1, "each"),
    (1100, 40, 24, 8, 7, BF16, 1, 1, 1, "each"),
    (2500, 32, 36, 4, 3, F32, 1, 1, 1, "runs"),
    (9, 128, 96, 8, 3, BF16, 12, 4, 1, "each"),
    (90, 64, 32, 8, 2, F16, 16, 6, 1, "runs"),
    (33, 96, 80, 20, 2, BF16, 8, 2, 2, "each"),
    (300, 32, 48, 6, 4, BF16, 64, 6, 6, "each"),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "T%d_k%d_rows%d_r%d_n%d_E%d" % (s[0], s[1], s[2], s[3], s[4], s[6]))
def test_forward_matches_the_definition(ex, shape):
    T, k, rows, rank, n, dtype, E, slots, x_rows, adapters = shape
    c = Case(T * 7 + k, T, k, rows, rank, n, dtype, E, slots, x_rows, adapters)
    want, bound = c.forward()
    got = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base, ids=c.d_ids)
    torch.cuda.synchronize()
    close(got, want, bound, "forward")
    none = torch.from_numpy(c.ad < 0).to(DEV)
    assert torch.equal(got[none], c.d_base[none])                       # rows without an adapter: the base's bits
    again = c.d_base.clone()
    assert ex.lora_apply(c.lora, c.d_x, c.d_ad, again, ids=c.d_ids, out=again) is again
    assert torch.equal(again, got)                                      # in place: the same bits
    alone = ex.lora_apply(c.lora, c.d_x, c.d_ad, ids=c.d_ids, out=torch.full_like(got, float("nan")))
    close(alone, want - c.base, bound, "without a base")
    hip_ok()


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "T%d_k%d_rows%d_r%d_n%d_E%d" % (s[0], s[1], s[2], s[3], s[4], s[6]))
def test_backward_matches_the_definition(ex, shape):
    T, k, rows, rank, n, dtype, E, slots, x_rows, adapters = shape
    c = Case(T * 11 + k, T, k, rows, rank, n, dtype, E, slots, x_rows, adapters)
    want, bound = c.backward()
    nan = float("nan")
    dx = torch.full((T, slots, k), nan, device=DEV)
    da, db = torch.full(c.lora.a.shape, nan, device=DEV), torch.full(c.lora.b.shape, nan, device=DEV)
    got = ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy, ids=c.d_ids, dx=dx, da=da, db=db)
    torch.cuda.synchronize()
    for g, w, b, what in zip(got, want, bound, ("dx", "da", "db")):
        close(g, w, b, what)
    first = [g.clone() for g in got]
    again = ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy, ids=c.d_ids)
    assert all(torch.equal(g, f) for g, f in zip(again, first))         # the same bits again
    # added to what is there: one more rounding
    adds = [torch.ones_like(g) for g in first]
    ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy, ids=c.d_ids, dx=adds[0], da=adds[1], db=adds[2], add_dx=True,
                     add_dw=True)
    for g, w, b, what in zip(adds, want, bound, ("dx", "da", "db")):
        close(g, w + 1.0, b + 2 * ref.U * (np.abs(w) + 1.0), "added " + what)
    # each gradient alone
    only = ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy, ids=c.d_ids, need_dw=False)
    assert torch.equal(only[0], first[0]) and only[1] is None and only[2] is None
    only = ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy, ids=c.d_ids, need_dx=False)
    assert only[0] is None and torch.equal(only[1], first[1]) and torch.equal(only[2], first[2])
    hip_ok()


def hip_ok():
    from sabah.runtime import rt
    rt.check(rt.lib().sabah_rt_check_errors(), "no call read an id out of range")


@pytest.mark.parametrize("T", [5, 90, 1200])
def test_gradients_against_differences(ex, T):
    """<dy, y> is bilinear in x, A and B, so a difference along any direction is exact but
    for the roundings of y: (L(+h) - L(-h)) / 2h equals the gradient along it."""
    c = Case(T, T, 48, 40, 6, 3, F32, adapters="runs")
    dx, da, db = ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy)
    g = torch.Generator(device=DEV).manual_seed(T)
    h = 0.5
    for t, grad in ((c.d_x, dx), (c.lora.a, da), (c.lora.b, db)):
        way = torch.randn(t.shape, generator=g, device=DEV)
        kept = t.clone()
        L, size = [], 0.0
        for sign in (h, -h):
            t.copy_(kept + sign * way)
            y = ex.lora_apply(c.lora, c.d_x, c.d_ad)
            L.append((y.double() * c.d_dy.double().view(y.shape)).sum().item())
            size += (y.double() * c.d_dy.double().view(y.shape)).abs().sum().item()
        t.copy_(kept)
        got, want = (grad.double() * way.double()).sum().item(), (L[0] - L[1]) / (2 * h)
        # y's roundings (at most 100 u of its terms' sizes, itself within 16 of y's here) on both sides, the
        # displaced operand's own rounding, and the gradient's
        bound = ref.U * 100 * 16 * size / (2 * h) + ref.U * 200 * (grad.double().abs() * way.double().abs()).sum().item()
        assert abs(got - want) <= bound, (got, want, bound)


def test_an_adapter_of_a_lower_rank_ignores_what_lies_past_it(ex):
    c = Case(3, 80, 96, 70, 24, 4, BF16, adapters="each", ranks=[24, 7, 0, 300])
    for n, r in ((1, 7), (2, 0)):                                       # past the rank: NaN and infinities
        c.lora.a[n, :, r:] = float("nan")
        c.lora.b[n, :, :, r:] = float("inf")
    a, b, scale, ranks = c.weights()
    want, bound = ref.lora_forward(c.x.astype(np.float64), c.ad, None, np.nan_to_num(a, nan=0, posinf=0),
                                   np.nan_to_num(b, nan=0, posinf=0), scale, ranks, c.base.astype(np.float64))
    got = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base)
    close(got, want, bound, "forward")
    want, bound = ref.lora_backward(c.x.astype(np.float64), c.ad, None, np.nan_to_num(a, nan=0, posinf=0),
                                    np.nan_to_num(b, nan=0, posinf=0), scale, ranks, c.dy.astype(np.float64))
    for g, w, bd, what in zip(ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy), want, bound, ("dx", "da", "db")):
        close(g, w, bd, what)


@pytest.mark.parametrize("T", [6, 150, 1300])
def test_a_row_of_nan_or_infinity_stays_its_own(ex, T):
    """One row's NaN, another's infinity and another's largest finite values touch no other
    row, with the same adapter or another; infinity gives infinity or NaN as the sums do."""
    c = Case(T + 1, T, 96, 40, 16, 2, BF16, adapters=[t % 2 for t in range(T)])
    clean = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base)
    x = c.d_x.clone()
    x[1, 0, 5], x[2, 0, 7], x[3, 0, 2] = float("nan"), float("inf"), 3.0e38
    got = ex.lora_apply(c.lora, x, c.d_ad, c.d_base)
    rest = torch.ones(T, dtype=torch.bool, device=DEV)
    rest[1:4] = False
    assert torch.equal(got[rest], clean[rest])
    assert got[1].isnan().all()
    a, b = c.lora.a[0, 0, :, 7].double(), c.lora.b[0, 0].double()
    assert not got[2].isfinite().any()
    one = b[:, 0] * 0 + 0
    # every s is an infinity of the sign of A's column; a row's sum is infinite where all its terms agree, else NaN
    signs = torch.sign(b * a[None, :] * c.lora.scale[0].double())
    agree = (signs != 0).all(dim=1) & (signs.min(dim=1).values == signs.max(dim=1).values)
    want = torch.where(agree, signs[:, 0] * float("inf"), torch.full_like(one, float("nan")))
    assert torch.equal(got[2, 0].double().nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))
    w = ref.lora_forward(x[3:4].double().cpu().numpy(), c.ad[3:4], None, *c.weights(), c.base[3:4].astype(np.float64))
    fits = np.abs(w[0]) + w[1] < 3.0e38
    assert (np.abs(got[3].double().cpu().numpy() - w[0][0])[fits[0]] <= w[1][0][fits[0]]).all()


def test_strides_and_rows_behind_the_last_token(ex):
    """x, ids, base and out inside larger tensors, off the 16-byte grid; what lies between
    and behind the rows stays as it was."""
    c = Case(5, 37, 45, 30, 6, 3, F16, E=8, slots=2, x_rows=2)
    want, bound = c.forward()
    xs = torch.zeros(37, 3, 53, device=DEV)
    xs[:, :2, 1:46] = c.d_x
    idw = torch.full((37, 7), 99, dtype=torch.int32, device=DEV)
    idw[:, 1:5:3] = c.d_ids
    bases = torch.full((40, 3, 37), 5.0, device=DEV)
    outs = torch.full((40, 3, 41), 7.0, device=DEV)
    bases[:37, :2, 3:33] = c.d_base
    got = ex.lora_apply(c.lora, xs[:, :2, 1:46], c.d_ad, bases[:37, :2, 3:33], ids=idw[:, 1:5:3],
                        out=outs[:37, :2, 5:35])
    close(got.contiguous(), want, bound, "strided")
    outs[:37, :2, 5:35] = 7.0
    assert bool((outs == 7.0).all())
    wantb, boundb = c.backward()
    dys = torch.zeros(37, 3, 33, device=DEV)
    dys[:, :2, 2:32] = c.d_dy
    dxs = torch.full((38, 3, 50), 7.0, device=DEV)
    g = ex.lora_backward(c.lora, xs[:, :2, 1:46], c.d_ad, dys[:, :2, 2:32], ids=idw[:, 1:5:3], dx=dxs[:37, :2, 3:48])
    for a, w, b, what in zip((g[0].contiguous(), g[1], g[2]), wantb, boundb, ("dx", "da", "db")):
        close(a, w, b, what)
    dxs[:37, :2, 3:48] = 7.0
    assert bool((dxs == 7.0).all())


@pytest.mark.parametrize("T", [0, 7, 200, 1200])
def test_no_token_has_an_adapter(ex, T):
    c = Case(9, T, 64, 48, 8, 2, BF16, adapters=[-1] * T)
    got = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base)
    assert torch.equal(got, c.d_base)
    dx, da, db = ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy)
    assert not dx.any() and not da.any() and not db.any()
    assert da.shape == c.lora.a.shape and db.shape == c.lora.b.shape


@pytest.mark.parametrize("T,E", [(6, 1), (6, 8), (300, 1), (300, 8), (1500, 1)])
def test_an_id_out_of_range_makes_its_row_nan_and_fails_the_next_call(ex, hip_rt, T, E):
    slots = 2 if E > 1 else 1
    c = Case(T + E, T, 64, 40, 8, 3, BF16, E=E, slots=slots, adapters=[t % 3 for t in range(T)])
    clean = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base, ids=c.d_ids)
    ad, ids = c.d_ad.clone(), None if E == 1 else c.d_ids.clone()
    bad = torch.zeros(T, slots, dtype=torch.bool, device=DEV)
    ad[1], bad[1] = 3, True
    ad[4], bad[4] = -2, True
    if E > 1:
        ids[2, 1], bad[2, 1] = 8, True
        ids[3, 0], bad[3, 0] = -1, True
    got = ex.lora_apply(c.lora, c.d_x, ad, c.d_base, ids=ids)
    torch.cuda.synchronize()
    assert got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])
    with pytest.raises(hip_rt.SabahRuntimeError, match="adapter id"):
        ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base, ids=c.d_ids)
    keep = torch.where(bad.any(dim=1), -1, c.d_ad) if E == 1 else None
    dx, da, db = ex.lora_backward(c.lora, c.d_x, ad, c.d_dy, ids=ids)
    torch.cuda.synchronize()
    assert dx.view(T, slots, -1)[bad].isnan().all() and dx.view(T, slots, -1)[~bad].isfinite().all()
    assert da.isfinite().all() and db.isfinite().all()
    with pytest.raises(hip_rt.SabahRuntimeError, match="adapter id"):
        hip_rt.check(hip_rt.lib().sabah_rt_check_errors(), "sticky")
    if keep is not None:                                                # the bad rows give no part of the weights' gradients
        _, wa, wb = ex.lora_backward(c.lora, c.d_x, keep.to(torch.int32), c.d_dy)
        close(da, wa.double().cpu().numpy(), 1e-5 * np.abs(wa.double().cpu().numpy()) + 1e-5, "da")
        close(db, wb.double().cpu().numpy(), 1e-5 * np.abs(wb.double().cpu().numpy()) + 1e-5, "db")


@pytest.mark.parametrize("T,E,slots", [(3, 1, 1), (260, 1, 1), (1300, 1, 1), (24, 8, 2)])
def test_captured_calls_replay(ex, T, E, slots):
    """Forward and backward captured into two graphs, replayed in turn with other inputs
    and eager work between: every replay equals the eager call."""
    c = Case(T, T, 96, 64, 16, 4, BF16, E=E, slots=slots, adapters="each")
    out = torch.empty_like(c.d_base)
    dx, da, db = (torch.empty(s, device=DEV) for s in ((T, slots, 96), c.lora.a.shape, c.lora.b.shape))

    def forward():
        return ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base, ids=c.d_ids, out=out)

    def backward():
        return ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy, ids=c.d_ids, dx=dx, da=da, db=db)
    graphs = []
    for call in (forward, backward):
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
    rng = torch.Generator(device=DEV).manual_seed(T)
    for rep in range(4):
        c.d_x.copy_(torch.randn(c.d_x.shape, generator=rng, device=DEV))
        c.d_ad.copy_(torch.randint(-1, 4, (T,), generator=rng, device=DEV))
        want = [v.clone() for v in (forward(), *backward())]
        torch.cuda.synchronize()
        for t in (out, dx, da, db):
            t.fill_(float("nan"))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, dx, da, db), want)), "replay %d" % rep
        (c.d_x * 2).sum().item()


def test_calls_on_two_streams_share_nothing(ex):
    cs = [Case(i, 700, 256, 256, 32, 4, BF16, adapters="runs") for i in range(2)]
    want = [(ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base), *ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy)) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(5):
        got = []
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                got.append((ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base),
                            *ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy)))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_load_places_an_adapter_of_a_lower_rank(ex):
    from sabah.runtime.lora import LoraBank
    g = torch.Generator(device=DEV).manual_seed(0)
    lora = LoraBank(3, 8, 40, 24, n_experts=2, dtype=F32, device="cuda:0")
    a, b = torch.randn(2, 5, 40, generator=g, device=DEV), torch.randn(2, 24, 5, generator=g, device=DEV)
    lora.load(1, a, b, scale=0.5)
    x = torch.randn(4, 40, generator=g, device=DEV)
    ids = torch.tensor([[0], [1], [1], [0]], dtype=torch.int32, device=DEV)
    y = ex.lora_apply(lora, x, torch.tensor([1, 1, -1, 1], dtype=torch.int32, device=DEV), ids=ids)
    want = torch.stack([0.5 * b[e].double() @ (a[e].double() @ x[t].double()) * (t != 2)
                        for t, e in enumerate((0, 1, 1, 0))])
    mag = torch.stack([0.5 * b[e].abs().double() @ (a[e].abs().double() @ x[t].abs().double())
                       for t, e in enumerate((0, 1, 1, 0))])
    assert ((y[:, 0].double() - want).abs() <= ref.U * 60 * mag).all()
    for bad in ((a[:, :, :39], b), (a, b[:, :, :4]), (torch.zeros(2, 9, 40), torch.zeros(2, 24, 9))):
        with pytest.raises(ValueError):
            lora.load(0, *bad)
    with pytest.raises(IndexError):
        lora.load(3, a, b)


def test_refusals_of_the_executor(ex):
    c = Case(2, 5, 64, 48, 8, 2, BF16)
    ok = (c.lora, c.d_x, c.d_ad)
    for bad in (dict(x=c.d_x[:, :, :63]), dict(x=c.d_x.double()), dict(x=c.d_x[:4]), dict(x=c.d_x.cpu()),
                dict(adapters=c.d_ad.long()), dict(base=c.d_base[:, :, :47]), dict(base=c.d_base.half()),
                dict(out=torch.empty(5, 2, 48, device=DEV)), dict(ids=torch.zeros(5, 1, device=DEV)),
                dict(x=torch.zeros(5, 1, 128, device=DEV)[:, :, ::2])):
        kw = dict(lora=ok[0], x=ok[1], adapters=ok[2], base=c.d_base)
        kw.update(bad)
        with pytest.raises((ValueError, RuntimeError)):
            ex.lora_apply(**kw)
    with pytest.raises(ValueError):
        ex.lora_backward(*ok, c.d_dy[:, :, :47])
    with pytest.raises(ValueError):
        ex.lora_backward(*ok, c.d_dy, add_dx=True)
    with pytest.raises(ValueError):
        ex.lora_backward(*ok, c.d_dy, da=torch.empty(2, 1, 8, 63, device=DEV))


def test_mul_mat_id_adds_each_tokens_adapter(ex, hip_rt, orc):
    """The expert product with adapters, one pair for all experts and one per expert, is
    the product and then the adapters; the product alone keeps its bits."""
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    from sabah.runtime.lora import LoraBank
    E, D, F, K, T = 16, 512, 256, 3, 20
    bank = ExpertBank(1, E, D, F, {"gate": 8, "up": 8, "down": 8}, device="cuda:0")
    bank.fill_synthetic(4)
    m = MoEExecutor(bank, max_used=K)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(T, 1, D, generator=g, device=DEV)
    ids = torch.rand(T, E, generator=g, device=DEV).topk(K, dim=1).indices.to(torch.int32)
    ad = torch.randint(-1, 4, (T,), generator=g, device=DEV).to(torch.int32)
    plain = m.mul_mat_id(0, "gate", x, ids)
    for n_experts in (1, E):
        lora = LoraBank(4, 8, D, F, n_experts=n_experts, dtype=BF16, device="cuda:0")
        lora.a.copy_(torch.randn(lora.a.shape, generator=g, device=DEV) / 16)
        lora.b.copy_(torch.randn(lora.b.shape, generator=g, device=DEV))
        got = m.mul_mat_id(0, "gate", x, ids, lora=lora, adapters=ad)
        want, bound = ref.lora_forward(x.double().cpu().numpy(), ad.cpu().numpy(), ids.cpu().numpy() % n_experts,
                                       lora.a.double().cpu().numpy(), lora.b.double().cpu().numpy(), np.ones(4),
                                       np.full(4, 8), plain.double().cpu().numpy())
        close(got, want, bound, "product and adapters")
        assert torch.equal(m.mul_mat_id(0, "gate", x, ids), plain)
    with pytest.raises(ValueError):
        m.mul_mat_id(0, "gate", x, ids, lora=LoraBank(1, 8, D, F, n_experts=2), adapters=ad)
