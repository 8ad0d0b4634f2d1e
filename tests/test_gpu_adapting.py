"""The operators that adapt a frozen bank used together, and at the edges of
their ranges: long batches, many adapters, memory beyond 2^32 bytes (needs an
MI355X).  Against the 64-bit forms of adapt_refs.py within their counted roundings."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import adapt_refs as ref
from test_gpu_lora import BF16, DEV, F16, F32, Case, close, hip_ok

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex(hip_rt):
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    return MoEExecutor(ExpertBank(1, 8, 256, 256, {"gate": 21, "up": 21, "down": 21}, device="cuda:0"))


def f64(t):
    return t.double().cpu().numpy()


class Step:
    """One training step of a router and of per-expert adapters beside a frozen projection:
    route, losses, product with adapters, the gradients back to x, the adapters and the logits."""

    def __init__(self, ex, E, D, F, K, T, groups, n_experts, seed):
        from sabah.runtime.lora import LoraBank
        self.ex, self.E, self.K, self.T, self.groups = ex, E, K, T, groups
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.g = g
        self.lora = LoraBank(3, 8, D, F, n_experts=n_experts, dtype=F16, device="cuda:0")
        self.lora.a.copy_(torch.randn(self.lora.a.shape, generator=g, device=DEV) / 16)
        self.lora.b.copy_(torch.randn(self.lora.b.shape, generator=g, device=DEV) / 4)
        self.lora.scale.copy_(torch.tensor([0.5, 2.0, -1.0]))
        self.logits, self.x = torch.empty(T, E, device=DEV), torch.empty(T, 1, D, device=DEV)
        self.v = torch.empty(T, K, F, device=DEV)
        self.ad = torch.empty(T, dtype=torch.int32, device=DEV)
        self.mask = torch.empty(T, dtype=torch.bool, device=DEV)
        self.fill()

    def fill(self):
        self.logits.copy_(torch.randn(self.T, self.E, generator=self.g, device=DEV) * 2)
        self.x.copy_(torch.randn(self.x.shape, generator=self.g, device=DEV))
        self.v.copy_(torch.randn(self.v.shape, generator=self.g, device=DEV))
        self.mask.copy_(torch.rand(self.T, generator=self.g, device=DEV) > 0.2)
        # a padded token has no adapter
        ad = torch.randint(-1, 3, (self.T,), generator=self.g, device=DEV)
        self.ad.copy_(torch.where(self.mask, ad, torch.full_like(ad, -1)))

    def run(self):
        ex = self.ex
        ids, w = ex.route(self.logits, self.K)
        stats = ex.balance(self.logits, ids, mask=self.mask, n_groups=self.groups)
        y = ex.mul_mat_id(0, "gate", self.x, ids, lora=self.lora, adapters=self.ad)
        dw = (y * self.v).sum(dim=2)                        # of sum w <y, v>
        dy = w[:, :, None] * self.v
        lids = ids if self.lora.n_experts > 1 else None
        dx, da, db = ex.lora_backward(self.lora, self.x, self.ad, dy, ids=lids)
        dl = ex.route_backward(self.logits, ids, dw, stats, 0.01, 0.001, mask=self.mask)
        return ids, w, stats.counts, stats.mean_p, stats.losses, y, dw, dy, dx, da, db, dl


@pytest.mark.parametrize("T,groups,shared", [(12, 1, False), (96, 4, False), (700, 2, False), (700, 2, True)])
def test_a_training_step_of_router_and_adapters(hip_rt, T, groups, shared):
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    E, D, F, K = 16, 512, 256, 3
    bank = ExpertBank(1, E, D, F, {"gate": 8, "up": 8, "down": 8}, device="cuda:0")
    bank.fill_synthetic(5)
    ex = MoEExecutor(bank, max_used=K)
    s = Step(ex, E, D, F, K, T, groups, 1 if shared else E, T)
    ids, w, counts, mean_p, losses, y, dw, dy, dx, da, db, dl = s.run()
    plain = ex.mul_mat_id(0, "gate", s.x, ids)
    torch.cuda.synchronize()
    hip_ok()
    hi, hm, had = ids.cpu().numpy(), s.mask.cpu().numpy(), s.ad.cpu().numpy()
    lw = (f64(s.lora.a), f64(s.lora.b), f64(s.lora.scale), s.lora.ranks.cpu().numpy())
    eids = hi * 0 if shared else hi
    want, bound = ref.lora_forward(f64(s.x), had, eids, *lw, f64(plain))
    close(y, want, bound, "product and adapters")
    c64, p64, l64, _, valid, pb, lb = ref.router_losses(f64(s.logits), hi, hm, groups)
    assert np.array_equal(counts.cpu().numpy(), c64)
    close(mean_p, p64, pb, "mean_p")
    close(losses, l64, lb, "losses")
    want, bound = ref.router_gradient(f64(s.logits), hi, valid, groups, f64(dw), True, 1.0, 0.01, 0.001)
    close(dl, want, bound, "dlogits")
    wants, bounds = ref.lora_backward(f64(s.x), had, eids, *lw, f64(dy))
    for got, want, bound, what in zip((dx, da, db), wants, bounds, ("dx", "da", "db")):
        close(got, want, bound, what)
    assert all(torch.equal(a, b) for a, b in zip(s.run(), (ids, w, counts, mean_p, losses, y, dw, dy, dx, da, db, dl)))


def test_a_captured_training_step_replays(hip_rt):
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    bank = ExpertBank(1, 16, 512, 256, {"gate": 8, "up": 8, "down": 8}, device="cuda:0")
    bank.fill_synthetic(5)
    s = Step(MoEExecutor(bank, max_used=3), 16, 512, 256, 3, 24, 2, 16, 1)
    s.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.run()
    for rep in range(4):
        s.fill()
        want = [t.clone() for t in s.run()]
        torch.cuda.synchronize()
        for t in out:
            t.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), "replay %d" % rep


@pytest.mark.parametrize("T,k,rows,rank,dtype", [(4099, 40, 68, 16, BF16), (4099, 33, 20, 40, BF16), (4500, 32, 12, 64, F16),
                                                 (5000, 36, 24, 128, F32)])
def test_long_batches_with_bad_rows(ex, hip_rt, T, k, rows, rank, dtype):
    """Batches whose tiles are shrunk and expanded at once: values, a row of NaN, of an
    infinity and of a bad id that touch no other row, no base, the same bits in place."""
    c = Case(T + rank, T, k, rows, rank, 3, dtype, adapters="each")
    want, bound = c.forward()
    got = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base)
    close(got, want, bound, "forward")
    close(ex.lora_apply(c.lora, c.d_x, c.d_ad), want - c.base, bound, "without a base")
    again = c.d_base.clone()
    ex.lora_apply(c.lora, c.d_x, c.d_ad, again, out=again)
    assert torch.equal(again, got)
    hip_ok()
    x, ad = c.d_x.clone(), c.d_ad.clone()
    ad[7:10] = torch.tensor([0, 1, 5], dtype=torch.int32)
    x[7, 0, 3], x[8, 0, k - 1] = float("nan"), float("-inf")
    bad = ex.lora_apply(c.lora, x, ad, c.d_base)
    torch.cuda.synchronize()
    rest = torch.ones(T, dtype=torch.bool, device=DEV)
    rest[7:10] = False
    assert torch.equal(bad[rest], got[rest])
    assert bad[7].isnan().all() and not bad[8].isfinite().any() and bad[9].isnan().all()
    with pytest.raises(hip_rt.SabahRuntimeError, match="adapter id"):
        hip_rt.check(hip_rt.lib().sabah_rt_check_errors(), "sticky")


@pytest.mark.parametrize("T,k,rows,rank,dtype,adapters", [
    (9300, 24, 20, 16, BF16, "each"), (9300, 20, 70, 64, BF16, "runs"), (3000, 66, 12, 128, F16, "runs"),
    (2049, 36, 40, 40, F32, "each"), (2048, 36, 40, 40, F32, "each"), (4099, 72, 8, 32, F16, "runs")])
def test_gradients_over_many_windows(ex, T, k, rows, rank, dtype, adapters):
    c = Case(T + rank, T, k, rows, rank, 5, dtype, adapters=adapters)
    want, bound = c.backward()
    for g, w, b, what in zip(ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy), want, bound, ("dx", "da", "db")):
        close(g, w, b, what)
    hip_ok()


@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 47, 63, 65])
def test_tiles_that_end_anywhere(ex, n):
    """Keys of n rows, at ranks with tiles of 16 and of 32 rows, one window and several."""
    for T, rank in ((max(260, 4 * n), 48), (max(260, 4 * n), 8), (2100, 80)):
        c = Case(n, T, 36, 20, rank, 3, BF16, adapters=[0] * n + [1] * (n + 1) + [2] * (T - 2 * n - 1))
        want, bound = c.forward()
        close(ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base), want, bound, "forward")
        want, bound = c.backward()
        for g, w, b, what in zip(ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy), want, bound, ("dx", "da", "db")):
            close(g, w, b, what)


@pytest.mark.parametrize("T", [9, 1500, 2600])
def test_infinities_in_training_stay_with_their_pair(ex, T):
    """An infinity of x or dy leaves its pair's gradients not finite, where they are the adapter's own
    rank's; past it they are zeros, and other pairs and rows keep their bits."""
    c = Case(T, T, 40, 24, 16, 4, BF16, adapters=[t % 4 for t in range(T)], ranks=[16, 5, 16, 16])
    dx, da, db = ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy)
    x, dy = c.d_x.clone(), c.d_dy.clone()
    x[1, 0, 3], dy[5, 0, 2] = float("inf"), float("-inf")   # both rows of adapter 1
    gx, ga, gb = ex.lora_backward(c.lora, x, c.d_ad, dy)
    rows = torch.ones(T, dtype=torch.bool, device=DEV)
    rows[5] = False                                         # dx of row 1 does not depend on x
    assert torch.equal(gx[rows], dx[rows]) and not gx[5].isfinite().all()
    for n in (0, 2, 3):
        assert torch.equal(ga[n], da[n]) and torch.equal(gb[n], db[n])
    assert not ga[1, 0, :5].isfinite().all() and not gb[1, 0, :, :5].isfinite().all()
    assert not ga[1, 0, 5:].any() and not gb[1, 0, :, 5:].any()
    # rows without an adapter are not read
    ad = c.d_ad.clone()
    ad[1] = ad[5] = -1
    want = ex.lora_backward(c.lora, c.d_x, ad, c.d_dy)
    got = ex.lora_backward(c.lora, x, ad, dy)
    assert all(torch.equal(g, w) for g, w in zip(got, want)) and got[1].isfinite().all()


def test_an_expert_named_twice_and_broadcast_rows(ex):
    """The same expert in two slots of a token, a base and dy shared by all tokens, one x for all."""
    c = Case(6, 50, 64, 40, 8, 3, BF16, E=8, slots=3)
    c.ids[:, 2] = c.ids[:, 0]
    c.x[:], c.base[:], c.dy[:] = c.x[:1], c.base[:1], c.dy[:1]
    ids = torch.from_numpy(c.ids).to(DEV)
    x, base, dy = (torch.from_numpy(v[:1]).to(DEV).expand(v.shape) for v in (c.x, c.base, c.dy))
    want, bound = c.forward()
    got = ex.lora_apply(c.lora, x, c.d_ad, base, ids=ids)
    close(got, want, bound, "forward")
    want, bound = c.backward()
    for g, w, b, what in zip(ex.lora_backward(c.lora, x, c.d_ad, dy, ids=ids), want, bound, ("dx", "da", "db")):
        close(g, w, b, what)


@pytest.mark.parametrize("T", [3, 300, 4200])
def test_as_many_adapters_as_a_call_takes(ex, T):
    n = 1 << 21
    g = np.random.default_rng(T)
    ad = g.integers(-1, n, T)
    ad[0], ad[-1] = n - 1, 0
    c = Case(T, T, 4, 3, 1, 1, F32, adapters=[0] * T)
    from sabah.runtime.lora import LoraBank
    c.lora = LoraBank(n, 1, 4, 3, dtype=F32, device="cuda:0")
    gen = torch.Generator(device=DEV).manual_seed(T)
    c.lora.a.normal_(generator=gen)
    c.lora.b.normal_(generator=gen)
    c.ad = ad.astype(np.int32)
    want, bound = c.forward()
    close(ex.lora_apply(c.lora, c.d_x, torch.from_numpy(c.ad).to(DEV), c.d_base), want, bound, "forward")
    with pytest.raises(Exception, match="pairs"):
        ex.lora_backward(c.lora, c.d_x, torch.from_numpy(c.ad).to(DEV), c.d_dy)
    n = 1 << 15
    c.lora = LoraBank(n, 1, 4, 3, dtype=F32, device="cuda:0")
    c.lora.a.normal_(generator=gen)
    c.lora.b.normal_(generator=gen)
    c.ad = np.where(c.ad < 0, -1, c.ad % n).astype(np.int32)
    want, bound = c.backward()
    for gr, w, b, what in zip(ex.lora_backward(c.lora, c.d_x, torch.from_numpy(c.ad).to(DEV), c.d_dy), want, bound,
                              ("dx", "da", "db")):
        close(gr, w, b, what)


@pytest.mark.parametrize("T,step", [(3, 1 << 29), (300, 1 << 22)])
def test_rows_beyond_four_gigabytes(ex, T, step):
    """Rows 2 GiB and 16 MiB apart (the last one past 2^32 bytes): x, base, out, dy and dx in one
    allocation; logits and their gradient in it too."""
    k, rows = 64, 48
    room = torch.empty((T - 1) * step + 4096, device=DEV)
    at = lambda o, w: torch.as_strided(room, (T, w), (step, 1), o)
    x, base, out, dy, dx, logits, dl = (at(500 * i, w) for i, w in enumerate((k, rows, rows, rows, k, 40, 40)))
    c = Case(T, T, k, rows, 8, 2, BF16, adapters="each")
    x.copy_(c.d_x[:, 0])
    base.copy_(c.d_base[:, 0])
    dy.copy_(c.d_dy[:, 0])
    want, bound = c.forward()
    got = ex.lora_apply(c.lora, x, c.d_ad, base, out=out)
    close(got.contiguous(), want, bound, "forward")
    want, bound = c.backward()
    for g, w, b, what in zip(ex.lora_backward(c.lora, x, c.d_ad, dy, dx=dx), want, bound, ("dx", "da", "db")):
        close(g.contiguous(), w, b, what)
    logits.copy_(torch.randn(T, 40, generator=torch.Generator(device=DEV).manual_seed(T), device=DEV))
    dense = logits.contiguous()
    ids, _ = ex.route(dense, 4)
    a, b = ex.balance(logits, ids), ex.balance(dense, ids)
    assert torch.equal(a.counts, b.counts) and torch.equal(a.mean_p, b.mean_p) and torch.equal(a.losses, b.losses)
    assert torch.equal(ex.route_backward(logits, ids, None, a, 0.5, 0.5, out=dl).contiguous(),
                       ex.route_backward(dense, ids, None, b, 0.5, 0.5))


def test_adapters_beyond_four_gigabytes(ex):
    """A bank of 10 GiB: the last pair's elements lie past 2^32."""
    c = Case(8, 40, 8192, 16, 128, 1, BF16)
    from sabah.runtime.lora import LoraBank
    big = LoraBank(40, 128, 8192, 16, n_experts=128, device="cuda:0")
    big.a[39, 127], big.b[39, 127] = c.lora.a[0, 0], c.lora.b[0, 0]
    big.scale[39] = c.lora.scale[0]
    ad = torch.where(c.d_ad == 0, 39, -1).to(torch.int32)
    ids = torch.full((40, 1), 127, dtype=torch.int32, device=DEV)
    want, bound = c.forward()
    close(ex.lora_apply(big, c.d_x, ad, c.d_base, ids=ids), want, bound, "forward")
    want, bound = c.backward()
    dx, da, db = ex.lora_backward(big, c.d_x, ad, c.d_dy, ids=ids)
    close(dx, want[0], bound[0], "dx")
    close(da[39, 127], want[1][0, 0], bound[1][0, 0], "da")
    close(db[39, 127], want[2][0, 0], bound[2][0, 0], "db")
    assert not da[:39].any() and not da[39, :127].any() and not db[:39].any() and not db[39, :127].any()


def test_calls_refuse_what_would_overwrite_their_inputs(ex, hip_rt):
    c = Case(4, 6, 48, 48, 8, 2, BF16)
    for call in (lambda: ex.lora_apply(c.lora, c.d_x, c.d_ad, out=c.d_x),
                 lambda: ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy, dx=c.d_dy),
                 lambda: ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy, dx=c.d_x)):
        with pytest.raises(hip_rt.SabahRuntimeError, match="overwrite"):
            call()
    with pytest.raises(ValueError):
        ex.mul_mat_id(0, "gate", torch.zeros(2, 1, 256, device=DEV), torch.zeros(2, 1, dtype=torch.int32, device=DEV),
                      lora=c.lora)


def test_the_losses_of_another_device_are_refused(ex):
    from sabah.runtime.executor import RouterBalance
    logits, ids = torch.zeros(4, 16, device=DEV), torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    away = RouterBalance(16, 1, device="cpu")
    with pytest.raises(ValueError):
        ex.balance(logits, ids, out=away)
    with pytest.raises(ValueError):
        ex.route_backward(logits, ids, None, away, 1.0, 1.0)


def test_the_current_stream_orders_the_calls(ex):
    """On a stream of its own, behind work that fills the inputs there, a call reads what that work wrote."""
    c = Case(12, 300, 256, 128, 16, 3, BF16, adapters="runs")
    want, bound = c.forward()
    x = torch.zeros_like(c.d_x)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        busy = torch.randn(2048, 2048, device=DEV)
        for _ in range(4):
            busy = busy @ busy * 1e-3
        x.copy_(c.d_x + busy[0, 0].nan_to_num(0, 0, 0) * 0)
        got = ex.lora_apply(c.lora, x, c.d_ad, c.d_base)
        dx, da, db = ex.lora_backward(c.lora, x, c.d_ad, c.d_dy)
    s.synchronize()
    close(got, want, bound, "forward")
    wants, bounds = c.backward()
    for g, w, b, what in zip((dx, da, db), wants, bounds, ("dx", "da", "db")):
        close(g, w, b, what)


@pytest.mark.parametrize("T", [5, 300, 2100, 5000])
@pytest.mark.parametrize("fill", [0, 255])
def test_the_workspace_may_hold_anything_and_each_gradient_may_be_left_out(ex, hip_rt, T, fill):
    """The calls of the C interface with a workspace full of zeros, or of ones (NaN, -1), and with
    one output at a time: the executor's bits."""
    lib = hip_rt.lib()
    c = Case(T, T, 72, 40, 20, 5, BF16, adapters="each")
    y = ex.lora_apply(c.lora, c.d_x, c.d_ad, c.d_base)
    dx, da, db = ex.lora_backward(c.lora, c.d_x, c.d_ad, c.d_dy)
    _, slots, rows = ex._lora_rows(c.lora, c.d_x, c.d_ad, None, c.d_base)
    stream = torch.cuda.current_stream().cuda_stream
    n = c.lora.space(lib, slots, T)
    ws = torch.full((max(n, 16),), fill, dtype=torch.uint8, device=DEV)
    got = torch.full_like(y, 3.0)
    rc = lib.sabah_lora_apply(c.lora.ref, *rows, *ex._lora_y("base", c.d_base, T, 1, 40),
                              *ex._lora_y("out", got, T, 1, 40), ws.data_ptr(), n, stream)
    hip_rt.check(rc, "apply")
    assert torch.equal(got, y)
    n = c.lora.space(lib, slots, T, 1)
    for which in range(3):
        ws = torch.full((n,), fill, dtype=torch.uint8, device=DEV)
        outs = [torch.full_like(g, 3.0) if i == which else None for i, g in enumerate((dx, da, db))]
        d = ex._lora_y("dx", outs[0], T, 1, 72) if which == 0 else (None, 0, 0)
        rc = lib.sabah_lora_backward(c.lora.ref, *rows, *ex._lora_y("dy", c.d_dy, T, 1, 40), *d, 0,
                                     outs[1].data_ptr() if which == 1 else None,
                                     outs[2].data_ptr() if which == 2 else None, 0, ws.data_ptr(), n, stream)
        hip_rt.check(rc, "backward")
        assert torch.equal(outs[which], (dx, da, db)[which]), which


@pytest.mark.parametrize("T,E,groups", [(3, 8, 1), (96, 300, 8), (4000, 512, 4)])
def test_the_losses_workspace_may_hold_anything(ex, hip_rt, T, E, groups):
    lib = hip_rt.lib()
    logits = torch.randn(T, E, generator=torch.Generator(device=DEV).manual_seed(T), device=DEV)
    ids, _ = ex.route(logits, 4)
    want = ex.balance(logits, ids, n_groups=groups)
    n = lib.sabah_moe_balance_workspace(T, E, groups)
    for fill in (0, 255):
        ws = torch.full((n,), fill, dtype=torch.uint8, device=DEV)
        got = [torch.full_like(t, 7) for t in (want.counts, want.mean_p, want.losses, want.n_valid)]
        rc = lib.sabah_moe_balance(logits.data_ptr(), E * 4, ids.data_ptr(), None, T, E, 4, groups,
                                   *(t.data_ptr() for t in got), ws.data_ptr(), n,
                                   torch.cuda.current_stream().cuda_stream)
        hip_rt.check(rc, "balance")
        assert all(torch.equal(a, b) for a, b in zip(got, (want.counts, want.mean_p, want.losses, want.n_valid)))
