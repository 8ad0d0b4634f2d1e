"""MoEExecutor.block_norm and block_norm_backward against the 64-bit forms of train_refs."""
import pytest
import torch

import train_refs as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS, SCALE = 1e-6, 0.5


@pytest.fixture(scope="module")
def ex(hip_rt):
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    return MoEExecutor(ExpertBank(1, 8, 256, 256, {"gate": 21, "up": 21, "down": 21}, device=DEV))


def make(T, D, dtype, after, before, gate, seed=1, y=True):
    from sabah.runtime.norm import BlockNorm
    g = torch.Generator().manual_seed(seed)
    n = BlockNorm(D, after=after, before=before, eps=EPS, scale=SCALE, device=DEV)
    for w in (n.w_after, n.w_before):
        if w is not None:
            w.copy_(1 + 0.3 * torch.randn(D, generator=g))
    t = dict(x=torch.randn(T, D, generator=g) * 2, y=torch.randn(T, D, generator=g) if y else None,
             dout=torch.randn(T, D, generator=g), dh=torch.randn(T, D, generator=g) if before else None)
    t = {k: v.to(dtype).to(DEV) if v is not None else None for k, v in t.items()}
    t["gate"] = torch.randn(T, generator=g).to(DEV) if gate else None
    return n, t


def cpu(t):
    return t.cpu() if t is not None else None


def check_forward(n, t, out, h):
    dtype = t["x"].dtype
    if t["y"] is not None:
        want, branch = R.norm(cpu(t["x"]), cpu(t["y"]), cpu(t["gate"]), cpu(n.w_after), None, EPS, SCALE)
        R.close(out, want, 34 * R.U * branch + R.U * want.abs() + R.half_step(want, dtype), "out")
    if n.w_before is not None:
        want = R.norm_h(cpu(out if t["y"] is not None else t["x"]), cpu(n.w_before), EPS)
        R.close(h, want, 32 * R.U * want.abs() + R.half_step(want, dtype), "h")


def check_backward(n, t, out, got):
    dtype = out.dtype
    want = R.norm_back(cpu(out), cpu(t["y"]), cpu(t["gate"]), cpu(n.w_after) if t["y"] is not None else None, cpu(n.w_before),
                       cpu(t["dout"]), cpu(t["dh"]), EPS, SCALE)
    for name, g in zip(("dx", "dy", "dgate", "dw_after", "dw_before"), got):
        if name not in want:
            assert g is None or (name == "dx" and g is t["dout"])
            continue
        v, tol = want[name]
        R.close(g, v, tol + (R.half_step(v, dtype) if name in ("dx", "dy") else 0), name)


FORMS = [(True, True, True, True), (False, True, False, True), (True, False, True, True), (False, True, False, False),
         (False, False, True, True), (True, True, False, True)]     # after, before, gate, y


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("T,D", [(1, 1), (3, 5), (7, 511), (5, 640), (4, 1025), (130, 2048), (9, 2560), (5, 2559), (3, 2561), (6, 1000), (3, 4097), (2, 8189), (1, 8192)])
def test_forward_and_backward(ex, T, D, form, dtype):
    n, t = make(T, D, TYPES[dtype], *form[:3], y=form[3])
    out, h = ex.block_norm(n, t["x"], t["y"], t["gate"])
    assert (out is None) == (t["y"] is None) and (h is None) == (n.w_before is None)
    check_forward(n, t, out, h)
    kept = out if out is not None else t["x"]
    got = ex.block_norm_backward(n, kept, t["y"], t["gate"], dout=t["dout"], dh=t["dh"])
    check_backward(n, t, kept, got)


@pytest.mark.parametrize("T", [64, 1023, 1025, 4100, 70000])
def test_many_tokens(ex, T):
    """Parts of one token, of several, and more parts than fill the chip."""
    n, t = make(T, 40, torch.float32, True, True, True)
    out, h = ex.block_norm(n, t["x"], t["y"], t["gate"])
    check_forward(n, t, out, h)
    check_backward(n, t, out, ex.block_norm_backward(n, out, t["y"], t["gate"], dout=t["dout"], dh=t["dh"]))


def test_gradients_against_differences(ex):
    """The whole pass in f32 against central differences of the 64-bit form."""
    T, D = 3, 24
    n, t = make(T, D, torch.float32, True, True, True, seed=4)
    out, h = ex.block_norm(n, t["x"], t["y"], t["gate"])
    got = ex.block_norm_backward(n, out, t["y"], t["gate"], dout=t["dout"], dh=t["dh"])
    p = {"x": cpu(t["x"]).double(), "y": cpu(t["y"]).double(), "gate": cpu(t["gate"]).double(), "w_after": cpu(n.w_after).double(),
         "w_before": cpu(n.w_before).double()}

    def loss(p):
        o, _ = R.norm(p["x"], p["y"], p["gate"], p["w_after"], None, EPS, SCALE)
        return ((o * cpu(t["dout"]).double()).sum() + (R.norm_h(o, p["w_before"], EPS) * cpu(t["dh"]).double()).sum()).item()
    for name, g in zip(("x", "y", "gate", "w_after", "w_before"), got):
        flat = p[name].reshape(-1)
        for i in range(0, flat.numel(), 7):
            keep, e = flat[i].item(), 1e-5
            flat[i] = keep + e
            up = loss(p)
            flat[i] = keep - e
            down = loss(p)
            flat[i] = keep
            # e^2 times third derivatives of at most some tens, the loss's own rounding over 2 e, and f32's error of out
            assert abs((up - down) / (2 * e) - g.reshape(-1)[i].item()) < 2e-5, (name, i)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_in_place_and_rows_behind(ex, dtype):
    """Rows of wider tensors, out in place of x, dx in place of dout; what lies beside the rows stays."""
    T, D, W = 6, 333, 401
    n, t = make(T, D, TYPES[dtype], True, True, True)
    plain = ex.block_norm(n, t["x"], t["y"], t["gate"])
    want = ex.block_norm_backward(n, plain[0], t["y"], t["gate"], dout=t["dout"], dh=t["dh"])
    wide = {k: torch.full((T + 1, W), 7.0, dtype=TYPES[dtype], device=DEV) for k in ("x", "y", "dout", "dh", "h", "dy")}
    rows = {k: w[:T, 3:3 + D] for k, w in wide.items()}
    for k in ("x", "y", "dout", "dh"):
        rows[k].copy_(t[k])
    out, h = ex.block_norm(n, rows["x"], rows["y"], t["gate"], out=rows["x"], h=rows["h"])
    assert out is rows["x"] and torch.equal(out, plain[0]) and torch.equal(h, plain[1])
    got = ex.block_norm_backward(n, out, rows["y"], t["gate"], dout=rows["dout"], dh=rows["dh"], dx=rows["dout"], dy=rows["dy"])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for w in wide.values():
        assert (w[T] == 7).all() and (w[:, :3] == 7).all() and (w[:, 3 + D:] == 7).all()


def test_weight_gradients_are_added(ex):
    n, t = make(50, 96, torch.float32, True, True, False)
    out, _ = ex.block_norm(n, t["x"], t["y"])
    one = ex.block_norm_backward(n, out, t["y"], dout=t["dout"], dh=t["dh"])
    a, b = torch.full((96,), 3.0, device=DEV), torch.full((96,), -2.0, device=DEV)
    ex.block_norm_backward(n, out, t["y"], dout=t["dout"], dh=t["dh"], dw_after=a, dw_before=b, add_dw=True)
    for got, base, part in ((a, 3.0, one[3]), (b, -2.0, one[4])):
        want = base + part.double()
        R.close(got, want, 2 * R.U * (abs(base) + part.double().abs()) + R.U * want.abs())


def test_no_tokens(ex):
    n, t = make(0, 64, torch.bfloat16, True, True, True)
    out, h = ex.block_norm(n, t["x"], t["y"], t["gate"])
    assert out.shape == h.shape == (0, 64)
    a, b = torch.full((64,), 5.0, device=DEV), torch.full((64,), 5.0, device=DEV)
    got = ex.block_norm_backward(n, out, t["y"], t["gate"], dout=t["dout"], dh=t["dh"], dw_after=a, dw_before=b, add_dw=True)
    assert (a == 5).all() and (b == 5).all()
    got = ex.block_norm_backward(n, out, t["y"], t["gate"], dout=t["dout"], dh=t["dh"])
    assert (got[3] == 0).all() and (got[4] == 0).all()


def test_nan_and_infinity_stay_in_their_rows(ex):
    n, t = make(40, 700, torch.float32, True, True, True)
    out0, h0 = ex.block_norm(n, t["x"], t["y"], t["gate"])
    t["x"][3, 5], t["y"][7, 9], t["gate"][11] = float("nan"), float("inf"), float("nan")
    t["gate"][12], t["gate"][13] = -200.0, 200.0
    out, h = ex.block_norm(n, t["x"], t["y"], t["gate"])
    sick = torch.zeros(40, dtype=torch.bool)
    sick[[3, 7, 11]] = True
    same = ~sick
    same[[12, 13]] = False
    assert torch.equal(out[same.to(DEV)], out0[same.to(DEV)]) and torch.equal(h[same.to(DEV)], h0[same.to(DEV)])
    assert h[3].isnan().all() and h[11].isnan().all() and not out[~sick.to(DEV)].isnan().any()
    assert torch.equal(out[12], t["x"][12])                      # a gate shut wholly
    dx, dy, dgate, _, _ = ex.block_norm_backward(n, out, t["y"], t["gate"], dout=t["dout"], dh=t["dh"])
    assert not dx[~sick.to(DEV)].isnan().any() and not dy[~sick.to(DEV)].isnan().any()
    assert (dy[12] == 0).all() and dgate[12] == 0 and dgate[13] == 0


def test_more_threads_than_a_launch_takes_along_x(ex):
    """2^22 + 3 tokens of 1,024 threads each are more than 2^32."""
    from sabah.runtime.norm import BlockNorm
    T, D = (1 << 22) + 3, 4097
    n = BlockNorm(D, after=False, eps=EPS, device=DEV)
    x = torch.empty(T, D, dtype=torch.bfloat16, device=DEV)
    x.fill_(2.0)
    x[T - 1] = 4.0
    _, h = ex.block_norm(n, x)
    for rows in (h[:2], h[(1 << 20) - 1:(1 << 20) + 2], h[T - 2:]):
        assert (rows == 1).all()                              # of equal values: rounded to bf16, 1 exactly
    del x, h
    torch.cuda.empty_cache()


def test_rows_of_zeros(ex):
    """The mean is zero and eps alone divides."""
    n, t = make(4, 100, torch.float32, True, True, False)
    t["x"].zero_()
    t["y"].zero_()
    out, h = ex.block_norm(n, t["x"], t["y"])
    assert (out == 0).all() and (h == 0).all()
    check_backward(n, t, out, ex.block_norm_backward(n, out, t["y"], dout=t["dout"], dh=t["dh"]))


def test_captured_and_replayed_on_another_stream(ex):
    n, t = make(200, 1536, torch.bfloat16, True, True, True)

    def both():
        out, h = ex.block_norm(n, t["x"], t["y"], t["gate"])
        return (out, h) + ex.block_norm_backward(n, out, t["y"], t["gate"], dout=t["dout"], dh=t["dh"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [w.clone() for w in both()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(3):
        t["x"].copy_(t["x"] + i)
        graph.replay()
        want = both()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
