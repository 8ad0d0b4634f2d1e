"""AdamW against the 64-bit forms of train_refs."""
import math

import pytest
import torch

import train_refs as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8)
SIZES = [1, 3, 255, 256, 257, 2048, 2049, 5000]


def make(sizes, p_types, g_types, seed=1, **kw):
    from sabah.runtime.adamw import AdamW
    g = torch.Generator().manual_seed(seed)
    ps = [torch.randn(n, generator=g).to(p_types[i % len(p_types)]).to(DEV) for i, n in enumerate(sizes)]
    gs = [(torch.randn(n, generator=g) * 10.0 ** (i % 5 - 3)).to(g_types[i % len(g_types)]).to(DEV) for i, n in enumerate(sizes)]
    decay = [0.0 if i % 2 else 0.1 for i in range(len(sizes))]
    return AdamW(ps, gs, weight_decay=decay, **HYPER, **kw), ps, gs, decay


def tensors(opt, flat):
    return [flat[at:at + p.numel()].cpu() for p, at in zip(opt.params, opt.starts)]


def check_step(opt, before, gs, decay, t, c=1.0):
    """One step from the state `before` (of p or master, m, v as values, m_scale and v_scale): f32 operations, each off by u."""
    ms, vs = (tensors(opt, f) for f in opt.moments())
    lr, eps = HYPER["lr"], HYPER["eps"]
    for i, p in enumerate(opt.params):
        p0, m0, v0 = before[0][i], before[1][i], before[2][i]
        g = gs[i].cpu().double() * c
        want, m, v, step = R.adamw(p0, gs[i].cpu(), m0, v0, t, lr, HYPER["betas"], eps, decay[i], c)
        # c, g c, two products and a sum; v with a square: at most 4 and 6 roundings of each part
        tm = 6 * R.U * (m0.double().abs() + g.abs()) + 1e-44
        tv = 8 * R.U * (v0.double().abs() + g * g) + 1e-44
        if opt.bits == 32:
            R.close(ms[i], m, tm, "m")
            R.close(vs[i], v, tv, "v")
        # m's own error, half of v's relative one, and 8 roundings of the step; 3 of the rest
        scale = lr / (1 - HYPER["betas"][0] ** t) / ((v / (1 - HYPER["betas"][1] ** t)).sqrt() + eps)
        tp = scale * tm + step.abs() * (12 * R.U + tv / v.clamp(min=1e-300)).clamp(max=1) + 3 * R.U * (p0.double().abs() + step.abs())
        got = opt.master[opt.starts[i]:opt.starts[i] + p.numel()].cpu() if opt.master is not None and p.dtype != F32 else p.cpu()
        R.close(got, want, tp + (R.half_step(want, p.dtype) if got.dtype != F32 else 0), "p")
        if got.dtype == F32 and p.dtype != F32:
            assert torch.equal(p.cpu(), got.to(p.dtype))


def state(opt):
    ps = tensors(opt, opt.master) if opt.master is not None else [p.cpu().clone() for p in opt.params]
    ps = [p.cpu().clone() if q.dtype == F32 else m for p, q, m in zip(opt.params, opt.params, ps)]
    m, v = opt.moments()
    return ps, [t.clone() for t in tensors(opt, m)], [t.clone() for t in tensors(opt, v)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("p_types,g_types,master", [((F32,), (F32,), False), ((BF16,), (F32,), True), ((F16,), (F16,), False),
                                                    ((F32, BF16, F16), (BF16, F32, F16), True), ((BF16,), (BF16,), False)])
def test_steps(hip_rt, bits, p_types, g_types, master):
    opt, ps, gs, decay = make(SIZES, p_types, g_types, bits=bits, master=master)
    for t in range(1, 5):
        before = state(opt)
        opt.step()
        torch.cuda.synchronize()
        assert opt.step_count.item() == t
        check_step(opt, before, gs, decay, t)
        for g in gs:
            g.mul_(-0.7)


def test_moments_of_8_bits_are_the_nearest_codes(hip_rt):
    """Codes and scales against the 64-bit forms; a value within 1e-9 steps of a border may take either code."""
    opt, ps, gs, _ = make([70000], (F32,), (F32,), bits=8)
    for _ in range(3):
        m0, v0 = (f.double().cpu() for f in opt.moments())
        # the values in 64 bits, from the codes themselves
        m0 = (R.m_value(opt.m.cpu()).reshape(-1, 256) * opt.m_scale.cpu().double()[:, None])
        v0 = (R.v_value(opt.v.cpu()).reshape(-1, 256) * opt.v_scale.cpu().double()[:, None])
        g = torch.zeros(opt.n_values, dtype=torch.float64)
        g[:70000] = gs[0].cpu().double()
        g = g.reshape(-1, 256)
        opt.step()
        torch.cuda.synchronize()
        b1, b2 = HYPER["betas"]
        m, v = m0 * b1 + g * (1 - b1), v0 * b2 + g * g * (1 - b2)
        for value, scale, code, find in ((m, opt.m_scale, opt.m, R.m_code), (v, opt.v_scale, opt.v, R.v_code)):
            s = value.abs().amax(1).float()
            assert torch.equal(scale.cpu(), s)
            want, border = find(value, s[:, None])
            differ = code.cpu().reshape(-1, 256).double() != want
            assert not (differ & (border > 1e-9)).any(), int(differ.sum())
        gs[0].mul_(-1.3)


def test_reading_and_writing_moments_of_8_bits(hip_rt):
    """Every code goes to its value and back; zeros, infinities and NaN."""
    opt, _, _, _ = make([256 * 64], (F32,), (F32,), bits=8)
    g = torch.Generator().manual_seed(3)
    mc = torch.randint(-127, 128, (64, 256), generator=g)
    vc = torch.randint(0, 256, (64, 256), generator=g)
    mc[:, 0], vc[:, 0] = -127, 255
    ms = torch.exp(torch.randn(64, generator=g) * 20).float()
    vs = torch.exp(torch.randn(64, generator=g) * 20).float()
    m = (R.m_value(mc) * ms.double()[:, None]).float()
    v = (R.v_value(vc) * vs.double()[:, None]).float()
    opt.load_moments(m.reshape(-1).to(DEV), v.reshape(-1).to(DEV), 7)
    assert opt.step_count.item() == 7
    assert torch.equal(opt.m.cpu().reshape(64, 256).long(), mc) and torch.equal(opt.v.cpu().reshape(64, 256).long(), vc)
    rm, rv = opt.moments()
    assert torch.equal(rm.cpu().reshape(64, 256), m) and torch.equal(rv.cpu().reshape(64, 256), v)
    m, v = m * 0, v * 0
    v[1, 5], v[2, 9], m[3, 1], m[4, 2], m[4, 3] = 1e-38, float("inf"), float("nan"), float("-inf"), 1.0
    v[1, 6] = 1e-45                                             # f32's smallest: 255 (1.4e-45 / 1e-38)^(1/4) = 4.93
    v[5, 0], v[5, 1] = 1.0, 1e-30
    opt.load_moments(m.reshape(-1).to(DEV), v.reshape(-1).to(DEV), 0)
    rm, rv = (f.cpu().reshape(64, 256) for f in opt.moments())
    assert (rm[0] == 0).all() and (rv[0] == 0).all() and rm[3].isnan().all() and rv[3].isnan().all()
    assert rv[1, 5] == 1e-38 or abs(rv[1, 5] - 1e-38) < 1e-44
    assert opt.v[256 + 6] == 5
    assert opt.v[5 * 256 + 1] == 1 and rv[5, 1] > 0             # above 0 stays above 0
    most = torch.finfo(F32).max
    assert rv[2, 9] == most and rv[2].isfinite().all() and rm[4, 2] == -most and rm[4].isfinite().all()


@pytest.mark.parametrize("bits", [32, 8])
def test_norm_and_clipping(hip_rt, bits):
    opt, ps, gs, decay = make(SIZES, (F32,), (F32, BF16), bits=bits, max_norm=0.5)
    for t, scale in ((1, 1.0), (2, 0.125), (3, 1e-6)):
        before = state(opt)
        opt.step(grad_scale=scale)
        torch.cuda.synchronize()
        norm = scale * math.sqrt(sum(g.double().square().sum().item() for g in gs))
        assert abs(opt.grad_norm.item() - norm) <= 2 * R.U * norm
        check_step(opt, before, gs, decay, t, scale * min(1.0, 0.5 / (norm + 1e-6)))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_step_without_a_finite_norm_changes_nothing(hip_rt, bits, bad):
    opt, ps, gs, _ = make(SIZES, (BF16, F32), (F32,), bits=bits, master=True, max_norm=1.0)
    opt.step()
    keep = [t.clone() for t in ps + [opt.m, opt.v, opt.master, opt.step_count]]
    gs[3][17] = bad
    opt.step()
    torch.cuda.synchronize()
    assert not math.isfinite(opt.grad_norm.item())
    for a, b in zip(ps + [opt.m, opt.v, opt.master, opt.step_count], keep):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [32, 8])
def test_without_clipping_nan_stays_in_its_value_or_block(hip_rt, bits):
    opt, ps, gs, _ = make([1000, 700], (F32,), (F32,), bits=bits)
    other, qs, hs, _ = make([1000, 700], (F32,), (F32,), bits=bits)
    gs[0][300] = float("nan")
    for o in (opt, other):
        o.step()
        o.step()
    torch.cuda.synchronize()
    sick = torch.zeros(1000, dtype=torch.bool)
    sick[300] = True
    if bits == 8:
        sick[256:512] = True                                    # the second step reads the block's NaN
    ok = ~sick.to(DEV)
    assert torch.equal(ps[0][ok], qs[0][ok]) and torch.equal(ps[1], qs[1]) and ps[0][300].isnan()


def test_large_and_small_gradients(hip_rt):
    """Squares that leave f32: v infinite (32 bits: no change of p), or the scale's largest value (8 bits)."""
    for bits in (32, 8):
        opt, ps, gs, _ = make([512], (F32,), (F32,), bits=bits)
        gs[0].fill_(1e30)
        gs[0][256:] = 1e-30
        p0 = ps[0].clone()
        opt.step()
        torch.cuda.synchronize()
        assert ps[0].isfinite().all()
        assert (ps[0] - p0 * (1 - HYPER["lr"] * 0.1)).abs().max() <= HYPER["lr"] * 1.001 + 1e-6
        assert opt.moments()[0].isfinite().all()


def test_views_at_any_address_and_what_lies_beside_them(hip_rt):
    from sabah.runtime.adamw import AdamW
    flat, grads = torch.full((4000,), 2.0, device=DEV, dtype=BF16), torch.full((4000,), 0.5, device=DEV, dtype=BF16)
    cuts = [(1, 1302), (1303, 1304), (1307, 3999)]
    opt = AdamW([flat[a:b] for a, b in cuts], [grads[a:b] for a, b in cuts], lr=0.25, weight_decay=0.0)
    opt.step()
    torch.cuda.synchronize()
    want = torch.full((4000,), 2.0, dtype=BF16)
    for a, b in cuts:
        want[a:b] = 1.75
    assert torch.equal(flat.cpu(), want)
    assert opt.starts == [0, 1536, 1792] and opt.n_values == 1792 + 2816
    assert (opt.m[1301:1536] == 0).all() and (opt.m[1537:1792] == 0).all()


def test_many_small_tensors_and_empty_ones(hip_rt):
    sizes = [(i * 37) % 90 for i in range(1500)]
    opt, ps, gs, decay = make(sizes, (F32, BF16), (F32,))
    before = state(opt)
    opt.step()
    torch.cuda.synchronize()
    check_step(opt, before, gs, decay, 1)
    opt, _, _, _ = make([0, 0], (F32,), (F32,), max_norm=1.0)
    opt.step()
    torch.cuda.synchronize()
    assert opt.grad_norm.item() == 0 and opt.step_count.item() == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_follow_gradients_and_rate(hip_rt, bits):
    """A replayed step against an eager one from the same state, with a rate that is read on the device."""
    lr = torch.tensor([1e-2], device=DEV)
    kw = dict(bits=bits, max_norm=3.0, master=True)
    from sabah.runtime.adamw import AdamW
    g = torch.Generator().manual_seed(5)
    start = [torch.randn(n, generator=g).to(BF16) for n in SIZES]
    pa, pb = [t.to(DEV) for t in start], [t.to(DEV) for t in start]
    gs = [torch.randn(n, generator=g).to(DEV) for n in SIZES]
    a, b = AdamW(pa, gs, lr=lr, **kw), AdamW(pb, gs, lr=lr, **kw)
    a.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    b.step()
    for i in range(3):
        lr.mul_(0.5)
        for t in gs:
            t.mul_(-0.9)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert a.step_count.item() == b.step_count.item() == i + 2
        for x, y in zip(pa + [a.m, a.v, a.master, a.grad_norm], pb + [b.m, b.v, b.master, b.grad_norm]):
            assert torch.equal(x, y)


def test_rate_and_norm_set_between_steps(hip_rt):
    """What lr and max_norm are when step() is called counts: each step equals that of an optimizer made with them."""
    from sabah.runtime.adamw import AdamW
    g = torch.Generator().manual_seed(6)
    start, grad = torch.randn(700, generator=g), torch.randn(700, generator=g).to(DEV)
    a = AdamW([start.to(DEV)], [grad], lr=1e-2, max_norm=1.0)
    for lr, max_norm in ((torch.tensor([3e-2], device=DEV), 1.0), (5e-3, 4.0), (torch.tensor([1e-3], device=DEV), 0.5)):
        b = AdamW([a.params[0].clone()], [grad], lr=lr, max_norm=max_norm)
        b.load_moments(a.m, a.v, int(a.step_count.item()))
        a.lr, a.max_norm = lr, max_norm
        a.step()
        b.step()
        torch.cuda.synchronize()
        for x, y in zip(a.params + [a.m, a.v, a.grad_norm], b.params + [b.m, b.v, b.grad_norm]):
            assert torch.equal(x, y)
    a.max_norm = None
    with pytest.raises(ValueError, match="max_norm"):
        a.step()
    a.max_norm, a.lr = 1.0, torch.zeros(2, device=DEV)
    with pytest.raises(ValueError, match="lr"):
        a.step()


def test_a_longer_run_of_8_bits_stays_near_32(hip_rt):
    """A noisy quadratic: with 8 bits the weights come as near to its minimum as with 32 (within twice the distance)."""
    far = {}
    for bits in (32, 8):
        g = torch.Generator(device=DEV).manual_seed(9)
        target = torch.randn(4096, generator=g, device=DEV)
        p, grad = torch.zeros(4096, device=DEV), torch.zeros(4096, device=DEV)
        from sabah.runtime.adamw import AdamW
        opt = AdamW([p], [grad], lr=1e-2, weight_decay=0.0, bits=bits)
        for _ in range(600):
            grad.copy_(p - target + 0.3 * torch.randn(4096, generator=g, device=DEV))
            opt.step()
        far[bits] = (p - target).square().mean().sqrt().item()
    assert far[8] < 2 * far[32] + 1e-3, far
