"""A block's norms, experts' products and AdamW where the training tests' ordinary values do not reach, against the 64-bit
forms of train_refs."""
import math

import pytest
import torch

import train_refs as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = {"f32": F32, "f16": F16, "bf16": BF16}


@pytest.fixture(scope="module")
def ex(hip_rt):
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    return MoEExecutor(ExpertBank(1, 8, 256, 256, {"gate": 21, "up": 21, "down": 21}, device=DEV))


# ---- norms -------------------------------------------------------------------
@pytest.mark.parametrize("after", [True, False])
@pytest.mark.parametrize("D", [24, 700])
def test_gates_far_from_zero(ex, after, D):
    """dgate has sigmoid(-gate), which is far below the steps of 1 - sigmoid(gate) where a gate is wide open."""
    from sabah.runtime.norm import BlockNorm
    eps, scale = 1e-6, 0.5
    gate = torch.linspace(-87.0, 87.0, 349)
    T = gate.numel()
    g = torch.Generator().manual_seed(3)
    n = BlockNorm(D, after=after, before=True, eps=eps, scale=scale, device=DEV)
    x, y, dout, dh = (torch.randn(T, D, generator=g) for _ in range(4))
    out, _ = ex.block_norm(n, x.to(DEV), y.to(DEV), gate.to(DEV))
    _, _, dgate, _, _ = ex.block_norm_backward(n, out, y.to(DEV), gate.to(DEV), dout=dout.to(DEV), dh=dh.to(DEV))
    one = torch.ones(D)
    d, tol = R.norm_back(out.cpu(), None, None, None, one, dout, dh, eps, scale)["dx"]
    branch = y.double()
    if after:
        branch = branch / torch.sqrt(branch.square().mean(1, keepdim=True) + eps)
    c = scale * torch.sigmoid(gate.double()) * torch.sigmoid(-gate.double())
    size = (tol / (80 * R.U) * branch.abs()).sum(1)
    # the bound of train_refs (an exp and a quotient more are within it), and steps of 2^-149 where factors are below 2^-126
    R.close(dgate, c * (d * branch).sum(1), 200 * R.U * c * size + 2.0 ** -147 * (1 + size), "dgate")


# ---- AdamW -------------------------------------------------------------------
def adamw(p, grad, **kw):
    from sabah.runtime.adamw import AdamW
    return AdamW([p.to(DEV)], [grad.to(DEV)], **{**dict(lr=3e-3, betas=(0.9, 0.99), weight_decay=0.0), **kw})


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("size,scale,max_norm", [(1e38, 1.0, 1e-4), (1e38, 1.0, 1e-9), (1e38, 1e-42, None), (1e-39, 1e39, None), (1e-39, 1e41, 10.0)])
def test_factors_of_the_gradients_beyond_f32(hip_rt, size, scale, max_norm, bits):
    """What gradients are multiplied by may lie outside f32's numbers where the products do not."""
    g = torch.Generator().manual_seed(2)
    grad = torch.randn(700, generator=g).clamp(-3, 3) * size
    p = torch.randn(700, generator=g)
    opt = adamw(p, grad, bits=bits, max_norm=max_norm)
    opt.step(grad_scale=scale)
    torch.cuda.synchronize()
    c = scale
    if max_norm is not None:
        c *= min(1.0, max_norm / (scale * grad.double().norm().item() + 1e-6))
    want, m, v, step = R.adamw(p, grad, torch.zeros(700), torch.zeros(700), 1, 3e-3, (0.9, 0.99), 1e-8, 0.0, c)
    q = grad.double().abs() * c
    tm, tv = 6 * R.U * q + 1e-44, 8 * R.U * q * q + 1e-44
    if bits == 32:
        R.close(opt.m[:700], m, tm, "m")
        R.close(opt.v[:700], v, tv, "v")
    # m's error, half of v's relative one, 12 roundings of the step and 3 of the rest; one more where the whole step is tiny
    tp = step.abs() * (12 * R.U + tm / m.abs().clamp(min=1e-300) + tv / v.clamp(min=1e-300)).clamp(max=1) + 3 * R.U * (p.double().abs() + step.abs())
    R.close(opt.params[0], want, tp, "p")


@pytest.mark.parametrize("bits", [32, 8])
def test_a_finite_norm_beyond_f32(hip_rt, bits):
    """A step that is made says so: its norm, which f32 cannot hold, is f32's largest number and not infinite."""
    grad = torch.tensor([3e38, -3e38, 1e38])
    opt = adamw(torch.zeros(3), grad, bits=bits, max_norm=1.0)
    opt.step()
    torch.cuda.synchronize()
    assert opt.step_count.item() == 1 and opt.grad_norm.item() == torch.finfo(F32).max
    want, _, _, step = R.adamw(torch.zeros(3), grad, torch.zeros(3), torch.zeros(3), 1, 3e-3, (0.9, 0.99), 1e-8, 0.0,
                               1.0 / grad.double().norm().item())
    R.close(opt.params[0], want, 20 * R.U * step.abs(), "p")
    for bad in (float("inf"), float("nan")):
        opt.grads[0][1] = bad
        opt.step()
        torch.cuda.synchronize()
        assert opt.step_count.item() == 1 and not opt.grad_norm.isfinite().item()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("lr,decay", [(1e-5, 0.01), (3e-5, 0.01), (1e-4, 0.1), (1e-2, 0.1)])
def test_a_small_decay_is_not_rounded_to_steps_of_one(hip_rt, lr, decay, bits):
    """p (1 - lr decay) rounded once: lr decay next to 1 would be a whole number of steps of 2^-24."""
    p = 1 + torch.rand(5000, generator=torch.Generator().manual_seed(4))
    opt = adamw(p, torch.zeros(5000), lr=lr, weight_decay=decay, bits=bits)
    opt.step()
    torch.cuda.synchronize()
    # the sum's rounding, half a step of numbers below 2, and those of lr decay and its product
    R.close(opt.params[0], p.double() * (1 - lr * decay), R.U * (1 + 4 * p.double() * lr * decay), "p")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("size", [1e-12, 1e-17, 1e-18, 1e-19, 1e-20])
def test_squares_below_f32_normal_numbers(hip_rt, size, bits):
    """v of gradients whose squares are below 2^-126 still divides m, down to f32's steps of 2^-149."""
    g = torch.Generator().manual_seed(5)
    grad = (1 + torch.rand(700, generator=g)) * size * torch.where(torch.rand(700, generator=g) < 0.5, -1.0, 1.0)
    opt = adamw(torch.zeros(700), grad, bits=bits, eps=1e-30)
    opt.step()
    torch.cuda.synchronize()
    want, m, v, step = R.adamw(torch.zeros(700), grad, torch.zeros(700), torch.zeros(700), 1, 3e-3, (0.9, 0.99), 1e-30, 0.0, 1.0)
    # f32's steps of a square, its product and v: 3 of 2^-149, of which the root takes half
    R.close(opt.params[0], want, step.abs() * (16 * R.U + 3 * 2.0 ** -149 / v), "p")


# ---- experts -----------------------------------------------------------------
@pytest.mark.parametrize("T", [5, 200])
def test_inputs_and_results_as_columns_of_one_buffer(ex, T):
    """x beside y and dy beside dx in the rows of [T, slots, k + rows]: the same as apart, and nothing else changes."""
    from sabah.runtime.experts import FloatExperts
    g = torch.Generator().manual_seed(8)
    k, rows = 72, 88
    e = FloatExperts(4, k, rows, dtype=BF16, device=DEV)
    e.w.copy_(torch.randint(-3, 4, (4, rows, k), generator=g))
    ids = torch.randint(-1, 4, (T, 2), generator=g, dtype=torch.int32).to(DEV)
    x, dy = (torch.randint(-3, 4, (T, 2, n), generator=g).to(BF16).to(DEV) for n in (k, rows))
    groups = ex.group_rows(ids, 4)
    want = ex.expert_mul(e, x, groups), ex.expert_mul_backward(e, x, groups, dy)
    buf = torch.full((T, 2, k + rows), 9.0, dtype=BF16, device=DEV)
    buf[:, :, :k] = x
    y = ex.expert_mul(e, buf[:, :, :k], groups, out=buf[:, :, k:])
    assert torch.equal(y, want[0]) and torch.equal(buf[:, :, :k], x)
    buf[:, :, k:] = dy
    dx, dw = ex.expert_mul_backward(e, x, groups, buf[:, :, k:], dx=buf[:, :, :k])
    assert torch.equal(dx, want[1][0]) and torch.equal(dw, want[1][1]) and torch.equal(buf[:, :, k:], dy)


# ---- unbiased moments of 8 bits ------------------------------------------------
def unbiased(p, grad, **kw):
    return adamw(p, grad, bits=8, unbiased=True, **kw)


def test_unbiased_codes_are_the_two_around_a_value_in_proportion(hip_rt):
    """Against the 64-bit values of the same step: below or above, by shares that fit (six standard deviations of that many
    independent choices), another choice in another step, and codes that a value hits exactly kept."""
    n = 1 << 16
    g = torch.Generator().manual_seed(11)
    opt = unbiased(torch.zeros(n), torch.randn(n, generator=g), betas=(0.9, 0.999))
    for _ in range(3):
        opt.step()
    kept = [t.clone() for t in (opt.m, opt.v, opt.m_scale, opt.v_scale)]
    ups = []
    for steps in (3, 4):
        for t, k in zip((opt.m, opt.v, opt.m_scale, opt.v_scale), kept):
            t.copy_(k)
        opt.step_count.fill_(steps)
        opt.step()
        torch.cuda.synchronize()
        m0 = R.m_value(kept[0].cpu()).reshape(-1, 256) * kept[2].cpu().double()[:, None]
        v0 = R.v_value(kept[1].cpu()).reshape(-1, 256) * kept[3].cpu().double()[:, None]
        grad = opt.grads[0].cpu().double().reshape(-1, 256)
        m, v = 0.9 * m0 + 0.1 * grad, 0.999 * v0 + 0.001 * grad * grad
        for x, scale, code, top, power in ((m, opt.m_scale, opt.m, 127, 2), (v, opt.v_scale, opt.v, 255, 4)):
            s = scale.cpu()
            # 0.9 s + 0.1 g of f32's numbers is often half way between two of them, where an error of 64 bits decides: half a step
            assert ((s.double() - x.abs().amax(1)).abs() <= R.U * (1 + 1e-6) * s.double()).all()
            t = (x.abs() / s.double()[:, None]).clamp(max=1) * top ** power
            low = torch.floor((t * (1 + 1e-12)).pow(1 / power)).clamp(max=top - 1)
            share = ((t - low ** power) / ((low + 1) ** power - low ** power)).clamp(0, 1)
            code = code.cpu().reshape(-1, 256).double()
            assert ((code == 0) | (torch.sign(code) == torch.sign(x))).all()
            up = code.abs() - low
            edge = (share < 1e-9) | (share > 1 - 1e-9) | ((low == 0) if power == 4 else (low < 0))   # v above 0 never becomes 0
            assert (((up == 0) | (up == 1)) | edge).all() and (up[share > 1 - 1e-9] == 1).all()
            if power == 4:
                assert (code[x > 0] >= 1).all()
            u, q = up[~edge], share[~edge]
            assert (u - q).sum().abs() <= 6 * (q * (1 - q)).sum().sqrt()
            for part in (q < 0.1, q > 0.9):                 # and where one of them is likely
                assert (u - q)[part].sum().abs() <= 6 * (q * (1 - q))[part].sum().sqrt()
            ups.append((up, share))
    for a, b in ((0, 2), (1, 3), (0, 1)):                  # m in two steps, v in two steps, m and v: no common choice
        (x, p), (y, q) = ups[a], ups[b]
        r = (x - p) * (y - q)
        assert r.sum().abs() <= 6 * (p * (1 - p) * q * (1 - q)).sum().sqrt() + 1e-3 * n ** 0.5


@pytest.mark.parametrize("largest", [False, True])
def test_unbiased_second_moments_over_thousands_of_steps(hip_rt, largest):
    """The mean of v against the unrounded recurrence, at beta2 = 0.999: even noise; and one value of each block that stays
    while the gradients of the others become a tenth.  A step moves v by 0.001 of itself; the choice between two codes 4 / k
    apart then has a variance of at most 0.004 / k of v^2, which later steps forget by 0.998: 2 / k.  While v falls, nothing is forgotten
    relative to v: 6,000 times 0.004 / k more.  k >= 128 under even noise (all values within 16 times), >= 80 at the end of the fall.  Over n values six
    standard deviations of their mean; the values' choices are independent."""
    n = 64 * 256
    g = torch.Generator(device=DEV).manual_seed(12)
    grad = torch.zeros(n, device=DEV)
    opt = unbiased(torch.zeros(n), grad, betas=(0.9, 0.999))
    grad, want = opt.grads[0], torch.zeros(n, dtype=torch.float64, device=DEV)
    first = torch.arange(n, device=DEV) % 256 == 0
    for step in range(8000 if largest else 5000):
        grad.normal_(generator=g)
        if largest and step >= 2000:
            grad.mul_(torch.where(first, 1.0, 0.1))
        opt.step()
        want.mul_(0.999).add_(grad.double().square(), alpha=0.001)
    v = opt.moments()[1].double()
    far = (v[~first].mean() / want[~first].mean() - 1).abs().item()
    spread = math.sqrt(2 / 80 + 6000 * 0.004 / 80) if largest else math.sqrt(2 / 128)
    assert far <= 6 * spread / math.sqrt(n - 64), far


def test_unbiased_steps_repeat_and_replay(hip_rt):
    """The same bits from the same state, eager or replayed; a step by R.adamw's rule from the values of the codes."""
    from sabah.runtime.adamw import AdamW
    g = torch.Generator().manual_seed(13)
    sizes = [1, 255, 257, 5000]
    start, gs = [torch.randn(n, generator=g).to(BF16) for n in sizes], [torch.randn(n, generator=g).to(DEV) for n in sizes]
    a, b = (AdamW([t.to(DEV) for t in start], gs, bits=8, unbiased=True, max_norm=3.0, master=True) for _ in range(2))
    a.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    b.step()
    for i in range(3):
        for t in gs:
            t.mul_(-0.9)
        m0, v0 = (t.clone() for t in b.moments())
        p0 = b.master.clone()
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        for x, y in zip(a.params + [a.m, a.v, a.m_scale, a.v_scale, a.master, a.grad_norm, a.step_count],
                        b.params + [b.m, b.v, b.m_scale, b.v_scale, b.master, b.grad_norm, b.step_count]):
            assert torch.equal(x, y)
        c = min(1.0, 3.0 / (math.sqrt(sum(t.double().square().sum().item() for t in gs)) + 1e-6))
        for j, (n, at) in enumerate(zip(sizes, b.starts)):
            rows = slice(at, at + n)
            want, _, v, step = R.adamw(p0[rows].cpu(), gs[j].cpu(), m0[rows].cpu(), v0[rows].cpu(), i + 2, 1e-3, (0.9, 0.999), 1e-8, 0.01, c)
            q = gs[j].cpu().double().abs() * c
            tm = 6 * R.U * (m0[rows].cpu().double().abs() + q) + 1e-44
            scale = 1e-3 / (1 - 0.9 ** (i + 2)) / ((v / (1 - 0.999 ** (i + 2))).sqrt() + 1e-8)
            R.close(b.master[rows], want, scale * tm + 20 * R.U * step.abs() + 3 * R.U * (p0[rows].cpu().double().abs() + step.abs()), "p")


def test_unbiased_moments_of_zeros_and_nan(hip_rt):
    """Values without a gradient keep moments of 0; a NaN becomes its block's; other blocks and what lies behind the tensor stay."""
    grad = torch.zeros(1000)
    grad[256:512], grad[600] = 1.0, float("nan")
    opt = unbiased(torch.ones(1000), grad)
    for _ in range(3):
        opt.step()
    torch.cuda.synchronize()
    m, v = (t.cpu() for t in opt.moments())
    assert (m[:256] == 0).all() and (v[:256] == 0).all() and (opt.params[0][:256] == 1).all()
    assert (opt.m[256:512] == 127).all() and (opt.v[256:512] == 255).all()      # all at the block's largest: exact
    assert m[512:768].isnan().all() and (m[768:] == 0).all() and (v[768:] == 0).all()


# ---- experts: stages and the ends of the types --------------------------------
def products(ex, w, x, ids, dy):
    """(y, dx, dw) on the device."""
    from sabah.runtime import rt
    from sabah.runtime.experts import FloatExperts
    e = FloatExperts(w.shape[0], w.shape[2], w.shape[1], dtype=w.dtype, device=DEV)
    e.w.copy_(w)
    groups = ex.group_rows(ids.to(DEV), e.n_experts)
    y = ex.expert_mul(e, x.to(DEV), groups)
    dx, dw = ex.expert_mul_backward(e, x.to(DEV), groups, dy.to(DEV))
    torch.cuda.synchronize()
    rt.check(rt.lib().sabah_rt_check_errors(), "experts")
    return y, dx, dw


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("last,k", [(1, 640), (33, 648), (70, 1024), (100, 72), (129, 640), (225, 1000)])
def test_sums_of_many_stages_in_tiles_of_256_rows(ex, last, k, dtype):
    """Two experts of more than 384 rows each on average and 24 x 8 tiles: the largest form, its three stages used again and again, by
    tiles of all numbers of 32-row results.  Whole numbers: sums are exact, results equal."""
    from sabah.runtime.experts import FloatExperts
    g = torch.Generator().manual_seed(last)
    T, rows = 6144 + last, 2048
    w = torch.randint(-3, 4, (2, rows, k), generator=g).to(TYPES[dtype])
    x = torch.randint(-3, 4, (T, k), generator=g).to(TYPES[dtype])
    ids = torch.zeros(T, 1, dtype=torch.int32)
    ids[torch.randperm(T, generator=g)[:last]] = 1
    e = FloatExperts(2, k, rows, dtype=TYPES[dtype], device=DEV)
    e.w.copy_(w)
    y = ex.expert_mul(e, x.to(DEV), ex.group_rows(ids.to(DEV), 2))
    torch.cuda.synchronize()
    want = torch.empty(T, rows, dtype=torch.float64)
    for i in (0, 1):
        at = ids[:, 0] == i
        want[at] = x[at].double() @ w[i].double().t()
    assert torch.equal(y[:, 0].cpu(), want.to(TYPES[dtype]))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,k,rows", [(5, 64, 96), (5, 63, 35), (90, 72, 128), (90, 71, 35)])
@pytest.mark.parametrize("what", ["subnormal", "large and small"])
def test_products_at_the_ends_of_their_types(ex, T, k, rows, dtype, what):
    """Operands below the type's normal numbers, and factors far from 1 whose products are not; in the streamed, the direct and
    the staged form.  Every product is a whole number of one unit and each sum exact in f32, so results equal."""
    t = TYPES[dtype]
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, 3, (T, 2), generator=g, dtype=torch.int32)
    step = torch.finfo(t).smallest_normal * torch.finfo(t).eps
    up = {"f32": 100, "f16": 12, "bf16": 100}[dtype]
    a, b = (step, 1.0) if what == "subnormal" else (2.0 ** up, 2.0 ** -up)

    def whole(*shape):
        return torch.randint(-3, 4, shape, generator=g).double()
    for small in ("w", "x"):                       # which operand has the far values; dy goes with the other one's
        w = (whole(3, rows, k) * (a if small == "w" else b)).to(t)
        x = (whole(T, 1, k) * (a if small == "x" else b)).to(t)
        dy = (whole(T, 2, rows) * (a if small == "x" else b)).to(t)
        y, dx, _ = products(ex, w, x, ids, dy)
        assert torch.equal(y.cpu(), R.expert_mul(w, x, ids)[0].to(t)), ("y", small)
        (wx, _), _ = R.expert_back(w, x, ids, dy)
        assert torch.equal(dx.cpu(), wx.to(t)), ("dx", small)
        dy = whole(T, 2, rows).mul(b if small == "x" else a).to(t)
        _, _, dw = products(ex, w, x, ids, dy)
        _, (ww, _) = R.expert_back(w, x, ids, dy)
        assert torch.equal(dw.cpu().double(), ww), ("dw", small)
