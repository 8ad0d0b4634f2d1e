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
