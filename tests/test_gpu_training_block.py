"""One training step of a MoE block through the operators together, as a program would make it: norm, router,
experts, the sum of the slots, the norm after the block with its residual, and back; then AdamW.  The whole
gradient is compared with one of plain 64-bit autograd on the same weights."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ex(hip_rt):
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    return MoEExecutor(ExpertBank(1, 8, 256, 256, {"gate": 21, "up": 21, "down": 21}, device=DEV))


T, D, F, E, K = 70, 96, 56, 8, 2
EPS, SCALE = 1e-6, 0.5


def block():
    from sabah.runtime.experts import FloatExperts
    from sabah.runtime.norm import BlockNorm
    g = torch.Generator().manual_seed(2)
    pre, post = BlockNorm(D, after=False, eps=EPS, device=DEV), BlockNorm(D, before=False, eps=EPS, scale=SCALE, device=DEV)
    mats = {n: FloatExperts(E, k, r, dtype=torch.float32, device=DEV) for n, (k, r) in
            {"gate": (D, F), "up": (D, F), "down": (F, D)}.items()}
    for m in mats.values():
        m.w.copy_(torch.randn(m.w.shape, generator=g) * 0.2)
    router = (torch.randn(E, D, generator=g) * 0.3).to(DEV)
    return pre, post, mats, router, torch.randn(T, D, generator=g).to(DEV), torch.randn(T, D, generator=g).to(DEV)


def own_step(ex, b):
    pre, post, mats, router, x, dout = b
    _, h = ex.block_norm(pre, x)
    logits = h @ router.t()
    ids, w = ex.route(logits, K)
    groups = ex.group_rows(ids, E)
    gate, up = ex.expert_mul(mats["gate"], h, groups), ex.expert_mul(mats["up"], h, groups)
    s = torch.sigmoid(gate)
    act = gate * s * up
    y = ex.expert_mul(mats["down"], act, groups)
    z = (y * w[:, :, None]).sum(1)
    out, _ = ex.block_norm(post, x, z)
    # back
    dxo, dz, _, dwa, _ = ex.block_norm_backward(post, out, z, dout=dout)
    dy, dw = dz[:, None] * w[:, :, None], (dz[:, None] * y).sum(2)
    dact, d_down = ex.expert_mul_backward(mats["down"], act, groups, dy)
    dgate, dup = dact * up * (s + gate * s * (1 - s)), dact * gate * s
    dh1, d_gate = ex.expert_mul_backward(mats["gate"], h, groups, dgate)
    dh2, d_up = ex.expert_mul_backward(mats["up"], h, groups, dup)
    dlogits = ex.route_backward(logits, ids, dw.contiguous())
    dh = (dh1 + dh2).sum(1) + dlogits @ router
    dx, _, _, _, dwb = ex.block_norm_backward(pre, x, dout=dxo, dh=dh)
    return out, ids, dict(x=dx, gate=d_gate, up=d_up, down=d_down, router=dlogits.t() @ h, w_after=dwa, w_before=dwb)


def plain_step(b, ids):
    pre, post, mats, router, x, dout = b
    p = {n: m.w.double().cpu().requires_grad_() for n, m in mats.items()}
    p.update(router=router.double().cpu().requires_grad_(), x=x.double().cpu().requires_grad_(),
             w_after=post.w_after.double().cpu().requires_grad_(), w_before=pre.w_before.double().cpu().requires_grad_())

    def n(v, w):
        return v / torch.sqrt(v.square().mean(1, keepdim=True) + EPS) * w
    h = n(p["x"], p["w_before"])
    pr = torch.softmax(h @ p["router"].t(), 1).gather(1, ids)
    w = pr / pr.sum(1, keepdim=True)
    z = torch.zeros(T, D, dtype=torch.float64)
    for j in range(K):
        gate = (p["gate"][ids[:, j]] @ h[:, :, None])[:, :, 0]
        up = (p["up"][ids[:, j]] @ h[:, :, None])[:, :, 0]
        act = torch.nn.functional.silu(gate) * up
        z = z + w[:, j, None] * (p["down"][ids[:, j]] @ act[:, :, None])[:, :, 0]
    out = p["x"] + SCALE * n(z, p["w_after"])
    out.backward(dout.double().cpu())
    return out.detach(), {k: v.grad for k, v in p.items()}


def test_a_step_of_a_block(ex):
    b = block()
    out, ids, grads = own_step(ex, b)
    want_out, want = plain_step(b, ids.cpu().long())

    def far(got, ref):
        return ((got.double().cpu() - ref).norm() / ref.norm()).item()
    # a chain of about ten sums of up to 100 f32 terms: 10 * sqrt(100) roundings of 2^-24, with room for their growth
    assert far(out, want_out) < 2e-5
    for name, g in grads.items():
        assert far(g, want[name]) < 2e-5, name


def test_training_lowers_nothing_but_moves_by_the_rule(ex):
    """Two steps with AdamW over all of the block's weights: each weight moves by at most lr (1 + decay |p|) in a first step."""
    from sabah.runtime.adamw import AdamW
    b = block()
    pre, post, mats, router, x, dout = b
    params = {n: m.w for n, m in mats.items()}
    params.update(router=router, w_after=post.w_after, w_before=pre.w_before)
    bufs = {n: torch.zeros_like(p) for n, p in params.items()}
    opt = AdamW([params[n] for n in params], [bufs[n] for n in params], lr=1e-2, weight_decay=0.0, bits=8, max_norm=1.0)
    for _ in range(2):
        keep = {n: p.clone() for n, p in params.items()}
        _, _, grads = own_step(ex, b)
        for n, g in bufs.items():
            g.copy_(grads[n])
        opt.step()
        torch.cuda.synchronize()
        assert opt.grad_norm.isfinite().all()
        for n, p in params.items():
            moved = (p - keep[n]).abs()
            assert moved.max() <= 2.3e-2 and ((moved > 0) == (grads[n] != 0)).float().mean() > 0.9, n
