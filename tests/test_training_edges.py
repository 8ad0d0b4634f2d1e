"""AdamW's and the experts' host side where the training tests' ordinary calls do not reach (no GPU)."""
import copy

import pytest
import torch

import train_refs as R
from test_train_refusals import P, expert_desc, fails, mul, mul_back, step


def test_master_copies_of_trainable_parameters_are_no_part_of_a_graph():
    from sabah.runtime.adamw import AdamW
    ps = [torch.nn.Parameter(torch.randn(n).to(torch.bfloat16)) for n in (10, 300)]
    opt = AdamW(ps, [torch.zeros_like(p) for p in ps], master=True)
    assert not opt.master.requires_grad and opt.master.grad_fn is None
    assert torch.equal(copy.deepcopy(opt.master), opt.master)
    for p, at in zip(ps, opt.starts):
        assert (opt.master[at:at + p.numel()].numpy() == p.detach().float().numpy()).all()


# x [3][2] of 128 bytes and y [3][2] of 96 in rows of one buffer, 256 bytes a slot, in either order of its axes; None: apart
COLUMNS = [
    (dict(y=P + 128), None), (dict(y=P + 160), None), (dict(y=P + 126), "overwrite"), (dict(y=P + 162), "overwrite"),
    (dict(y=P + 256 + 128), None), (dict(y=P + 256 + 126), "overwrite"), (dict(x=P + 96, y=P), None), (dict(x=P + 94, y=P), "overwrite"),
    (dict(xi=768, xt=256, yi=768, yt=256, y=P + 128), None), (dict(xi=768, xt=256, yi=768, yt=256, y=P + 162), "overwrite"),
    (dict(yi=768, yt=256, y=P + 128), None),
    # one row of x for a token, in the first slot's
    (dict(xr=1, xi=0, y=P + 128), None), (dict(xr=1, xi=0, y=P + 126), "overwrite"),
    # slots of 224 bytes: no columns of x's 256, and some meet
    (dict(yi=224, yt=448, y=P + 128), "overwrite")]


@pytest.mark.parametrize("kw,msg", COLUMNS)
def test_experts_take_columns_of_one_buffer(kw, msg):
    v = {**dict(xi=256, xr=2, xt=512, yi=256, yt=512), **kw}
    fails(mul(expert_desc(w=32 * P), **v, g=None), msg or "groups must")    # the check that follows
    # backward the same of dx, in x's rows, beside dy, in y's
    back = dict(dx=v.get("x", P), di=v["xi"], dt=v["xt"], y=v["y"], yi=v["yi"], yt=v["yt"], xi=128, xr=2, xt=256)
    if v["xr"] == 2:
        fails(mul_back(expert_desc(w=32 * P), **back, x=8 * P, dw=None, g=None), msg or "groups must")


def group(ids=P, g=2 * P, si=4, st=8, T=3):
    from sabah.runtime import rt
    return rt.lib().sabah_expert_group(ids, si, st, 2, T, 4, g, 1 << 40, None)


# groups of [3][2] rows over 4 experts at 2 P; y, dx and ids of 3 tokens' two rows, dw of 49,152 bytes
@pytest.mark.parametrize("call,own,msg", [
    (mul, dict(y=2 * P), "groups"), (mul, dict(y=2 * P - 574), "groups"), (mul, dict(y=2 * P - 576), None), (mul, dict(y=2 * P + 16), "groups"),
    (mul_back, dict(dx=2 * P - 766), "groups"), (mul_back, dict(dx=2 * P - 768), None), (mul_back, dict(dx=None, dw=2 * P), "groups"),
    (mul_back, dict(dw=2 * P - 49148), "groups"), (mul_back, dict(dw=2 * P - 49152), None),
    (group, dict(ids=2 * P), "ids"), (group, dict(ids=2 * P - 20), "ids"), (group, dict(ids=2 * P - 24), None), (group, dict(ids=2 * P, T=0), None)])
def test_nothing_is_written_over_the_groups(call, own, msg):
    """Rows' numbers that were overwritten would send kernels anywhere."""
    from sabah.runtime import rt
    n = rt.lib().sabah_expert_groups_bytes(2, 3, 4)
    if msg is None and torch.cuda.device_count():
        pytest.skip("with a device an accepted call would use the addresses")
    rc = call(**own) if call is group else call(expert_desc(w=32 * P), **{**dict(x=8 * P, y=9 * P, g=2 * P), **own})
    fails(rc, msg or "sabah_rt_init")
    if call is not group and "y" in own and own["y"] == 2 * P:           # the groups' last bytes, and what follows them
        fails(mul(expert_desc(w=32 * P), x=8 * P, y=2 * P + n - 2), "groups")
        if not torch.cuda.device_count():
            fails(mul(expert_desc(w=32 * P), x=8 * P, y=2 * P + n), "sabah_rt_init")


def test_unbiased_codes_are_of_8_bits():
    from sabah.runtime import rt
    from sabah.runtime.adamw import AdamW
    flag = rt.ADAMW_UNBIASED
    for bits in (32 | flag, 16 | flag, flag, 8 | flag << 1):
        fails(step(bits=bits), "bits")
    fails(step(bits=8 | flag, m_scale=None), "null")
    with pytest.raises(ValueError, match="unbiased"):
        AdamW([torch.zeros(4)], [torch.zeros(4)], unbiased=True)
    a = AdamW([torch.zeros(4)], [torch.zeros(4)], bits=8, unbiased=True)
    assert a.desc.bits == 8 | flag and a.m.dtype == torch.int8


def nearest(v, top):
    return R.v_value(R.v_code(v, top)[0]) * top


@pytest.mark.parametrize("beta2,least,most", [(0.999, 1.1, 1.9), (0.99, 0.99, 1.02)])
def test_what_nearest_codes_make_of_even_noise(beta2, least, most):
    """The limit that AdamW's documentation names, by the 64-bit forms: after 5,000 steps the mean of v is about 1.4 times the unrounded
    recurrence's at beta2 = 0.999, and right at 0.99.  By how much goes with a block's largest value, which sets when its codes
    fall: 1.4 with a standard deviation of 0.45 over 64 blocks, so 8 of them within 3 x 0.16 of it."""
    g = torch.Generator().manual_seed(1)
    coded, v = torch.zeros(8, 256, dtype=torch.float64), torch.zeros(8, 256, dtype=torch.float64)
    for _ in range(5000):
        q = (1 - beta2) * torch.randn(8, 256, generator=g, dtype=torch.float64).square()
        v, coded = beta2 * v + q, beta2 * coded + q
        coded = nearest(coded, coded.amax(1, keepdim=True).float().double())
    assert least < (coded.mean() / v.mean()).item() < most


def test_what_nearest_codes_make_of_gradients_that_become_small():
    """255 (1 - 0.999^(1/4)) = 0.064 of a code: beside a value that keeps the block's scale, codes do not fall at all."""
    v = torch.full((256,), 0.5, dtype=torch.float64)
    v[0] = 1.0
    v = before = nearest(v, v.max())
    for _ in range(3000):
        v = 0.999 * v
        v[0] = 1.0
        v = nearest(v, v.max())
    assert torch.equal(v, before)
