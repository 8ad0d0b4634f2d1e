"""AdamW's and the experts' host side where the training tests' ordinary calls do not reach (no GPU)."""
import copy

import pytest
import torch

from test_train_refusals import P, expert_desc, fails, mul, mul_back


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
