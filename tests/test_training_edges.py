"""AdamW's and the experts' host side where the training tests' ordinary calls do not reach (no GPU)."""
import copy

import torch


def test_master_copies_of_trainable_parameters_are_no_part_of_a_graph():
    from sabah.runtime.adamw import AdamW
    ps = [torch.nn.Parameter(torch.randn(n).to(torch.bfloat16)) for n in (10, 300)]
    opt = AdamW(ps, [torch.zeros_like(p) for p in ps], master=True)
    assert not opt.master.requires_grad and opt.master.grad_fn is None
    assert torch.equal(copy.deepcopy(opt.master), opt.master)
    for p, at in zip(ps, opt.starts):
        assert (opt.master[at:at + p.numel()].numpy() == p.detach().float().numpy()).all()
