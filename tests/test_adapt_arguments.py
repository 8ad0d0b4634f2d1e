"""Arguments of the adapters' and the router's calls that the executor and the C entry points
must refuse, or must not, seen before the device is touched (no GPU)."""
import pytest
import torch

from test_adapt_refusals import P, apply, desc


@pytest.fixture
def ex():
    """The executor's checks without its bank; a CPU tensor's device index is -1."""
    from sabah.runtime.executor import MoEExecutor
    e = MoEExecutor.__new__(MoEExecutor)
    e.device, e._index = torch.device("cpu"), -1
    return e


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_rows_have_two_or_three_dimensions(ex):
    """One row given flat, as long as there are tokens, would be read as tokens four bytes apart."""
    from sabah.runtime.lora import LoraBank
    lora, pairs = LoraBank(2, 4, 8, 6, device="cpu"), LoraBank(2, 4, 8, 6, n_experts=3, device="cpu")
    for x in (torch.zeros(8), torch.zeros(8, 1, 1, 8), torch.zeros(())):
        with pytest.raises(ValueError, match="adapters"):
            ex._lora_rows(lora, x, i32(8), None, None)
    for ids in (i32(8), i32(8, 2, 5), i32()):
        with pytest.raises(ValueError, match="adapters"):
            ex._lora_rows(pairs, torch.zeros(8, 8), i32(8), ids, None)
    for y in (torch.zeros(8), torch.zeros(()), torch.zeros(8, 1, 1, 6)):
        with pytest.raises(ValueError, match="adapters"):
            ex._lora_y("out", y, 8, 1, 6)
    T, slots, rows = ex._lora_rows(pairs, torch.zeros(8, 8), i32(8), i32(8, 2), None)
    assert (T, slots) == (8, 2) and rows[1:4] == (0, 1, 32)
    T, slots, rows = ex._lora_rows(pairs, torch.zeros(8, 2, 8), i32(8), i32(8, 2), None)
    assert (T, slots) == (8, 2) and rows[1:4] == (32, 2, 64)


def test_router_tensors_have_two_dimensions(ex):
    for logits, ids in ((torch.zeros(6), i32(6, 2)), (torch.zeros(6, 2, 8), i32(6, 2)), (torch.zeros(6, 8), i32(6)),
                        (torch.zeros(6, 8), i32(6, 2, 3)), (torch.zeros(()), i32(6, 2)), (torch.zeros(6, 8), i32())):
        with pytest.raises(ValueError, match="router"):
            ex._router_rows(logits, ids, None, 1)
    assert ex._router_rows(torch.zeros(6, 8), i32(6, 2), None, 1) == (6, 8, 2)


def test_in_place_where_a_stride_is_never_used():
    """Base and dst are the same rows whatever the slots' stride of one slot, or the tokens' of one token:
    the next check (a missing workspace) is what refuses these calls."""
    from sabah.runtime import rt
    L = rt.lib()
    many = dict(ws=None, nws=0, base=P)
    assert apply(L, desc(), T=5000, bi=0, di=192, bt=192, dt=192, **many) == -1 and "workspace" in rt.last_error()
    assert apply(L, desc(), T=1, n=5000, bi=192, di=192, bt=0, dt=192 * 5000, **many) == -1 and "workspace" in rt.last_error()
    assert apply(L, desc(), T=5000, bi=0, di=0, bt=96, dt=192, **many) == -1 and "in place" in rt.last_error()
    assert apply(L, desc(), T=1, n=5000, bi=96, di=192, bt=0, dt=0, **many) == -1 and "in place" in rt.last_error()
