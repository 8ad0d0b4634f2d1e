"""What the adapters' and the router's training entry points refuse before the
device is touched (no GPU)."""
import ctypes

import pytest

vp = ctypes.c_void_p
P = 0x10000                                        # never dereferenced: the checks come first


def desc(**kw):
    from sabah.runtime import rt
    v = dict(a=P, b=P, scale=None, ranks=None, type=30, n_adapters=4, n_experts=1, rank=16, k=64, rows=48)
    v.update(kw)
    return rt.LoraDesc(*(v[f] for f, _ in rt.LoraDesc._fields_))


def apply(L, d, **kw):
    v = dict(x=P, xi=0, xr=1, xt=256, ad=P, ids=None, ii=0, it=0, n=1, T=3, base=None, bi=0, bt=0, dst=P, di=0, dt=192,
             ws=P, nws=1 << 40, st=None)
    v.update(kw)
    return L.sabah_lora_apply(ctypes.byref(d), *v.values())


def backward(L, d, **kw):
    v = dict(x=P, xi=0, xr=1, xt=256, ad=P, ids=None, ii=0, it=0, n=1, T=3, dy=P, yi=0, yt=192, dx=P, di=0, dt=256,
             add_dx=0, da=P, db=P, add_dw=0, ws=P, nws=1 << 40, st=None)
    v.update(kw)
    return L.sabah_lora_backward(ctypes.byref(d), *v.values())


@pytest.mark.parametrize("call", [apply, backward])
@pytest.mark.parametrize("bank,kw,msg", [
    (dict(a=None), {}, "null adapter bank"), (dict(b=None), {}, "null adapter bank"), (dict(type=8), {}, "type"),
    (dict(rank=0), {}, "rank"), (dict(rank=129), {}, "rank"), (dict(n_adapters=0), {}, "geometry"),
    (dict(k=0), {}, "geometry"), (dict(rows=-1), {}, "geometry"), (dict(n_experts=2), {}, "need ids"),
    (dict(n_adapters=1 << 20, n_experts=1 << 10), {}, "geometry"), ({}, dict(x=None), "null pointer"),
    ({}, dict(ad=None), "null pointer"), ({}, dict(n=0), "rows"), ({}, dict(T=-1), "rows"),
    ({}, dict(n=4096, T=4097), "rows"), ({}, dict(n=4, xr=2), "input rows"), ({}, dict(xt=255), "multiples of 4"),
    ({}, dict(dt=191), "multiples of 4"), ({}, dict(ids=P, it=2), "multiples of 4")])
def test_adapters_refuse(call, bank, kw, msg):
    from sabah.runtime import rt
    assert call(rt.lib(), desc(**bank), **kw) == -1
    assert msg in rt.last_error()


def test_adapters_refuse_their_own_arguments():
    from sabah.runtime import rt
    L = rt.lib()
    assert apply(L, desc(), dst=None) == -1 and "null pointer" in rt.last_error()
    assert apply(L, desc(), base=P, bt=96) == -1 and "in place" in rt.last_error()
    assert backward(L, desc(), dy=None) == -1 and "null pointer" in rt.last_error()
    n = L.sabah_lora_workspace(ctypes.byref(desc()), 1, 3, 1)
    assert n > 0
    for bad in (dict(ws=None), dict(nws=n - 1), dict(ws=P + 8)):
        assert backward(L, desc(), **bad) == -1 and "workspace" in rt.last_error()
    m = L.sabah_lora_workspace(ctypes.byref(desc()), 1, 5000, 0)
    for bad in (dict(ws=None), dict(nws=m - 1), dict(ws=P + 8)):
        if m:
            assert apply(L, desc(), T=5000, **bad) == -1 and "workspace" in rt.last_error()
    assert L.sabah_lora_workspace(ctypes.byref(desc(rank=200)), 1, 3, 1) == 0


def balance(L, **kw):
    v = dict(l=P, s=256, ids=P, mask=None, T=12, E=64, k=8, g=1, c=P, p=P, loss=P, n=P, ws=P, nws=1 << 40, st=None)
    v.update(kw)
    return L.sabah_moe_balance(*v.values())


def gradient(L, **kw):
    v = dict(l=P, s=256, ids=P, mask=None, T=12, E=64, k=8, norm=1, scale=1.0, dw=P, c=P, n=P, g=1, cb=0.1, cz=0.1, d=P,
             ds=256, st=None)
    v.update(kw)
    return L.sabah_moe_route_backward(*v.values())


@pytest.mark.parametrize("call", [balance, gradient])
@pytest.mark.parametrize("kw,msg", [
    (dict(E=0), "n_experts"), (dict(E=4097, s=1 << 20, ds=1 << 20), "n_experts"), (dict(k=0), "n_used"),
    (dict(k=65), "n_used"), (dict(E=7, k=8), "n_used"), (dict(T=-1), "n_tokens"), (dict(T=(1 << 24) + 1), "n_tokens"),
    (dict(g=0), "n_groups"), (dict(g=5), "n_groups"), (dict(l=None), "null pointer"), (dict(ids=None), "null pointer"),
    (dict(s=252), "stride"), (dict(s=258), "stride")])
def test_router_calls_refuse(call, kw, msg):
    from sabah.runtime import rt
    L = rt.lib()
    if call is balance:
        kw = {k: v for k, v in kw.items() if k != "ds"}
    assert call(L, **kw) == -1
    assert msg in rt.last_error()


def test_router_calls_refuse_their_own_arguments():
    from sabah.runtime import rt
    L = rt.lib()
    for bad in (dict(c=None), dict(p=None), dict(loss=None), dict(n=None)):
        assert balance(L, **bad) == -1 and "null pointer" in rt.last_error()
    n = L.sabah_moe_balance_workspace(12, 64, 1)
    for bad in (dict(ws=None), dict(nws=n - 1), dict(ws=P + 4)):
        assert balance(L, **bad) == -1 and "workspace" in rt.last_error()
    assert L.sabah_moe_balance_workspace(12, 64, 5) == 0
    for bad in (dict(c=None), dict(n=None)):
        assert gradient(L, **bad) == -1 and "counts" in rt.last_error()
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert gradient(L, scale=scale) == -1 and "w_scale" in rt.last_error()
    assert gradient(L, d=None) == -1 and "null pointer" in rt.last_error()


def test_they_need_init():
    from sabah.runtime import rt
    if rt._initialised is not None:
        pytest.skip("runtime already initialised in this process")
    for rc in (apply(rt.lib(), desc()), backward(rt.lib(), desc()), balance(rt.lib()), gradient(rt.lib())):
        assert rc == -1 and "sabah_rt_init" in rt.last_error()


def test_adapter_bank_refuses_types_and_sizes():
    import torch
    from sabah.runtime.lora import LoraBank
    with pytest.raises(ValueError):
        LoraBank(2, 8, 16, 16, dtype=torch.float64, device="cpu")
    for bad in ((0, 8, 16, 16), (2, 129, 16, 16), (2, 8, 0, 16), (2, 8, 16, -1)):
        with pytest.raises(ValueError):
            LoraBank(*bad, device="cpu")
