"""What the norms', experts' and AdamW's entry points, and the classes around them, refuse before
the device is touched (no GPU)."""
import ctypes

import pytest
import torch

vp = ctypes.c_void_p
P = 0x10000                                        # never dereferenced: the checks come first


def addresses(v):
    return [vp(a) if isinstance(a, int) and a >= P and a % P == 0 and a < 64 * P else a for a in v]


def fails(rc, msg):
    from sabah.runtime import rt
    assert rc == -1 and msg in rt.last_error(), rt.last_error()


# ---- norms -------------------------------------------------------------------
def norm_desc(**kw):
    from sabah.runtime import rt
    v = dict(w_after=P, w_before=P, type=30, width=64, eps=1e-6, scale=1.0)
    v.update(kw)
    return rt.NormDesc(*(v[f] for f, _ in rt.NormDesc._fields_))


def norm(d, **kw):
    from sabah.runtime import rt
    v = dict(x=P, xs=128, y=2 * P, ys=128, gate=None, T=3, out=3 * P, os=128, h=4 * P, hs=128, st=None)
    v.update(kw)
    return rt.lib().sabah_block_norm(ctypes.byref(d), *v.values())


def norm_back(d, **kw):
    from sabah.runtime import rt
    v = dict(out=P, os=128, y=2 * P, ys=128, gate=None, T=3, dout=3 * P, dos=128, dh=4 * P, dhs=128, dx=5 * P, dxs=128,
             dy=6 * P, dys=128, dgate=None, dwa=7 * P, dwb=8 * P, add=0, ws=9 * P, n=1 << 40, st=None)
    v.update(kw)
    return rt.lib().sabah_block_norm_backward(ctypes.byref(d), *v.values())


@pytest.mark.parametrize("call", [norm, norm_back])
@pytest.mark.parametrize("d,kw,msg", [
    (dict(type=2), {}, "type"), (dict(width=0), {}, "width"), (dict(width=8193), {}, "width"), ({}, dict(T=-1), "n_tokens"),
    ({}, dict(T=(1 << 24) + 1), "n_tokens"), (dict(eps=-1.0), {}, "eps"), (dict(eps=float("nan")), {}, "eps"),
    ({}, dict(ys=126), "stride"), ({}, dict(ys=129), "stride"), ({}, dict(os=64), "stride")])
def test_norms_refuse(call, d, kw, msg):
    fails(call(norm_desc(**d), **kw), msg)


def test_norms_refuse_their_own_arguments():
    from sabah.runtime import rt
    d, bare = norm_desc(), norm_desc(w_after=None, w_before=None)
    fails(norm(d, x=None), "null")
    fails(norm(d, out=None), "null")
    fails(norm(d, h=None), "null")
    fails(norm(d, y=None), "needs y")
    fails(norm(bare, y=None), "neither")
    fails(norm(norm_desc(w_after=None), y=None, gate=P), "needs y")
    fails(norm(d, h=P), "overwrite")
    fails(norm(d, h=3 * P), "overwrite")
    fails(norm(d, out=2 * P), "overwrite")
    fails(norm(d, out=P, os=256), "overwrite")
    fails(norm_back(d, out=None), "null")
    fails(norm_back(d, dh=None), "null")
    fails(norm_back(d, dx=None), "null")
    fails(norm_back(d, y=None), "null")
    fails(norm_back(d, gate=P), "null")
    fails(norm_back(d, dwa=None), "null")
    fails(norm_back(d, dwb=None), "null")
    fails(norm_back(norm_desc(w_before=None), dout=None), "null")
    fails(norm_back(d, dy=None), "needs dy")
    fails(norm_back(bare, dy=None), "neither")
    fails(norm_back(d, dx=P), "overwrite")
    fails(norm_back(d, dy=5 * P), "overwrite")
    fails(norm_back(d, dx=3 * P, dxs=256), "in place")
    n = rt.lib().sabah_block_norm_workspace(64, 3)
    for bad in (dict(ws=None), dict(n=n - 1), dict(ws=9 * P + 8)):
        fails(norm_back(d, **bad), "workspace")
    assert rt.lib().sabah_block_norm_workspace(0, 3) == 0


# three rows of 128 bytes at P, 2 P ..: one value, the last byte's and other rows' overlaps, and columns of one buffer
@pytest.mark.parametrize("kw,msg", [
    (dict(out=P + 2), "overwrite"), (dict(out=P + 128), "overwrite"), (dict(out=2 * P - 382), "overwrite"), (dict(out=2 * P - 384), None),
    (dict(out=2 * P + 382), "overwrite"), (dict(out=2 * P + 384), None), (dict(out=P), None), (dict(h=P + 382), "overwrite"),
    (dict(h=3 * P + 2), "overwrite"), (dict(x=P, xs=512, out=P + 128, os=512, y=P + 256, ys=512, h=P + 384, hs=512), None),
    (dict(x=P, xs=512, h=P + 126, hs=512), "overwrite"), (dict(x=P, xs=512, h=P + 386, hs=512), "overwrite"),
    (dict(x=P, xs=512, h=P + 384 + 512, hs=512), None), (dict(x=P, xs=512, h=P + 128, hs=256), "overwrite"),
    (dict(x=P, xs=512, h=P + 128, hs=256, T=1), None), (dict(x=P, h=P + 126, T=1), "overwrite"), (dict(x=P, h=P + 2, T=0), None)])
def test_norms_refuse_results_over_other_rows(kw, msg):
    if torch.cuda.device_count():
        pytest.skip("with a device an accepted call would use the addresses")
    fails(norm(norm_desc(), **kw), msg or "sabah_rt_init")


@pytest.mark.parametrize("kw,msg", [
    (dict(dx=P + 2), "overwrite"), (dict(dx=4 * P + 128), "overwrite"), (dict(dy=3 * P + 382), "overwrite"), (dict(dy=5 * P + 2), "overwrite"),
    (dict(dx=3 * P), None), (dict(dx=3 * P + 128), "in place"), (dict(dwb=7 * P), "each other"), (dict(dwb=7 * P + 252), "each other"),
    (dict(dwb=7 * P + 256), None)])
def test_norms_backward_refuses_results_over_other_rows(kw, msg):
    fails(norm_back(norm_desc(), **kw, ws=None), msg or "workspace")       # the check that follows


# ---- experts -----------------------------------------------------------------
def expert_desc(**kw):
    from sabah.runtime import rt
    v = dict(w=P, type=30, n_experts=4, k=64, rows=48)
    v.update(kw)
    return rt.ExpertDesc(*(v[f] for f, _ in rt.ExpertDesc._fields_))


def mul(d, **kw):
    from sabah.runtime import rt
    v = dict(x=P, xi=0, xr=1, xt=128, g=2 * P, ng=1 << 40, n=2, T=3, y=3 * P, yi=96, yt=192, st=None)
    v.update(kw)
    return rt.lib().sabah_expert_mul(ctypes.byref(d), *v.values())


def mul_back(d, **kw):
    from sabah.runtime import rt
    v = dict(x=P, xi=0, xr=1, xt=128, g=2 * P, ng=1 << 40, n=2, T=3, y=3 * P, yi=96, yt=192, dx=4 * P, di=128, dt=256, dw=5 * P,
             add=0, st=None)
    v.update(kw)
    return rt.lib().sabah_expert_mul_backward(ctypes.byref(d), *v.values())


@pytest.mark.parametrize("call", [mul, mul_back])
@pytest.mark.parametrize("d,kw,msg", [
    (dict(w=None), {}, "null experts"), (dict(type=8), {}, "type"), (dict(n_experts=0), {}, "n_experts"),
    (dict(n_experts=4097), {}, "n_experts"), (dict(k=0), {}, "geometry"), (dict(rows=(1 << 20) + 1), {}, "geometry"),
    ({}, dict(x=None), "null"), ({}, dict(y=None), "null"), ({}, dict(n=0), "rows"), ({}, dict(T=-1), "rows"),
    ({}, dict(n=4096, T=4097, xr=1), "rows"), ({}, dict(xr=3), "input rows"), ({}, dict(xt=127), "whole values"),
    ({}, dict(yi=95), "whole values"), ({}, dict(g=None), "groups"), ({}, dict(ng=64), "groups"), ({}, dict(g=P + 8), "groups")])
def test_experts_refuse(call, d, kw, msg):
    fails(call(expert_desc(**d), **kw), msg)


def test_experts_refuse_their_own_arguments():
    from sabah.runtime import rt
    L = rt.lib()
    fails(mul(expert_desc(), y=P), "overwrite")
    fails(mul_back(expert_desc(), dx=P), "overwrite")
    fails(mul_back(expert_desc(), dx=3 * P), "overwrite")
    n = L.sabah_expert_groups_bytes(2, 3, 4)
    assert n > 0 and L.sabah_expert_groups_bytes(0, 3, 4) == 0 and L.sabah_expert_groups_bytes(2, 3, 5000) == 0
    fails(mul(expert_desc(), ng=n - 1), "groups")

    def group(ids=P, si=4, st=8, n_ids=2, T=3, E=4, g=2 * P, ng=1 << 40):
        return L.sabah_expert_group(ids, si, st, n_ids, T, E, g, ng, None)
    fails(group(ids=None), "null")
    fails(group(si=2), "multiples of 4")
    fails(group(st=6), "multiples of 4")
    fails(group(E=0), "n_experts")
    fails(group(T=-1), "rows")
    fails(group(ng=n - 1), "groups")
    fails(group(g=2 * P + 4), "groups")


# x: three rows of 128 bytes at P (the weights' 24,576 lie at 32 P); y: [3][2] rows of 96 bytes
@pytest.mark.parametrize("kw,msg", [
    (dict(yi=94), "overlap"), (dict(yt=190), "overlap"), (dict(yi=0), "overlap"), (dict(yt=0), "overlap"), (dict(yi=288, yt=96), None),
    (dict(yi=286, yt=96), "overlap"), (dict(n=1, yi=0, yt=96), None), (dict(T=1, yt=0), None), (dict(y=P + 382), "overwrite"),
    (dict(y=P + 384), None), (dict(xt=512, y=P + 128, yt=512), None), (dict(xt=512, y=P + 126, yt=512), "overwrite"),
    (dict(xt=512, y=P + 322, yt=512), "overwrite"), (dict(xt=0, y=P + 126), "overwrite"), (dict(xt=0, y=P + 128), None),
    (dict(y=32 * P + 24574), "overwrite"), (dict(y=32 * P + 24576), None)])
def test_experts_refuse_results_over_other_rows(kw, msg):
    fails(mul(expert_desc(w=32 * P), **kw, g=None), msg or "groups must")  # the check that follows


@pytest.mark.parametrize("kw,msg", [
    (dict(di=126), "overlap"), (dict(dt=254), "overlap"), (dict(dx=P + 382), "overwrite"), (dict(dx=3 * P + 574), "overwrite"),
    (dict(dx=3 * P + 576), None), (dict(dx=32 * P), "overwrite"), (dict(dw=32 * P + 24572), "overwrite"), (dict(dw=4 * P + 764), "overwrite"),
    (dict(dw=4 * P + 768), None), (dict(dw=3 * P), "overwrite"), (dict(dw=None), None), (dict(dx=None, di=0, dt=0), None),
    (dict(T=0, dx=None, dw=32 * P), "overwrite")])
def test_experts_backward_refuses_results_over_other_rows(kw, msg):
    fails(mul_back(expert_desc(w=32 * P), **kw, g=None), msg or "groups must")


# ---- AdamW -------------------------------------------------------------------
def table(*ts):
    from sabah.runtime import rt
    arr = (rt.AdamWTensor * max(1, len(ts)))()
    for i, t in enumerate(ts):
        v = dict(p=(1 + 8 * i) * P, g=(5 + 8 * i) * P, master=None, decay=0.1, n=100, p_type=0, g_type=0)
        v.update(t)
        arr[i] = rt.AdamWTensor(*(v[f] for f, _ in rt.AdamWTensor._fields_))
    n = ctypes.c_longlong(-1)
    return rt.lib().sabah_adamw_table_bytes(arr, len(ts), ctypes.byref(n)), n.value, arr


def test_adamw_tables():
    from sabah.runtime import rt
    size, n, arr = table({}, dict(n=0, p=None, g=None), dict(n=2049))
    assert n == 256 + 2304 and size == 256 + 8 * (1 + 0 + 2)
    buf = ctypes.create_string_buffer(size)
    assert rt.lib().sabah_adamw_table(arr, 3, buf, size) == 0
    fails(rt.lib().sabah_adamw_table(arr, 3, buf, size - 8), "bytes")
    fails(rt.lib().sabah_adamw_table(arr, 3, None, size), "bytes")


@pytest.mark.parametrize("ts,msg", [
    ([], "tensors"), ([dict(p_type=8)], "types"), ([dict(g_type=2)], "types"), ([dict(n=-1)], "values"), ([dict(p=None)], "null"),
    ([dict(g=None)], "null"), ([dict(master=2 * P)], "master"), ([dict(decay=-0.1)], "decay"), ([dict(decay=float("nan"))], "decay"),
    ([dict(p=P + 2)], "aligned"), ([{}, dict(p=P + 396)], "shares memory"), ([dict(g=P)], "shares memory"),
    ([dict(p_type=30, master=5 * P + 16)], "shares memory"), ([{}, {}, dict(p=P, n=1)], "shares memory")])
def test_adamw_tables_refuse(ts, msg):
    from sabah.runtime import rt
    size, _, _ = table(*ts)
    assert size == 0 and msg in rt.last_error(), rt.last_error()


def test_a_gradient_may_serve_two_tensors():
    assert table({}, dict(g=5 * P))[0] > 0


def step(**kw):
    from sabah.runtime import rt
    v = dict(table=P, table_bytes=256 + 8, n_tensors=1, bits=8, m=2 * P, v=3 * P, m_scale=4 * P, v_scale=5 * P, lr=1e-3, beta1=0.9,
             beta2=0.999, eps=1e-8, grad_scale=1.0, max_norm=1.0, d_lr=None, step=6 * P, norm=7 * P, workspace=8 * P,
             workspace_bytes=1 << 20)
    v.update(kw)
    return rt.lib().sabah_adamw_step(ctypes.byref(rt.AdamWDesc(*(v[f] for f, _ in rt.AdamWDesc._fields_))), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(table=None), "null"), (dict(step=None), "null"), (dict(m=None), "null"), (dict(v_scale=None), "null"), (dict(bits=16), "bits"),
    (dict(m=2 * P + 4), "aligned"), (dict(beta1=1.0), "betas"), (dict(beta2=-0.1), "betas"), (dict(eps=0.0), "eps"), (dict(eps=1e-60), "eps"),
    (dict(lr=float("nan")), "lr"), (dict(lr=-1.0), "lr"), (dict(grad_scale=0.0), "grad_scale"), (dict(max_norm=0.0), "max_norm"),
    (dict(table_bytes=260), "table"), (dict(table_bytes=100), "table"), (dict(n_tensors=0), "table"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=64), "workspace"), (dict(workspace=8 * P + 8), "workspace")])
def test_adamw_refuses(kw, msg):
    fails(step(**kw), msg)


def test_moments_refuse():
    from sabah.runtime import rt
    L = rt.lib()
    fails(L.sabah_adamw_moments_read(P, 2 * P, 3 * P, 4 * P, 255, 5 * P, 6 * P, None), "whole blocks")
    fails(L.sabah_adamw_moments_read(P, 2 * P, 3 * P, 4 * P, 256, None, 6 * P, None), "null")
    fails(L.sabah_adamw_moments_write(P, 2 * P, 256, 3 * P + 2, 4 * P, 5 * P, 6 * P, None), "aligned")


# ---- the classes -------------------------------------------------------------
@pytest.fixture
def ex():
    """The executor's checks without its bank; a CPU tensor's device index is -1."""
    from sabah.runtime.executor import MoEExecutor
    e = MoEExecutor.__new__(MoEExecutor)
    e.device, e._index = torch.device("cpu"), -1
    return e


def test_norm_tensors(ex):
    from sabah.runtime.norm import BlockNorm
    n = BlockNorm(8, device="cpu")
    x = torch.zeros(5, 8)
    for bad in (dict(x=torch.zeros(5, 7)), dict(x=torch.zeros(8)), dict(y=torch.zeros(5, 8, dtype=torch.float16)), dict(y=torch.zeros(4, 8)),
                dict(y=torch.zeros(8, 5).t()), dict(gate=torch.zeros(4)), dict(gate=torch.zeros(5, dtype=torch.float64)),
                dict(out=torch.zeros(5, 9)), dict(h=torch.zeros(5, 16)[:, ::2]), dict(y=None, gate=torch.zeros(5))):
        with pytest.raises(ValueError, match="block_norm"):
            ex.block_norm(n, **{**dict(x=x, y=x.clone()), **bad})
    for bad in (dict(dh=None), dict(add_dw=True), dict(dw_after=torch.zeros(7)), dict(dw_before=torch.zeros(8, dtype=torch.float16)),
                dict(dout=torch.zeros(5, 9)), dict(dx=torch.zeros(8, 5).t())):
        with pytest.raises(ValueError, match="block_norm"):
            ex.block_norm_backward(n, **{**dict(out=x, y=x.clone(), dout=x.clone(), dh=x.clone()), **bad})
    with pytest.raises(ValueError):
        ex.block_norm(n, x.double(), x.double())
    with pytest.raises(ValueError):
        BlockNorm(0, device="cpu")
    with pytest.raises(ValueError):
        BlockNorm(8193, device="cpu")


def test_expert_tensors(ex):
    from sabah.runtime.experts import FloatExperts, RowGroups
    e, g = FloatExperts(4, 8, 6, device="cpu"), RowGroups(5, 2, 4, device="cpu")
    x, dy = torch.zeros(5, 8, dtype=torch.bfloat16), torch.zeros(5, 2, 6, dtype=torch.bfloat16)
    for bad in (dict(x=x.float()), dict(x=x[:4]), dict(x=x[:, :7]), dict(x=x.reshape(40)), dict(x=torch.zeros(5, 3, 8, dtype=torch.bfloat16)),
                dict(x=torch.zeros(8, 5, dtype=torch.bfloat16).t()), dict(groups=RowGroups(5, 2, 5, device="cpu")),
                dict(out=dy.float()), dict(out=dy[:, :1]), dict(out=torch.zeros(5, 2, 12, dtype=torch.bfloat16)[:, :, ::2])):
        with pytest.raises(ValueError, match="experts"):
            ex.expert_mul(e, **{**dict(x=x, groups=g), **bad})
    for bad in (dict(dy=dy.float()), dict(dx=dy), dict(dw=torch.zeros(4, 6, 8, dtype=torch.bfloat16)), dict(dw=torch.zeros(4, 8, 6)),
                dict(add_dw=True)):
        with pytest.raises(ValueError, match="expert"):
            ex.expert_mul_backward(e, **{**dict(x=x, groups=g, dy=dy), **bad})
    for bad in (torch.zeros(5, 2, dtype=torch.int64), torch.zeros(5, dtype=torch.int32), torch.zeros(5, 3, dtype=torch.int32)):
        with pytest.raises(ValueError, match="group_rows"):
            ex.group_rows(bad, out=g)
    for bad in (dict(n_experts=0), dict(k=0), dict(dtype=torch.float64)):
        with pytest.raises(ValueError):
            FloatExperts(**{**dict(n_experts=4, k=8, rows=6, device="cpu"), **bad})


def test_adamw_tensors():
    from sabah.runtime.adamw import AdamW
    from sabah.runtime import rt
    p, g = torch.zeros(10), torch.zeros(10)
    for bad in (dict(params=[]), dict(grads=[]), dict(grads=[torch.zeros(9)]), dict(params=[torch.zeros(10, dtype=torch.float64)]),
                dict(params=[torch.zeros(5, 4)[:, ::2]]), dict(bits=16), dict(weight_decay=[0.1, 0.1]), dict(lr=torch.zeros(2))):
        with pytest.raises(ValueError, match="adamw"):
            AdamW(**{**dict(params=[p], grads=[g]), **bad})
    for bad in (dict(grads=[p]), dict(params=[p, p[3:]], grads=[g, g[3:]]), dict(weight_decay=-1.0)):
        with pytest.raises(rt.SabahRuntimeError, match="adamw"):
            AdamW(**{**dict(params=[p], grads=[g]), **bad})
    a = AdamW([p, torch.zeros(300)], [g, torch.zeros(300)], bits=8)
    assert a.starts == [0, 256] and a.n_values == 768 and a.m.dtype == torch.int8 and a.m_scale.shape == (3,)
    for bad in (torch.zeros(767), torch.zeros(768, dtype=torch.float64)):
        with pytest.raises(ValueError, match="moments"):
            a.load_moments(bad, bad, 0)
    with pytest.raises(ValueError, match="steps"):
        a.load_moments(torch.zeros(768), torch.zeros(768), -1)
    for call in (a.step, a.moments, lambda: a.load_moments(torch.zeros(768), torch.zeros(768), 0)):
        with pytest.raises(ValueError, match="GPU"):           # kernels are never given a host address
            call()
