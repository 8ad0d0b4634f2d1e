"""MoEExecutor.group_rows, expert_mul and expert_mul_backward against the 64-bit forms of train_refs."""
import pytest
import torch

import train_refs as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ex(hip_rt):
    from sabah.runtime.bank import ExpertBank
    from sabah.runtime.executor import MoEExecutor
    return MoEExecutor(ExpertBank(1, 8, 256, 256, {"gate": 21, "up": 21, "down": 21}, device=DEV))


def experts_of(w, dtype):
    from sabah.runtime.experts import FloatExperts
    e = FloatExperts(w.shape[0], w.shape[2], w.shape[1], dtype=dtype, device=DEV)
    e.w.copy_(w)
    return e


def draw(T, E, K, k, rows, dtype, spread="even", each=False, none=0.0, whole=True, seed=1):
    """whole: small whole numbers, whose products' sums are exact, so that a result is the sum rounded once."""
    g = torch.Generator().manual_seed(seed)
    if spread == "even":
        ids = torch.rand(T, E, generator=g).topk(min(K, E), dim=1).indices.to(torch.int32)
        if K > E:
            ids = torch.randint(0, E, (T, K), generator=g, dtype=torch.int32)
    elif spread == "one":                                    # all rows with one expert, named again and again by a token
        ids = torch.full((T, K), E - 1, dtype=torch.int32)
    else:
        ids = (torch.rand(T, K, generator=g).pow(4) * E).to(torch.int32).clamp(max=E - 1)
    ids[torch.rand(T, K, generator=g) < none] = -1

    def values(*shape, scale=1.0):
        if whole:
            return torch.randint(-3, 4, shape, generator=g).float()
        return torch.randn(*shape, generator=g) * scale
    x, w, dy = values(T, K if each else 1, k), values(E, rows, k, scale=0.1), values(T, K, rows, scale=0.1)
    return ids, x.to(dtype), w.to(dtype), dy.to(dtype)


def run(ex, ids, x, w, dy, dtype):
    e = experts_of(w, dtype)
    groups = ex.group_rows(ids.to(DEV), e.n_experts)
    xd = x.to(DEV)
    y = ex.expert_mul(e, xd, groups)
    dx, dw = ex.expert_mul_backward(e, xd, groups, dy.to(DEV))
    ex_check(ex)
    return y, dx, dw


def ex_check(ex):
    from sabah.runtime import rt
    torch.cuda.synchronize()
    rt.check(rt.lib().sabah_rt_check_errors(), "experts")


def check(got, ids, x, w, dy, dtype, whole):
    y, dx, dw = got
    wy, ty = R.expert_mul(w, x, ids)
    (wx, tx), (ww, tw) = R.expert_back(w, x, ids, dy)
    if whole:
        assert torch.equal(y.cpu(), wy.to(dtype)), "y"
        assert torch.equal(dx.cpu(), wx.to(dtype)), "dx"
        assert torch.equal(dw.cpu().double(), ww), "dw"
    else:
        R.close(y, wy, ty + R.half_step(wy, dtype) * 1.001, "y")
        R.close(dx, wx, tx + R.half_step(wx, dtype) * 1.001, "dx")
        R.close(dw, ww, tw, "dw")


SIZES = [(1, 1, 1, 1, 1), (2, 3, 2, 5, 7), (1, 16, 4, 64, 48), (3, 8, 2, 17, 33), (40, 5, 3, 130, 70), (200, 4, 2, 256, 136),
         (300, 3, 2, 96, 129), (64, 64, 6, 128, 200), (129, 2, 1, 72, 260), (33, 7, 9, 40, 24)]     # T, E, K, k, rows


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,E,K,k,rows", SIZES)
@pytest.mark.parametrize("whole", [True, False])
def test_products_and_gradients(ex, T, E, K, k, rows, dtype, whole):
    for each, none in ((False, 0.0), (True, 0.3)):
        args = draw(T, E, K, k, rows, TYPES[dtype], "even" if K <= E else "skewed", each, none, whole)
        check(run(ex, *args, TYPES[dtype]), *args, TYPES[dtype], whole)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("spread", ["one", "skewed"])
def test_uneven_groups(ex, dtype, spread):
    """All rows with one expert, which a token names several times, and groups from none to many tiles."""
    args = draw(150, 9, 4, 80, 152, TYPES[dtype], spread, True)
    check(run(ex, *args, TYPES[dtype]), *args, TYPES[dtype], True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,E,K,k,rows", [(117, 64, 6, 704, 712), (6300, 4, 1, 64, 2048), (3500, 2, 2, 2560, 40), (5000, 3, 1, 48, 1000)])
def test_every_tile(ex, T, E, K, k, rows, dtype):
    """Calls that fill the card with tiles of 128 x 256, or of 256 x 256, and their last tiles of any number of rows; sums over
    more rows than LDS holds the places of."""
    args = draw(T, E, K, k, rows, TYPES[dtype], "skewed")
    check(run(ex, *args, TYPES[dtype]), *args, TYPES[dtype], True)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("last", [1, 31, 32, 33, 64, 65, 97, 128, 129, 200, 255])
def test_last_tiles_of_any_number_of_rows(ex, last, dtype):
    """Groups that end inside each of a tile's 32-row results, in both large forms."""
    for T0, rows in ((6144, 2048), (1280, 2048)):
        T = T0 + last
        ids, x, w, dy = draw(T, 2, 1, 32, rows, TYPES[dtype])
        ids[:] = 0
        ids[:last] = 1
        e = experts_of(w, TYPES[dtype])
        y = ex.expert_mul(e, x.to(DEV), ex.group_rows(ids.to(DEV), 2))
        assert torch.equal(y.cpu(), R.expert_mul(w, x, ids)[0].to(TYPES[dtype]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("k,rows", [(2048, 768), (640, 2560), (1000, 300)])
def test_model_sizes(ex, k, rows, dtype):
    for T in (1, 30, 700):
        args = draw(T, 6, 2, k, rows, TYPES[dtype], whole=T != 30)
        check(run(ex, *args, TYPES[dtype]), *args, TYPES[dtype], T != 30)


@pytest.mark.parametrize("R_,E,K", [(1, 1, 1), (5, 4096, 5), (64, 3, 1), (60, 512, 10), (64, 70, 8), (65, 4, 5), (4096, 512, 8), (4097, 7, 1), (20000, 60, 10),
                                     (70000, 4096, 7), (9000, 2, 3), (300000, 100, 3)])
def test_groups_are_stable_and_whole(ex, R_, E, K):
    """The buffer's order, offsets and tiles against a stable sort, with -1 and bad ids at the end."""
    from sabah.runtime import rt
    T = R_ // K
    g = torch.Generator().manual_seed(R_)
    ids = torch.randint(-1, E, (T, K), generator=g, dtype=torch.int32)
    bad = T > 10
    if bad:
        ids[T // 2, 0], ids[0, K - 1] = E, -7
    groups = ex.group_rows(ids.to(DEV), E)
    torch.cuda.synchronize()
    if bad:
        with pytest.raises(rt.SabahRuntimeError, match="expert id"):
            rt.check(rt.lib().sabah_rt_check_errors(), "groups")
    words = groups.buffer.cpu().view(torch.int32)
    n = T * K
    assert words[1] == n and words[3] == E
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, torch.where(flat == -1, E, E + 1))
    counts = torch.bincount(key, minlength=E + 2)
    start = torch.cumsum(counts, 0) - counts
    off = words[16:16 + E + 3].long()
    assert torch.equal(off[:E + 2], start) and off[E + 2] == n
    at = 16 + (E + 3 + 3) // 4 * 4
    assert torch.equal(words[at:at + n].long(), torch.argsort(key, stable=True))
    at += (n + 3) // 4 * 4
    for rows, count in ((16, int(words[4])), (128, int(words[5])), (256, int(words[6]))):
        if rows == 16 and n > 10 * E:                          # for products over few rows alone
            assert count == 0
            continue
        want = [(e if e < E else E - 1 - e, int(start[e]) + o, min(rows, int(counts[e]) - o), 0)
                for e in torch.nonzero(counts)[:, 0].tolist() for o in range(0, int(counts[e]), rows)]
        most = n // rows + min(n, E + 2)
        assert count == len(want) <= most
        assert words[at:at + 4 * count].reshape(-1, 4).tolist() == [list(w) for w in want]
        at += most * 4


def test_ids_with_strides(ex):
    ids, x, w, dy = draw(50, 6, 3, 64, 40, torch.bfloat16)
    wide = torch.full((50, 9), -1, dtype=torch.int32)
    wide[:, 1::3] = ids
    e = experts_of(w, torch.bfloat16)
    a = ex.group_rows(ids.to(DEV), 6)
    b = ex.group_rows(wide.to(DEV)[:, 1::3], 6)
    c = ex.group_rows(ids.t().contiguous().to(DEV).t(), 6)
    ys = [ex.expert_mul(e, x.to(DEV), g) for g in (a, b, c)]
    assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])


@pytest.mark.parametrize("T", [4, 90])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_strided_rows_and_what_lies_beside_them(ex, T, dtype):
    """x, y, dy and dx inside wider tensors, at addresses that are no multiple of 16."""
    dt = TYPES[dtype]
    ids, x, w, dy = draw(T, 5, 2, 72, 88, dt, each=True, none=0.2)
    e = experts_of(w, dt)
    groups = ex.group_rows(ids.to(DEV), 5)
    want = ex.expert_mul(e, x.to(DEV), groups), ex.expert_mul_backward(e, x.to(DEV), groups, dy.to(DEV))

    def wide(width):
        t = torch.full((T + 1, 3, width + 5), 9.0, dtype=dt, device=DEV)
        return t, t[:T, :2, 1:1 + width]
    (_, xs), (yw, ys), (_, ds), (dw, dxs) = wide(72), wide(88), wide(88), wide(72)
    xs.copy_(x)
    ds.copy_(dy)
    y = ex.expert_mul(e, xs, groups, out=ys)
    dx, g = ex.expert_mul_backward(e, xs, groups, ds, dx=dxs)
    assert torch.equal(y, want[0]) and torch.equal(dx, want[1][0]) and torch.equal(g, want[1][1])
    for t, inner in ((yw, 88), (dw, 72)):
        assert (t[T] == 9).all() and (t[:, 2] == 9).all() and (t[:, :, 0] == 9).all() and (t[:, :, 1 + inner:] == 9).all()
    one = x[:1, :1].to(DEV).expand(T, 1, 72)                   # one row for all tokens: strides of 0
    full = one.contiguous()
    assert torch.equal(ex.expert_mul(e, one, groups), ex.expert_mul(e, full, groups))


@pytest.mark.parametrize("T", [5, 200])
def test_rows_without_an_expert_and_bad_ids(ex, T):
    from sabah.runtime import rt
    ids, x, w, dy = draw(T, 4, 2, 64, 96, torch.float32)
    ids[0, 0], ids[1, 1], ids[2, 0], ids[3] = -1, 4, -2, -1
    e = experts_of(w, torch.float32)
    out = torch.full((T, 2, 96), 5.0, device=DEV)
    groups = ex.group_rows(ids.to(DEV), 4)
    torch.cuda.synchronize()
    with pytest.raises(rt.SabahRuntimeError, match="expert id"):
        ex.expert_mul(e, x.to(DEV), groups, out=out)
    y = ex.expert_mul(e, x.to(DEV), groups, out=out)
    dx, dw = ex.expert_mul_backward(e, x.to(DEV), groups, dy.to(DEV))
    wy, _ = R.expert_mul(w, x, ids)
    (wx, _), (ww, _) = R.expert_back(w, x, ids, dy)
    for got, want in ((y, wy), (dx, wx)):
        assert torch.equal(got.cpu().double().nan_to_num(nan=1e9), want.nan_to_num(nan=1e9))
    assert torch.equal(dw.cpu().double(), ww)


def test_no_rows_at_all(ex):
    for T in (0, 6):
        ids, x, w, dy = draw(max(T, 1), 3, 2, 40, 24, torch.bfloat16, none=2.0)
        ids, x, dy = ids[:T], x[:T], dy[:T]
        y, dx, dw = run(ex, ids, x, w, dy, torch.bfloat16)
        assert y.shape == (T, 2, 24) and (y == 0).all() and (dx == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("T", [3, 100])
def test_weight_gradients_are_added_and_others_left_alone(ex, T):
    ids, x, w, dy = draw(T, 8, 2, 48, 56, torch.bfloat16, "skewed")
    ids[ids == 5] = 4
    e = experts_of(w, torch.bfloat16)
    groups = ex.group_rows(ids.to(DEV), 8)
    base = torch.randint(-9, 10, (8, 56, 48)).float()
    base[5, 3, 7] = float("nan")                               # of an expert without rows: not read
    dw = base.to(DEV)
    dx, got = ex.expert_mul_backward(e, x.to(DEV), groups, dy.to(DEV), dw=dw, add_dw=True, need_dx=False)
    assert dx is None and got is dw
    (_, _), (ww, _) = R.expert_back(w, x, ids, dy)
    want = base.double() + ww
    assert torch.equal(dw.cpu().double().nan_to_num(nan=1e9), want.nan_to_num(nan=1e9))
    dx, got = ex.expert_mul_backward(e, x.to(DEV), groups, dy.to(DEV), need_dw=False)
    assert got is None and dx.shape == (T, 2, 48)


@pytest.mark.parametrize("T", [6, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_nan_and_infinity_stay_where_they_belong(ex, T, dtype):
    """A row's NaN reaches its own y and its expert's dw alone; an expert's NaN its own rows alone."""
    dt = TYPES[dtype]
    ids, x, w, dy = draw(T, 4, 2, 72, 100, dt, each=True)
    ids = ids % 4
    clean = run(ex, ids, x, w, dy, dt)
    x2, w2, dy2 = x.clone(), w.clone(), dy.clone()
    ids_c = ids.clone()
    ids_c[ids_c == 3] = 2
    ids_c[0, 0], ids_c[1, 1] = 3, 0                            # expert 3 has one row
    clean = run(ex, ids_c, x, w, dy, dt)
    x2[0, 0, 5], w2[3, 7, 9], dy2[0, 0, 50] = float("inf"), float("nan"), float("nan")
    y, dx, dw = run(ex, ids_c, x2, w2, dy2, dt)
    other = torch.ones(T, 2, dtype=torch.bool)
    other[0, 0] = False
    other = other.to(DEV)
    assert torch.equal(y[other], clean[0][other]) and torch.equal(dx[other], clean[1][other])
    assert torch.equal(dw[:3], clean[2][:3]) and not y[0, 0].isfinite().all()


def test_groups_of_another_call_are_refused(ex):
    """On the host by their sizes, and by the kernels where a buffer was never made for them."""
    from sabah.runtime import rt
    from sabah.runtime.experts import RowGroups
    ids, x, w, dy = draw(12, 4, 2, 64, 64, torch.float32)
    e = experts_of(w, torch.float32)
    groups = ex.group_rows(ids.to(DEV), 4)
    with pytest.raises(ValueError):
        ex.expert_mul(e, x[:11].to(DEV), groups)
    with pytest.raises(ValueError):
        ex.expert_mul(e, x.to(DEV), ex.group_rows(ids.to(DEV), 5))
    empty = RowGroups(12, 2, 4, device=DEV)
    out = torch.full((12, 2, 64), 5.0, device=DEV)
    ex.expert_mul(e, x.to(DEV), empty, out=out)
    torch.cuda.synchronize()
    assert (out == 5).all()
    with pytest.raises(rt.SabahRuntimeError, match="groups"):
        rt.check(rt.lib().sabah_rt_check_errors(), "experts")
    ex_check(ex)


@pytest.mark.parametrize("T", [2, 300])
def test_captured_and_replayed_on_another_stream(ex, T):
    ids, x, w, dy = (t.to(DEV) for t in draw(T, 8, 2, 200, 120, torch.bfloat16, whole=False))
    e = experts_of(w, torch.bfloat16)

    def all_of_it():
        groups = ex.group_rows(ids, 8)
        return (ex.expert_mul(e, x, groups),) + ex.expert_mul_backward(e, x, groups, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        all_of_it()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = all_of_it()
    for i in range(3):
        ids.copy_((ids + 1 + i) % 8)
        x.copy_(x * 0.5 + 1)
        graph.replay()
        want = all_of_it()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    ex_check(ex)
