"""Layer norm and its gradients on a B200 against 64 bits, element by element.

The bounds follow from how the kernels compute.  E is the unit roundoff of
fp32, 2^-24.  A row's sum is taken by chains of at most 32 additions in a
thread and 10 more over the threads: DEPTH roundings, one for the division."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
DEPTH = 44


@pytest.fixture(autouse=True)
def _lib(libapk):
    return libapk


def _rand(*shape, seed, scale=1.0, mean=0.0, dtype="bf16"):
    import torch
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return torch.empty(shape, dtype={"bf16": torch.bfloat16, "f32": torch.float32}[dtype], device="cuda").normal_(mean, scale, generator=g)


def _make(D, w="f32", bias=True, out="bf16", seed=0, **kw):
    import apk_b200
    return apk_b200.LayerNorm(_rand(D, seed=seed + 1, mean=1.0, scale=0.3, dtype=w),
                              _rand(D, seed=seed + 2, dtype=w) if bias else None, out_dtype=out, **kw)


def _round(err, want, dtype):
    import torch
    return err + (2.0 ** -8 if dtype == torch.bfloat16 else E) * (want.abs() + err) + 2.0 ** -120


def _forward_bounds(norm, x):
    """(y, bound), (mean, bound), (rstd, bound) in 64 bits."""
    x = x.double()
    mean, size = x.mean(-1, keepdim=True), x.abs().mean(-1, keepdim=True)
    c = x - mean
    var = c.square().mean(-1, keepdim=True)
    rstd = (var + norm.eps).rsqrt()
    em = DEPTH * E * size + E * mean.abs()
    ec = em + E * (c.abs() + em)
    dv = (2 * c.abs() * ec + ec * ec).mean(-1, keepdim=True)
    er = rstd * (dv / (var + norm.eps) + (DEPTH + 8) * E)  # (twice the half that the root takes; rsqrtf within 2 ulp)
    w = norm.weight.double()
    y = c * rstd * w
    ey = w.abs() * (rstd * ec + c.abs() * er) + 3 * E * y.abs()
    if norm.bias is not None:
        y = y + norm.bias.double()
        ey = ey + E * (y.abs() + norm.bias.double().abs())
    return (y, _round(ey, y, norm.out_dtype)), (mean, em), (rstd, er)


def _check_forward(norm, x):
    import layer_bounds as lb
    import torch
    y, stats = norm.forward(x, save_stats=True)
    (want, by), (mean, bm), (rstd, br) = _forward_bounds(norm, x)
    assert y.shape == x.shape and y.dtype == norm.out_dtype and stats.shape == (*x.shape[:-1], 2)
    lb.check(y, want, by, "y")
    lb.check(stats[..., :1], mean, bm, "mean")
    lb.check(stats[..., 1:], rstd, br, "rstd")
    assert torch.equal(norm.forward(x), y), "a second call differs"
    return stats


def _check_backward(norm, x, dy, stats, res=None):
    import layer_bounds as lb
    import torch
    got = norm.backward(dy, x, stats, residual_grad=res)
    D, M = x.shape[-1], x.numel() // max(1, x.shape[-1])
    m, r = stats[..., :1].double(), stats[..., 1:].double()
    n = (x.double() - m) * r
    en = 3 * E * n.abs()
    d = dy.double()
    g = d * norm.weight.double()
    a, b = g.mean(-1, keepdim=True), (g * n).mean(-1, keepdim=True)
    ea = (DEPTH + 2) * E * g.abs().mean(-1, keepdim=True)
    eb = (DEPTH + 6) * E * (g * n).abs().mean(-1, keepdim=True)
    dx = r * (g - a - n * b)
    ex = r * (E * g.abs() + ea + n.abs() * eb + en * b.abs() + 4 * E * (g.abs() + a.abs() + (n * b).abs()))
    if res is not None:
        dx = dx + res.double()
        ex = ex + E * (dx.abs() + res.double().abs())
    lb.check(got[0], dx, _round(ex, dx, x.dtype), "dx")
    lead = tuple(range(x.dim() - 1))
    for t, want, size, what in ((got[1], d * n, (d * n).abs(), "dw"), (got[2], d, d.abs(), "db")):
        if t is None:
            assert what == "db" and norm.bias is None
            continue
        lb.check(t, want.sum(lead), _round((M + 16) * E * size.sum(lead), want.sum(lead), t.dtype), what)
    again = norm.backward(dy, x, stats, residual_grad=res)
    assert all(p is q is None or torch.equal(p, q) for p, q in zip(got, again)), "a second call differs"


# each way of laying a row over threads, with its borders; one row to many
SHAPES = [(1, 1), (3, 2), (1, 7), (9, 8), (5, 255), (17, 256), (2, 264), (130, 512), (7, 520), (33, 1001), (400, 1024),
          (3, 1032), (1, 2048), (160, 2056), (37, 4096), (2, 4099), (5, 4104), (3, 8191), (300, 8192), (2, 16383), (3, 16384)]
TYPES = [("bf16", "f32", "bf16", True), ("f32", "bf16", "f32", False), ("f32", "f32", "bf16", True), ("bf16", "bf16", "f32", True)]


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(map(str, t)))
@pytest.mark.parametrize("M,D", SHAPES)
def test_shapes(M, D, types):
    xt, w, other, bias = types
    norm = _make(D, w, bias, other, seed=D)
    x = _rand(M, D, seed=D + 3, scale=2.0, mean=0.5, dtype=xt)
    stats = _check_forward(norm, x)
    res = _rand(M, D, seed=D + 5, dtype=xt) if M % 2 else None
    _check_backward(norm, x, _rand(M, D, seed=D + 4, dtype=other), stats, res)


# more rows than go by the gradient's form for few (three an SM)
MANY = [(500, 1), (460, 7), (500, 255), (450, 256), (600, 264), (449, 512), (500, 520), (450, 1000), (446, 1024), (470, 1032),
        (600, 2056), (446, 4096), (450, 4099), (460, 4104), (446, 8191), (500, 8192), (449, 16383), (446, 16384)]


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(map(str, t)))
@pytest.mark.parametrize("M,D", MANY)
def test_shapes_of_many_rows(M, D, types):
    xt, w, other, bias = types
    norm = _make(D, w, bias, other, seed=D)
    x = _rand(M, D, seed=D + 3, scale=2.0, mean=0.5, dtype=xt)
    stats = _check_forward(norm, x)
    _check_backward(norm, x, _rand(M, D, seed=D + 4, dtype=other), stats, _rand(M, D, seed=D + 5, dtype=xt) if D % 3 else None)


@pytest.mark.parametrize("D", [64, 1001, 2048])
def test_many_rows(D):
    norm = _make(D)
    x = _rand(9001, D, seed=1, scale=3.0)
    _check_backward(norm, x, _rand(9001, D, seed=2), _check_forward(norm, x))


def test_rows_whose_mean_is_far_from_zero_and_constant_rows():
    import torch
    norm = _make(1536, out="f32", eps=1e-3)
    x = _rand(64, 1536, seed=1, dtype="f32")
    x += torch.linspace(-300, 300, 64, device="cuda")[:, None]
    x[5] = 0.0
    x[6] = 0.375
    stats = _check_forward(norm, x)
    assert torch.equal(norm.forward(x)[5:7], norm.bias.expand(2, -1))
    _check_backward(norm, x, _rand(64, 1536, seed=2), stats)


def test_rows_with_nan_or_infinity_do_not_touch_others():
    import torch
    norm = _make(768)
    x = _rand(40, 768, seed=1)
    dy = _rand(40, 768, seed=2)
    want, stats = norm.forward(x, save_stats=True)
    wx, _, _ = norm.backward(dy, x, stats)
    bad = x.clone()
    bad[3, 5], bad[4, 700], bad[39, 0] = float("nan"), float("inf"), -float("inf")
    y, st = norm.forward(bad, save_stats=True)
    dx, dw, db = norm.backward(dy, bad, st)
    rows = torch.tensor([3, 4, 39], device="cuda")
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[rows] = False
    assert y[rows].isnan().all() and torch.equal(y[keep], want[keep])
    assert dx[rows].isnan().all() and torch.equal(dx[keep], wx[keep])
    assert dw.isnan().all() and torch.isfinite(db).all()


@pytest.mark.parametrize("D,ld,at", [(256, 264, 8), (256, 259, 1), (1000, 1003, 3), (2048, 2056, 0), (2048, 2049, 1)])
def test_strided_and_unaligned_rows(D, ld, at):
    """Views into wider rows, as from a fused buffer: same results as of a copy, and nothing written beside them."""
    import torch
    norm = _make(D)
    wide = _rand(50, ld, seed=1)
    x = wide[:, at:at + D]
    room = _rand(50, ld, seed=7)
    kept = room.clone()
    out = room[:, at:at + D]
    if ld - at < D:
        pytest.skip("no room")
    _check_forward(norm, x)
    norm.forward(x, out=out)
    assert torch.equal(out, norm.forward(x))
    kept[:, at:at + D] = out
    assert torch.equal(room, kept)
    y, stats = norm.forward(x.contiguous(), save_stats=True)
    dyw, resw = _rand(50, ld, seed=3), _rand(50, ld, seed=4)
    _check_backward(norm, x, dyw[:, at:at + D], stats, resw[:, at:at + D])


def test_leading_axes_and_in_place():
    import torch
    norm = _make(320)
    x = _rand(2, 3, 5, 320, seed=1)
    stats = _check_forward(norm, x)
    _check_backward(norm, x, _rand(2, 3, 5, 320, seed=2), stats, _rand(2, 3, 5, 320, seed=3))
    want = norm.forward(x)
    assert norm.forward(x, out=x) is x and torch.equal(x, want)
    for D in (1001, 4096):
        norm, x = _make(D), _rand(333, D, seed=4)
        want = norm.forward(x)
        assert torch.equal(norm.forward(x, out=x), want)


@pytest.mark.parametrize("M,D", [(21, 96), (500, 96), (30, 1500), (600, 1500)])
def test_parts_of_the_gradient_and_no_rows(M, D):
    import torch
    norm = _make(D, "bf16")
    x, dy = _rand(M, D, seed=1), _rand(M, D, seed=2)
    _, stats = norm.forward(x, save_stats=True)
    full = norm.backward(dy, x, stats)
    for i in range(8):
        need = [bool(i >> j & 1) for j in range(3)]
        got = norm.backward(dy, x, stats, None, *need)
        for n, g, f in zip(need, got, full):
            assert (g is None) if not n else torch.equal(g, f)
    e = x[:0]
    y, st = norm.forward(e, save_stats=True)
    assert y.shape == (0, D) and st.shape == (0, 2)
    dx, dw, db = norm.backward(e, e, st)
    assert dx.shape == (0, D) and not dw.any() and not db.any()


def test_gradient_against_differences():
    """dx, dw and db along random directions against central differences of
    the definition in 64 bits (step 1e-5: truncation about 1e-10 of the values)."""
    import torch
    D, M = 77, 13
    norm = _make(D, out="f32")
    x, dy = _rand(M, D, seed=1, scale=1.5, dtype="f32"), _rand(M, D, seed=2, dtype="f32")
    _, stats = norm.forward(x, save_stats=True)
    got = norm.backward(dy, x, stats)

    def loss(x, w, b):
        c = x - x.mean(1, keepdim=True)
        return ((c * (c.square().mean(1, keepdim=True) + norm.eps).rsqrt() * w + b) * dy.double()).sum()

    at = [x.double(), norm.weight.double(), norm.bias.double()]
    for i, g in enumerate(got):
        for k in range(4):
            v = _rand(*g.shape, seed=10 * i + k, dtype="f32").double()
            up, down = list(at), list(at)
            up[i], down[i] = at[i] + 1e-5 * v, at[i] - 1e-5 * v
            want = float((loss(*up) - loss(*down)) / 2e-5)
            # each of the M D terms carries a few E of the sums behind it
            size = float((dy.double().abs() * norm.weight.double().abs()).sum()) * float(v.abs().max())
            assert abs(float((g.double() * v).sum()) - want) <= 64 * E * size + 1e-7 * size


def test_streams_devices_and_graphs():
    """On another stream than the inputs' own, from two streams at once, captured and replayed with new inputs."""
    import torch
    norm = _make(2048)
    xs = [_rand(700, 2048, seed=i) for i in range(4)]
    dys = [_rand(700, 2048, seed=10 + i) for i in range(4)]

    def f(x, dy):
        y, st = norm.forward(x, save_stats=True)
        return (y, st, *norm.backward(dy, x, st, residual_grad=x))

    want = [f(x, d) for x, d in zip(xs, dys)]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(4):
        with torch.cuda.stream(side[i % 2]):
            got.append(f(xs[i], dys[i]))
    torch.cuda.synchronize()
    x, dy = xs[0].clone(), dys[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f(x, dy)
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    for i in (2, 1, 3):
        x.copy_(xs[i])
        dy.copy_(dys[i])
        graph.replay()
        again = f(xs[0], dys[0])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[i])) and all(torch.equal(p, q) for p, q in zip(again, want[0]))


def test_first_calls_in_a_capture():
    """What needs no scratch may be captured before it was ever called; what does is refused, and works after one call."""
    import torch

    import apk_b200
    w, b = torch.rand(4096, device="cuda") + 0.5, torch.rand(4096, device="cuda")
    x, few = _rand(1000, 4096, seed=1), _rand(20, 4096, seed=2)
    norm, graph = apk_b200.LayerNorm(w, b), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, stats = norm.forward(x, save_stats=True)
        y2, stats2 = norm.forward(few, save_stats=True)
        d2 = norm.backward(few, few, stats2)
        with pytest.raises(apk_b200.ApkError, match="before the capture"):
            norm.backward(x, x, stats)
    graph.replay()
    torch.cuda.synchronize()
    other = apk_b200.LayerNorm(w, b)
    want, ws = other.forward(x, save_stats=True)
    assert torch.equal(y, want) and torch.equal(stats, ws) and torch.equal(y2, other.forward(few))
    assert all(torch.equal(p, q) for p, q in zip(d2, other.backward(few, few, stats2)))
    wd = other.backward(x, x, ws)
    norm.backward(x, x, ws)
    with torch.cuda.graph(graph := torch.cuda.CUDAGraph()):
        d = norm.backward(x, x, ws)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(d, wd))


def test_refusals():
    import torch

    import apk_b200
    from apk_b200 import _lib as L
    w = torch.ones(64, device="cuda")
    for bad in (dict(weight=w.double()), dict(weight=w[None]), dict(weight=w[::2]), dict(weight=w, bias=w[:32]),
                dict(weight=w, bias=w.cpu()), dict(weight=w, out_dtype="f16")):
        with pytest.raises(ValueError):
            apk_b200.LayerNorm(**bad)
    with pytest.raises(apk_b200.ApkError):
        apk_b200.LayerNorm(w, eps=0.0)
    with pytest.raises(apk_b200.ApkError):
        apk_b200.LayerNorm(torch.ones(16385, device="cuda"))
    norm = apk_b200.LayerNorm(w, w)
    x = _rand(6, 64, seed=1)
    y, stats = norm.forward(x, save_stats=True)
    for bad in (x.half(), x.cpu(), x[:, :32], x.t().contiguous().t(), x[0, 0]):
        with pytest.raises(ValueError):
            norm.forward(bad)
    with pytest.raises(ValueError):
        norm.forward(x, out=x.float())
    with pytest.raises(ValueError, match="shares memory"):
        flat = _rand(400, seed=2)
        norm.forward(flat[:320].view(5, 64), out=flat[8:328].view(5, 64))
    with pytest.raises(ValueError, match="shares memory"):
        flat = _rand(400, seed=2, dtype="f32")
        norm.forward(flat[:64].view(1, 64), out=flat[:64].view(torch.bfloat16)[:64].view(1, 64))
    with pytest.raises(apk_b200.ApkError):
        norm.forward(x[:1].expand(6, 64))          # rows of stride 0
    for kw in (dict(dy=y[:5]), dict(stats=stats[:5]), dict(stats=stats.double()), dict(residual_grad=x.float()),
               dict(residual_grad=x[:5])):
        with pytest.raises(ValueError):
            norm.backward(**{**dict(dy=y, x=x, stats=stats), **kw})
    p = w.data_ptr()
    for io in (dict(rows=-1), dict(rows=(1 << 30) + 1), dict(x=None), dict(y=None), dict(x_dtype=2), dict(ldx=63),
               dict(ldy=0), dict(x=p + 1), dict(stats=p + 4)):
        a = L.NormIO(**{**dict(x=p, ldx=64, rows=1, x_dtype=1, y_dtype=1, y=p, ldy=64), **io})
        assert norm._lib.apk_norm_forward(norm._h, ctypes.byref(a)) == L.APK_EINVAL
        assert norm._lib.apk_norm_last_error(norm._h)
    norm.weight = torch.ones(64, device="cuda")
    with pytest.raises(ValueError, match="other memory"):
        norm.forward(x)
    with pytest.raises(ValueError, match="other memory"):
        norm.backward(y, x, stats)


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(map(str, t)))
@pytest.mark.parametrize("D,ld,at", [(515, 515, 1), (1001, 1001, 0), (1003, 1010, 7), (2048, 2048, 5), (2051, 2057, 3), (4099, 4099, 6),
                                     (8191, 8193, 1)])
def test_rows_from_any_address(D, ld, at, types):
    """Many rows that start anywhere, the first one too: a NaN beside a row, or in another row, does not reach it."""
    import torch
    xt, w, other, bias = types
    norm = _make(D, w, bias, other, seed=D)
    M = 500

    def rows(dtype, seed):
        room = torch.full((at + M * ld,), float("nan"), device="cuda", dtype={"bf16": torch.bfloat16, "f32": torch.float32}[dtype])
        t = room[at:].as_strided((M, D), (ld, 1))
        t.copy_(_rand(M, D, seed=seed, scale=2.0, mean=0.5, dtype=dtype))
        return room, t

    (_, x), (_, dy), (_, res) = rows(xt, D + 3), rows(other, D + 4), rows(xt, D + 5)
    stats = _check_forward(norm, x)
    _check_backward(norm, x, dy, stats, res)
    _check_backward(norm, x, dy, stats)
    want = norm.forward(x)
    room, out = rows(other, D + 6)
    kept = room.clone()
    norm.forward(x, out=out)
    assert torch.equal(out, want)
    kept[at:].as_strided((M, D), (ld, 1)).copy_(want)
    assert torch.equal(room.nan_to_num(7.0), kept.nan_to_num(7.0)), "something beside the rows was written"
    dx = norm.backward(dy, x, stats)[0]
    bad = torch.arange(0, M, 3, device="cuda")
    clean = [i for i in range(M) if i % 3]
    x[bad] = float("nan")
    dy[bad] = float("inf")
    assert torch.equal(norm.forward(x)[clean], want[clean]) and norm.forward(x)[bad].isnan().all()
    assert torch.equal(norm.backward(dy, x, stats)[0][clean], dx[clean])
    if xt == other:
        x[bad] = 1.0
        want = norm.forward(x)
        assert torch.equal(norm.forward(x, out=x), want)


def _close_bounds(norm, x):
    """As _forward_bounds, for a mean that is corrected by the mean of the
    differences from it where it is larger than the deviation.  The first one is
    within e1 = (DEPTH + 1) E mean|x|; the differences, d = x - that, are within
    E |d|, their mean within (DEPTH + 3) E mean|d|, and |d| is up to |c| + e1.
    The variance is mean(d^2) less the square of mean(d), which is up to e1."""
    import torch
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    e1 = (DEPTH + 1) * E * x.abs().mean(-1, keepdim=True)
    d = c.abs() + e1
    var, size = c.square().mean(-1, keepdim=True), d.square().mean(-1, keepdim=True)
    em = (DEPTH + 3) * E * d.mean(-1, keepdim=True)
    em = torch.where(mean.abs() < 1.001 * var.sqrt(), e1 + em, em)
    ec = em + 2 * E * d
    dv = (DEPTH + 6) * E * size + 2 * e1 * em + 3 * E * e1.square()
    rstd = (var + norm.eps).rsqrt()
    er = rstd * (dv / (var + norm.eps) + 6 * E)  # (the root takes half of that; rsqrtf within 2 ulp)
    w = norm.weight.double()
    y = c * rstd * w
    ey = w.abs() * ((rstd + er) * ec + c.abs() * er) + 3 * E * y.abs()
    if norm.bias is not None:
        y = y + norm.bias.double()
        ey = ey + E * (y.abs() + norm.bias.double().abs())
    return (y, _round(ey, y, norm.out_dtype)), (mean, em + E * mean.abs()), (rstd, er)


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,D", [(12, 100), (12, 256), (12, 333), (12, 512), (12, 1000), (12, 1001), (300, 1001), (300, 1536), (12, 3000),
                                 (300, 4099), (12, 4096), (300, 8192), (12, 8191), (12, 16384), (300, 16383)])
def test_a_mean_far_from_zero_costs_no_digits(M, D, out):
    """Constant rows give the bias, and rows close to one value their own norm."""
    import layer_bounds as lb
    import torch
    norm = _make(D, out=out)
    x = _rand(M, D, seed=1, dtype="f32")
    at = torch.tensor([100.1, 5000.3, -77.7, 1.0e6 / 3, 0.1, -0.3], device="cuda")
    for i in range(6):
        x[i] = at[i]
        x[6 + i] = at[i] * (1 + x[6 + i] * 1e-5)
    x[12:] += torch.linspace(-3000, 3000, M - 12, device="cuda")[:, None]
    y, stats = norm.forward(x, save_stats=True)
    (want, by), (mean, bm), (rstd, br) = _close_bounds(norm, x)
    lb.check(y, want, by, "y")
    lb.check(stats[:, :1], mean, bm, "mean")
    lb.check(stats[:, 1:], rstd, br, "rstd")
    assert torch.equal(stats[:6, 0], at), "a constant row's mean"


def test_a_mean_far_from_zero_and_almost_no_eps():
    """The square of what the mean was off by may pass the mean of the squares: no NaN comes of it."""
    import torch
    for D in (200, 1001, 1536, 8191):
        norm = _make(D, out="f32", eps=1e-30)
        x = torch.full((64, D), 1.0, device="cuda") * torch.linspace(100.1, 9999.7, 64, device="cuda")[:, None]
        y, stats = norm.forward(x, save_stats=True)
        assert torch.isfinite(y).all() and torch.isfinite(stats).all()
        x[3, 5] = float("nan")
        y, stats = norm.forward(x, save_stats=True)
        assert y[3].isnan().all() and stats[3].isnan().all() and torch.isfinite(y[[2, 4]]).all()
