"""The linear layer and its gradients on a B200 against 64 bits, element by
element, with bounds derived from the arithmetic (layer_bounds.py)."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu

ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


@pytest.fixture(autouse=True)
def _lib(libapk):
    return libapk


def _rand(*shape, seed, scale=1.0, dtype=None):
    import torch
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return torch.empty(shape, dtype=dtype or torch.bfloat16, device="cuda").normal_(0.0, scale, generator=g)


def _layer(K, N, layout="kn", act="none", bias="f32", out="bf16", seed=0, **kw):
    import torch

    import apk_b200
    w = _rand(*((K, N) if layout == "kn" else (N, K)), seed=seed + 1, scale=K ** -0.5)
    b = None if bias is None else _rand(N, seed=seed + 2, dtype={"f32": torch.float32, "bf16": torch.bfloat16}[bias])
    return apk_b200.Linear(w, b, act=act, layout=layout, out_dtype=out, **kw), (w if layout == "kn" else w.t())


def _check_forward(M, K, N, layout, act, bias, residual, out, x=None, seed=0):
    import layer_bounds as lb
    import torch
    lin, w = _layer(K, N, layout, act, bias, out, seed)
    x = _rand(M, K, seed=seed + 3) if x is None else x
    r = None if residual is None else _rand(M, N, seed=seed + 4, dtype=residual)
    y, z = lin.forward(x, residual=r, save_preact=True)
    y2 = lin.forward(x, residual=r)
    assert y.dtype == {"bf16": torch.bfloat16, "f32": torch.float32}[out] and y.shape == (M, N)
    want, by, wz, bz = lb.linear(x, w, lin.bias, act, r, y.dtype)
    lb.check(y, want, by, "y")
    lb.check(z, wz, bz, "preact")
    assert torch.equal(y, y2), "a second call differs"
    assert lin.status() == 0


# every tile variant: rows of one token to several pair tiles, K from less than a
# stage to long sums, columns that end inside a tile, odd strides
SHAPES = [(1, 1, 1), (1, 2048, 2048), (2, 64, 8), (7, 33, 65), (8, 520, 1000), (9, 128, 130), (16, 4096, 256),
          (17, 72, 40), (33, 4096, 128), (64, 1024, 1024), (65, 1001, 129), (128, 8, 2000), (130, 2048, 512),
          (257, 136, 257), (300, 5000, 96), (513, 264, 1048), (1024, 192, 4104), (2000, 1100, 1031)]


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_forward_shapes(M, K, N, layout):
    import torch
    i = SHAPES.index((M, K, N))
    _check_forward(M, K, N, layout, ACTS[i % 5], (None, "f32", "bf16")[i % 3], (None, torch.bfloat16, torch.float32)[i % 3],
                   ("bf16", "f32")[(i + (layout == "nk")) % 2], seed=10 * i)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [4, 100, 700])
def test_forward_activations(M, act):
    import torch
    _check_forward(M, 264, 520, "kn", act, "f32", torch.bfloat16, "f32", seed=1)
    _check_forward(M, 264, 520, "nk", act, "bf16", None, "bf16", seed=2)


def test_large_tiles_both_kinds_and_fp32_of_a_long_sum():
    import torch
    _check_forward(4096, 4096, 1536, "kn", "gelu_tanh", "f32", torch.bfloat16, "bf16")  # 512 x 256 pair tiles
    _check_forward(1030, 8192, 1030, "nk", "none", None, None, "f32")                  # accumulators of 512 k
    _check_forward(5, 8192, 48, "kn", "none", None, None, "f32")
    _check_forward(40, 8192, 160, "kn", "silu", "f32", None, "f32")                    # split over a cluster


def test_forward_views_of_other_strides_and_alignments():
    import layer_bounds as lb
    import torch

    import apk_b200
    for M in (3, 50, 300):
        big = _rand(M, 515, seed=5)
        x = big[:, 3:3 + 264]                       # rows off the 16-byte grid
        wide = _rand(300, 417, seed=6, scale=0.06)
        for layout, w in (("kn", wide[:264, 1:201]), ("nk", wide[:200, 2:266])):
            lin = apk_b200.Linear(w, act="silu", layout=layout)
            out = torch.full((M, 333), 7.0, dtype=torch.bfloat16, device="cuda")
            res = _rand(M, 250, seed=7)[:, 5:205]
            y = lin.forward(x, residual=res, out=out[:, 10:210])
            want, by, _, _ = lb.linear(x, w if layout == "kn" else w.t(), None, "silu", res, torch.bfloat16)
            lb.check(y, want, by, f"{M} {layout}")
            assert bool((out[:, :10] == 7).all()) and bool((out[:, 210:] == 7).all()), "wrote outside its view"


def test_more_axes_in_place_residual_and_no_rows():
    import layer_bounds as lb
    import torch
    lin, w = _layer(96, 64, act="gelu", bias="bf16")
    x = _rand(2, 3, 5, 96, seed=3)
    assert torch.equal(lin.forward(x), lin.forward(x.reshape(30, 96)).reshape(2, 3, 5, 64))
    for m in (5, 40, 600):
        x, r = _rand(m, 96, seed=4), _rand(m, 64, seed=5)
        want, by, _, _ = lb.linear(x, w, lin.bias, "gelu", r, torch.bfloat16)
        y = lin.forward(x, residual=r, out=r)       # added where it stands
        assert y.data_ptr() == r.data_ptr()
        lb.check(y, want, by, "in place")
    y = lin.forward(x[:0])
    assert y.shape == (0, 64)
    dx, dw, db = lin.backward(y, x[:0], preact=y)
    assert dx.shape == (0, 96) and not dw.any() and not db.any()


@pytest.mark.parametrize("M", [6, 40, 300])
def test_special_values_stay_in_their_rows_and_columns(M):
    import torch
    lin, w = _layer(200, 136, act="relu", bias="f32")
    x, r = _rand(M, 200, seed=3), _rand(M, 136, seed=4)
    clean = lin.forward(x, residual=r)
    x[1, 7], x[2, 0], r[3, 5], r[4, 9] = float("nan"), float("inf"), float("-inf"), float("nan")
    y = lin.forward(x, residual=r)
    assert bool(torch.isnan(y[1]).all())
    assert bool((torch.isinf(y[2]) | torch.isnan(y[2]) | (y[2] == r[2])).all())  # inf * w, or relu of -inf
    assert float(y[3, 5]) == float("-inf") and bool(torch.isnan(y[4, 9]))
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[1] = keep[2] = False
    keep[3, 5] = keep[4, 9] = False
    assert torch.equal(y[keep], clean[keep])


GRADS = [(1, 1, 1), (1, 64, 200), (5, 33, 65), (16, 512, 128), (64, 1024, 1024), (100, 1001, 130), (128, 2048, 72),
         (333, 520, 1037), (1000, 96, 2048), (2048, 1032, 768)]


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("M,K,N", GRADS)
def test_gradients_against_the_formulas(M, K, N, layout):
    import layer_bounds as lb
    import torch
    i = GRADS.index((M, K, N))
    act, bias, wdt = ACTS[(i + 2 * (layout == "nk")) % 5], ("f32", "bf16")[i % 2], ("bf16", "f32")[i // 2 % 2]
    lin, w = _layer(K, N, layout, act, bias, seed=10 * i)
    x, dy, z = _rand(M, K, seed=3), _rand(M, N, seed=4), _rand(M, N, seed=5, scale=2.0)
    got = lin.backward(dy, x, preact=z, dw_dtype=wdt)
    want = lb.linear_grads(x, w, z, act, dy, got[1].dtype, got[2].dtype)
    lb.check(got[0], *want[0], "dx")
    lb.check(got[1] if layout == "kn" else got[1].t(), *want[1], "dw")
    lb.check(got[2], *want[2], "db")
    again = lin.backward(dy, x, preact=z, dw_dtype=wdt)
    assert all(torch.equal(a, b) for a, b in zip(got, again)), "a second call differs"
    for k, need in enumerate(("need_dx", "need_dw", "need_db")):
        one = lin.backward(dy, x, preact=z, dw_dtype=wdt, **{n: n == need for n in ("need_dx", "need_dw", "need_db")})
        assert [g is not None for g in one] == [j == k for j in range(3)]
        alone = want[k][0] if not (k == 1 and layout == "nk") else want[1][0].t()
        lb.check(one[k], alone, want[k][1] if not (k == 1 and layout == "nk") else want[1][1].t(), need)
    assert lin.status() == 0


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(act):
    """<gradient, direction> against central differences of <dy, forward> in 64 bits."""
    import layer_bounds as lb
    import torch
    M, K, N = 20, 48, 40
    lin, w = _layer(K, N, "kn", act, "f32", seed=3)
    x, dy = _rand(M, K, seed=6), _rand(M, N, seed=7)
    # away from relu's corner, where a difference is no derivative
    z64 = x.double() @ w.double() + lin.bias.double()
    z = z64.to(torch.bfloat16)
    dx, dw, db = lin.backward(dy, x, preact=z, dw_dtype="f32")
    (_, ex), (_, ew), (_, eb) = lb.linear_grads(x, w, z, act, dy, torch.float32)
    # the stored pre-activation is rounded: its slope moves by at most 2 U |z| (second derivatives are below 2)
    ez = torch.zeros_like(z64) if act == "none" else 2 * lb.U * z64.abs() * dy.double().abs()
    if act == "relu":
        ez = torch.zeros_like(z64)
    ex, ew, eb = ex + ez @ w.t().double().abs(), ew + x.t().double().abs() @ ez, eb + ez.sum(0)
    g = torch.Generator("cuda")
    g.manual_seed(11)

    def loss(x_, w_, b_):
        return (dy.double() * lb.act(act, x_ @ w_ + b_)).sum()

    for grad, err, which in ((dx, ex, 0), (dw, ew, 1), (db, eb, 2)):
        at = [x.double(), w.double(), lin.bias.double()]
        for _ in range(4):
            v = torch.empty_like(at[which]).normal_(generator=g)
            h = 1e-6
            up, down = list(at), list(at)
            up[which], down[which] = at[which] + h * v, at[which] - h * v
            diff = float((loss(*up) - loss(*down)) / (2 * h))
            tol = float((err * v.abs()).sum()) + 1e-4 * float((grad.double().abs() * v.abs()).sum())
            assert abs(float((grad.double() * v).sum()) - diff) <= tol


def test_gradients_of_extreme_preactivations():
    import torch
    z = torch.tensor([[-3e38, -1e20, -200.0, -30.0, 0.0, 30.0, 200.0, 1e20, 3e38]], device="cuda").bfloat16()
    dy = torch.ones_like(z)
    for act in ("gelu", "gelu_tanh", "silu", "relu"):
        lin, _ = _layer(8, 9, act=act, bias="f32")
        _, _, db = lin.backward(dy, _rand(1, 8, seed=1), preact=z)
        want = torch.tensor([0, 0, 0, 0, 0.0 if act == "relu" else 0.5, 1, 1, 1, 1.0], device="cuda")
        assert float((db - want).abs().max()) < 1e-6, (act, db)
        _, _, db = lin.backward(dy, _rand(1, 8, seed=1), preact=torch.full_like(z, float("nan")))
        assert act == "relu" or bool(torch.isnan(db).all())


def test_another_stream_two_streams_in_turn_and_a_graph():
    import torch
    lin, _ = _layer(1001, 333, act="silu", bias="f32")  # odd rows: the scratch is used by every call
    x, dy = _rand(200, 1001, seed=3), _rand(200, 333, seed=4)
    y, z = lin.forward(x, save_preact=True)
    want = lin.backward(dy, x, preact=z)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append((lin.forward(x), lin.backward(dy, x, preact=z)))
    torch.cuda.synchronize()
    for y2, g2 in outs:
        assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(want, g2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg = lin.forward(x)
        gg = lin.backward(dy, x, preact=z)
    for _ in range(3):
        yg.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, yg) and all(torch.equal(a, b) for a, b in zip(want, gg))
    # scratch cannot grow inside a capture
    import apk_b200
    from apk_b200 import _lib as L
    lin2, _ = _layer(1001, 333, act="silu")
    with pytest.raises(apk_b200.ApkError) as e:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            lin2.forward(x)
    assert e.value.status == L.APK_ESTATE
    torch.cuda.synchronize()
    assert lin2.forward(x).shape == (200, 333)


def test_weights_updated_in_place_are_seen():
    import torch
    lin, w = _layer(128, 64, bias="f32")
    x = _rand(30, 128, seed=3)
    y = lin.forward(x)
    w.mul_(2)
    lin.bias.mul_(2)
    assert torch.equal(lin.forward(x), (y.float() * 2).bfloat16())


def test_fewer_sms_give_the_same_values():
    import torch
    import layer_bounds as lb
    for sms in (1, 2, 7, 100):
        lin, w = _layer(520, 700, act="silu", sms=sms)
        x = _rand(400, 520, seed=3)
        want, by, _, _ = lb.linear(x, w, lin.bias, "silu", None, torch.bfloat16)
        lb.check(lin.forward(x), want, by, f"{sms} SMs")


def test_refusals():
    import torch

    import apk_b200
    from apk_b200 import _lib as L
    w = _rand(64, 32, seed=1)
    for bad in (w.float(), w.cpu(), w[0], w.t(), "w"):
        with pytest.raises(ValueError):
            apk_b200.Linear(bad)
    for kw in (dict(act="tanh"), dict(layout="mn"), dict(out_dtype="f16"), dict(bias=w[0, :31]),
               dict(bias=w[0].half()), dict(bias=w[:, 0][:32])):
        with pytest.raises(ValueError):
            apk_b200.Linear(w, **kw)
    with pytest.raises(apk_b200.ApkError) as e:
        apk_b200.Linear(w, sms=10_000)
    assert e.value.status == L.APK_EINVAL
    lin = apk_b200.Linear(w, act="silu")
    x = _rand(4, 64, seed=2)
    for bad in (x[:, :63], x.float(), x.cpu(), _rand(64, 4, seed=3).t()):
        with pytest.raises(ValueError):
            lin.forward(bad)
    for kw in (dict(residual=x), dict(residual=_rand(4, 32, seed=3).half()),
               dict(out=torch.empty(4, 32, device="cuda")), dict(out=torch.empty(3, 32, device="cuda").bfloat16())):
        with pytest.raises(ValueError):
            lin.forward(x, **kw)
    y = lin.forward(x)
    with pytest.raises(ValueError):
        lin.backward(y, x)                          # no pre-activation
    with pytest.raises(ValueError):
        lin.backward(y[:3], x, preact=y)
    with pytest.raises(apk_b200.ApkError) as e:     # rows that lie on one another
        lin.forward(x[:1].expand(4, 64))
    assert e.value.status == L.APK_EINVAL
    assert torch.equal(lin.forward(x), y)           # still usable


def test_c_entry_refuses_what_python_cannot_send():
    import torch

    import apk_b200
    from apk_b200 import _lib as L
    lin, _ = _layer(64, 32, act="silu", bias=None)
    x, y = _rand(4, 64, seed=1), torch.empty(4, 32, device="cuda").bfloat16()
    f, b, lib = lin._lib.apk_linear_forward, lin._lib.apk_linear_backward, lin._lib
    good = dict(x=x.data_ptr(), ldx=64, rows=4, y=y.data_ptr(), ldy=32, y_dtype=L.APK_BF16)
    assert f(lin._h, ctypes.byref(L.LinearIO(**good))) == L.APK_OK
    for bad in (dict(rows=-1), dict(x=None), dict(y=None), dict(ldx=63), dict(ldy=31), dict(y_dtype=2),
                dict(x=x.data_ptr() + 1), dict(y=y.data_ptr() + 1), dict(residual=y.data_ptr(), ld_residual=32,
                                                                        residual_dtype=9)):
        assert f(lin._h, ctypes.byref(L.LinearIO(**{**good, **bad}))) == L.APK_EINVAL, bad
        assert lib.apk_linear_last_error(lin._h)
    dx = torch.empty_like(x)
    good = dict(dy=y.data_ptr(), ld_dy=32, x=x.data_ptr(), ldx=64, preact=y.data_ptr(), ld_preact=32, rows=4,
                dx=dx.data_ptr(), ld_dx=64)
    assert b(lin._h, ctypes.byref(L.LinearGrads(**good))) == L.APK_OK
    for bad in (dict(dx=None), dict(db=dx.data_ptr()), dict(preact=None), dict(dy=None), dict(ld_dx=1),
                dict(dw=dx.data_ptr(), ld_dw=1), dict(dw=dx.data_ptr(), ld_dw=32, dw_dtype=5)):
        assert b(lin._h, ctypes.byref(L.LinearGrads(**{**good, **bad}))) == L.APK_EINVAL, bad
    assert f(None, None) == L.APK_EINVAL and b(lin._h, None) == L.APK_EINVAL
    torch.cuda.synchronize()
    assert lin.status() == 0


def test_a_graph_keeps_its_scratch_when_it_grows():
    import torch
    lin, _ = _layer(1001, 333, act="silu", bias="f32")
    x, dy = _rand(40, 1001, seed=3), _rand(40, 333, seed=4)
    y, z = lin.forward(x, save_preact=True)
    want = lin.backward(dy, x, preact=z)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg = lin.forward(x)
        gg = lin.backward(dy, x, preact=z)
    big, dbig = _rand(900, 1001, seed=5), _rand(900, 333, seed=6)
    for _ in range(3):
        lin.backward(dbig, big, preact=lin.forward(big, save_preact=True)[1])
        filler = torch.full((1 << 22,), -1, dtype=torch.int32, device="cuda")  # would reuse freed memory
        yg.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(yg, y) and all(torch.equal(a, b) for a, b in zip(gg, want))
        assert bool((filler == -1).all())


def test_threads_share_a_layer():
    import threading

    import torch
    lin, _ = _layer(264, 136, act="gelu", bias="bf16")
    xs = [_rand(10 + 30 * i, 264, seed=i) for i in range(4)]
    want = [lin.forward(x) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(200):
                y = lin.forward(xs[i])
            torch.cuda.current_stream().synchronize()
            if not torch.equal(y, want[i]):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and lin.status() == 0


def test_no_rows_one_gradient_at_a_time():
    lin, _ = _layer(16, 8, bias="f32")
    x, dy = _rand(0, 16, seed=1), _rand(0, 8, seed=2)
    for need in ("need_dx", "need_dw", "need_db"):
        got = lin.backward(dy, x, **{n: n == need for n in ("need_dx", "need_dw", "need_db")})
        assert [g is not None for g in got] == [n == need for n in ("need_dx", "need_dw", "need_db")]
        assert not any(bool(g.any()) for g in got if g is not None)
