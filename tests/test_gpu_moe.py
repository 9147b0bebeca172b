"""The mixture-of-experts layer on a B200 against 64 bits, element by element,
with bounds derived from the arithmetic (layer_bounds.py)."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(libapk):
    return libapk


def _rand(*shape, seed, scale=1.0):
    import torch
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0.0, scale, generator=g)


def _layer(E, k, D, F, act="silu", gated=True, renorm=True, out="bf16", seed=0, router=None, **kw):
    import apk_b200
    return apk_b200.MoE(_rand(E, D, seed=seed + 1, scale=D ** -0.5) if router is None else router,
                        _rand(E, 2 * F if gated else F, D, seed=seed + 2, scale=D ** -0.5),
                        _rand(E, D, F, seed=seed + 3, scale=F ** -0.5), top_k=k, act=act, gated=gated,
                        renormalize=renorm, out_dtype=out, **kw)


def _check(moe, x, act, gated, renorm):
    """The choice must be a top_k one within the logits' error; values follow from that choice."""
    import layer_bounds as lb
    import torch
    y, ids, probs = moe.forward(x, return_routing=True)
    assert torch.equal(y, moe.forward(x)), "a second call differs"
    assert moe.status() == 0
    want, ey, p, rel, logits, el = lb.moe(x, moe.router, moe.w_in, moe.w_out, ids.long(), act, gated, renorm)
    assert all(len(set(row)) == moe.top_k for row in ids.tolist())
    chosen = logits.gather(1, ids.long())
    kth = logits.topk(moe.top_k, 1).values
    slack = 2 * el.amax(1, keepdim=True)
    assert bool(((chosen - kth).abs() <= slack).all()), "not the largest logits, or not in their order"
    lb.check(probs, p, (rel + 2.0 ** -20) * p + lb.TINY, "weights")
    lb.check(y, want, lb.rounded(want, ey, y.dtype), "y")


CASES = [  # T, E, k, D, F, act, gated, renorm
    (1, 1, 1, 8, 8, "none", True, True), (1, 8, 2, 1024, 2048, "silu", True, True), (1, 7, 7, 264, 72, "gelu", False, False),
    (1, 512, 16, 136, 1000, "silu", True, True), (2, 4, 1, 7168, 8, "relu", False, True),
    (3, 60, 4, 1032, 520, "gelu_tanh", True, False), (5, 64, 6, 512, 1408, "silu", True, False),
    (8, 3, 2, 64, 128, "gelu", True, True), (9, 16, 3, 2048, 136, "silu", False, True), (16, 128, 8, 512, 256, "silu", True, True),
    (17, 33, 5, 200, 264, "gelu", True, False), (31, 256, 8, 256, 64, "relu", True, True),
    (33, 5, 1, 520, 1000, "silu", False, False), (48, 20, 12, 128, 96, "gelu_tanh", True, True),
    (64, 1, 1, 256, 512, "silu", True, True), (64, 8, 8, 136, 72, "silu", True, True), (64, 128, 8, 1024, 256, "silu", True, True),
    (64, 512, 16, 64, 16, "gelu", False, True)]


@pytest.mark.parametrize("T,E,k,D,F,act,gated,renorm", CASES)
def test_layer(T, E, k, D, F, act, gated, renorm):
    moe = _layer(E, k, D, F, act, gated, renorm, out="f32" if T % 2 else "bf16", seed=T)
    _check(moe, _rand(T, D, seed=99), act, gated, renorm)


def test_ties_go_to_the_lowest_index_and_tokens_crowd_one_expert():
    import torch
    E, k, D, F = 40, 3, 64, 32
    router = torch.zeros(E, D, device="cuda").bfloat16()
    for T in (1, 10, 64):
        x = _rand(T, D, seed=5)
        moe = _layer(E, k, D, F, router=router)
        _, ids, probs = moe.forward(x, return_routing=True)
        assert ids.tolist() == [[0, 1, 2]] * T
        assert float((probs - 1 / 3).abs().max()) < 1e-6
        _check(moe, x, "silu", True, True)
    router[17] = 1.0                                 # one expert above or below all others, the rest tied
    x = torch.ones(64, D, device="cuda").bfloat16()
    x[::2] = -1.0
    _, ids, _ = _layer(E, k, D, F, router=router).forward(x, return_routing=True)
    assert ids.tolist() == [[0, 1, 2], [17, 0, 1]] * 32


def test_special_values_stay_with_their_tokens():
    import torch
    for T in (4, 20, 64):
        moe = _layer(16, 4, 128, 64)
        x = _rand(T, 128, seed=3)
        clean = moe.forward(x)
        x[1, 5], x[2, 9] = float("nan"), float("inf")
        y, ids, _ = moe.forward(x, return_routing=True)
        assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[2]).all())
        assert all(len(set(r)) == 4 and min(r) >= 0 and max(r) < 16 for r in ids.tolist())
        keep = [t for t in range(T) if t not in (1, 2)]
        assert torch.equal(y[keep], clean[keep])
        assert moe.status() == 0
    # an expert that no token chooses may hold anything
    router = torch.zeros(4, 128, device="cuda").bfloat16()
    for T in (1, 30):
        moe = _layer(4, 2, 128, 64, router=router)
        clean = moe.forward(_rand(T, 128, seed=3))
        moe.w_in[2:].fill_(float("nan"))
        moe.w_out[2:].fill_(float("inf"))
        assert torch.equal(moe.forward(_rand(T, 128, seed=3)), clean)


def test_views_axes_streams_and_a_graph():
    import torch
    moe = _layer(32, 4, 256, 128)
    x = _rand(24, 256, seed=3)
    y = moe.forward(x)
    wide = torch.zeros(24, 520, device="cuda").bfloat16()
    wide[:, 8:264] = x
    assert torch.equal(moe.forward(wide[:, 8:264]), y)
    assert torch.equal(moe.forward(x.reshape(2, 3, 4, 256)).reshape(24, 256), y)
    assert moe.forward(x[:0]).shape == (0, 256)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(moe.forward(x))
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg = moe.forward(x)
    for _ in range(3):
        yg.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(yg, y) and torch.equal(moe.forward(x), y)


@pytest.mark.parametrize("sms", [1, 3, 40])
def test_fewer_sms(sms):
    for T in (1, 7, 40):
        moe = _layer(12, 3, 264, 136, sms=sms)
        _check(moe, _rand(T, 264, seed=3), "silu", True, True)


def test_refusals():
    import torch

    import apk_b200
    from apk_b200 import _lib as L
    r, wi, wo = _rand(4, 64, seed=1), _rand(4, 64, 64, seed=2), _rand(4, 64, 32, seed=3)
    make = lambda *a, **kw: apk_b200.MoE(*a, **{"top_k": 2, **kw})  # noqa: E731
    for a in ((r.float(), wi, wo), (r, wi.cpu(), wo), (r[:3], wi, wo), (r, wi[:, :63], wo), (r, wo, wi),
              (r, wi.transpose(1, 2), wo)):
        with pytest.raises(ValueError):
            make(*a)
    for kw in (dict(act="x"), dict(out_dtype="f64"), dict(gated=False)):
        with pytest.raises(ValueError):
            make(r, wi, wo, **kw)
    for kw in (dict(top_k=0), dict(top_k=5), dict(sms=10_000)):
        with pytest.raises(apk_b200.ApkError) as e:
            make(r, wi, wo, **kw)
        assert e.value.status == L.APK_EINVAL
    odd = _rand(4, 60, seed=1), _rand(4, 64, 60, seed=2), _rand(4, 60, 32, seed=3)
    with pytest.raises(apk_b200.ApkError):           # d_model not a multiple of 8
        make(*odd)
    moe = make(r, wi, wo)
    x = _rand(65, 64, seed=4)
    for bad in (x, x.float()[:2], x[:2, :63], x[:2].cpu()):
        with pytest.raises((ValueError, apk_b200.ApkError)):
            moe.forward(bad)
    off = _rand(2, 80, seed=4)[:, 1:65]              # rows off the 16-byte grid
    with pytest.raises(apk_b200.ApkError) as e:
        moe.forward(off)
    assert e.value.status == L.APK_EINVAL
    y = moe.forward(x[:2])
    io = dict(x=x.data_ptr(), ldx=64, tokens=2, y=y.data_ptr(), ldy=64, y_dtype=L.APK_BF16)
    f = moe._lib.apk_moe_forward
    for bad in (dict(tokens=-1), dict(x=None), dict(y=None), dict(ldx=63), dict(ldy=63), dict(y_dtype=7), dict(ldx=65),
                dict(ids=y.data_ptr() + 2), dict(y=y.data_ptr() + 1)):
        assert f(moe._h, ctypes.byref(L.MoeIO(**{**io, **bad}))) == L.APK_EINVAL, bad
    assert f(None, None) == L.APK_EINVAL
    torch.cuda.synchronize()
    assert torch.equal(moe.forward(x[:2]), y) and moe.status() == 0
