"""Log probabilities, entropies, alternatives and their gradient on a B200
against 64 bits, element by element.

Bounds, with E = 2^-24 the unit roundoff of fp32, d = x - m, p = exp(l), and
D1, D2 the sums of p |d| and p d^2: an exponential is off by 3 E |d| + 4 E of
itself (the difference, its product with log2(e), and that constant; the
hardware's 2^x 4 E); a thread adds at most V / 256 + 8 of them, 16 more
additions join threads, warps and parts, and a running sum is scaled at most
once in a round of 2048, which costs 6 E (4 E, and 3 E |Delta| of a part that
is exp(-Delta) of the sum).  The sums are taken against a reference that may be
2 below the maximum: there the terms p d, and with them what additions round,
are up to p (|d| + 2), in all D1 + 2."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


@pytest.fixture(autouse=True)
def _lib(libapk):
    return libapk


def _rand(*shape, seed, scale=1.0, dtype="f32"):
    import torch
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return torch.empty(shape, dtype={"bf16": torch.bfloat16, "f32": torch.float32}[dtype], device="cuda").normal_(0.0, scale, generator=g)


def _tokens(M, V, seed, dtype=None):
    import torch
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return torch.randint(0, V, (M,), device="cuda", generator=g, dtype=dtype or torch.int64)


def _reference(x):
    """m, l, p, H and the bounds of log S and H, for finite maxima."""
    import torch
    x = x.double()
    V = x.shape[-1]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = d.exp()
    s = e.sum(-1, keepdim=True)
    l, p = d - s.log(), e / s
    pd = torch.where(p > 0, p * d, 0.0)
    d1, d2 = -pd.sum(-1), torch.where(p > 0, pd * d, 0.0).sum(-1)
    h = s.log()[..., 0] + d1
    adds = V / 256 + 24 + 6 * (V / 2048 + 2)
    rel = E * (adds + 4 + 3 * d1)
    els = rel + 2 * E * s.log()[..., 0] + 1e-30
    eh = els + E * (3 * (d2 + 2 * d1) + (adds + 6) * (d1 + 2)) + d1 * (rel + 2 * E) + E * h.abs()
    return m, l, p, h, els, eh


def _check(x, tokens=None, top=0):
    import layer_bounds as lb
    import torch

    import apk_b200
    lp = apk_b200.LogProbs(top=top)
    logprob, entropy, ids, tops, stats = lp.forward(x, tokens, save_stats=True)
    m, l, p, h, els, eh = _reference(x)
    lb.check(entropy, h, eh, "entropy")
    lb.check(stats[..., :1], m, torch.zeros_like(m), "m")
    lb.check(stats[..., 1], (x.double() - m).exp().sum(-1).log(), els, "log S")
    d = (x.double() - m)

    def bound(at):
        want, dist = l.gather(-1, at), d.gather(-1, at).abs()
        err = E * dist + els[..., None] + E * want.abs()
        return want, torch.where(want.isinf(), 0.0, err)

    if tokens is not None:
        want, err = bound(tokens.long().clamp(0, x.shape[-1] - 1)[..., None])
        assert torch.equal(logprob[tokens < 0], torch.zeros_like(logprob[tokens < 0]))
        real = (tokens >= 0) & ~want[..., 0].isinf()
        lb.check(logprob[real], want[..., 0][real], err[..., 0][real], "logprob")
        gone = (tokens >= 0) & want[..., 0].isinf()
        assert bool((logprob[gone] == -math.inf).all())
    else:
        assert logprob is None
    if top:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top]
        assert torch.equal(ids, order.int()), "ids"
        want, err = bound(order)
        fine = ~want.isinf()
        lb.check(tops[fine], want[fine], err[fine], "tops")
        assert bool((tops[~fine] == -math.inf).all())
    else:
        assert ids is None and tops is None
    again = lp.forward(x, tokens, save_stats=True)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(again, (logprob, entropy, ids, tops, stats)))
    return stats, entropy


def _check_grad(x, tokens, stats, entropy, dlp, dh):
    import layer_bounds as lb
    import torch

    import apk_b200
    got = apk_b200.LogProbs().backward(dlp, x, tokens, stats, dentropy=dh, entropy=entropy if dh is not None else None)
    st = stats.double()
    d = x.double() - st[..., :1]
    l = d - st[..., 1:]
    p = l.exp()
    a = torch.zeros_like(entropy).double() if dlp is None else torch.where(tokens < 0, 0.0, dlp.double())
    hot = torch.zeros_like(p)
    if dlp is not None:
        hot.scatter_(-1, tokens.long().clamp(min=0)[..., None], (tokens >= 0).double()[..., None])
    a, g = a[..., None], (0.0 if dh is None else dh.double()[..., None])
    H = entropy.double()[..., None]
    inner = torch.where(p > 0, a + g * (l + H), 0.0)
    want = a * hot - p * inner
    lf = torch.where(p > 0, l, 0.0).abs()
    el = E * torch.where(p > 0, d, 0.0).abs() + E * lf
    size = abs(a) + abs(g) * (lf + H.abs())
    err = p * size * (el + 2 * E * lf + 4 * E) + p * (abs(g) * el + 4 * E * size) + 3 * E * abs(a) * hot
    # an exponential below 2^-126, the least normal value, is 0: what it was a factor of is lost
    err = err + 2.0 ** -126 * size
    u = 2.0 ** -8 if x.dtype == torch.bfloat16 else E
    lb.check(got, want, err + u * (want.abs() + err) + 2.0 ** -120, "dlogits")
    return got


VOCABULARIES = [1, 2, 7, 33, 255, 2040, 2048, 2049, 4096, 4111, 8192, 10007, 32768, 100003, 131072]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", VOCABULARIES)
def test_sizes(V, dtype):
    import torch
    for M, top, scale in ((1, 20, 3.0), (3, 5, 1.0), (37, 1, 10.0), (150, 32, 3.0), (301, 0, 2.0)):
        if M * V > 2.1e7:
            continue
        x = _rand(M, V, seed=V + M, scale=scale, dtype=dtype)
        tokens = _tokens(M, V, M, torch.int32 if M == 3 else torch.int64)
        tokens[M // 2::5] = -100
        stats, entropy = _check(x, tokens, min(top, V))
        _check_grad(x, tokens, stats, entropy, _rand(M, seed=1), _rand(M, seed=2, scale=0.1))


def test_many_rows_and_every_top():
    for top in range(33):
        _check(_rand(200, 997 + 101 * top, seed=top, scale=4.0, dtype="bf16"), _tokens(200, 997, top), top)


@pytest.mark.parametrize("M,V", [(1, 131072), (2, 50000), (160, 30011), (3, 2047)])
def test_orders_and_ties(M, V):
    """Rows in which everything, or nothing, passes the running bound; equal values go to the lowest index."""
    import torch
    up = torch.arange(V, device="cuda").float().expand(M, V) * (16.0 / V)
    half = up.clone()
    half[:, :V // 2] = 0.0
    steps = (up * 2).floor()
    few = torch.zeros(M, V, device="cuda")
    few[:, V - 5:] = 1.0
    waves = (up * 200).sin()
    for x in (up.contiguous(), up.flip(1), half, torch.zeros(M, V, device="cuda"), steps, steps.flip(1), few, waves):
        for top in (1, 20, 32):
            _check(x.contiguous(), _tokens(M, V, 1), top)
            _check(x.bfloat16().contiguous(), _tokens(M, V, 1), top)


def test_few_allowed_tokens():
    """Rows in which fewer values than alternatives are not masked, as constrained decoding leaves them."""
    import torch
    for V in (300, 5000, 20000, 131072):
        for left in (1, 2, 7):
            x = torch.full((4, V), -math.inf, device="cuda")
            at = torch.randperm(V, device="cuda", generator=torch.Generator("cuda").manual_seed(V))[:left]
            x[:, at] = _rand(4, left, seed=left)
            t = at[:1].expand(4).contiguous()
            for top in (1, 5, 32):
                _check(x, t, top)
                _check(x.bfloat16(), t, top)


def test_masked_logits():
    """-inf, and a type's lowest value, as masks: few values left, at either end, one, and many."""
    import torch
    for dtype in ("f32", "bf16"):
        for V in (40, 5000, 70001):
            x = _rand(6, V, seed=V, dtype=dtype)
            for fill in (-math.inf, torch.finfo(x.dtype).min):
                y = x.clone()
                y[0, 7:] = fill                      # the first ones are left
                y[1, :V - 9] = fill                  # the last ones
                y[2, :] = fill
                y[2, V // 2] = -50.0                 # one
                y[3, ::2] = fill
                y[4, V // 3:] = fill
                t = torch.tensor([3, V - 2, V // 2, 1, 0, 5], device="cuda")
                stats, entropy = _check(y, t, 20)
                g = _check_grad(y, t, stats, entropy, _rand(6, seed=1), _rand(6, seed=2))
                assert not g[0, 7:].any() and not g[1, :V - 9].any()
                _check(y, torch.tensor([20, 0, 0, 0, V - 1, 5], device="cuda"), 1)    # masked tokens
            y = torch.full((3, V), torch.finfo(x.dtype).min, dtype=x.dtype, device="cuda")    # even: all the same
            _check(y, _tokens(3, V, 1), 5)


def test_rows_with_nothing_left_nan_and_infinity():
    import torch

    import apk_b200
    for V in (33, 9000, 70001):
        x = _rand(8, V, seed=V)
        lp = apk_b200.LogProbs(top=4)
        t = torch.tensor([1, 2, -1, 3, 4, 5, V, 7], device="cuda")
        want = lp.forward(x, t, save_stats=True)
        y = x.clone()
        y[1], y[2] = -math.inf, -math.inf
        y[3, 17], y[5, 20], y[4, 30] = math.nan, math.inf, -math.nan
        got = lp.forward(y, t, save_stats=True)
        bad = torch.tensor([1, 3, 4, 5], device="cuda")
        assert got[0][bad].isnan().all() and float(got[0][2]) == 0.0 and math.isnan(float(got[0][6]))
        assert got[1][[1, 2, 3, 4, 5]].isnan().all() and got[3][[1, 2, 3, 4, 5]].isnan().all()
        assert got[2][1].tolist() == [0, 1, 2, 3] and int(got[2][3, 0]) == 17 and int(got[2][4, 0]) == 30 and int(got[2][5, 0]) == 20
        for g, w in zip(got, want):
            assert torch.equal(g[[0, 7]], w[[0, 7]])
        # their gradients: NaN where a coefficient is not 0, zeros where all are
        ones = torch.ones(8, device="cuda")
        d = lp.backward(ones, y, t, got[4])
        assert d[[1, 3, 4, 5, 6]].isnan().all(1).all() and not d[2].any() and torch.isfinite(d[[0, 7]]).all()
        assert not lp.backward(0 * ones, y, torch.zeros_like(t), got[4], dentropy=0 * ones, entropy=got[1]).any()


def test_logits_far_from_zero():
    for shift in (-3e4, 1e4, -9.9e7, -1.3e8, 9.9e7, 1.5e8, 3e20, -1e30):
        x = _rand(5, 30000, seed=1, scale=2.0) * max(1.0, abs(shift) * 1e-7) + shift
        stats, entropy = _check(x, _tokens(5, 30000, 2), 8)
        _check_grad(x, _tokens(5, 30000, 2), stats, entropy, _rand(5, seed=3), _rand(5, seed=4))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_rows_and_gradients_in_place(dtype):
    """Rows inside wider ones, and gradients over them: bitwise as of copies, nothing written beside."""
    import torch

    import apk_b200
    lp = apk_b200.LogProbs(top=3)
    for V, ld, at in ((1000, 1003, 1), (5001, 5008, 5), (4096, 4104, 8)):
        wide = _rand(9, ld, seed=V, scale=2.0, dtype=dtype)
        x, t = wide[:, at:at + V], _tokens(9, V, 1)
        a, b = lp.forward(x, t, True), lp.forward(x.contiguous(), t, True)
        assert torch.equal(a[2], b[2])
        stats, entropy = _check(x, t, 3)
        dlp, dh = _rand(9, seed=2), _rand(9, seed=3)
        want = _check_grad(x, t, stats, entropy, dlp, dh)
        room = _rand(9, ld + 3, seed=5, dtype=dtype)
        for to in (0, 1, 3):
            kept = room.clone()
            lp.backward(dlp, x, t, stats, dentropy=dh, entropy=entropy, out=room[:, to:to + V])
            kept[:, to:to + V] = want
            assert torch.equal(room, kept)
        kept = wide.clone()
        kept[:, at:at + V] = want
        assert lp.backward(dlp, x, t, stats, dentropy=dh, entropy=entropy, out=x).data_ptr() == x.data_ptr()
        assert torch.equal(wide, kept)


def test_leading_axes_parts_and_no_rows():
    import torch

    import apk_b200
    x, t = _rand(2, 3, 500, seed=1, dtype="bf16"), _tokens(6, 500, 1).view(2, 3)
    stats, entropy = _check(x, t, 4)
    _check(x[0, 0], t[0, 0], 2)                        # one row without leading axes
    _check(x, None, 4)
    dlp, dh = _rand(2, 3, seed=2), _rand(2, 3, seed=3)
    _check_grad(x, t, stats, entropy, dlp, dh)
    _check_grad(x, t, stats, entropy, dlp, None)
    _check_grad(x, None, stats, entropy, None, dh)
    lp = apk_b200.LogProbs(top=4)
    e = lp.forward(x[:0], t[:0], True)
    assert [tuple(v.shape) for v in e] == [(0, 3), (0, 3), (0, 3, 4), (0, 3, 4), (0, 3, 2)]
    assert lp.backward(dlp[:0], x[:0], t[:0], e[4]).shape == (0, 3, 500)


def test_gradient_against_differences():
    """Against central differences of the definition in 64 bits (step 1e-5: truncation about 1e-9 of the values)."""
    import torch

    import apk_b200
    x, t = _rand(7, 300, seed=1, scale=2.0), _tokens(7, 300, 1)
    dlp, dh = _rand(7, seed=2), _rand(7, seed=3)
    lp = apk_b200.LogProbs()
    _, entropy, _, _, stats = lp.forward(x, t, True)
    got = lp.backward(dlp, x, t, stats, dentropy=dh, entropy=entropy).double()

    def loss(x):
        l = x - x.logsumexp(1, keepdim=True)
        return (dlp.double() * l.gather(1, t[:, None])[:, 0]).sum() - (dh.double() * (l.exp() * l).sum(1)).sum()

    for k in range(8):
        v = _rand(7, 300, seed=10 + k).double()
        want = float((loss(x.double() + 1e-5 * v) - loss(x.double() - 1e-5 * v)) / 2e-5)
        # elements are off by a few tens of E of p (|a| + |h| (|l| + H)): summed over rows, of these sizes
        size = float((dlp.double().abs() + 20 * dh.double().abs()).sum()) * float(v.abs().max())
        assert abs(float((got * v).sum()) - want) <= 100 * E * size + 1e-7 * size


def test_streams_and_graphs():
    import torch

    import apk_b200
    lp = apk_b200.LogProbs(top=20)
    xs = [_rand(2, 60000, seed=i, scale=3.0) for i in range(4)]
    t = _tokens(2, 60000, 1)
    one = torch.ones(2, device="cuda")

    def f(x):
        a = lp.forward(x, t, True)
        return (*a, lp.backward(one, x, t, a[4], dentropy=one, entropy=a[1]))

    want = [f(x) for x in xs]
    torch.cuda.synchronize()
    side, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i in range(4):
        with torch.cuda.stream(side[i % 2]):
            got.append(f(xs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for a, b in zip(got, want) for p, q in zip(a, b))
    graphs = []
    for _ in range(2):
        x = xs[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f(x)
        graphs.append((x, graph, out))
    for i, j in ((1, 2), (3, 0), (2, 2)):
        graphs[0][0].copy_(xs[i])
        graphs[1][0].copy_(xs[j])
        torch.cuda.synchronize()
        with torch.cuda.stream(side[0]):
            graphs[0][1].replay()
        with torch.cuda.stream(side[1]):
            graphs[1][1].replay()
        again = f(xs[3])
        torch.cuda.synchronize()
        for out, w in ((graphs[0][2], want[i]), (graphs[1][2], want[j]), (again, want[3])):
            assert all(torch.equal(p, q) for p, q in zip(out, w))


def test_refusals():
    import torch

    import apk_b200
    from apk_b200 import _lib as L
    lp = apk_b200.LogProbs(top=5)
    x, t = _rand(6, 64, seed=1), _tokens(6, 64, 1)
    _, entropy, _, _, stats = lp.forward(x, t, True)
    for bad in (x.double(), x.cpu(), x[:, :4], x.t(), x[:, ::2], 3.0):
        with pytest.raises(ValueError):
            lp.forward(bad, t)
    for bad in (t[:5], t.cpu(), t.float(), t[:, None], t.repeat(2)[::2], x):
        with pytest.raises(ValueError):
            lp.forward(x, bad)
    one = torch.ones(6, device="cuda")
    good = dict(dlogprob=one, logits=x, tokens=t, stats=stats)
    for bad in (dict(dlogprob=None), dict(dlogprob=one.double()), dict(dlogprob=one[:1].expand(6)), dict(tokens=None),
                dict(stats=stats[:5]), dict(stats=None), dict(dentropy=one), dict(dentropy=one, entropy=entropy[:3]),
                dict(out=x.bfloat16()), dict(out=x[:5]), dict(out=3)):
        with pytest.raises(ValueError):
            lp.backward(**{**good, **bad})
    flat = _rand(400, seed=2)
    with pytest.raises(ValueError, match="shares memory"):
        lp.backward(**{**good, "logits": flat[:384].view(6, 64), "out": flat[8:392].view(6, 64)})
    p = x.data_ptr()
    for bad in (dict(rows=-1), dict(rows=(1 << 30) + 1), dict(vocabulary=0), dict(vocabulary=4), dict(vocabulary=(1 << 30) + 1),
                dict(dtype=2), dict(ld=63), dict(logits=None), dict(logits=p + 2), dict(top_ids=None), dict(top_logprobs=None),
                dict(tokens=None), dict(tokens=p + 4), dict(logprob=p + 1), dict(entropy=p + 2), dict(stats=p + 4)):
        a = L.LogprobsIO(**{**dict(logits=p, ld=64, rows=1, vocabulary=64, dtype=0, tokens_64=1, tokens=t.data_ptr(), logprob=p,
                                   entropy=p, top_ids=p, top_logprobs=p), **bad})
        assert lp._lib.apk_logprobs_forward(lp._h, ctypes.byref(a)) == L.APK_EINVAL and lp._lib.apk_logprobs_last_error(lp._h)
    for bad in (dict(rows=-1), dict(vocabulary=0), dict(ld=3), dict(ld_d=63), dict(dlogits=None), dict(stats=None), dict(dlogprob=None),
                dict(tokens=None), dict(dentropy=p), dict(dlogits=p + 1), dict(rows=1 << 30, vocabulary=1 << 30, ld=1 << 30, ld_d=1 << 30)):
        a = L.LogprobsGrads(**{**dict(logits=p, ld=64, rows=1, vocabulary=64, dtype=0, tokens_64=1, tokens=t.data_ptr(), dlogprob=p,
                                      stats=p, dlogits=p, ld_d=64), **bad})
        assert lp._lib.apk_logprobs_backward(lp._h, ctypes.byref(a)) == L.APK_EINVAL and lp._lib.apk_logprobs_last_error(lp._h)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [33, 300, 1000, 2041, 5000])
def test_more_equal_values_than_a_short_row_keeps(V, dtype):
    """Rows of equal values, of NaN, and with a NaN at the first place, at the
    last and between: NaN by index, then values by size and index."""
    import torch

    import apk_b200
    nan = math.nan
    x = torch.zeros(7, V, device="cuda")
    x[1] = nan
    x[2, 0] = nan
    x[3, 0], x[3, V // 2], x[3, V - 1] = nan, nan, nan
    x[4] = torch.arange(V, device="cuda") * 0.25 - 5.0
    x[5, 1:] = nan
    x[6] = -math.inf
    x[6, 0] = nan
    x = x.to({"bf16": torch.bfloat16, "f32": torch.float32}[dtype])
    order = torch.sort(x, dim=1, descending=True, stable=True).indices  # (a NaN is the largest there too)
    for top in (1, 5, 20, 27, 32):
        _, entropy, ids, tops = apk_b200.LogProbs(top=top).forward(x)
        assert torch.equal(ids, order[:, :top].int()), top
        assert tops[[1, 2, 3, 5, 6]].isnan().all() and entropy[[1, 2, 3, 5, 6]].isnan().all()
        _check(x[[0, 4]], _tokens(2, V, 1), top)


@pytest.mark.parametrize("V", [300, 5000, 20001])
def test_gradient_of_tokens_outside_the_vocabulary(V):
    """Their log probability is NaN, and so is the gradient by it; where that counts nothing, the row gets zeros, or
    the entropy's gradient alone."""
    import torch

    import apk_b200
    lp = apk_b200.LogProbs()
    x = _rand(6, V, seed=1, dtype="bf16")
    t = torch.tensor([1, V, V + 7, 3, -1, V], device="cuda")
    logprob, entropy, _, _, stats = lp.forward(x, t, True)
    assert logprob.isnan().tolist() == [False, True, True, False, False, True]
    a = torch.tensor([1.0, 0.0, 2.0, 0.0, 1.0, -0.0], device="cuda")
    none = torch.zeros(6, device="cuda")
    for to in (None, torch.empty(6, V + 1, dtype=torch.bfloat16, device="cuda")[:, 1:]):
        for dh in (None, none):
            d = lp.backward(a, x, t, stats, dentropy=dh, entropy=entropy, out=to)
            assert torch.isfinite(d[0]).all() and d[0].any() and d[2].isnan().all() and not d[[1, 3, 4, 5]].any()
        h = _rand(6, seed=2)
        d = lp.backward(a, x, t, stats, dentropy=h, entropy=entropy, out=to)
        alone = lp.backward(None, x, None, stats, dentropy=h, entropy=entropy)
        assert d[2].isnan().all() and torch.equal(d[[1, 3, 4, 5]], alone[[1, 3, 4, 5]])
