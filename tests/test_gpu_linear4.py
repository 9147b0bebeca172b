"""Linear layers with 4-bit weights on a B200 against 64 bits, element by
element, with the linear layers' bounds (layer_bounds.py): weights are whole
numbers times a scale, products of whole numbers and bf16 are exact, and a
group's sum is scaled in fp32 (two more roundings, for which those bounds have
room).  Above 64 rows a weight is first rounded to bf16 (2^-8 of itself), for
an fp32 result to two bf16 terms (2^-16)."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(libapk):
    return libapk


def _rand(*shape, seed, scale=1.0, dtype=None):
    import torch
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return torch.empty(shape, dtype=dtype or torch.bfloat16, device="cuda").normal_(0.0, scale, generator=g)


def _layer(K, N, group=128, zeros=False, scale="bf16", act="none", bias=None, out="bf16", seed=0, **kw):
    """(the layer, its weights as [K, N] in 64 bits)."""
    import torch

    import apk_b200
    g = torch.Generator("cuda")
    g.manual_seed(seed + 1)
    groups = -(-K // group)
    w = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device="cuda", generator=g)
    s = (_rand(N, groups, seed=seed + 2).float().abs() * K ** -0.5 / 4 + 1e-3).to({"bf16": torch.bfloat16, "f32": torch.float32}[scale])
    z = torch.randint(0, 16, (N, groups), dtype=torch.uint8, device="cuda", generator=g) if zeros else None
    b = None if bias is None else _rand(N, seed=seed + 3, dtype=bias)
    lin = apk_b200.Linear4(w, s, zeros=z, bias=b, group=group, act=act, out_dtype=out, **kw)
    q = torch.stack((w & 15, w >> 4), 2).view(N, K).double()
    at = torch.arange(K, device="cuda") // group
    return lin, ((q - (8.0 if z is None else z.double()[:, at])) * s.double()[:, at]).t()


def _bounds(lin, w, x, r):
    import layer_bounds as lb
    import torch
    z, size = x.double() @ w, x.double().abs() @ w.abs()
    if lin.bias is not None:
        z, size = z + lin.bias.double(), size + lin.bias.double().abs()
    f32 = lin.out_dtype == torch.float32
    ez = (lb.sum_err(2 * x.shape[-1]) + (0.0 if x.shape[0] <= 64 else 2.0 ** -16 if f32 else lb.U)) * size
    y = lb.act(lin.act, z)
    ey = lb.LIP * ez + lb.ACT_REL * (z.abs() + y.abs())
    if r is not None:
        y = y + r.double()
        ey = ey + 2.0 ** -23 * (y.abs() + r.double().abs())
    return y, lb.rounded(y, ey, lin.out_dtype), z, lb.rounded(z, ez, torch.bfloat16)


def _check(lin, w, x, r=None):
    import layer_bounds as lb
    import torch
    y, z = lin.forward(x, residual=r, save_preact=True)
    want, by, wz, bz = _bounds(lin, w, x, r)
    lb.check(y, want, by, "y")
    lb.check(z, wz, bz, "preact")
    assert torch.equal(lin.forward(x, residual=r), y), "a second call differs"
    assert lin.status() == 0


SHAPES = [(1, 32, 1), (1, 4096, 2048), (2, 64, 8), (3, 160, 33), (7, 1024, 65), (8, 2080, 1000), (9, 96, 130), (16, 8192, 256),
          (17, 992, 40), (33, 4096, 128), (64, 1056, 300), (65, 1056, 129), (130, 2048, 512), (500, 160, 96), (1000, 1120, 1031)]


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_shapes(M, K, N, group):
    import torch
    i = SHAPES.index((M, K, N)) + group // 32
    lin, w = _layer(K, N, group, zeros=i % 2 == 0, scale=("bf16", "f32")[i % 3 == 0], act=("none", "silu", "gelu_tanh", "relu", "gelu")[i % 5],
                    bias=(None, torch.float32, torch.bfloat16)[i % 3], out=("bf16", "f32")[i % 4 == 1], seed=i)
    r = None if i % 2 else _rand(M, N, seed=5, dtype=(torch.bfloat16, torch.float32)[i % 4 == 0])
    _check(lin, w, _rand(M, K, seed=4), r)


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("M", [1, 13, 64, 200])
def test_long_sums_and_results(M, out):
    lin, w = _layer(16384, 96, 128, out=out)
    x = _rand(M, 16384, seed=1).abs()       # of one sign: nothing hides a bias of the sums
    _check(lin, w, x)


def test_every_nibble_and_zero_point_is_exact():
    """One weight at a time against one value of x: the layer returns it exactly."""
    import torch

    import apk_b200
    K = 256
    q = (torch.arange(16 * K, device="cuda").view(16, K) * 7 // 3 % 16).to(torch.uint8)
    w = q[:, 0::2] | (q[:, 1::2] << 4)
    x = torch.eye(K, dtype=torch.bfloat16, device="cuda")
    for group in (32, 64, 128):
        z = (torch.arange(16 * (K // group), device="cuda") % 16).to(torch.uint8).view(16, -1)
        s = torch.full((16, K // group), 0.5, device="cuda")
        lin = apk_b200.Linear4(w, s, zeros=z, group=group, out_dtype="f32")
        want = (q.float() - z.float().repeat_interleave(group, 1)).t() * 0.5
        for rows in (x.split(8), x.split(16), x.split(64), (x,)):
            assert torch.equal(torch.cat([lin.forward(r) for r in rows]), want)
        high = apk_b200.Linear4(w, s, zeros=z | 0xF0, group=group, out_dtype="f32")     # the low four bits count
        assert torch.equal(high.forward(x[:8]), want[:8]) and torch.equal(high.forward(x), want)


@pytest.mark.parametrize("M", [1, 5, 20, 100])
def test_strides_alignment_and_leading_axes(M):
    import torch
    K, N = 416, 77
    lin, w = _layer(K, N, 32, zeros=True, act="silu", bias=torch.float32)
    for ld, at in ((K, 0), (K + 1, 1), (K + 8, 8), (K + 6, 2)):
        wide = _rand(M, ld, seed=ld)
        x = wide[:, at:at + K] if ld > K else wide
        room = _rand(M, N + 9, seed=2)
        kept = room.clone()
        _check(lin, w, x, room[:, :N])
        y = lin.forward(x, residual=room[:, :N])
        assert lin.forward(x, residual=room[:, :N], out=room[:, :N]) is not None
        kept[:, :N] = y
        assert torch.equal(room, kept)
    x = _rand(2, 3, K, seed=3)
    assert torch.equal(lin.forward(x).view(6, N), lin.forward(x.view(6, K))) and lin.forward(x[0, 0]).shape == (N,)
    assert lin.forward(x[:0]).shape == (0, 3, N)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_scales_and_zeros_at_odd_addresses(group):
    """Scales, zero points and bias behind an odd element: the same results as on their own boundaries."""
    import torch

    import apk_b200
    K, N = 512, 70
    lin, _ = _layer(K, N, group, zeros=True, bias=torch.float32, act="silu")

    def moved(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        room[1:].copy_(t.flatten())
        return room[1:].view(t.shape)

    other = apk_b200.Linear4(lin.weight, moved(lin.scales), zeros=moved(lin.zeros), bias=moved(lin.bias), group=group, act="silu")
    for M in (1, 12, 30, 64, 90):
        x = _rand(M, K, seed=M)
        assert torch.equal(lin.forward(x), other.forward(x))


def test_long_rows_in_slices():
    """x of 64 rows that shared memory holds a part of at a time, whole chunks or not."""
    for K, group in ((20480, 128), (9056, 32)):
        lin, w = _layer(K, 48, group, zeros=True)
        _check(lin, w, _rand(64, K, seed=1))
        _check(lin, w, _rand(9, K, seed=2))


def test_weights_in_wider_rows_and_updated_in_place():
    import torch

    import apk_b200
    g = torch.Generator("cuda").manual_seed(1)
    wide = torch.randint(0, 256, (40, 96), dtype=torch.uint8, device="cuda", generator=g)
    s = torch.rand(40, 2, device="cuda", generator=g)
    lin = apk_b200.Linear4(wide[:, 16:80], s, group=64)
    copy = apk_b200.Linear4(wide[:, 16:80].contiguous(), s, group=64)
    for M in (3, 100):
        x = _rand(M, 128, seed=M)
        assert torch.equal(lin.forward(x), copy.forward(x))
    wide.zero_()
    s.fill_(1.0)
    assert torch.allclose(lin.forward(x), -8 * x.float().sum(1, keepdim=True).bfloat16().expand(-1, 40), rtol=2.0 ** -6, atol=0.5)


def test_values_that_are_not_finite_stay_in_their_rows():
    import torch
    for M in (5, 90):
        lin, w = _layer(352, 50, 32, zeros=True)
        x = _rand(M, 352, seed=1)
        want = lin.forward(x)
        x[1, 351], x[3, 0] = float("nan"), float("inf")
        y = lin.forward(x)
        keep = [i for i in range(M) if i not in (1, 3)]
        assert y[1].isnan().all() and not torch.isfinite(y[3]).any() and torch.equal(y[keep], want[keep])


def test_streams_and_graphs():
    import torch
    lin, _ = _layer(1024, 500, 64, zeros=True, act="silu")
    xs = [_rand(M, 1024, seed=M) for M in (1, 40, 300, 200)]
    want = [lin.forward(x) for x in xs]
    torch.cuda.synchronize()
    side, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i in range(8):
        with torch.cuda.stream(side[i % 2]):
            got.append(lin.forward(xs[i % 4]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 4]) for i, y in enumerate(got))
    held = [x.clone() for x in xs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [lin.forward(x) for x in held]
    for _ in range(3):
        for o in out:
            o.zero_()
        graph.replay()
        again = lin.forward(xs[2])
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(out, want)) and torch.equal(again, want[2])
    big, other = _rand(3000, 1024, seed=9), _layer(1024, 500, 64)[0]
    with pytest.raises(Exception, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            lin.forward(held[0])
            other.forward(big)
    assert lin.status() == 0


def test_refusals():
    import torch

    import apk_b200
    from apk_b200 import _lib as L
    w = torch.zeros(24, 64, dtype=torch.uint8, device="cuda")
    s = torch.ones(24, 1, dtype=torch.bfloat16, device="cuda")
    good = dict(weight=w, scales=s, group=128)
    for bad in (dict(weight=w.cpu()), dict(weight=w.int()), dict(weight=w[0]), dict(weight=w.t()), dict(scales=s[:5]), dict(scales=s.half()),
                dict(scales=s.cpu()), dict(group=64), dict(group=0), dict(zeros=s), dict(zeros=w[:, :2]), dict(bias=s), dict(bias=s[:5, 0]),
                dict(act="tanh"), dict(out_dtype="f16")):
        with pytest.raises(ValueError):
            apk_b200.Linear4(**{**good, **bad})
    for bad in (dict(weight=w[:, 1:49].contiguous(), scales=s, group=100), dict(weight=w[:, 8:40]), dict(weight=torch.zeros(24, 40, dtype=torch.uint8, device="cuda")),
                dict(sms=1000)):
        with pytest.raises(apk_b200.ApkError):
            apk_b200.Linear4(**{**good, **bad})
    lin = apk_b200.Linear4(**good)
    x = _rand(6, 128, seed=1)
    for bad in (x.float(), x.cpu(), x[:, :64], x.t()):
        with pytest.raises(ValueError):
            lin.forward(bad)
    for kw in (dict(residual=x), dict(out=x), dict(out=_rand(6, 24, seed=2, dtype=torch.float32)), dict(out=x.view(-1)[8:152].view(6, 24)),
               dict(residual=x.view(-1)[:144].view(6, 24), out=x.view(-1)[8:152].view(6, 24))):
        with pytest.raises(ValueError):
            lin.forward(x, **kw)
    p = x.data_ptr()
    for bad in (dict(rows=-1), dict(rows=(1 << 30) + 1), dict(x=None), dict(y=None), dict(y_dtype=3), dict(ldx=127), dict(ldy=23),
                dict(x=p + 1), dict(residual=p, ld_residual=3), dict(preact=p, ld_preact=3)):
        a = L.LinearIO(**{**dict(x=p, ldx=128, rows=1, y=p, ldy=24, y_dtype=1), **bad})
        assert lin._lib.apk_linear4_forward(lin._h, ctypes.byref(a)) == L.APK_EINVAL and lin._lib.apk_linear4_last_error(lin._h)
    lin.scales = s.clone()
    with pytest.raises(ValueError, match="other memory"):
        lin.forward(x)
    torch.cuda.synchronize()


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("M", [3, 64, 65, 130])
def test_infinite_values_of_x(M, out):
    """An infinite x times a weight is infinite, times 0 NaN, whatever the form that the rows take; other rows stay
    as they are."""
    import torch
    lin, w = _layer(256, 72, group=32, zeros=True, out=out)
    x = _rand(M, 256, seed=1)
    want = lin.forward(x)
    bad = x.clone()
    bad[0, 5], bad[1, 200], bad[2, 31], bad[2, 64] = float("inf"), -float("inf"), float("nan"), float("inf")
    got = lin.forward(bad)
    rows = bad[:2].double()
    ref = torch.where(rows.isinf(), rows, torch.zeros_like(rows)) @ w  # (0 * inf is NaN here too)
    inf = torch.zeros(2, 72, dtype=torch.float64, device="cuda")
    inf[0], inf[1] = float("inf") * w[5], -float("inf") * w[200]
    assert torch.equal(ref.isnan(), inf.isnan()) and inf.isnan().any() and inf.isinf().any()
    assert torch.equal(got[:2].isnan(), inf.isnan()) and torch.equal(got[:2].double().nan_to_num(7.0), inf.nan_to_num(7.0))
    assert got[2].isnan().all() and torch.equal(got[3:], want[3:])
