"""The norm of many gradients and their clipping on a B200 against 64 bits.

Bounds, E = 2^-24 the unit roundoff of fp32: squares are added in fp32 over at
most 32 values in chains of 8 and a sum of 4 (12 roundings with the squares'
own), so the norm is within 6 E, and one more for its own rounding.  A factor
carries the same and one more, a product one more."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


@pytest.fixture(autouse=True)
def _lib(libapk):
    return libapk


def _rand(n, seed, dtype="f32", scale=1.0, at=0):
    """n values that start `at` elements behind a 16-byte boundary."""
    import torch
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    t = torch.empty(n + at, dtype={"bf16": torch.bfloat16, "f32": torch.float32}[dtype], device="cuda")
    return t.normal_(0.0, scale, generator=g)[at:]


def _want(grads, max_norm):
    norm = math.sqrt(math.fsum(float(t.double().square().sum()) for t in grads))
    return norm, min(1.0, max_norm / (norm + 1e-6))


def _check(grads, max_norm=1.0):
    import layer_bounds as lb
    import torch

    import apk_b200
    clip = apk_b200.GradClip(max_norm)
    kept = [t.clone() for t in grads]
    norm, c = _want(grads, max_norm)
    got = clip.norm(grads)
    assert got.shape == () and got.dtype == torch.float32
    assert abs(float(got) - norm) <= 7 * E * norm
    out = [torch.full_like(t, 7.0) for t in grads]
    assert torch.equal(clip.clip(grads, out=out), got)
    assert all(torch.equal(t, k) for t, k in zip(grads, kept)), "the inputs changed"
    for t, o in zip(grads, out):
        want = t.double() * c
        lb.check(o, want, want.abs() * (9 * E + (2.0 ** -8 if t.dtype == torch.bfloat16 else E)) + 2.0 ** -126, "out")
    assert torch.equal(clip.clip(grads), got)
    assert all(torch.equal(t, o) for t, o in zip(grads, out)), "in place differs"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 9, 255, 4095, 4096, 4097, 8191, 8192, 100003, 2500001])
def test_sizes_and_starts(n, dtype):
    for at in (0, 1, 3, 4, 7):
        _check([_rand(n, n + at, dtype, at=at)], max_norm=0.3 * n ** 0.5)


@pytest.mark.parametrize("count", [2, 59, 60, 61, 300, 999, 1000, 1001, 2300])
def test_many_tensors(count):
    _check([_rand(1 + 37 * i % 6000, i, "bf16" if i % 3 else "f32", scale=0.1, at=i % 5) for i in range(count)], 2.5)


def test_large_and_small_tensors_of_both_types():
    _check([_rand(n, n, t) for n, t in ((30000000, "f32"), (1, "bf16"), (0, "f32"), (20000001, "bf16"), (5, "f32"))], 100.0)


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-18, 1e-13, 1e13, 1e18, 1e30])
def test_squares_beyond_fp32(scale):
    for dtype in ("f32", "bf16"):
        _check([_rand(5000, 1, dtype, scale), _rand(77, 2, dtype, scale)], max_norm=10 * scale)
    # far apart in one vector, and in one call
    t = _rand(4000, 3)
    t[::5] *= scale
    _check([t, _rand(1000, 4, "bf16", scale)])


def test_denormals_zeros_and_the_largest_values():
    import torch

    import apk_b200
    clip = apk_b200.GradClip(1.0)
    tiny = torch.full((1000,), 2.0 ** -149, device="cuda")
    assert float(clip.norm([tiny])) == pytest.approx(2.0 ** -149 * 1000 ** 0.5, rel=0.05)  # (a denormal itself: steps of 2^-149)
    most = torch.full((100,), 3.0e38, device="cuda")
    assert float(clip.norm([most])) == math.inf                      # 3e39 is not an fp32 value
    clip.clip([most])
    assert torch.allclose(most, torch.full_like(most, 0.1), rtol=3e-6)    # the factor, 3e-40, has steps of 2^-149
    zero = torch.zeros(5000, device="cuda")
    assert float(clip.clip([zero])) == 0.0 and not zero.any()
    assert float(clip.norm([])) == 0.0 and float(clip.clip([])) == 0.0 and float(clip.norm([zero[:0]])) == 0.0


def test_a_norm_below_the_bound_leaves_every_bit():
    import torch

    import apk_b200
    clip = apk_b200.GradClip(1000.0)
    for dtype in ("f32", "bf16"):
        t = _rand(10001, 1, dtype, at=1)
        kept, out = t.clone(), torch.empty_like(t)
        clip.clip([t], out=[out])
        clip.clip([t])
        assert torch.equal(t, kept) and torch.equal(out, kept)
    clip.max_norm = math.inf
    clip.clip([t])
    assert torch.equal(t, kept)
    clip.max_norm = 0.0
    clip.clip([t])
    assert not t.any()


def test_infinite_and_nan_norms():
    import torch

    import apk_b200
    clip = apk_b200.GradClip(1.0)
    t, u = _rand(5000, 1), _rand(300, 2, "bf16")
    t[17] = math.inf
    assert float(clip.clip([t, u])) == math.inf
    assert bool(t[17].isnan()) and int((t != 0).sum()) == 1 and not u.any()
    t, u = _rand(5000, 1), _rand(300, 2, "bf16")
    u[299] = math.nan
    assert math.isnan(float(clip.clip([t, u]))) and t.isnan().all() and u.isnan().all()


def test_orders_of_axes_and_nones():
    import torch

    import apk_b200
    clip = apk_b200.GradClip(1.0)
    a = _rand(24 * 40, 1).view(24, 40).t()
    b = _rand(6 * 7 * 8, 2, "bf16").view(6, 7, 8).permute(1, 2, 0)
    norm, c = _want([a, b], 1.0)
    out = [torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda") for t in (a, b)]
    assert abs(float(clip.clip([a, None, b], out=[out[0], None, out[1]])) - norm) <= 7 * E * norm
    assert torch.allclose(out[0].double(), a.double() * c, rtol=1e-6, atol=0)
    assert torch.allclose(out[1].double(), b.double() * c, rtol=2.0 ** -7, atol=0)


def test_outputs_that_start_elsewhere():
    """An input and an output whose places within 16 bytes differ."""
    import torch

    import apk_b200
    clip = apk_b200.GradClip(0.5)
    for dtype in ("f32", "bf16"):
        for n in (5, 4097, 30000):
            for at in (1, 2, 3):
                t, room = _rand(n, n, dtype, at=at), _rand(n + 16, 1, dtype)
                for to in (0, 1, 2, 5):
                    kept = room.clone()
                    clip.clip([t], out=[room[to:to + n]])
                    want = t.clone()
                    clip.clip([want])
                    kept[to:to + n] = want
                    assert torch.equal(room, kept), "something beside the output was written"


def test_streams_and_graphs():
    import torch

    import apk_b200
    clip = apk_b200.GradClip(1.0)
    lists = [[_rand(50000 + 1000 * i, 10 * i + j, "f32" if j else "bf16") for j in range(5)] for i in range(4)]
    want = [(clip.norm(g), [torch.empty_like(t) for t in g]) for g in lists]
    for g, (_, o) in zip(lists, want):
        clip.clip(g, out=o)
    torch.cuda.synchronize()
    side, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i, g in enumerate(lists):
        with torch.cuda.stream(side[i % 2]):
            o = [torch.empty_like(t) for t in g]
            got.append((clip.clip(g, out=o), o))
    torch.cuda.synchronize()
    for (n, o), (m, p) in zip(got, want):
        assert torch.equal(n, m) and all(torch.equal(x, y) for x, y in zip(o, p))
    held = [t.clone() for t in lists[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip.clip(held)
    for _ in range(3):
        for t, s in zip(held, lists[0]):
            t.copy_(s)
        graph.replay()
        other = clip.norm(lists[1])
        torch.cuda.synchronize()
        assert torch.equal(norm, want[0][0]) and torch.equal(other, want[1][0])
        assert all(torch.equal(x, y) for x, y in zip(held, want[0][1]))


def test_refusals():
    import torch

    import apk_b200
    from apk_b200 import _lib as L
    clip = apk_b200.GradClip(1.0)
    t = _rand(64, 1)
    for bad in ([t.double()], [t, t.cpu()], [t[::2]], [t, 3.0], [t.view(8, 8)[:, :4]], [t.half()]):
        with pytest.raises(ValueError):
            clip.norm(bad)
        with pytest.raises(ValueError):
            clip.clip(bad)
    for out in ([], [t, t], [t[:32]], [t.bfloat16()], [t.view(8, 8)]):
        with pytest.raises(ValueError):
            clip.clip([t], out=out)
    with pytest.raises(ValueError):
        clip.clip([t.view(8, 8)], out=[torch.empty(8, 8, device="cuda").t()])
    other = _rand(64, 2)
    for grads, out in (([t, t], None), ([t, t[5:9]], None), ([t[:32], t[31:]], None), ([t, other], [other, t]),
                       ([t[:40]], [t[8:48]]), ([t[:32], t[32:]], [other[:32], other[:32]]), ([t, other], [t, t])):
        with pytest.raises(apk_b200.ApkError, match="memory"):
            clip.clip(grads, out=out)
    assert float(clip.norm([t, t])) == pytest.approx(2 ** 0.5 * float(clip.norm([t])), rel=1e-6)    # counted twice
    clip.clip([t[:32], t[32:]], out=[other[32:], other[:32]])                                       # apart
    clip.max_norm = math.nan
    with pytest.raises(ValueError):
        clip.clip([t])
    p = (ctypes.c_longlong * 1)(t.data_ptr())
    n, kind = (ctypes.c_longlong * 1)(64), (ctypes.c_int * 1)(0)
    good = dict(count=1, in_=ctypes.addressof(p), out=ctypes.addressof(p), n=ctypes.addressof(n), dtype=ctypes.addressof(kind),
                max_norm=1.0, norm=other.data_ptr())
    for bad in (dict(count=-1), dict(in_=None), dict(out=None), dict(n=None), dict(dtype=None), dict(max_norm=-1.0),
                dict(max_norm=math.nan), dict(norm=None), dict(norm=other.data_ptr() + 1)):
        a = L.ClipIO(**{**good, **bad})
        assert clip._lib.apk_clip_scale(clip._h, ctypes.byref(a)) == L.APK_EINVAL
        assert clip._lib.apk_clip_last_error(clip._h)
    for array, value in ((n, -1), (n, (1 << 40) + 1), (kind, 2), (p, 0), (p, t.data_ptr() + 2)):
        kept, array[0] = array[0], value
        assert clip._lib.apk_clip_norm(clip._h, ctypes.byref(L.ClipIO(**good))) == L.APK_EINVAL
        array[0] = kept
    torch.cuda.synchronize()
