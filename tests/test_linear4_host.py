"""Linear layers with 4-bit weights without a GPU: refusals that come before
any device call, and the weights' quantization."""
import ctypes

import pytest

from conftest import has_gpu


def _linear4(libapk, **kw):
    from apk_b200 import _lib as L
    cfg = dict(device=0, in_features=256, out_features=16, group=128, act=L.APK_ACT_NONE, scale_dtype=L.APK_BF16,
               bias_dtype=L.APK_F32, W=4096, ldw=128, scales=4096, zeros=None, bias=None)
    cfg.update(kw)
    h = ctypes.c_void_p()
    return libapk.apk_linear4_create(ctypes.byref(L.Linear4Config(**cfg)), ctypes.byref(h)), h


@pytest.mark.parametrize("bad", [dict(in_features=0), dict(in_features=16), dict(in_features=100), dict(in_features=(1 << 30) + 32, ldw=1 << 30),
                                 dict(out_features=0), dict(out_features=(1 << 30) + 1), dict(group=0), dict(group=16), dict(group=96),
                                 dict(group=192), dict(group=-128), dict(act=5), dict(act=-1), dict(W=None), dict(W=4104),
                                 dict(ldw=112), dict(ldw=136), dict(scales=None), dict(scales=4097), dict(scale_dtype=2),
                                 dict(scale_dtype=0, scales=4098), dict(bias=4098), dict(bias=4096, bias_dtype=3), dict(wait_limit_ns=-1)])
def test_create_refuses(libapk, bad):
    from apk_b200 import _lib as L
    st, h = _linear4(libapk, **bad)
    assert st == L.APK_EINVAL and h.value and libapk.apk_linear4_last_error(h)
    # a handle whose create failed is refused by every call
    assert libapk.apk_linear4_forward(h, ctypes.byref(L.LinearIO())) == L.APK_EINVAL
    assert libapk.apk_linear4_status(h, None, ctypes.byref(ctypes.c_int())) == L.APK_EINVAL
    assert libapk.apk_linear4_destroy(h) == L.APK_OK


def test_null_arguments(libapk):
    from apk_b200 import _lib as L
    h = ctypes.c_void_p()
    assert libapk.apk_linear4_create(None, ctypes.byref(h)) == L.APK_EINVAL and h.value
    assert libapk.apk_linear4_destroy(h) == L.APK_OK and libapk.apk_linear4_destroy(None) == L.APK_OK
    assert libapk.apk_linear4_create(None, None) == L.APK_EINVAL and libapk.apk_linear4_last_error(None)


@pytest.mark.skipif(has_gpu(), reason="checks the no-device failure path")
def test_create_fails_cleanly_without_gpu(libapk):
    from apk_b200 import _lib as L
    st, h = _linear4(libapk)
    assert st == L.APK_ECUDA and b"device" in libapk.apk_linear4_last_error(h)
    libapk.apk_linear4_destroy(h)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("k,group", [(256, 32), (256, 128), (160, 64), (96, 128)])
def test_quantize(k, group, zeros):
    """Within half a step of the weight, or of what the scale's rounding moves the ends by."""
    torch = pytest.importorskip("torch")
    import apk_b200
    w = torch.randn(24, k, generator=torch.Generator().manual_seed(1)) + 0.3
    w[3] = 0.0
    q, s, z = apk_b200.Linear4.quantize(w, group=group, zeros=zeros)
    assert q.shape == (24, k // 2) and q.dtype == torch.uint8 and s.shape == (24, -(-k // group)) and (z is None) != zeros
    full = torch.stack((q & 15, q >> 4), 2).view(24, k).double()
    at = torch.arange(k) // group
    s_k = s.double()[:, at]
    got = (full - (z.double()[:, at] if zeros else 8.0)) * s_k
    # the zero point is rounded to half a step, and the scale by 2^-8 of up to 15 steps
    step = 0.5 + (0.5 + 15 * 2.0 ** -8 if zeros else 7 * 2.0 ** -8)
    assert bool(((got - w.double()).abs() <= step * s_k + 1e-6).all()) and not got[3].any()


@pytest.mark.parametrize("group", [1 << 31, (1 << 32) + 128, 1 << 40, 0, -128])
def test_groups_past_32_bits(group):
    """(1 << 32) + 128 would reach the library as 128, whose scales are not there."""
    torch = pytest.importorskip("torch")
    import apk_b200
    with pytest.raises(ValueError, match="group"):
        apk_b200.Linear4(torch.zeros(16, 128, dtype=torch.uint8), torch.ones(16, 1), group=group)
