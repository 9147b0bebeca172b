"""Layer norm without a GPU: refusals that come before any device call."""
import ctypes

import pytest

from conftest import has_gpu


def _norm(libapk, **kw):
    from apk_b200 import _lib as L
    cfg = dict(device=0, features=16, eps=1e-5, weight_dtype=L.APK_F32, bias_dtype=L.APK_F32, weight=4096, bias=None)
    cfg.update(kw)
    h = ctypes.c_void_p()
    return libapk.apk_norm_create(ctypes.byref(L.NormConfig(**cfg)), ctypes.byref(h)), h


@pytest.mark.parametrize("bad", [dict(features=0), dict(features=-1), dict(features=16385), dict(features=(1 << 31) - 1),
                                 dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
                                 dict(weight=None), dict(weight=4098), dict(weight_dtype=2), dict(bias=4096, bias_dtype=-1),
                                 dict(bias=4097, bias_dtype=1)])
def test_create_refuses(libapk, bad):
    from apk_b200 import _lib as L
    st, h = _norm(libapk, **bad)
    assert st == L.APK_EINVAL and h.value and libapk.apk_norm_last_error(h)
    # a handle whose create failed is refused by every call
    assert libapk.apk_norm_forward(h, ctypes.byref(L.NormIO())) == L.APK_EINVAL
    assert libapk.apk_norm_backward(h, ctypes.byref(L.NormGrads())) == L.APK_EINVAL
    assert libapk.apk_norm_destroy(h) == L.APK_OK


def test_null_arguments(libapk):
    from apk_b200 import _lib as L
    h = ctypes.c_void_p()
    assert libapk.apk_norm_create(None, ctypes.byref(h)) == L.APK_EINVAL and h.value
    assert libapk.apk_norm_destroy(h) == L.APK_OK and libapk.apk_norm_destroy(None) == L.APK_OK
    assert libapk.apk_norm_create(None, None) == L.APK_EINVAL
    assert libapk.apk_norm_forward(None, None) == L.APK_EINVAL and libapk.apk_norm_last_error(None)


@pytest.mark.skipif(has_gpu(), reason="checks the no-device failure path")
def test_create_fails_cleanly_without_gpu(libapk):
    from apk_b200 import _lib as L
    st, h = _norm(libapk)
    assert st == L.APK_ECUDA and b"device" in libapk.apk_norm_last_error(h)
    libapk.apk_norm_destroy(h)


def test_python_refuses_host_tensors(libapk):
    torch = pytest.importorskip("torch")
    import apk_b200
    with pytest.raises(ValueError, match="CUDA"):
        apk_b200.LayerNorm(torch.zeros(8))
