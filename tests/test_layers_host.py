"""Layer operators without a GPU: refusals that come before any device call,
handles that failed, and the Python layer's argument checks."""
import ctypes

import pytest

from conftest import has_gpu


def _linear(libapk, **kw):
    from apk_b200 import _lib as L
    cfg = dict(device=0, in_features=16, out_features=16, w_layout=L.APK_W_KN, act=L.APK_ACT_NONE,
               bias_dtype=L.APK_F32, W=4096, ldw=16, bias=None)
    cfg.update(kw)
    h = ctypes.c_void_p()
    st = libapk.apk_linear_create(ctypes.byref(L.LinearConfig(**cfg)), ctypes.byref(h))
    return st, h


def _moe(libapk, **kw):
    from apk_b200 import _lib as L
    cfg = dict(device=0, experts=4, top_k=2, d_model=16, d_ff=16, act=L.APK_ACT_SILU, gated=1, renormalize=1,
               router=4096, w_in=4096, w_out=4096)
    cfg.update(kw)
    h = ctypes.c_void_p()
    st = libapk.apk_moe_create(ctypes.byref(L.MoeConfig(**cfg)), ctypes.byref(h))
    return st, h


@pytest.mark.parametrize("bad", [dict(in_features=0), dict(out_features=-3), dict(w_layout=2), dict(act=5), dict(act=-1),
                                 dict(W=None), dict(ldw=15), dict(W=4097), dict(bias=4096, bias_dtype=2),
                                 dict(bias=4098), dict(wait_limit_ns=-1)])
def test_linear_create_refuses(libapk, bad):
    from apk_b200 import _lib as L
    st, h = _linear(libapk, **bad)
    assert st == L.APK_EINVAL and h.value
    assert libapk.apk_linear_last_error(h)
    # a handle whose create failed is refused by every call
    assert libapk.apk_linear_forward(h, ctypes.byref(L.LinearIO())) == L.APK_EINVAL
    assert libapk.apk_linear_backward(h, ctypes.byref(L.LinearGrads())) == L.APK_EINVAL
    assert libapk.apk_linear_status(h, None, ctypes.byref(ctypes.c_int())) == L.APK_EINVAL
    assert libapk.apk_linear_destroy(h) == L.APK_OK


@pytest.mark.parametrize("bad", [dict(experts=0), dict(experts=513), dict(top_k=0), dict(top_k=5), dict(experts=40, top_k=17),
                                 dict(d_model=0), dict(d_model=12), dict(d_ff=4), dict(act=9), dict(router=None),
                                 dict(w_in=None), dict(w_out=None), dict(router=4104), dict(wait_limit_ns=-1)])
def test_moe_create_refuses(libapk, bad):
    from apk_b200 import _lib as L
    st, h = _moe(libapk, **bad)
    assert st == L.APK_EINVAL and h.value
    assert libapk.apk_moe_last_error(h)
    assert libapk.apk_moe_forward(h, ctypes.byref(L.MoeIO())) == L.APK_EINVAL
    assert libapk.apk_moe_status(h, None, ctypes.byref(ctypes.c_int())) == L.APK_EINVAL
    assert libapk.apk_moe_destroy(h) == L.APK_OK


def test_null_arguments(libapk):
    from apk_b200 import _lib as L
    h = ctypes.c_void_p()
    assert libapk.apk_linear_create(None, ctypes.byref(h)) == L.APK_EINVAL and h.value
    libapk.apk_linear_destroy(h)
    assert libapk.apk_moe_create(None, ctypes.byref(h)) == L.APK_EINVAL and h.value
    libapk.apk_moe_destroy(h)
    for f in (libapk.apk_linear_destroy, libapk.apk_moe_destroy):
        assert f(None) == L.APK_OK
    assert libapk.apk_linear_last_error(None) and libapk.apk_moe_last_error(None)


@pytest.mark.skipif(has_gpu(), reason="checks the no-device failure path")
def test_create_fails_cleanly_without_gpu(libapk):
    from apk_b200 import _lib as L
    for make, err, gone in ((_linear, libapk.apk_linear_last_error, libapk.apk_linear_destroy),
                            (_moe, libapk.apk_moe_last_error, libapk.apk_moe_destroy)):
        st, h = make(libapk)
        assert st == L.APK_ECUDA and b"device" in err(h)
        gone(h)


def test_python_refuses_host_tensors(libapk):
    torch = pytest.importorskip("torch")
    import apk_b200
    w = torch.zeros(8, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        apk_b200.Linear(w)
    with pytest.raises(ValueError, match="CUDA"):
        apk_b200.MoE(w, w, w, top_k=1)
    with pytest.raises(AttributeError):
        apk_b200.NoSuchLayer
