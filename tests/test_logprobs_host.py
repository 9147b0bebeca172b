"""Log probabilities without a GPU: refusals that come before any device call."""
import ctypes

import pytest

from conftest import has_gpu


def _make(libapk, top):
    from apk_b200 import _lib as L
    h = ctypes.c_void_p()
    return libapk.apk_logprobs_create(ctypes.byref(L.LogprobsConfig(0, top)), ctypes.byref(h)), h


@pytest.mark.parametrize("top", [-1, 33, 1 << 30])
def test_create_refuses(libapk, top):
    from apk_b200 import _lib as L
    st, h = _make(libapk, top)
    assert st == L.APK_EINVAL and h.value and b"top" in libapk.apk_logprobs_last_error(h)
    # a handle whose create failed is refused by every call
    assert libapk.apk_logprobs_forward(h, ctypes.byref(L.LogprobsIO())) == L.APK_EINVAL
    assert libapk.apk_logprobs_backward(h, ctypes.byref(L.LogprobsGrads())) == L.APK_EINVAL
    assert libapk.apk_logprobs_destroy(h) == L.APK_OK


def test_null_arguments(libapk):
    from apk_b200 import _lib as L
    h = ctypes.c_void_p()
    assert libapk.apk_logprobs_create(None, ctypes.byref(h)) == L.APK_EINVAL and h.value
    assert libapk.apk_logprobs_destroy(h) == L.APK_OK and libapk.apk_logprobs_destroy(None) == L.APK_OK
    assert libapk.apk_logprobs_create(None, None) == L.APK_EINVAL and libapk.apk_logprobs_last_error(None)
    assert libapk.apk_logprobs_forward(None, None) == L.APK_EINVAL
    assert libapk.apk_logprobs_backward(None, None) == L.APK_EINVAL


@pytest.mark.skipif(has_gpu(), reason="checks the no-device failure path")
def test_create_fails_cleanly_without_gpu(libapk):
    from apk_b200 import _lib as L
    st, h = _make(libapk, 5)
    assert st == L.APK_ECUDA and b"device" in libapk.apk_logprobs_last_error(h)
    libapk.apk_logprobs_destroy(h)


def test_python_refusals(libapk):
    pytest.importorskip("torch")
    import apk_b200
    for bad in (-1, 33, 2.5, None):
        with pytest.raises(ValueError, match="top"):
            apk_b200.LogProbs(top=bad, device="cuda:0")
    with pytest.raises(ValueError, match="CUDA"):
        apk_b200.LogProbs(device="cpu")
