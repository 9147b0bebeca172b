"""Gradient norm and clipping without a GPU: refusals that come before any device call."""
import ctypes

import pytest

from conftest import has_gpu


def test_null_arguments(libapk):
    from apk_b200 import _lib as L
    h = ctypes.c_void_p()
    assert libapk.apk_clip_create(None, ctypes.byref(h)) == L.APK_EINVAL and h.value
    # a handle whose create failed is refused by every call
    for f in (libapk.apk_clip_norm, libapk.apk_clip_scale):
        assert f(h, ctypes.byref(L.ClipIO())) == L.APK_EINVAL
        assert f(None, ctypes.byref(L.ClipIO())) == L.APK_EINVAL
    assert libapk.apk_clip_destroy(h) == L.APK_OK and libapk.apk_clip_destroy(None) == L.APK_OK
    assert libapk.apk_clip_create(None, None) == L.APK_EINVAL and libapk.apk_clip_last_error(None)


@pytest.mark.skipif(has_gpu(), reason="checks the no-device failure path")
def test_create_fails_cleanly_without_gpu(libapk):
    from apk_b200 import _lib as L
    h = ctypes.c_void_p()
    assert libapk.apk_clip_create(ctypes.byref(L.ClipConfig(0)), ctypes.byref(h)) == L.APK_ECUDA
    assert b"device" in libapk.apk_clip_last_error(h)
    libapk.apk_clip_destroy(h)


def test_python_refusals(libapk):
    pytest.importorskip("torch")
    import apk_b200
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            apk_b200.GradClip(bad, device="cuda:0")
    with pytest.raises(ValueError, match="CUDA"):
        apk_b200.GradClip(1.0, device="cpu")


def test_dense():
    torch = pytest.importorskip("torch")
    from apk_b200.training import _dense
    t = torch.zeros(4, 6, 8)
    for yes in (t, t.permute(2, 0, 1), t[1], t[:, 0:1][0], t[:0], torch.zeros(()), t[1:3], t[0].t(), t.transpose(1, 2)):
        assert _dense(yes)
    for no in (t[:, ::2], t[..., :7], t[:, 0], t[0, 0].expand(3, 8), t[::2]):
        assert not _dense(no)


def test_status_of_what_has_nothing_to_report():
    """Code that asks every layer for its status may ask these too."""
    pytest.importorskip("torch")
    import apk_b200
    for kind in (apk_b200.LayerNorm, apk_b200.GradClip, apk_b200.LogProbs):
        assert kind.__new__(kind).status() == 0
