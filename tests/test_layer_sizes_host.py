"""Sizes that the layer kernels' 32-bit counts cannot step past are refused."""
import ctypes

import pytest

from test_layers_host import _linear, _moe


@pytest.mark.parametrize("size", [(1 << 30) + 1, (1 << 31) - 1])
@pytest.mark.parametrize("which", ["in_features", "out_features"])
@pytest.mark.parametrize("layout", [0, 1])
def test_linear_refuses(libapk, which, size, layout):
    from apk_b200 import _lib as L
    st, h = _linear(libapk, **{which: size}, w_layout=layout, ldw=1 << 31)
    assert st == L.APK_EINVAL and b"2^30" in libapk.apk_linear_last_error(h)
    libapk.apk_linear_destroy(h)


@pytest.mark.parametrize("which", ["d_model", "d_ff"])
def test_moe_refuses(libapk, which):
    from apk_b200 import _lib as L
    for size in ((1 << 26) + 8, (1 << 31) - 8):
        st, h = _moe(libapk, **{which: size})
        assert st == L.APK_EINVAL and b"2^26" in libapk.apk_moe_last_error(h)
        libapk.apk_moe_destroy(h)


@pytest.mark.gpu
def test_rows_are_refused(libapk):
    import torch

    import apk_b200
    from apk_b200 import _lib as L
    w = torch.zeros(64, 32, dtype=torch.bfloat16, device="cuda")
    lin = apk_b200.Linear(w, torch.zeros(32, device="cuda"))
    p = w.data_ptr()
    for rows in ((1 << 30) + 1, (1 << 31) - 1):
        io = L.LinearIO(x=p, ldx=64, rows=rows, y=p, ldy=32, y_dtype=L.APK_BF16)
        assert lin._lib.apk_linear_forward(lin._h, ctypes.byref(io)) == L.APK_EINVAL
        g = L.LinearGrads(dy=p, ld_dy=32, x=p, ldx=64, rows=rows, dx=p, ld_dx=64)
        assert lin._lib.apk_linear_backward(lin._h, ctypes.byref(g)) == L.APK_EINVAL
    torch.cuda.synchronize()
    assert lin.status() == 0
