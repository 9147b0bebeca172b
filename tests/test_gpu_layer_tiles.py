"""The linear layer and its gradients at the sizes of ordinary layers, element
by element against 64 bits: CTA pairs with either operand's axis contiguous,
two accumulators a tile, two products dealt out over pairs, accumulators of
512 k in pairs, and streaming products whose warps take more than 512 k."""
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


# M, K, N, act, dtype of dw.  On 148 SMs these reach, with every combination of
# contiguous axes: pairs of 512 x 256 and 256 x 256 tiles for one product and
# for two, pairs with accumulators of 512 k likewise, one CTA with them, and two
# products apart.
GRADS = [(2048, 1024, 4096, "gelu_tanh", "bf16"), (2048, 1024, 4096, "none", "f32"), (4096, 2048, 4096, "silu", "bf16"),
         (4096, 2048, 4096, "relu", "f32"), (4096, 4096, 8192, "gelu", "bf16"), (512, 1024, 4096, "silu", "bf16"),
         (2001, 1025, 4099, "relu", "bf16"), (1000, 264, 520, "gelu", "f32"), (600, 96, 72, "none", "f32"),
         (2048, 512, 264, "silu", "f32")]


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("M,K,N,act,wdt", GRADS)
def test_gradients(M, K, N, act, wdt, layout):
    import layer_bounds as lb
    import torch

    import apk_b200
    w = _rand(*((K, N) if layout == "kn" else (N, K)), seed=1, scale=K ** -0.5)
    lin = apk_b200.Linear(w, torch.zeros(N, device="cuda"), act=act, layout=layout)
    x, dy, z = _rand(M, K, seed=3), _rand(M, N, seed=4), _rand(M, N, seed=5, scale=2.0)
    want = lb.linear_grads(x, w if layout == "kn" else w.t(), z, act, dy, {"f32": torch.float32, "bf16": torch.bfloat16}[wdt])
    whole = lin.backward(dy, x, preact=z, dw_dtype=wdt)
    again = lin.backward(dy, x, preact=z, dw_dtype=wdt)
    assert all(torch.equal(a, b) for a, b in zip(whole, again)), "a second call differs"
    for got, what in ((whole, "together"),
                      (lin.backward(dy, x, preact=z, need_dw=False, need_db=False), "dx alone"),
                      (lin.backward(dy, x, preact=z, need_dx=False, need_db=False, dw_dtype=wdt), "dw alone")):
        if got[0] is not None:
            lb.check(got[0], *want[0], f"dx, {what}")
        if got[1] is not None:
            lb.check(got[1] if layout == "kn" else got[1].t(), *want[1], f"dw, {what}")
    lb.check(whole[2], *want[2], "db")
    assert lin.status() == 0


FORWARD = [(4096, 4096, 1536, "bf16"), (2048, 512, 2048, "bf16"), (1500, 1000, 3000, "bf16"), (4096, 1024, 4096, "f32"),
           (5, 16400, 2500, "f32"), (5, 16400, 2500, "bf16"), (12, 9000, 1200, "f32"), (3, 16400, 500, "f32")]


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("M,K,N,out", FORWARD)
def test_forward(M, K, N, out, layout):
    import layer_bounds as lb
    import torch

    import apk_b200
    w = _rand(*((K, N) if layout == "kn" else (N, K)), seed=1, scale=K ** -0.5)
    bias, x, r = _rand(N, seed=2), _rand(M, K, seed=3), _rand(M, N, seed=4)
    lin = apk_b200.Linear(w, bias, act="silu", layout=layout, out_dtype=out)
    y, z = lin.forward(x, residual=r, save_preact=True)
    want, by, wz, bz = lb.linear(x, w if layout == "kn" else w.t(), bias, "silu", r, y.dtype)
    lb.check(y, want, by, "y")
    lb.check(z, wz, bz, "preact")
    assert torch.equal(y, lin.forward(x, residual=r)) and lin.status() == 0


def test_streaming_with_long_shares_of_k():
    """One SM's worth of CTAs: a warp takes 4096 k of 12 rows' product."""
    import layer_bounds as lb
    import torch

    import apk_b200
    for layout in ("kn", "nk"):
        for out in ("f32", "bf16"):
            w = _rand(*((32768, 48) if layout == "kn" else (48, 32768)), seed=1, scale=2.0 ** -7.5)
            x = _rand(12, 32768, seed=2)
            lin = apk_b200.Linear(w, layout=layout, out_dtype=out, sms=1)
            want, by, _, _ = lb.linear(x, w if layout == "kn" else w.t(), None, "none", None, lin.out_dtype)
            lb.check(lin.forward(x), want, by, f"{layout} {out}")
            assert torch.equal(lin.forward(x), lin.forward(x))
