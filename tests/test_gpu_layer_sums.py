"""fp32 results of long sums of one sign, where the tensor core's truncation is
a bias: about 1e-9 per k of the result in one accumulator (3e-5 at 32768 k).

Bound: an accumulator takes 512 k in 32 truncating steps, each at most 2^-23 of
the partial sum, which grows evenly: 16.5 x 2^-23 of the piece.  The pieces,
then warps or ranks, are added with rounding, 2^-24 of a partial sum each:
n / 4 x 2^-23 for n of them.  Two more for the ends."""
import pytest

pytestmark = pytest.mark.gpu


def bound(adds):
    return (16.5 + adds / 4 + 2) * 2.0 ** -23


@pytest.fixture(autouse=True)
def _lib(libapk):
    return libapk


def _positive(*shape, seed, scale=1.0):
    import torch
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0.0, scale, generator=g).abs_()


def _check(got, want, adds, what):
    rel = float(((got.double() - want).abs() / want).max())
    assert rel <= bound(adds), f"{what}: {rel:.3g}, bound {bound(adds):.3g}"


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("M,N,sms", [(40, 96, 0), (200, 160, 0), (200, 160, 1), (900, 520, 0)])
def test_linear(M, N, sms, layout):
    import torch

    import apk_b200
    K = 32768
    x, w = _positive(M, K, seed=1), _positive(*((K, N) if layout == "kn" else (N, K)), seed=2, scale=1 / K)
    lin = apk_b200.Linear(w, layout=layout, out_dtype="f32", sms=sms)
    want = x.double() @ (w if layout == "kn" else w.t()).double()
    assert lin.forward(x).dtype == torch.float32
    _check(lin.forward(x), want, K / 512 + 8, "y")


@pytest.mark.parametrize("rows", [1, 8, 12])
@pytest.mark.parametrize("layout,K,N,warps", [("nk", 1 << 18, 32, 16), ("kn", 1 << 17, 40, 8), ("nk", (1 << 18) - 3, 32, 16)])
def test_linear_of_a_few_rows(rows, layout, K, N, warps):
    """One SM's worth of CTAs: K is split over a CTA's warps alone."""
    import apk_b200
    x, w = _positive(rows, K, seed=1), _positive(*((K, N) if layout == "kn" else (N, K)), seed=2, scale=1 / K)
    lin = apk_b200.Linear(w, layout=layout, out_dtype="f32", sms=1)
    want = x.double() @ (w if layout == "kn" else w.t()).double()
    # [K][N] weights of 9 rows go through the tensor memory from 4 MB on
    adds = K / 512 if layout == "kn" and rows > 8 else K / warps / 512 + warps
    _check(lin.forward(x), want, adds, "y")


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("K,N", [(64, 96), (520, 264), (1024, 768)])
def test_weight_gradients(K, N, layout):
    import apk_b200
    M = 32768
    x, dy = _positive(M, K, seed=1), _positive(M, N, seed=2, scale=1 / M)
    w = _positive(*((K, N) if layout == "kn" else (N, K)), seed=3)
    lin = apk_b200.Linear(w, layout=layout)
    want = x.double().t() @ dy.double()
    for need_dx in (True, False):
        dw = lin.backward(dy, x, need_dx=need_dx, dw_dtype="f32")[1]
        _check(dw if layout == "kn" else dw.t(), want, M / 512 + 8, "dw")


@pytest.mark.parametrize("T", [2, 12, 30, 64])
@pytest.mark.parametrize("sms", [1, 0])
def test_experts(T, sms):
    """The hidden values are w_in's (x picks a column): exact, so that only the
    second product's sums are off."""
    import torch

    import apk_b200
    D, F = 256, 32768
    w_in, w_out = _positive(1, F, D, seed=1), _positive(1, D, F, seed=2, scale=1 / F)
    moe = apk_b200.MoE(_positive(1, D, seed=3), w_in, w_out, top_k=1, act="none", gated=False, out_dtype="f32", sms=sms)
    x = torch.eye(D, dtype=torch.bfloat16, device="cuda")[:T].contiguous()
    want = w_in[0, :, :T].t().double() @ w_out[0].t().double()
    _check(moe.forward(x), want, F / 512 + 16, "y")
    assert moe.status() == 0


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("T,E,k,D,F", [(1, 8, 2, 1024, 2048), (1, 4, 3, 8192, 264), (3, 60, 4, 1032, 520), (12, 16, 2, 2048, 1408),
                                       (30, 8, 4, 512, 4096), (64, 4, 2, 1024, 2048)])
def test_experts_of_an_fp32_result(T, E, k, D, F, gated):
    """The hidden values are two bf16 terms: each is off by at most 2^-17 of
    itself, the weights by the softmax's 2^-18 or so, the sums by less; a single
    bf16 term would be off by 2^-10 in the 2-norm."""
    import layer_bounds as lb
    import torch

    import apk_b200

    def rnd(*shape, seed, scale=1.0):
        g = torch.Generator("cuda").manual_seed(seed)
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0.0, scale, generator=g)

    router, w_in = rnd(E, D, seed=1, scale=D ** -0.5), rnd(E, 2 * F if gated else F, D, seed=2, scale=D ** -0.5)
    w_out, x = rnd(E, D, F, seed=3, scale=F ** -0.5), rnd(T, D, seed=4)
    moe = apk_b200.MoE(router, w_in, w_out, top_k=k, act="silu", gated=gated, out_dtype="f32")
    y, ids, _ = moe.forward(x, return_routing=True)
    want = lb.moe(x, router, w_in, w_out, ids.long(), "silu", gated, True)[0]
    assert float((y.double() - want).norm() / want.norm()) <= 2.0 ** -16 + 2.0 ** -18
    half = apk_b200.MoE(router, w_in, w_out, top_k=k, act="silu", gated=gated).forward(x)
    assert float((half.double() - want).norm() / want.norm()) <= 2.0 ** -7


@pytest.mark.parametrize("T", [1, 5, 40])
def test_infinite_hidden_values_of_an_fp32_result(T):
    """An infinity is one term, its rest none: it stays infinite."""
    import torch

    import apk_b200
    w_in = torch.zeros(1, 8, 8, dtype=torch.bfloat16, device="cuda")
    w_in[0, 0, 0] = 2.0 ** 100
    w_out = torch.zeros(1, 8, 8, dtype=torch.bfloat16, device="cuda")
    w_out[0, 0, 0] = 1.0
    x = torch.zeros(T, 8, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = 2.0 ** 100
    for out in ("f32", "bf16"):
        moe = apk_b200.MoE(torch.zeros(1, 8, dtype=torch.bfloat16, device="cuda"), w_in, w_out, top_k=1, act="none",
                           gated=False, out_dtype=out)
        y = moe.forward(x)
        assert bool((y[:, 0] == float("inf")).all())
        assert bool(torch.isnan(y[:, 1:]).all())      # 0 x inf
