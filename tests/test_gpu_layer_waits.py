"""Layer operators whose device waits run out.  A limit of one nanosecond makes
ordinary waits give up (nothing is faulted or held up): the kernel has to end
by itself, report a status and leave the GPU as it found it."""
import time

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


# sums long enough that the epilogue's wait for the first accumulator runs out:
# one CTA, a CTA pair, accumulators of 512 k, K split over a cluster
FORWARD = [(128, 128, 1 << 20, "kn", "bf16", 1), (128, 128, 1 << 20, "nk", "bf16", 1), (512, 512, 1 << 18, "kn", "bf16", 2),
           (512, 512, 1 << 18, "nk", "bf16", 2), (512, 256, 1 << 18, "kn", "f32", 2), (64, 64, 1 << 20, "kn", "bf16", 8)]


@pytest.mark.parametrize("M,N,K,layout,out,sms", FORWARD)
def test_a_product_that_gives_up_ends_and_leaves_no_trace(M, N, K, layout, out, sms):
    import layer_bounds as lb
    import torch

    import apk_b200
    w = _rand(*((K, N) if layout == "kn" else (N, K)), seed=1, scale=K ** -0.5)
    x = _rand(M, K, seed=2)
    short = apk_b200.Linear(w, act="silu", layout=layout, out_dtype=out, sms=sms, wait_limit_ns=1)
    torch.cuda.synchronize()
    began = time.monotonic()
    for _ in range(3):
        short.forward(x)
        # (an fp32 result's waits, for 512 k each, may be met before they are looked at)
        assert short.status() in ((1, 2) if out == "bf16" else (0, 1, 2)) and short.status() == 0
    assert time.monotonic() - began < 10          # unwinding is bounded by a second each
    lin = apk_b200.Linear(w[:520] if layout == "kn" else w[:, :520], act="silu", layout=layout, out_dtype=out, sms=sms)
    for rows in (5, M):                           # the same SMs, their tensor memory and shared memory
        want, by, _, _ = lb.linear(x[:rows, :520], w[:520] if layout == "kn" else w[:, :520].t(), None, "silu", None,
                                   lin.out_dtype)
        lb.check(lin.forward(x[:rows, :520]), want, by, "a call that follows")
    assert lin.status() == 0


@pytest.mark.parametrize("layout,sms", [("kn", 2), ("nk", 1)])
def test_gradients_that_give_up_end(layout, sms):
    import layer_bounds as lb
    import torch

    import apk_b200
    M, K, N = 1 << 18, 512, 256
    w = _rand(*((K, N) if layout == "kn" else (N, K)), seed=1, scale=K ** -0.5)
    x, dy = _rand(M, K, seed=2), _rand(M, N, seed=3)
    bias = torch.zeros(N, device="cuda")
    short = apk_b200.Linear(w, bias, act="silu", layout=layout, sms=sms, wait_limit_ns=1)
    short.backward(dy, x, preact=dy)
    assert short.status() in (1, 2) and short.status() == 0
    # db is summed before the products, without a wait
    _, _, db = short.backward(dy[:300], x[:300], preact=dy[:300])
    short.status()
    (_, _), (_, _), (want, eb) = lb.linear_grads(x[:300], w if layout == "kn" else w.t(), dy[:300], "silu", dy[:300])
    lb.check(db, want, eb, "db")
    lin = apk_b200.Linear(w, bias, act="silu", layout=layout, sms=sms)
    got = lin.backward(dy[:300], x[:300], preact=dy[:300])
    want = lb.linear_grads(x[:300], w if layout == "kn" else w.t(), dy[:300], "silu", dy[:300])
    for g, (ref, bound), what in zip((got[0], got[1] if layout == "kn" else got[1].t(), got[2]), want, ("dx", "dw", "db")):
        lb.check(g, ref, bound, what)
    assert lin.status() == 0
