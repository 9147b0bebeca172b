"""Layer operators whose device waits run out.  A limit of one nanosecond makes
ordinary waits give up (nothing is faulted or held up): the kernel has to end
by itself, report a status and leave the GPU as it found it."""
import ctypes
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


def _slow_moe(wait_limit_ns, tokens=1):
    """One expert of 8 hidden values over 2^20 inputs: one CTA reads it for a
    few hundred microseconds while the others wait at the grid barrier."""
    import apk_b200
    D = 1 << 20
    moe = apk_b200.MoE(_rand(1, D, seed=1, scale=D ** -0.5), _rand(1, 16, D, seed=2, scale=D ** -0.5),
                       _rand(1, D, 8, seed=3, scale=8 ** -0.5), top_k=1, wait_limit_ns=wait_limit_ns)
    return moe, _rand(tokens, D, seed=4)


@pytest.mark.parametrize("tokens", [1, 3, 20])
def test_a_grid_barrier_that_gives_up_every_time(tokens):
    import torch

    from apk_b200 import _lib as L
    moe, x = _slow_moe(1, tokens)
    for _ in range(3):
        # a barrier whose words were left half counted would let a second call pass
        moe.forward(x)
        assert moe.status() == 3 and moe.status() == 0
    # until status() has been asked, further calls touch no output
    moe.forward(x)
    y, ids, probs = moe.forward(x, return_routing=True)
    y.fill_(7.0)
    io = L.MoeIO(x=x.data_ptr(), ldx=x.shape[1], tokens=tokens, y=y.data_ptr(), ldy=x.shape[1], y_dtype=L.APK_BF16,
                 stream=torch.cuda.current_stream().cuda_stream)
    assert moe._lib.apk_moe_forward(moe._h, ctypes.byref(io)) == L.APK_OK
    torch.cuda.synchronize()
    assert bool((y == 7.0).all())
    assert moe.status() == 3
    ok, _ = _slow_moe(0, tokens)
    first = ok.forward(x)
    assert bool(torch.isfinite(first).all()) and torch.equal(first, ok.forward(x)) and ok.status() == 0


def test_a_graph_whose_barrier_gave_up_starts_anew():
    import torch
    moe, x = _slow_moe(1)
    moe.forward(x)
    assert moe.status() == 3
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moe.forward(x)
    more = _rand(20, x.shape[1], seed=5)
    moe.forward(more)                                # the scratch grows: the graph has a buffer of its own
    assert moe.status() == 3
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert moe.status() == 3 and moe.status() == 0
