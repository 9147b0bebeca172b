"""Layer operators in CUDA graphs: what else runs at the same time, or is gone
by then, changes no result."""
import gc

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


def _linear(M=1500):
    """A layer whose every call uses scratch (odd rows, an activation), and a
    call of it: a forward and a backward pass over one of eight inputs."""
    import torch

    import apk_b200
    K, N = 1001, 333
    lin = apk_b200.Linear(_rand(K, N, seed=1, scale=K ** -0.5), torch.zeros(N, device="cuda"), act="silu")
    xs = [_rand(M, K, seed=10 + i) for i in range(8)]
    dys = [_rand(M, N, seed=30 + i) for i in range(8)]
    zs = [_rand(M, N, seed=50 + i) for i in range(8)]
    return lin, lambda i: (lin.forward(xs[i]), *lin.backward(dys[i], xs[i], preact=zs[i]))


def _moe(T=40):
    import apk_b200
    E, D, F = 16, 512, 512
    moe = apk_b200.MoE(_rand(E, D, seed=1, scale=D ** -0.5), _rand(E, 2 * F, D, seed=2, scale=D ** -0.5),
                       _rand(E, D, F, seed=3, scale=F ** -0.5), top_k=4)
    xs = [_rand(T, D, seed=10 + i) for i in range(8)]
    return moe, lambda i: (moe.forward(xs[i]),)


MAKE = {"linear": _linear, "moe": _moe}


def _equal(a, b):
    import torch
    return all(torch.equal(x, y) for x, y in zip(a, b))


def _capture(f, *inputs):
    import torch
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [f(i) for i in inputs]
    return graph, outs


@pytest.mark.parametrize("kind", MAKE)
def test_parallel_branches_of_one_graph(kind):
    import torch
    layer, f = MAKE[kind]()
    want = [f(i) for i in range(8)]
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        other.wait_stream(main)
        outs = {}
        for i in range(4):
            outs[i] = f(i)
            with torch.cuda.stream(other):
                outs[4 + i] = f(4 + i)
        main.wait_stream(other)
    for _ in range(10):
        for o in outs.values():
            for t in o:
                t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(_equal(outs[i], want[i]) for i in range(8))
    assert layer.status() == 0


@pytest.mark.parametrize("kind", MAKE)
def test_replays_beside_calls_and_another_graph(kind):
    import torch
    layer, f = MAKE[kind]()
    want = [f(i) for i in range(8)]
    torch.cuda.synchronize()
    (g0, o0), (g1, o1) = _capture(f, 0, 1), _capture(f, 2, 3)
    s0, s1 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(s0):
            g0.replay()
        with torch.cuda.stream(s1):
            g1.replay()
        direct = [f(i) for i in range(4, 8)]
        torch.cuda.synchronize()
        assert all(_equal(a, b) for a, b in zip(o0 + o1 + direct, want))
        for t in (t for o in o0 + o1 for t in o):
            t.zero_()
    assert layer.status() == 0


@pytest.mark.parametrize("kind", MAKE)
def test_a_graph_outlives_its_layer(kind):
    import torch
    layer, f = MAKE[kind]()
    want = f(0)
    graph, (out,) = _capture(f, 0)
    weights = [v for v in vars(layer).values() if isinstance(v, torch.Tensor)]  # the caller's to keep
    layer.close()
    del layer
    gc.collect()
    # the library's next allocations would reuse what it had freed, and clear it
    others = [MAKE[kind]() for _ in range(3)]
    for _, g in others:
        again = g(1)
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert _equal(out, want)
    assert weights and _equal(others[0][1](1), again)


def test_capturing_again_and_again_keeps_no_memory():
    import torch
    layer, f = _linear(6000)                         # 16 MB of scratch a capture
    want = f(0)

    def once():
        graph, (out,) = _capture(f, 0)
        graph.replay()
        torch.cuda.synchronize()
        assert _equal(out, want)
        del graph, out
        gc.collect()
        torch.cuda.empty_cache()

    for _ in range(3):
        once()
    before = torch.cuda.mem_get_info()[0]
    for _ in range(20):
        once()
    assert before - torch.cuda.mem_get_info()[0] < 64 << 20
    layer.close()
