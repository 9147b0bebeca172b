"""Streaming linear layers in a row: each may start while the one before it
still runs, and reads what that one writes."""
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


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("rows,d", [(1, 512), (8, 1024), (16, 1001)])
def test_a_chain_through_the_same_buffers(rows, d, layout):
    """x -> a -> b -> a -> b ... in place of fresh tensors: a value that is read
    too early is the last step's."""
    import torch

    import apk_b200
    layers = [apk_b200.Linear(_rand(d, d, seed=i, scale=d ** -0.5), act="silu", layout=layout) for i in range(6)]
    x = _rand(rows, d, seed=99)
    want = [x]
    for lin in layers:                               # one at a time
        torch.cuda.synchronize()
        want.append(lin.forward(want[-1]))
    torch.cuda.synchronize()
    a, b = torch.empty_like(x), torch.empty_like(x)

    def chain():
        a.copy_(x)
        src, dst = a, b
        for lin in layers:
            lin.forward(src, out=dst)
            src, dst = dst, src
        return src

    for _ in range(100):
        last = chain()
    torch.cuda.synchronize()
    assert torch.equal(last, want[-1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(20):
            last = chain()
    for _ in range(10):
        last.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(last, want[-1])


def test_weights_written_by_the_layer_before():
    import torch

    import apk_b200
    first = apk_b200.Linear(_rand(256, 2048, seed=1, scale=1 / 16))
    w = torch.empty(16, 2048, dtype=torch.bfloat16, device="cuda")
    second = {"nk": apk_b200.Linear(w, layout="nk"), "kn": apk_b200.Linear(w, layout="kn")}
    v = {"nk": _rand(3, 2048, seed=2), "kn": _rand(3, 16, seed=3)}
    xs = [_rand(16, 256, seed=10 + i) for i in range(2)]
    want = []
    for x in xs:
        first.forward(x, out=w)
        torch.cuda.synchronize()
        want.append({k: second[k].forward(v[k]) for k in second})
        torch.cuda.synchronize()
    for i in range(200):
        k = "nk" if i & 2 else "kn"
        first.forward(xs[i & 1], out=w)
        got = second[k].forward(v[k])
        assert torch.equal(got, want[i & 1][k]), i
