"""The layers hold their weights' addresses: weights that have moved are
refused, not read where they were."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(libapk):
    return libapk


def _rand(*shape, seed):
    import torch
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)


def _set(layer, name, w):
    setattr(layer, name, w)


def _data(layer, name, w):
    getattr(layer, name).data = w


def _freed(layer, name, w):
    getattr(layer, name).untyped_storage().resize_(0)


@pytest.mark.parametrize("move", [_set, _data, _freed])
@pytest.mark.parametrize("name", ["weight", "bias"])
def test_linear(name, move):
    import apk_b200
    w, b = _rand(64, 32, seed=1), _rand(32, seed=2)
    lin = apk_b200.Linear(w, b)
    x = _rand(5, 64, seed=3)
    y = lin.forward(x)
    move(lin, name, _rand(*{"weight": (64, 32), "bias": (32,)}[name], seed=4))
    with pytest.raises(ValueError, match="new layer"):
        lin.forward(x)
    with pytest.raises(ValueError, match="new layer"):
        lin.backward(y, x)


def test_linear_without_the_bias_it_was_made_with():
    import apk_b200
    lin = apk_b200.Linear(_rand(64, 32, seed=1), _rand(32, seed=2))
    lin.bias = None
    with pytest.raises(ValueError, match="new layer"):
        lin.forward(_rand(5, 64, seed=3))


@pytest.mark.parametrize("move", [_set, _data, _freed])
@pytest.mark.parametrize("name", ["router", "w_in", "w_out"])
def test_moe(name, move):
    import apk_b200
    shapes = {"router": (4, 64), "w_in": (4, 64, 64), "w_out": (4, 64, 32)}
    moe = apk_b200.MoE(*(_rand(*s, seed=i) for i, s in enumerate(shapes.values())), top_k=2)
    x = _rand(3, 64, seed=9)
    moe.forward(x)
    move(moe, name, _rand(*shapes[name], seed=7))
    with pytest.raises(ValueError, match="new layer"):
        moe.forward(x)


def test_a_weight_transposed_in_place_keeps_the_gradients_shape():
    """dw has the shape that the layer was made with: rows of another length
    would be written past their end."""
    import torch

    import apk_b200
    w, x, dy = _rand(96, 32, seed=1), _rand(5, 96, seed=2), _rand(5, 32, seed=3)
    lin = apk_b200.Linear(w)
    want = lin.backward(dy, x)[1]
    w.t_()
    got = lin.backward(dy, x)[1]
    assert got.shape == (96, 32) and torch.equal(got, want)


def test_shorter_views_at_the_same_address():
    """The memory has not moved, and gradients have the size that the layer was made with."""
    import torch

    import apk_b200
    w, b, x, dy = _rand(64, 32, seed=1), _rand(32, seed=2), _rand(500, 64, seed=3), _rand(500, 32, seed=4)
    lin = apk_b200.Linear(w, b)
    want = lin.backward(dy, x)
    lin.weight, lin.bias = w[:8], b[:3]
    assert all(torch.equal(p, q) for p, q in zip(lin.backward(dy, x), want))
    g, c = _rand(64, seed=5), _rand(64, seed=6)
    norm = apk_b200.LayerNorm(g, c)
    y, stats = norm.forward(x, save_stats=True)
    for rows in (5, 500):
        want = norm.backward(x[:rows], x[:rows], stats[:rows])
        norm.weight, norm.bias = g[:8], c[:3]
        got = norm.backward(x[:rows], x[:rows], stats[:rows])
        assert [tuple(t.shape) for t in got] == [(rows, 64), (64,), (64,)] and all(torch.equal(p, q) for p, q in zip(got, want))
        norm.weight, norm.bias = g, c
