"""forward(out=...) over its own operands: refused where a value would be read
after it was written, allowed where views only lie side by side."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(libapk):
    return libapk


def _layer(K, N):
    import torch

    import apk_b200
    g = torch.Generator("cuda").manual_seed(1)
    return apk_b200.Linear(torch.empty(K, N, dtype=torch.bfloat16, device="cuda").normal_(0.0, K ** -0.5, generator=g))


def _rand(*shape, seed=2):
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)


def test_refused():
    lin = _layer(64, 64)
    for rows in (3, 200):
        flat = _rand(rows * 200)
        x = flat[:rows * 64].view(rows, 64)
        wide = flat.view(rows, 200)
        other = _rand(rows, 64, seed=3)
        for x_, out in ((x, x), (x, flat[8:8 + rows * 64].view(rows, 64)), (wide[:, :64], wide[:, 60:124]),
                        (wide[:, 60:124], wide[:, :64]), (x, wide[:, 100:164])):
            with pytest.raises(ValueError, match="shares memory with x"):
                lin.forward(x_, out=out)
        for res, out in ((wide[:, :64], wide[:, 8:72]), (x, flat[64:64 + rows * 64].view(rows, 64))):
            with pytest.raises(ValueError, match="residual"):
                lin.forward(other, residual=res, out=out)


def test_allowed():
    import torch
    lin = _layer(64, 64)
    for rows in (1, 3, 200):
        flat = _rand(rows * 400)
        other = _rand(rows, 64, seed=3)
        want = lin.forward(other, residual=other)
        wide, pairs = flat.view(rows, 400), flat.view(2 * rows, 200)
        for x, res, out in ((wide[:, :64], wide[:, 64:128], wide[:, 128:192]), (wide[:, 336:], wide[:, 200:264], wide[:, :64]),
                            (pairs[0::2, :64], pairs[0::2, 64:128], pairs[1::2, :64]),
                            (pairs[1::2, 3:67], pairs[0::2, 70:134], pairs[0::2, 6:70])):
            x.copy_(other)
            res.copy_(other)
            assert torch.equal(lin.forward(x, residual=res, out=out), want)
            res.copy_(other)
            assert torch.equal(lin.forward(x, residual=res, out=res), want)     # in place
        assert lin.forward(other[:0], out=other[:0]).shape == (0, 64)
