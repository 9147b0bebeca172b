"""The layer operators together, as apk_b200/ffn.py uses them."""
import pytest

pytestmark = pytest.mark.gpu


def test_block_gradients_against_64_bit_autograd(libapk):
    """Through two layers and the residual.  Every value that is handed on is
    rounded to bf16 (h, z, dy, dh, dz): the sums of 64 or 96 such values stay
    within 5 roundings of the gradient's size in the 2-norm."""
    import layer_bounds as lb
    import torch

    from apk_b200.ffn import Block
    block = Block(64, 96, seed=3)
    x = torch.randn(200, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    dy = torch.randn(200, 64, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    y, saved = block.forward(x)
    dx, grads = block.backward(dy, saved)
    p = [t.double().requires_grad_(True) for t in (x, block.up.weight, block.up.bias, block.down.weight, block.down.bias)]
    want = p[0] + lb.act("gelu_tanh", p[0] @ p[1] + p[2]) @ p[3] + p[4]
    want.backward(dy.double())
    for got, ref in ((y, want.detach()), (dx, p[0].grad), *zip(grads, (t.grad for t in p[1:]))):
        assert float((got.double() - ref).norm() / ref.norm()) <= 5 * lb.U


def test_training_lowers_the_loss(libapk):
    from apk_b200.ffn import train
    losses, us = train(steps=40, rows=512, d_model=128, d_ff=256)
    assert losses[-1] < 0.7 * losses[0] and us > 0
    assert losses == train(steps=40, rows=512, d_model=128, d_ff=256)[0], "a second run differs"


def test_decoding_in_a_graph_repeats(libapk):
    from apk_b200.ffn import decode
    a, _ = decode(tokens=12, d_model=256, d_ff=128, experts=8, top_k=2, vocabulary=512)
    b, _ = decode(tokens=12, d_model=256, d_ff=128, experts=8, top_k=2, vocabulary=512)
    assert a == b and len(set(a)) > 1
