"""The operators together, as apk_b200/ffn.py uses them: a model trained on
tokens with clipped gradients, and decoding through a 4-bit head with scores."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(libapk):
    return libapk


def _reference(model, tokens, targets, dlp, dh):
    """64-bit autograd through the same formulas: (log probabilities,
    entropies, gradients in the order of master).  bf16 weights as they are."""
    import layer_bounds as lb
    import torch
    b = model.block
    p = [model.embedding.bfloat16(), model.head.weight, model.last.weight, model.last.bias, b.up.weight, b.up.bias,
         b.down.weight, b.down.bias, b.norm.weight, b.norm.bias]
    p = [t.double().requires_grad_(True) for t in p]
    emb, head, g2, c2, w1, b1, w2, b2, g1, c1 = p

    def norm(x, g, c):
        d = x - x.mean(1, keepdim=True)
        return d * (d.square().mean(1, keepdim=True) + 1e-5).rsqrt() * g + c

    x = emb[tokens]
    y = x + lb.act("gelu_tanh", norm(x, g1, c1) @ w1 + b1) @ w2 + b2
    l = torch.log_softmax(norm(y, g2, c2) @ head.t(), 1)
    logprob = l.gather(1, targets.clamp(min=0)[:, None])[:, 0] * (targets >= 0)
    entropy = -(l.exp() * l).sum(1)
    ((logprob * dlp.double()).sum() + (entropy * dh.double()).sum()).backward()
    return logprob.detach(), entropy.detach(), [t.grad for t in p]


def test_model_gradients_against_64_bit_autograd():
    """Every value that is handed on is rounded to bf16 (x, n, h, z, y, n, the
    logits, and their gradients back): ten roundings on the longest way, each
    2^-8 of a value at most and 2^-9.8 in the mean square, and what the logits'
    roundings move of the probabilities, which is of the logits' size, about 4,
    times theirs: within 16 of 2^-8 in the 2-norm."""
    import layer_bounds as lb
    import torch

    from apk_b200.ffn import TokenModel
    model = TokenModel(vocabulary=500, d_model=64, d_ff=96, seed=3)
    g = torch.Generator("cuda").manual_seed(5)
    tokens, targets = (torch.randint(0, 500, (300,), device="cuda", generator=g) for _ in range(2))
    targets[::7] = -1
    dlp = torch.empty(300, device="cuda").normal_(generator=g)
    dh = 0.1 * torch.empty(300, device="cuda").normal_(generator=g)
    logprob, entropy, saved = model.forward(tokens, targets)
    grads = model.backward(dlp, saved, dentropy=dh)
    want = _reference(model, tokens, targets, dlp, dh)
    for got, ref in zip((logprob, entropy, *grads), (want[0], want[1], *want[2])):
        assert float((got.double() - ref).norm() / ref.norm()) <= 16 * lb.U


def test_a_step_with_clipped_gradients():
    """One step against the same step taken from the gradients by hand."""
    import torch

    import apk_b200
    from apk_b200.ffn import TokenModel
    model = TokenModel(vocabulary=257, d_model=72, d_ff=40, seed=1)
    g = torch.Generator("cuda").manual_seed(2)
    tokens, targets = (torch.randint(0, 257, (130,), device="cuda", generator=g) for _ in range(2))
    _, _, saved = model.forward(tokens, targets)
    grads = model.backward(torch.full((130,), -1.0, device="cuda"), saved)
    kept, before = [t.clone() for t in grads], [p.clone() for p in model.master]
    norm = float(apk_b200.GradClip(0.5).clip(grads))
    want = float(torch.cat([t.double().flatten() for t in kept]).norm())
    assert abs(norm - want) <= 1e-6 * want and want > 0.5
    model.step(grads, lr=0.1)
    for p, b, t in zip(model.master, before, kept):
        assert torch.allclose(p.double(), b.double() - 0.1 * t.double() * (0.5 / (want + 1e-6)), rtol=1e-6, atol=1e-6)
    assert torch.equal(model.head.weight, model.master[1].bfloat16())
    assert torch.equal(model.block.up.weight, model.master[4].bfloat16())


def test_block_with_a_norm_and_training_repeat():
    from apk_b200.ffn import train, train_tokens
    kw = dict(steps=6, rows=256, d_model=128, d_ff=256)
    a, us = train(**kw, norm=True, max_norm=0.5)
    assert a == train(**kw, norm=True, max_norm=0.5)[0] and us > 0 and len(a) == 6
    a, norms, us = train_tokens(**kw, vocabulary=300)
    b, again, _ = train_tokens(**kw, vocabulary=300)
    assert len(a) == 6 and a[0] == b[0] and norms[0] == again[0] and us > 0    # (index_add_ of the embedding's gradient may order its sums anew)


def test_decoding_through_a_4_bit_head_with_scores():
    """What is said are the largest logits of the layers called one by one, and the scores are the distribution's."""
    import torch

    import apk_b200
    from apk_b200.ffn import decode
    kw = dict(tokens=10, d_model=256, d_ff=128, experts=8, top_k=2, vocabulary=512)
    said, us, logprob, entropy, ids, alternatives = decode(**kw, head_bits=4, top=5)
    again = decode(**kw, head_bits=4, top=5)
    assert said == again[0] and torch.equal(ids, again[4]) and torch.equal(alternatives, again[5])
    assert said == ids[:, 0].tolist() and us > 0 and decode(**kw, head_bits=4)[0] == said
    # the layers that decode() makes, called without a graph
    g = torch.Generator("cuda")
    g.manual_seed(0)

    def rnd(*shape, scale=1.0):
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0.0, scale, generator=g)

    embedding = rnd(512, 256)
    moe = apk_b200.MoE(rnd(8, 256, scale=1 / 16), rnd(8, 256, 256, scale=1 / 16), rnd(8, 256, 128, scale=128 ** -0.5), top_k=2)
    w4, s, _ = apk_b200.Linear4.quantize(rnd(512, 256, scale=1 / 16), group=64)
    full = (torch.stack((w4 & 15, w4 >> 4), 2).view(512, 256).double() - 8) * s.double().repeat_interleave(64, 1)
    token = 0
    for i, t in enumerate(said):
        e = embedding[token][None]
        l = torch.log_softmax((e + moe.forward(e)).double() @ full.t(), 1)[0]
        assert abs(float(l[t]) - float(logprob[i])) < 1e-4 and abs(float(-(l.exp() * l).sum()) - float(entropy[i])) < 1e-4
        assert float((l[ids[i].long()] - alternatives[i]).abs().max()) < 1e-4 and float(l.max() - l[t]) < 1e-4
        token = t
