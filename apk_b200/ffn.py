"""The layer operators as a program uses them: a feed-forward block trained
for a few steps, a small model trained on tokens, then a routed block that
decodes token by token.

    python -m apk_b200.ffn [--steps 30] [--rows 2048] [--d-model 1024] [--d-ff 4096] [--tokens 64]
                           [--norm] [--max-norm 1.0] [--vocabulary 4096] [--head-bits 4] [--top 5]

Training: y = x + act(x W1 + b1) W2 + b2 against a fixed random block of the
same shape, mean squared error, plain SGD on fp32 master weights.  The
forward pass keeps the pre-activation; the residual is added in the second
layer's epilogue.  With --norm the block's branch reads the layer norm of x,
with --max-norm gradients are clipped by their global norm.  Training on
tokens (with --norm): embedding, block, norm and head; the next token's log
probability is the loss, its gradient overwrites the logits.  Decoding:
h = e + moe(e), logits = h Wv; the largest logit names the next token.  With
--head-bits 4 the head has 4-bit weights; with --top every token is said with
its log probability, the distribution's entropy and alternatives.  The
decoding step is captured once in a CUDA graph.
No counterpart in the reference, which multiplies bare matrices
(src/tcyield.cu:91-356).
"""
from __future__ import annotations

import argparse
import math

import torch

import apk_b200


class Block:
    """x + act(n W1 + b1) W2 + b2 with fp32 master weights, n = x or with
    `norm` the layer norm of x."""

    def __init__(self, d_model: int, d_ff: int, seed: int, act: str = "gelu_tanh", norm: bool = False):
        g = torch.Generator("cuda")
        g.manual_seed(seed)

        def rnd(*shape, scale):
            return torch.empty(shape, device="cuda").normal_(0.0, scale, generator=g)

        self.master = [rnd(d_model, d_ff, scale=d_model ** -0.5), rnd(d_ff, scale=0.1),
                       rnd(d_ff, d_model, scale=d_ff ** -0.5), rnd(d_model, scale=0.1)]
        w1, b1, w2, b2 = self.master
        self.up = apk_b200.Linear(w1.bfloat16(), b1, act=act)
        self.down = apk_b200.Linear(w2.bfloat16(), b2)
        self.norm = None
        if norm:
            self.master += [1.0 + rnd(d_model, scale=0.1), rnd(d_model, scale=0.1)]
            self.norm = apk_b200.LayerNorm(*self.master[4:])

    def forward(self, x):
        n, stats = (x, None) if self.norm is None else self.norm.forward(x, save_stats=True)
        h, z = self.up.forward(n, save_preact=True)
        y = self.down.forward(h, residual=x)
        return y, (x, h, z) if self.norm is None else (x, h, z, n, stats)

    def backward(self, dy, saved):
        """(dx, the gradients in the order of `master`)."""
        x, h, z = saved[:3]
        dh, dw2, db2 = self.down.backward(dy, h, dw_dtype="f32")
        if self.norm is None:
            dx, dw1, db1 = self.up.backward(dh, x, preact=z, dw_dtype="f32")
            return dx + dy, [dw1, db1, dw2, db2]
        n, stats = saved[3:]
        dn, dw1, db1 = self.up.backward(dh, n, preact=z, dw_dtype="f32")
        dx, dg, db = self.norm.backward(dn, x, stats, residual_grad=dy)
        return dx, [dw1, db1, dw2, db2, dg, db]

    def step(self, grads, lr: float):
        for p, g in zip(self.master, grads):
            p.sub_(g, alpha=lr)
        # the layers keep pointers to their weights: updated where they stand
        self.up.weight.copy_(self.master[0])
        self.down.weight.copy_(self.master[2])


class TokenModel:
    """Embedding, a block with a norm, a last norm and a head over the
    vocabulary, with fp32 master weights."""

    def __init__(self, vocabulary: int, d_model: int, d_ff: int, seed: int):
        g = torch.Generator("cuda")
        g.manual_seed(seed)

        def rnd(*shape, scale):
            return torch.empty(shape, device="cuda").normal_(0.0, scale, generator=g)

        self.block = Block(d_model, d_ff, seed + 1, norm=True)
        self.embedding, head = rnd(vocabulary, d_model, scale=1.0), rnd(vocabulary, d_model, scale=d_model ** -0.5)
        last = [1.0 + rnd(d_model, scale=0.1), rnd(d_model, scale=0.1)]
        self.master = [self.embedding, head, *last, *self.block.master]
        self.head = apk_b200.Linear(head.bfloat16(), layout="nk")
        self.last = apk_b200.LayerNorm(*last)
        self.logprobs = apk_b200.LogProbs()

    def forward(self, tokens, targets):
        """(log probabilities of the targets, entropies, what backward() needs)."""
        y, block = self.block.forward(self.embedding[tokens].bfloat16())
        n, stats = self.last.forward(y, save_stats=True)
        logits = self.head.forward(n)
        logprob, entropy, _, _, sums = self.logprobs.forward(logits, targets, save_stats=True)
        return logprob, entropy, (tokens, targets, y, block, n, stats, logits, sums, entropy)

    def backward(self, dlogprob, saved, dentropy=None):
        """The gradients in the order of `master`.  Overwrites the logits."""
        tokens, targets, y, block, n, stats, logits, sums, entropy = saved
        dlogits = self.logprobs.backward(dlogprob, logits, targets, sums, dentropy=dentropy,
                                         entropy=None if dentropy is None else entropy, out=logits)
        dn, dhead, _ = self.head.backward(dlogits, n, dw_dtype="f32")
        dy, dg, db = self.last.backward(dn, y, stats)
        dx, grads = self.block.backward(dy, block)
        dembedding = torch.zeros_like(self.embedding).index_add_(0, tokens, dx.float())
        return [dembedding, dhead, dg, db, *grads]

    def step(self, grads, lr: float):
        for p, g in zip(self.master[:4], grads):
            p.sub_(g, alpha=lr)
        self.head.weight.copy_(self.master[1])
        self.block.step(grads[4:], lr)


def train(steps: int = 30, rows: int = 2048, d_model: int = 1024, d_ff: int = 4096, lr: float | None = None, seed: int = 0,
          norm: bool = False, max_norm: float | None = None):
    """Losses of `steps` steps on fresh random rows, and us per step.  The
    loss's curvature grows with the rows' squared length, d_model: so does the
    reciprocal of the default learning rate."""
    lr = 4.0 / d_model if lr is None else lr
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    block, teacher = Block(d_model, d_ff, seed + 1, norm=norm), Block(d_model, d_ff, seed + 2, norm=norm)
    clip = None if max_norm is None else apk_b200.GradClip(max_norm)
    losses, began, ended = [], torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for i in range(steps):
        if i == min(3, steps - 1):
            began.record()
        x = torch.empty(rows, d_model, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
        target, _ = teacher.forward(x)
        y, saved = block.forward(x)
        err = y.float() - target.float()
        losses.append(err.square().mean())
        _, grads = block.backward((err * (2.0 / rows)).bfloat16(), saved)
        if clip is not None:
            clip.clip(grads)
        block.step(grads, lr)
    ended.record()
    torch.cuda.synchronize()
    return [float(v) for v in losses], began.elapsed_time(ended) * 1e3 / max(1, steps - min(3, steps - 1))


def train_tokens(steps: int = 30, rows: int = 2048, vocabulary: int = 4096, d_model: int = 1024, d_ff: int = 4096,
                 lr: float = 1.0, max_norm: float = 1.0, seed: int = 0):
    """Losses, gradient norms before clipping, and us per step: every token is
    followed by the same other one, which the model learns."""
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    model, clip = TokenModel(vocabulary, d_model, d_ff, seed + 1), apk_b200.GradClip(max_norm)
    follows = torch.randperm(vocabulary, device="cuda", generator=g)
    dlogprob = torch.full((rows,), -1.0 / rows, device="cuda")
    losses, norms = [], []
    began, ended = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for i in range(steps):
        if i == min(3, steps - 1):
            began.record()
        tokens = torch.randint(0, vocabulary, (rows,), device="cuda", generator=g)
        logprob, _, saved = model.forward(tokens, follows[tokens])
        losses.append(-logprob.mean())
        grads = model.backward(dlogprob, saved)
        norms.append(clip.clip(grads))
        model.step(grads, lr)
    ended.record()
    torch.cuda.synchronize()
    us = began.elapsed_time(ended) * 1e3 / max(1, steps - min(3, steps - 1))
    return [float(v) for v in losses], [float(v) for v in norms], us


def decode(tokens: int = 64, d_model: int = 1024, d_ff: int = 1024, experts: int = 32, top_k: int = 4,
           vocabulary: int = 4096, seed: int = 0, head_bits: int = 16, top: int = 0):
    """The tokens that follow token 0, and us per token; with `top` also, for
    every token, its log probability, the entropy, and the alternatives with
    theirs."""
    g = torch.Generator("cuda")
    g.manual_seed(seed)

    def rnd(*shape, scale=1.0):
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0.0, scale, generator=g)

    embedding = rnd(vocabulary, d_model)
    moe = apk_b200.MoE(rnd(experts, d_model, scale=d_model ** -0.5), rnd(experts, 2 * d_ff, d_model, scale=d_model ** -0.5),
                       rnd(experts, d_model, d_ff, scale=d_ff ** -0.5), top_k=top_k)
    weight = rnd(vocabulary, d_model, scale=d_model ** -0.5)
    if head_bits == 4:
        w4, scales, _ = apk_b200.Linear4.quantize(weight, group=64)
        head = apk_b200.Linear4(w4, scales, group=64, out_dtype="f32")
    else:
        head = apk_b200.Linear(weight, layout="nk", out_dtype="f32")
    logprobs = apk_b200.LogProbs(top=top) if top else None
    token = torch.zeros(1, dtype=torch.int64, device="cuda")
    said = torch.empty(tokens, dtype=torch.int64, device="cuda")
    scores, now = [], None

    def step():
        e = embedding[token]
        logits = head.forward(e + moe.forward(e))
        if logprobs is None:
            token.copy_(logits.argmax(1))
            return None
        _, entropy, ids, alternatives = logprobs.forward(logits)  # the first alternative is what is said
        token.copy_(ids[:, 0])
        return entropy, ids, alternatives

    step()  # scratch is allocated by a first call, which a capture may not do
    torch.cuda.synchronize()
    token.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        now = step()
    began, ended = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    began.record()
    for i in range(tokens):
        graph.replay()
        said[i].copy_(token[0])
        if now is not None:
            scores.append([t[0].clone() for t in now])
    ended.record()
    torch.cuda.synchronize()
    assert moe.status() == 0 and head.status() == 0
    us = began.elapsed_time(ended) * 1e3 / tokens
    if not top:
        return said.tolist(), us
    entropy, ids, alternatives = (torch.stack(t) for t in zip(*scores))
    return said.tolist(), us, alternatives[:, 0], entropy, ids, alternatives


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("steps", 30), ("rows", 2048), ("d-model", 1024), ("d-ff", 4096), ("tokens", 64), ("vocabulary", 4096),
                        ("top", 0)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--norm", action="store_true")
    ap.add_argument("--max-norm", type=float)
    ap.add_argument("--head-bits", type=int, choices=(4, 16), default=16)
    a = ap.parse_args()
    losses, us = train(a.steps, a.rows, a.d_model, a.d_ff, norm=a.norm, max_norm=a.max_norm)
    flops = 2 * 2 * a.rows * a.d_model * a.d_ff * 4  # block: two layers forward and twice that back; teacher: forward
    print(f"train: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps, {us:.0f} us a step, "
          f"{flops / us / 1e6:.0f} TFLOP/s of products")
    if a.norm:
        losses, norms, us = train_tokens(a.steps, a.rows, a.vocabulary, a.d_model, a.d_ff, max_norm=1.0 if a.max_norm is None else a.max_norm)
        print(f"train on tokens: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps, {us:.0f} us a step, "
              f"gradient norm {norms[0]:.3f} -> {norms[-1]:.3f} before clipping")
    said, us, *scores = decode(a.tokens, a.d_model, vocabulary=a.vocabulary, head_bits=a.head_bits, top=a.top)
    print(f"decode: {a.tokens} tokens, {us:.1f} us a token, first ones {said[:8]}")
    if scores:
        logprob, entropy, ids, alternatives = (t.tolist() for t in scores)
        for i in range(min(4, a.tokens)):
            others = ", ".join(f"{j} {v:.3f}" for j, v in zip(ids[i], alternatives[i]))
            print(f"  {said[i]}: log probability {logprob[i]:.3f}, entropy {entropy[i]:.3f}, alternatives {others}")
    assert math.isfinite(losses[-1])


if __name__ == "__main__":
    main()
