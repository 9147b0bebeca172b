"""The layer operators as a program uses them: a feed-forward block trained
for a few steps, then a routed block that decodes token by token.

    python -m apk_b200.ffn [--steps 30] [--rows 2048] [--d-model 1024] [--d-ff 4096] [--tokens 64]

Training: y = x + act(x W1 + b1) W2 + b2 against a fixed random block of the
same shape, mean squared error, plain SGD on fp32 master weights.  The
forward pass keeps the pre-activation; the residual is added in the second
layer's epilogue.  Decoding: h = e + moe(e), logits = h Wv; the largest logit
names the next token.  The decoding step is captured once in a CUDA graph.
No counterpart in the reference, which multiplies bare matrices
(src/tcyield.cu:91-356).
"""
from __future__ import annotations

import argparse
import math

import torch

import apk_b200


class Block:
    """x + act(x W1 + b1) W2 + b2 with fp32 master weights."""

    def __init__(self, d_model: int, d_ff: int, seed: int, act: str = "gelu_tanh"):
        g = torch.Generator("cuda")
        g.manual_seed(seed)

        def rnd(*shape, scale):
            return torch.empty(shape, device="cuda").normal_(0.0, scale, generator=g)

        self.master = [rnd(d_model, d_ff, scale=d_model ** -0.5), rnd(d_ff, scale=0.1),
                       rnd(d_ff, d_model, scale=d_ff ** -0.5), rnd(d_model, scale=0.1)]
        w1, b1, w2, b2 = self.master
        self.up = apk_b200.Linear(w1.bfloat16(), b1, act=act)
        self.down = apk_b200.Linear(w2.bfloat16(), b2)

    def forward(self, x):
        h, z = self.up.forward(x, save_preact=True)
        return self.down.forward(h, residual=x), (x, h, z)

    def backward(self, dy, saved):
        """(dx, the gradients in the order of `master`)."""
        x, h, z = saved
        dh, dw2, db2 = self.down.backward(dy, h, dw_dtype="f32")
        dx, dw1, db1 = self.up.backward(dh, x, preact=z, dw_dtype="f32")
        return dx + dy, [dw1, db1, dw2, db2]

    def step(self, grads, lr: float):
        for p, g in zip(self.master, grads):
            p.sub_(g, alpha=lr)
        # the layers keep pointers to their weights: updated where they stand
        self.up.weight.copy_(self.master[0])
        self.down.weight.copy_(self.master[2])


def train(steps: int = 30, rows: int = 2048, d_model: int = 1024, d_ff: int = 4096, lr: float | None = None, seed: int = 0):
    """Losses of `steps` steps on fresh random rows, and us per step.  The
    loss's curvature grows with the rows' squared length, d_model: so does the
    reciprocal of the default learning rate."""
    lr = 4.0 / d_model if lr is None else lr
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    block, teacher = Block(d_model, d_ff, seed + 1), Block(d_model, d_ff, seed + 2)
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
        block.step(grads, lr)
    ended.record()
    torch.cuda.synchronize()
    return [float(v) for v in losses], began.elapsed_time(ended) * 1e3 / max(1, steps - min(3, steps - 1))


def decode(tokens: int = 64, d_model: int = 1024, d_ff: int = 1024, experts: int = 32, top_k: int = 4,
           vocabulary: int = 4096, seed: int = 0):
    """The tokens that follow token 0, and us per token."""
    g = torch.Generator("cuda")
    g.manual_seed(seed)

    def rnd(*shape, scale=1.0):
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0.0, scale, generator=g)

    embedding = rnd(vocabulary, d_model)
    moe = apk_b200.MoE(rnd(experts, d_model, scale=d_model ** -0.5), rnd(experts, 2 * d_ff, d_model, scale=d_model ** -0.5),
                       rnd(experts, d_model, d_ff, scale=d_ff ** -0.5), top_k=top_k)
    head = apk_b200.Linear(rnd(vocabulary, d_model, scale=d_model ** -0.5), layout="nk", out_dtype="f32")
    token = torch.zeros(1, dtype=torch.int64, device="cuda")
    said = torch.empty(tokens, dtype=torch.int64, device="cuda")

    def step():
        e = embedding[token]
        token.copy_(head.forward(e + moe.forward(e)).argmax(1))

    step()  # scratch is allocated by a first call, which a capture may not do
    torch.cuda.synchronize()
    token.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    began, ended = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    began.record()
    for i in range(tokens):
        graph.replay()
        said[i].copy_(token[0])
    ended.record()
    torch.cuda.synchronize()
    assert moe.status() == 0 and head.status() == 0
    return said.tolist(), began.elapsed_time(ended) * 1e3 / tokens


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("steps", 30), ("rows", 2048), ("d-model", 1024), ("d-ff", 4096), ("tokens", 64)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    losses, us = train(a.steps, a.rows, a.d_model, a.d_ff)
    flops = 2 * 2 * a.rows * a.d_model * a.d_ff * 4  # block: two layers forward and twice that back; teacher: forward
    print(f"train: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps, {us:.0f} us a step, "
          f"{flops / us / 1e6:.0f} TFLOP/s of products")
    said, us = decode(a.tokens, a.d_model)
    print(f"decode: {a.tokens} tokens, {us:.1f} us a token, first ones {said[:8]}")
    assert math.isfinite(losses[-1])


if __name__ == "__main__":
    main()
