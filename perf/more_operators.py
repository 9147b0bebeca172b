"""The operators around the feed-forward block as they are measured: layer
norm with its gradients, the clipping of gradients by their global norm, log
probabilities of given tokens, and a linear layer with 4-bit weights.

norm        n = (x - mean) rstd over the last axis, y = n w + b;  stats are (mean, rstd)
norm_bwd    g = dy w;  dx = rstd (g - mean(g) - n mean(g n)) + residual gradient,
            dw = sum over rows of dy n,  db = sum over rows of dy
grad_norm   sqrt of the sum of all squares of many tensors
clip        the same, and every tensor times min(1, max_norm / (norm + 1e-6))
logprobs    l = x - max - log S,  S = sum exp(x - max);  l[token] (0 for a negative token),
            the entropy, the largest logits' indices (ties to the lowest index) and their l
logprobs_bwd  dx_j = dlogprob ([j = token] - p_j) - dentropy p_j (l_j + entropy)
linear4     y = act(x W^T + b) + r,  W[n][k] = s[n][k / G] (q[n][k] - z[n][k / G]), q of 4 bits

Where `own` is false, run() computes them by elementary torch operations in
32 bits; where it is true, through this package's entry points.
"""
import math

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------- the cases
def _norm(name, M, D, x="bf16", w="f32", bias=True, out="bf16", stats=True):
    return {"name": name, "op": "norm", "M": M, "D": D, "x": x, "w": w, "bias": bias, "out": out, "stats": stats}


def _norm_bwd(name, M, D, x="bf16", dy="bf16", w="f32", bias=True, residual=True):
    return {"name": name, "op": "norm_bwd", "M": M, "D": D, "x": x, "dy": dy, "w": w, "bias": bias,
            "residual": residual}


def _clip(name, op, tensors, total, types="f32"):
    return {"name": name, "op": op, "tensors": tensors, "total": total, "types": types}


def _logprobs(name, op, M, V, dtype="f32", top=0, masked=0):
    return {"name": name, "op": op, "M": M, "V": V, "dtype": dtype, "top": top, "masked": masked}


def _lin4(name, M, K, N, group=128, zeros=False, act="none", bias="none", residual=False, out="bf16"):
    return {"name": name, "op": "linear4", "M": M, "K": K, "N": N, "group": group, "zeros": zeros, "act": act,
            "bias": bias, "residual": residual, "out": out}


def listed():
    return [
        # one token being decoded: latency alone
        _norm("norm_one_token", 1, 2048, stats=False),
        # a packed batch of odd size from an fp32 residual stream, its statistics kept for the backward pass
        _norm("norm_ragged", 1537, 1001, x="f32"),
        # a training step's norm, with the residual stream's gradient added to dx
        _norm_bwd("norm_bwd_train", 8192, 4096),
        # gradients at odd sizes, in a short batch
        _norm_bwd("norm_bwd_ragged", 333, 1001, w="bf16", residual=False),
        # the gradients of a small block, fp32 as the linear layers give them
        _clip("clip_block", "clip", 4, 8393728),
        # a whole model's gradients: many small tensors and a few large ones, of both types; only watched
        _clip("norm_of_many", "grad_norm", 300, 100000001, types="mixed"),
        # the same order of size, clipped into the optimizer's fp32 buffers
        _clip("clip_large", "clip", 48, 268435456),
        # one decoded token with the alternatives a server reports
        _logprobs("logprobs_one_token", "logprobs", 1, 131072, top=20),
        # scoring a long prompt from bf16 logits, the vocabulary odd and padded with masked entries
        _logprobs("logprobs_score", "logprobs", 2048, 100003, "bf16", top=5, masked=61),
        # the loss's gradient in a training step on tokens
        _logprobs("logprobs_bwd_train", "logprobs_bwd", 4096, 32768, "bf16"),
        # one token through a wide projection
        _lin4("linear4_one_token", 1, 4096, 8192, act="silu"),
        # a decoding batch, small groups with zero points, the block's residual stream
        _lin4("linear4_16_tokens", 16, 8192, 4096, group=32, zeros=True, bias="f32", residual=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size between lo and hi, even in its logarithm; one in three stays as odd as it falls, the others are multiples of 8."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 1 / 3 else max(lo, n // 8 * 8)


def draw(rng):
    op = rng.choice(("norm", "norm_bwd", "grad_norm", "clip", "logprobs", "logprobs", "logprobs_bwd", "linear4", "linear4"))
    if op in ("norm", "norm_bwd"):
        while True:
            M, D = _log(rng, 1, 16384), _size(rng, 16, 16384)
            if M * D <= 8192 * 4096:
                break
        x, w, other = (rng.choice(("bf16", "f32")) for _ in range(3))
        if op == "norm":
            c = _norm("", M, D, x, w, rng.random() < 0.75, other, rng.random() < 0.5)
        else:
            # fp32 on both sides moves twice the bytes
            c = _norm_bwd("", M if M * D <= 8192 * 2048 else (M + 1) // 2, D, x, other, w, rng.random() < 0.75,
                          rng.random() < 0.5)
    elif op == "grad_norm":
        n = _log(rng, 1, 400)
        c = _clip("", op, n, max(4 * n, _log(rng, 1000, 100000000)), rng.choice(("f32", "bf16", "mixed")))
    elif op == "clip":
        n = _log(rng, 1, 60)
        c = _clip("", op, n, max(4 * n, _log(rng, 1000, 268435456)), rng.choice(("f32", "bf16")))
    elif op == "logprobs":
        while True:
            M, V = _log(rng, 1, 4096), _size(rng, 32, 200000)
            if M * V <= 2048 * 100003:
                break
        dtype = rng.choice(("bf16", "f32")) if M * V <= 1024 * 100003 else "bf16"
        c = _logprobs("", op, M, V, dtype, rng.choice((0, 1, 5, 8, 20)), rng.choice((0, 0, V // 16)))
    elif op == "logprobs_bwd":
        while True:
            M, V = _log(rng, 1, 8192), _size(rng, 32, 200000)
            if M * V <= 4096 * 32768:
                break
        dtype = rng.choice(("bf16", "f32")) if M * V <= 2048 * 32768 else "bf16"
        c = _logprobs("", op, M, V, dtype, 0, rng.choice((0, 0, V // 16)))
    else:
        M = _log(rng, 1, 64) if rng.random() < 0.75 else _log(rng, 64, 512)
        while True:
            K, N = _log(rng, 256, 16384) // 32 * 32, _size(rng, 64, 16384)
            if K * N <= 4096 * 8192 and M * K * N <= 64 * 4096 * 8192:
                break
        c = _lin4("", M, K, N, rng.choice((32, 64, 128)), rng.random() < 0.5, rng.choice(("none", "relu", "gelu_tanh", "silu")),
                  rng.choice(("none", "f32", "bf16")), rng.random() < 0.5, "f32" if rng.random() < 0.2 else "bf16")
    del c["name"]
    return c


# ---------------------------------------------------------------- the inputs
def _sizes(case):
    """The tensors' sizes: two thirds of them vectors, the others matrices of one to sixteen shares of the rest, most of
    them of whole 64s.  The last matrix takes what is left over, the vectors are as odd as they fall."""
    n, left = case["tensors"], case["total"]
    small = [max(1, min(left // (4 * n), 1 + 257 * i % 8191)) for i in range(n - 1) if i % 3]
    left -= sum(small)
    shares = [1 + i * 7 % 16 for i in range(n - len(small))]
    sizes = [left * s // sum(shares) for s in shares]
    sizes = [max(1, k if k < 64 else k // 64 * 64) for k in sizes]
    sizes[-1] += max(0, left - sum(sizes))
    return sizes + small


def _inputs(case, seed):
    """The case's input tensors, on the GPU, from the seed alone."""
    g = torch.Generator(DEV)
    g.manual_seed(int(seed))

    def rnd(*shape, scale=1.0, mean=0.0, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device=DEV).normal_(mean, scale, generator=g)

    op = case["op"]
    if op in ("norm", "norm_bwd"):
        M, D = case["M"], case["D"]
        d = {"x": rnd(M, D, scale=2.0, mean=0.3, dtype=DT[case["x"]]), "w": rnd(D, scale=0.2, mean=1.0, dtype=DT[case["w"]]),
             "b": rnd(D, scale=0.2, dtype=DT[case["w"]]) if case["bias"] else None}
        if op == "norm_bwd":
            d["dy"] = rnd(M, D, dtype=DT[case["dy"]])
            d["r"] = rnd(M, D, dtype=DT[case["x"]]) if case["residual"] else None
            x = d["x"].double()
            mean = x.mean(1)
            d["stats"] = torch.stack((mean, (x.square().mean(1) - mean.square() + 1e-5).rsqrt()), 1).float()
        return d
    if op in ("grad_norm", "clip"):
        kinds = {"f32": ("f32",), "bf16": ("bf16",), "mixed": ("bf16", "f32", "bf16")}[case["types"]]
        return {"grads": [rnd(n, scale=0.01 * (1 + i % 5), dtype=DT[kinds[i % len(kinds)]])
                          for i, n in enumerate(_sizes(case))]}
    if op in ("logprobs", "logprobs_bwd"):
        M, V, masked = case["M"], case["V"], case["masked"]
        d = {"x": rnd(M, V, scale=3.0, dtype=DT[case["dtype"]])}
        if masked:
            d["x"][:, V - masked:] = -math.inf
        tokens = torch.randint(0, V - masked, (M,), device=DEV, generator=g)
        # a batch's padding: every eighth row, where there are as many
        d["tokens"] = torch.where(torch.arange(M, device=DEV) % 8 == 7, torch.full_like(tokens, -1), tokens)
        if op == "logprobs_bwd":
            d["dlogprob"], d["dentropy"] = rnd(M, dtype=torch.float32), rnd(M, scale=0.01, dtype=torch.float32)
            top, s, h = [], [], []
            for rows in d["x"].split(256):
                t = rows.double()
                m = t.amax(1, keepdim=True)
                e = (t - m).exp()
                top.append(m[:, 0])
                s.append(e.sum(1))
                h.append(s[-1].log() - torch.where(e > 0, e * (t - m), 0.0).sum(1) / s[-1])
            d["stats"] = torch.stack((torch.cat(top), torch.cat(s).log()), 1).float()
            d["entropy"] = torch.cat(h).float()
        return d
    M, K, N, G = case["M"], case["K"], case["N"], case["group"]
    groups = -(-K // G)
    w = torch.zeros(N, groups * G, device=DEV)
    w[:, :K].normal_(0.0, K ** -0.5, generator=g)
    w = w.view(N, groups, G)
    if case["zeros"]:
        low, high = w.amin(2).clamp(max=0), w.amax(2).clamp(min=0)
        s = ((high - low) / 15).bfloat16()
        z = torch.round(-low / s.float()).clamp(0, 15)
    else:
        s = (w.abs().amax(2) / 7).bfloat16()
        z = torch.full((N, groups), 8.0, device=DEV)
    q = torch.round(w / s.float()[:, :, None] + z[:, :, None]).clamp(0, 15).to(torch.uint8).view(N, -1)[:, :K]
    return {"x": rnd(M, K), "w": q[:, 0::2] | (q[:, 1::2] << 4), "s": s, "z": z.to(torch.uint8) if case["zeros"] else None,
            "b": None if case["bias"] == "none" else rnd(N, scale=0.5, dtype=DT[case["bias"]]),
            "r": rnd(M, N) if case["residual"] else None}


MAX_NORM = 1.0  # below the norm of every case's gradients of ordinary size


def prepare(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "clip":
        # the optimizer's own gradient buffer, of which the tensors' places are views
        d["flat"] = torch.empty(sum(t.numel() for t in d["grads"]), dtype=d["grads"][0].dtype, device=DEV)
        d["out"] = list(d["flat"].split([t.numel() for t in d["grads"]]))
    if not own:
        return case, d, None
    import apk_b200
    op = case["op"]
    if op in ("norm", "norm_bwd"):
        plan = apk_b200.LayerNorm(d["w"], d["b"], out_dtype=case.get("out", "bf16"))
    elif op in ("grad_norm", "clip"):
        plan = apk_b200.GradClip(MAX_NORM)
    elif op in ("logprobs", "logprobs_bwd"):
        plan = apk_b200.LogProbs(top=case["top"])
    else:
        plan = apk_b200.Linear4(d["w"], d["s"], zeros=d["z"], bias=d["b"], group=case["group"], act=case["act"],
                                out_dtype=case["out"])
    return case, d, plan


# ---------------------------------------------------------------- the plain forms
def _plain_norm(case, d):
    x = d["x"].float()
    mean = x.sum(1, keepdim=True) / case["D"]
    c = x - mean
    rstd = 1.0 / torch.sqrt((c * c).sum(1, keepdim=True) / case["D"] + 1e-5)
    y = c * rstd * d["w"].float()
    if d["b"] is not None:
        y = y + d["b"].float()
    y = y.to(DT[case["out"]])
    return (y, torch.cat((mean, rstd), 1)) if case["stats"] else y


def _plain_norm_bwd(case, d):
    mean, rstd = d["stats"][:, :1], d["stats"][:, 1:]
    n, dy = (d["x"].float() - mean) * rstd, d["dy"].float()
    g = dy * d["w"].float()
    dx = rstd * (g - g.sum(1, keepdim=True) / case["D"] - n * ((g * n).sum(1, keepdim=True) / case["D"]))
    if d["r"] is not None:
        dx = dx + d["r"].float()
    dw, db = (dy * n).sum(0), dy.sum(0)
    return dx.to(d["x"].dtype), dw.to(d["w"].dtype), None if d["b"] is None else db.to(d["b"].dtype)


def _plain_grad_norm(d):
    parts = [t.float() for t in d["grads"]]
    return torch.sqrt(torch.stack([(t * t).sum() for t in parts]).sum())


def _plain_clip(d):
    norm = _plain_grad_norm(d)
    c = torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)
    for t, out in zip(d["grads"], d["out"]):
        out.copy_(t.float() * c)
    return norm, d["flat"]


def _plain_logprobs(case, d):
    x, tokens = d["x"].float(), d["tokens"]
    m = x.amax(1, keepdim=True)
    t = x - m
    e = torch.exp(t)
    s = e.sum(1, keepdim=True)
    log_s = torch.log(s)
    at = tokens.clamp(min=0)[:, None]
    lp = torch.where(tokens < 0, 0.0, (t.gather(1, at) - log_s)[:, 0])
    entropy = (log_s - torch.where(e > 0, e * t, 0.0).sum(1, keepdim=True) / s)[:, 0]
    if not case["top"]:
        return lp, entropy, None, None
    # the largest by (value, lowest index): as integers that are ordered as the floats are, the index below them
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64) * 2 ** 32 - torch.arange(case["V"], device=DEV)
    ids = torch.topk(key, case["top"], dim=1).indices
    return lp, entropy, ids.to(torch.int32), t.gather(1, ids) - log_s


def _plain_logprobs_bwd(case, d):
    x, tokens = d["x"].float(), d["tokens"][:, None]
    lp = x - d["stats"][:, :1] - d["stats"][:, 1:]
    p = torch.exp(lp)
    dlp = torch.where(tokens < 0, 0.0, d["dlogprob"][:, None])
    dx = -dlp * p - d["dentropy"][:, None] * torch.where(p > 0, p * (lp + d["entropy"][:, None]), 0.0)
    return dx.scatter_add(1, tokens.clamp(min=0), dlp).to(d["x"].dtype)


def _act(name, z):
    if name == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), z)
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z / (1.0 + torch.exp(-z)) if name == "silu" else z


def _plain_linear4(case, d):
    N, K, G = case["N"], case["K"], case["group"]
    q = torch.stack((d["w"] & 15, d["w"] >> 4), 2).view(N, K).float()
    group = torch.arange(K, device=DEV) // G
    z = 8.0 if d["z"] is None else d["z"].float()[:, group]
    y = d["x"].float() @ ((q - z) * d["s"].float()[:, group]).t()
    if d["b"] is not None:
        y = y + d["b"].float()
    y = _act(case["act"], y)
    if d["r"] is not None:
        y = y + d["r"].float()
    return y.to(DT[case["out"]])


def run(state):
    case, d, plan = state
    op = case["op"]
    if op == "norm":
        return plan.forward(d["x"], save_stats=case["stats"]) if own else _plain_norm(case, d)
    if op == "norm_bwd":
        return plan.backward(d["dy"], d["x"], d["stats"], residual_grad=d["r"]) if own else _plain_norm_bwd(case, d)
    if op == "grad_norm":
        return plan.norm(d["grads"]) if own else _plain_grad_norm(d)
    if op == "clip":
        return (plan.clip(d["grads"], out=d["out"]), d["flat"]) if own else _plain_clip(d)
    if op == "logprobs":
        return plan.forward(d["x"], d["tokens"]) if own else _plain_logprobs(case, d)
    if op == "logprobs_bwd":
        if own:
            return plan.backward(d["dlogprob"], d["x"], d["tokens"], d["stats"], dentropy=d["dentropy"], entropy=d["entropy"])
        return _plain_logprobs_bwd(case, d)
    return plan.forward(d["x"], residual=d["r"]) if own else _plain_linear4(case, d)


# ---------------------------------------------------------------- what they cannot do without
SIZE = {"bf16": 2, "f32": 4}


def work(case):
    op = case["op"]
    if op in ("norm", "norm_bwd"):
        n, D, w = case["M"] * case["D"], case["D"], SIZE[case["w"]] * (1 + case["bias"])
        if op == "norm":
            return {"bytes": n * (SIZE[case["x"]] + SIZE[case["out"]]) + D * w + 8.0 * case["M"] * case["stats"], "flops": 8.0 * n}
        return {"bytes": n * (SIZE[case["x"]] * (2 + case["residual"]) + SIZE[case["dy"]]) + D * (2 * w - SIZE[case["w"]] * case["bias"])
                + 8.0 * case["M"], "flops": 14.0 * n}
    if op in ("grad_norm", "clip"):
        kinds = {"f32": (4,), "bf16": (2,), "mixed": (2, 4, 2)}[case["types"]]
        b = sum(n * kinds[i % len(kinds)] for i, n in enumerate(_sizes(case)))
        return {"bytes": b * (2.0 if op == "clip" else 1.0), "flops": 2.0 * case["total"]}
    if op in ("logprobs", "logprobs_bwd"):
        n = float(case["M"] * case["V"])
        return {"bytes": n * SIZE[case["dtype"]] * (1 if op == "logprobs" else 2) + case["M"] * (16 + 8 * case["top"]), "flops": 6.0 * n}
    M, K, N = case["M"], case["K"], case["N"]
    groups = -(-K // case["group"])
    return {"bytes": N * (0.5 * K + groups * (2 + case["zeros"])) + 2.0 * M * K + {"none": 0, "f32": 4, "bf16": 2}[case["bias"]] * N
            + M * N * (SIZE[case["out"]] + 2 * case["residual"]), "flops": 2.0 * M * K * N}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    d, op = _inputs(case, seed), case["op"]
    wide = {n: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for n, v in d.items()
            if op not in ("logprobs", "logprobs_bwd") or n != "x"}
    if op == "norm":
        x = wide["x"]
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + 1e-5) * wide["w"]
        y = y if d["b"] is None else y + wide["b"]
        return (y, torch.cat((mean, torch.rsqrt(var + 1e-5)), 1)) if case["stats"] else y
    if op == "norm_bwd":
        x, w = wide["x"].requires_grad_(), wide["w"].requires_grad_()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + 1e-5) * w
        y.backward(wide["dy"])
        dx = x.grad if d["r"] is None else x.grad + wide["r"]
        return dx, w.grad, None if d["b"] is None else torch.einsum("md->d", wide["dy"])
    if op in ("grad_norm", "clip"):
        norm = math.sqrt(math.fsum(float(torch.dot(t.double(), t.double())) for t in d["grads"]))
        norm_t = torch.tensor(norm, dtype=torch.float64, device=DEV)
        if op == "grad_norm":
            return norm_t
        return norm_t, torch.cat([t.double() * min(1.0, MAX_NORM / (norm + 1e-6)) for t in d["grads"]])
    if op in ("logprobs", "logprobs_bwd"):
        outs = []
        for i in range(0, case["M"], 128):  # 64-bit rows by the batch: they are large
            rows = slice(i, i + 128)
            lp = torch.log_softmax(d["x"][rows].double(), 1)
            p, tokens = lp.exp(), d["tokens"][rows]
            h = -torch.special.xlogy(p, p).sum(1)
            real = tokens >= 0
            hot = torch.zeros_like(lp)
            hot[real, tokens[real]] = 1.0
            if op == "logprobs_bwd":
                dl = wide["dlogprob"][rows] * real
                dx = dl[:, None] * (hot - p) - wide["dentropy"][rows][:, None] * (torch.special.xlogy(p, p) + p * h[:, None])
                outs.append((dx.float(),) if case["M"] > 128 else (dx,))  # (what is rounded here is far below bf16's)
                continue
            got = [(torch.where(hot > 0, lp, 0.0)).sum(1), h]
            if case["top"]:
                ids = torch.argsort(d["x"][rows], dim=1, descending=True, stable=True)[:, :case["top"]]
                got += [ids.int(), torch.take_along_dim(lp, ids, 1)]
            outs.append(got)
        outs = [torch.cat(o) for o in zip(*outs)]
        if op == "logprobs_bwd":
            return outs[0]
        return (*outs, None, None)[:4]
    q = torch.empty(case["N"], case["K"], dtype=torch.float64, device=DEV)
    q[:, 0::2], q[:, 1::2] = (d["w"] % 16).double(), torch.div(d["w"], 16, rounding_mode="floor").double()
    y = torch.zeros(case["M"], case["N"], dtype=torch.float64, device=DEV)
    for j in range(wide["s"].shape[1]):  # group by group, scaled behind the product
        ks = slice(j * case["group"], (j + 1) * case["group"])
        zero = 8.0 if d["z"] is None else d["z"][:, j, None].double()
        y += torch.einsum("mk,nk->mn", wide["x"][:, ks], q[:, ks] - zero) * wide["s"][:, j]
    y = y if d["b"] is None else y + wide["b"]
    if case["act"] == "relu":
        y = y.clamp(min=0)
    elif case["act"] == "gelu_tanh":
        y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
    elif case["act"] == "silu":
        y = y * torch.sigmoid(y)
    return y if d["r"] is None else y + wide["r"]
