"""The feed-forward operators as they are measured: a linear layer with its
epilogue, its backward pass, and a mixture-of-experts layer for a few tokens.

linear      y = act(x W + b) + r               x [M, K], W [K, N] ("kn") or [N, K] ("nk")
linear_bwd  dz = dy * act'(z),  dx = dz W^T,  dW = x^T dz (W's layout),  db = sum over rows of dz
moe         logits = x Wr^T;  the k largest (ties to the lowest index) with their softmax
            probabilities p (renormalised over the k, or not);
            y = sum_j p_j * (act(x G_j^T) * (x U_j^T)) D_j^T, or without U where not gated

Where `own` is false, run() computes them by elementary torch operations in
32 bits; where it is true, through this package's entry points.
"""
import math

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------- the cases
def _lin(name, M, K, N, layout="kn", act="none", bias="f32", residual=False, save=False, out="bf16"):
    return {"name": name, "op": "linear", "M": M, "K": K, "N": N, "layout": layout, "act": act, "bias": bias,
            "residual": residual, "save": save, "out": out}


def _bwd(name, M, K, N, layout="kn", act="none", bias="f32"):
    return {"name": name, "op": "linear_bwd", "M": M, "K": K, "N": N, "layout": layout, "act": act, "bias": bias}


def _moe(name, T, E, k, D, F, act="silu", gated=True, renorm=True):
    return {"name": name, "op": "moe", "T": T, "E": E, "k": k, "D": D, "F": F, "act": act, "gated": gated,
            "renorm": renorm}


def listed():
    return [
        # one token being decoded through a small projection: latency alone
        _lin("linear_one_token", 1, 2048, 2048, layout="nk", act="silu", bias="bf16"),
        # a decoding batch through a wide up-projection, weights as the GEMM runtime lays them out
        _lin("linear_8_tokens", 8, 4096, 8192, act="gelu_tanh", residual=True),
        # a short prompt with odd sizes: no row of x, W or y starts on a 16-byte boundary
        _lin("linear_ragged", 333, 1001, 1537, act="gelu", residual=True, save=True),
        # a training step's up-projection: the pre-activation is kept for the backward pass
        _lin("linear_train", 2048, 4096, 8192, act="gelu_tanh", save=True),
        # the runtime's largest background GEMM as a layer, with the block's residual stream
        _lin("linear_large", 8192, 8192, 8192, layout="nk", bias="bf16", residual=True),
        # gradients of a small layer in a small batch
        _bwd("linear_bwd_small", 128, 1024, 1024, layout="nk", act="relu", bias="bf16"),
        # gradients at odd sizes
        _bwd("linear_bwd_ragged", 777, 1001, 2050, act="silu"),
        # gradients of the training step's up-projection
        _bwd("linear_bwd_train", 4096, 4096, 8192, act="gelu_tanh"),
        # one token, a few coarse experts
        _moe("moe_one_token", 1, 8, 2, 1024, 2048),
        # a few tokens, many fine experts of which few are chosen
        _moe("moe_few_tokens", 5, 64, 6, 2048, 1408, renorm=False),
        # ungated experts
        _moe("moe_ungated", 16, 16, 2, 2048, 4096, act="gelu", gated=False),
        # the largest batch that still decodes token by token: nearly every expert is read
        _moe("moe_64_tokens", 64, 128, 8, 4096, 1536),
    ]


ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size between lo and hi, even in its logarithm; one in three stays as odd as it falls, the others are multiples of 8."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 1 / 3 else max(lo, n // 8 * 8)


def draw(rng):
    op = rng.choice(("linear", "linear", "linear_bwd", "moe"))
    if op == "moe":
        while True:
            c = _moe("", _log(rng, 1, 64), rng.choice((4, 8, 16, 32, 60, 64, 128, 160, 256)), rng.randint(1, 8),
                     _log(rng, 256, 7168) // 8 * 8, _log(rng, 256, 8192) // 8 * 8, act=rng.choice(ACTS[1:]),
                     gated=rng.random() < 0.75, renorm=rng.random() < 0.5)
            if c["k"] <= c["E"] and c["E"] * c["D"] * c["F"] <= 128 * 4096 * 1536:
                break
    else:
        most = 8192 ** 3 if op == "linear" else 4096 * 4096 * 8192
        while True:
            M = _log(rng, 1, 8192) if rng.random() < 0.75 else _log(rng, 1, 64)
            K, N = _size(rng, 64, 8192), _size(rng, 64, 8192)
            if 64 * 64 <= M * K * N <= most:
                break
        layout, act, bias = rng.choice(("kn", "nk")), rng.choice(ACTS), rng.choice(("none", "f32", "bf16"))
        if op == "linear":
            c = _lin("", M, K, N, layout, act, bias, rng.random() < 0.5, rng.random() < 0.3,
                     "f32" if rng.random() < 0.2 else "bf16")
        else:
            c = _bwd("", M, K, N, layout, act, bias)
    del c["name"]
    return c


# ---------------------------------------------------------------- the inputs
def _inputs(case, seed):
    """The case's input tensors, on the GPU, from the seed alone."""
    g = torch.Generator(DEV)
    g.manual_seed(int(seed))

    def rnd(*shape, scale=1.0, dtype=torch.bfloat16):
        t = torch.empty(shape, dtype=dtype, device=DEV)
        t.normal_(0.0, scale, generator=g)
        return t

    if case["op"] == "moe":
        T, E, D, F = case["T"], case["E"], case["D"], case["F"]
        return {"x": rnd(T, D), "router": rnd(E, D, scale=D ** -0.5),
                "w_in": rnd(E, 2 * F if case["gated"] else F, D, scale=D ** -0.5),
                "w_out": rnd(E, D, F, scale=F ** -0.5)}
    M, K, N = case["M"], case["K"], case["N"]
    d = {"x": rnd(M, K), "w": rnd(*((K, N) if case["layout"] == "kn" else (N, K)), scale=K ** -0.5),
         "bias": None if case["bias"] == "none" else rnd(N, scale=0.5, dtype=DT[case["bias"]])}
    if case["op"] == "linear":
        d["residual"] = rnd(M, N) if case["residual"] else None
    else:
        d["dy"] = rnd(M, N)
        d["z"] = None if case["act"] == "none" else rnd(M, N)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    if not own:
        return case, d, None
    import apk_b200
    if case["op"] == "moe":
        plan = apk_b200.MoE(d["router"], d["w_in"], d["w_out"], top_k=case["k"], act=case["act"], gated=case["gated"],
                            renormalize=case["renorm"])
    else:
        plan = apk_b200.Linear(d["w"], d["bias"], act=case["act"], layout=case["layout"],
                               out_dtype=case.get("out", "bf16"))
    return case, d, plan


# ---------------------------------------------------------------- the plain forms
def _act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), z)  # a NaN stays one
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z / (1.0 + torch.exp(-z))


def _act_grad(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    if name == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _plain_linear(case, d):
    w = d["w"].float()
    z = d["x"].float() @ (w if case["layout"] == "kn" else w.t())
    if d["bias"] is not None:
        z = z + d["bias"].float()
    y = _act(case["act"], z)
    if d["residual"] is not None:
        y = y + d["residual"].float()
    y = y.to(DT[case["out"]])
    return (y, z.to(torch.bfloat16)) if case["save"] else y


def _plain_linear_bwd(case, d):
    dz = d["dy"].float()
    if case["act"] != "none":
        dz = dz * _act_grad(case["act"], d["z"].float())
    w, x, b = d["w"].float(), d["x"].float(), torch.bfloat16
    if case["layout"] == "kn":
        dx, dw = dz @ w.t(), x.t() @ dz
    else:
        dx, dw = dz @ w, dz.t() @ x
    return dx.to(b), dw.to(b), None if d["bias"] is None else dz.sum(0).to(d["bias"].dtype)


def _plain_moe(case, d):
    x, k, F = d["x"].float(), case["k"], case["F"]
    logits = x @ d["router"].float().t()
    top = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    e = torch.exp(logits - logits.amax(1, keepdim=True))
    p = (e / e.sum(1, keepdim=True)).gather(1, top)
    if case["renorm"]:
        p = p / p.sum(1, keepdim=True)
    if case["T"] * k <= case["E"]:  # the chosen experts' weights, one set for each token and choice
        w_in, w_out = d["w_in"][top.reshape(-1)].float(), d["w_out"][top.reshape(-1)].float()
        a = (w_in @ x.repeat_interleave(k, 0).unsqueeze(2)).squeeze(2)
        h = _act(case["act"], a[:, :F]) * a[:, F:] if case["gated"] else _act(case["act"], a)
        o = (w_out @ h.unsqueeze(2)).reshape(case["T"], k, case["D"])
        return (o * p.unsqueeze(2)).sum(1).to(torch.bfloat16)
    a = x @ d["w_in"].float().transpose(1, 2)  # every token through every expert
    h = _act(case["act"], a[..., :F]) * a[..., F:] if case["gated"] else _act(case["act"], a)
    o = h @ d["w_out"].float().transpose(1, 2)
    share = torch.zeros_like(logits).scatter(1, top, p)
    return (o * share.t().unsqueeze(2)).sum(0).to(torch.bfloat16)


def run(state):
    case, d, plan = state
    if case["op"] == "moe":
        return plan.forward(d["x"]) if own else _plain_moe(case, d)
    if case["op"] == "linear":
        return plan.forward(d["x"], residual=d["residual"], save_preact=case["save"]) if own else _plain_linear(case, d)
    return plan.backward(d["dy"], d["x"], preact=d["z"]) if own else _plain_linear_bwd(case, d)


# ---------------------------------------------------------------- what they cannot do without
def work(case):
    if case["op"] == "moe":
        T, E, k, D, F = (case[n] for n in ("T", "E", "k", "D", "F"))
        per = (3 if case["gated"] else 2) * D * F
        active = E * (1.0 - (1.0 - k / E) ** T)  # experts that some token chooses, where all are as likely
        return {"bytes": 2.0 * (active * per + E * D + 2 * T * D), "flops": 2.0 * T * (k * per + E * D)}
    M, K, N = case["M"], case["K"], case["N"]
    b = {"none": 0, "f32": 4, "bf16": 2}[case["bias"]] * N
    if case["op"] == "linear":
        out = 4 if case["out"] == "f32" else 2
        return {"bytes": 2.0 * (M * K + K * N) + b + M * N * (out + 2 * case["residual"] + 2 * case["save"]),
                "flops": 2.0 * M * K * N}
    return {"bytes": 4.0 * (M * K + K * N) + 2 * b + M * N * (2 if case["act"] == "none" else 4),
            "flops": 4.0 * M * K * N}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_act(name, z):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
    return z * torch.sigmoid(z) if name == "silu" else z


def _exact_slope(name, z):
    if name == "none":
        return torch.ones_like(z)
    z = z.clone().requires_grad_(True)
    return torch.autograd.grad(_exact_act(name, z).sum(), z)[0]


def exact(case, seed):
    d = {n: None if v is None else v.double() for n, v in _inputs(case, seed).items() if n not in ("w_in", "w_out")}
    if case["op"] == "moe":
        whole = _inputs(case, seed)
        logits = torch.einsum("td,ed->te", d["x"], d["router"])
        y = torch.zeros_like(d["x"])
        for t in range(case["T"]):
            chosen = sorted(range(case["E"]), key=lambda e, row=logits[t].tolist(): (-row[e], e))[:case["k"]]
            p = torch.softmax(logits[t], 0)[chosen]
            p = p / p.sum() if case["renorm"] else p
            for e, share in zip(chosen, p):
                a = torch.mv(whole["w_in"][e].double(), d["x"][t])
                h = _exact_act(case["act"], a[:case["F"]])
                h = h * a[case["F"]:] if case["gated"] else h
                y[t] += share * torch.mv(whole["w_out"][e].double(), h)
        return y
    w = d["w"] if case["layout"] == "kn" else d["w"].t()
    if case["op"] == "linear":
        z = torch.einsum("mk,kn->mn", d["x"], w)
        z = z if d["bias"] is None else z + d["bias"]
        y = _exact_act(case["act"], z)
        y = y if d["residual"] is None else y + d["residual"]
        return (y, z) if case["save"] else y
    dz = d["dy"] if d["z"] is None else d["dy"] * _exact_slope(case["act"], d["z"])
    dx = torch.einsum("mn,kn->mk", dz, w)
    dw = torch.einsum("mk,mn->kn", d["x"], dz)
    return dx, dw if case["layout"] == "kn" else dw.t(), None if d["bias"] is None else dz.sum(0)
