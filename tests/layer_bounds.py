"""64-bit references of the layer operators with a bound for every element.

The bounds follow from how the kernels compute, before any run:
  U      unit roundoff of bf16 (8 significant bits): a result rounded once
  sum_err(k) * sum |a||b|   an fp32 sum of k exact products: the tensor core
         truncates (2^-23 a step) and pieces are added with rounding
  ACT_REL   the activations' hardware exponential and reciprocal, a few 2^-22
         of the argument's and result's size
"""
import torch

U = 2.0 ** -8
ACT_REL = 2.0 ** -19
LIP = 1.13  # largest slope of an activation (gelu: 1.129)
TINY = 2.0 ** -120


def sum_err(k):
    # chains of at most 512 products, 16 a step for the tensor core, then
    # pieces and ranks; one more for the bias and one for safety
    return (min(k, 512) + k / 512 + 16) * 2.0 ** -23


def act(name, z):
    if name == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3))
    return z * torch.sigmoid(z) if name == "silu" else z


def slope(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    z = z.clone().requires_grad_(True)
    return torch.autograd.grad(act(name, z).sum(), z)[0]


def rounded(y, err, dtype):
    """Bound of |result - y| where the value before rounding is within err."""
    u = U if dtype == torch.bfloat16 else 2.0 ** -23
    return err + u * (y.abs() + err) + TINY


def linear(x, w_kn, bias, name, residual, out_dtype):
    """(y, bound of y, z, bound of the stored z)."""
    x, w = x.double(), w_kn.double()
    z, size = x @ w, x.abs() @ w.abs()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    ez = sum_err(x.shape[-1]) * size
    y = act(name, z)
    ey = LIP * ez + ACT_REL * (z.abs() + y.abs())
    if residual is not None:
        y = y + residual.double()
        ey = ey + 2.0 ** -23 * (y.abs() + residual.double().abs())
    return y, rounded(y, ey, out_dtype), z, rounded(z, ez, torch.bfloat16)


def linear_grads(x, w_kn, z, name, dy, dw_dtype=torch.bfloat16, db_dtype=torch.float32):
    """((dx, bound), (dW as [K, N], bound), (db, bound))."""
    x, w, dy = x.double(), w_kn.double(), dy.double()
    dz = dy if name == "none" else dy * slope(name, z.double())
    edz = (0.0 if name == "none" else ACT_REL) * dy.abs()
    # the products' operand is rounded to bf16 (exact without an activation)
    eop = edz if name == "none" else edz + U * (dz.abs() + edz)
    size = dz.abs() + eop
    m, n = dy.shape
    dx = dz @ w.t()
    ex = eop @ w.t().abs() + sum_err(n) * (size @ w.t().abs())
    dw = x.t() @ dz
    ew = x.t().abs() @ eop + sum_err(m) * (x.t().abs() @ size)
    db = dz.sum(0)
    eb = edz.sum(0) + (m + 64) * 2.0 ** -24 * dz.abs().sum(0)
    return ((dx, rounded(dx, ex, torch.bfloat16)), (dw, rounded(dw, ew, dw_dtype)),
            (db, rounded(db, eb, db_dtype)))


def moe(x, router, w_in, w_out, ids, name, gated, renorm):
    """For the given choice of experts: (y, bound before rounding, weights,
    relative bound of the weights, logits, bound of the logits)."""
    x, r = x.double(), router.double()
    logits = x @ r.t()
    el = sum_err(x.shape[1]) * (x.abs() @ r.abs().t())
    p = torch.softmax(logits, 1).gather(1, ids)
    rel = 2 * el.amax(1, keepdim=True) + 2.0 ** -17  # exp of a difference of two logits, and the divisions
    if renorm:
        p, rel = p / p.sum(1, keepdim=True), 2 * rel
    y, ey = torch.zeros_like(x), torch.zeros_like(x)
    f = w_out.shape[2]
    for t in range(x.shape[0]):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            wi, wo = w_in[e].double(), w_out[e].double()
            a, ea = wi @ x[t], sum_err(x.shape[1]) * (wi.abs() @ x[t].abs())
            h = act(name, a[:f])
            eh = LIP * ea[:f] + ACT_REL * (a[:f].abs() + h.abs())
            if gated:
                eh = eh * (a[f:].abs() + ea[f:]) + h.abs() * ea[f:]
                h = h * a[f:]
            eh = eh + U * (h.abs() + eh)
            o, eo = wo @ h, wo.abs() @ eh + sum_err(f) * (wo.abs() @ (h.abs() + eh))
            y[t] += p[t, j] * o
            ey[t] += p[t, j] * (eo + (rel[t, 0] + 2.0 ** -22) * o.abs())
    return y, ey, p, rel, logits, el


def check(got, want, bound, what=""):
    d = (got.double() - want).abs()
    bad = ~(d <= bound)
    if bool(bad.any()):
        i = int(torch.argmax(torch.where(torch.isnan(d), torch.full_like(d, torch.inf), d / bound)))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; at {i} got {got.flatten()[i]} want "
                             f"{want.flatten()[i]} bound {bound.flatten()[i]:.3g}")
