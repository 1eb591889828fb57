"""The wide layers (vocabulary losses, gated feed-forward) in 64 bits from their definitions, with bounds on how far a
kernel may be off, counted rounding by rounding.

u = finfo(type).eps / 2 is the largest relative error of one rounding.  A dot product of n terms in fp32 is off by at
most n 2^-24 sum |a||b| (each partial sum is at most that large); fp32 operands of 22 bits add 3 2^-22 sum |a||b| (both
operands' and the dropped product of the low terms).
"""

import math

import torch

U32 = 2.0 ** -24


def u_of(dtype):
    return torch.finfo(dtype).eps / 2


def product_slack(n, dtype):
    """Relative to sum |a||b|: fp32 sums over n terms, and the operands' terms where they are fp32."""
    return n * U32 + (3 * 2.0 ** -22 if dtype == torch.float32 else 0.0)


def gradient_unit(dtype, rows):
    """Relative rounding of the gradient that the backward products take: the operands' type, or two terms of it (fp32: of
    fp16; the others: up to 256 rows)."""
    if dtype == torch.float32:
        return 2.0 ** -22
    return u_of(dtype) ** 2 if rows <= 256 else u_of(dtype)


def targets_of_labels(labels, ignore_index=-100):
    y = labels.flatten()
    live = y != ignore_index
    return torch.where(live, y, 0)[:, None], torch.ones_like(y, dtype=torch.float64)[:, None], live


def targets_of_teacher(logits, ids, temperature):
    t = logits.flatten(0, -2).double() / temperature
    i = ids.flatten(0, -2)
    held = (i >= 0) & (t != -math.inf)
    live = held.any(-1)
    t = torch.where(held, t, -math.inf)
    p = torch.softmax(torch.where(live[:, None], t, 0.0), -1) * held
    return torch.where(held, i, 0), p, live


def head(hidden, weight, ids, p, live, temperature, coef, rows=None):
    """Loss per row and gradients for sum_n coef[n] loss[n], with bounds: {name: (value, bound)}.  rows: of the call that
    these are a part of."""
    dtype = hidden.dtype
    X = torch.where(live[:, None], hidden.flatten(0, -2).double(), 0.0)
    W = weight.double()
    N, d = X.shape
    u, ug = u_of(dtype), gradient_unit(dtype, rows or N)
    z = X @ W.T / temperature
    lse = torch.logsumexp(z, -1, keepdim=True)
    log_q = z - lse
    q = log_q.exp()
    entropy = torch.special.xlogy(p, p).sum(-1)
    own = log_q.gather(1, ids)
    loss = temperature ** 2 * (entropy - (p * own).sum(-1)) * live
    # a logit's error: the product's, and a few fp32 roundings of the logit, of lse and of their difference
    size = (X.abs() @ W.abs().T).amax(-1, keepdim=True) / temperature
    top = z.abs().amax(-1, keepdim=True) + lse.abs()
    off = product_slack(d, dtype) * size + 8 * U32 * (top + 4.0)
    # p and ln p of a teacher: a few roundings each, of logits up to |t|
    off_p = 32 * U32 * (1.0 + (p > 0) * torch.log(p.clamp(min=1e-300)).abs())
    loss_bound = temperature ** 2 * (2 * off[:, 0] + (p * off_p * (2 + own.abs())).sum(-1)) + 64 * U32 * (
        loss.abs() + temperature ** 2 * (entropy.abs() + (p * own.abs()).sum(-1)))
    g = q.clone().scatter_add_(1, ids, -p * live[:, None])
    g_off = 2 * q * off
    g_off.scatter_add_(1, ids, p * off_p)
    scale = (coef * live * temperature)[:, None]
    # coef is formed in fp32 by a few roundings; G is rounded once, at worst to a quarter of the type's last step below
    # the smallest number kept (2^-40 of the largest coefficient)
    g_bound = (g_off + (ug + 8 * U32) * (g.abs() + g_off)) * scale.abs() + 2.0 ** -39 * scale.abs().amax()
    g = g * scale
    out = {"loss": (loss, loss_bound)}
    for name, a, b in (("dhidden", (g, g_bound), W), ("dweight", (g.T, g_bound.T), X)):
        value = a[0] @ b
        reach = a[0].abs() + a[1]
        bound = a[1] @ b.abs() + product_slack(reach.shape[1], dtype) * (reach @ b.abs())
        # the store's rounding, and the smallest subnormal of the type
        out[name] = (value, bound + u * (value.abs() + bound) + torch.finfo(dtype).smallest_normal * 2 * u)
    return out


def act_slope(g, activation):
    if activation == "silu":
        c = torch.sigmoid(g)
        return g * c, c * (1 + g * (1 - c))
    c = torch.special.ndtr(g)
    return g * c, c + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def gated(x, wg, wu, activation, dh=None, spread=1.0):
    dtype = x.dtype
    X, G, U = x.flatten(0, -2).double(), wg.double(), wu.double()
    d = X.shape[1]
    u_t, ug = u_of(dtype), gradient_unit(dtype, X.shape[0])
    g, u = X @ G.T, X @ U.T
    slack = product_slack(d, dtype)
    g_off, u_off = slack * (X.abs() @ G.abs().T), slack * (X.abs() @ U.abs().T)
    a, s = act_slope(g, activation)
    # |act'| < 1.13 and |act''| < 1 (silu: 0.5, gelu: 0.8); the activation itself: a cumulative value off by at most 1e-7
    # (erf's published form) and 16 roundings, of exponents up to |g| log2 e
    c_off = 1e-7 + 16 * U32 * (1 + g.abs())
    a_off = 1.13 * g_off + c_off * g.abs()
    s_off = g_off + c_off * (1 + g.abs())
    h = a * u
    h_bound = a_off * (u.abs() + u_off) + a.abs() * u_off
    tiny = torch.finfo(dtype).smallest_normal * 2 * u_t
    out = {"h": (h, h_bound + (u_t + 4 * U32) * (h.abs() + h_bound) + tiny)}
    if dh is None:
        return out
    D = dh.flatten(0, -2).double()
    dg, du = D * u * s, D * a
    dg_b = D.abs() * (u_off * (s.abs() + s_off) + u.abs() * s_off)
    du_b = D.abs() * a_off
    # one rounding of dg and du, relative, or of the smallest number kept: fp16 keeps 2^-24 beside a bound of 2^15
    # over every |dg| and |du|, max|dh| 1.15 max|x| max|w| (and a factor of two of the power of two); spread: how far the
    # kernel's max|x| max|w| lies over the norms
    floor = 2.0 ** -39 * 2 * 1.15 * float(D.abs().amax()) * float(X.norm(dim=1).amax()) * float(
        max(G.norm(dim=1).amax(), U.norm(dim=1).amax())) * 0.5 * spread if dtype != torch.bfloat16 else 0.0
    dg_b = dg_b + (ug + 8 * U32) * (dg.abs() + dg_b) + floor
    du_b = du_b + (ug + 8 * U32) * (du.abs() + du_b) + floor

    def product(terms):
        value = sum(p @ q for p, _, q in terms)
        bound = sum(b @ q.abs() for _, b, q in terms)
        n = sum(p.shape[1] for p, _, _ in terms)
        bound = bound + product_slack(n, dtype) * sum((p.abs() + b) @ q.abs() for p, b, q in terms)
        return value, bound + (u_t + 4 * U32) * (value.abs() + bound) + tiny

    out["dx"] = product([(dg, dg_b, G), (du, du_b, U)])
    out["dgate"] = product([(dg.T, dg_b.T, X)])
    out["dup"] = product([(du.T, du_b.T, X)])
    return out


def check(name, got, value, bound):
    got = got.detach().double().reshape(value.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(value)), f"{name}: finite places differ"
    over = (got - value).abs() - bound
    worst = float(torch.nan_to_num(over, nan=-1.0).amax()) if over.numel() else 0.0
    at = int(torch.nan_to_num(over, nan=-1.0).argmax()) if over.numel() else 0
    assert worst <= 0.0, (f"{name}: off by {float((got - value).abs().flatten()[at]):.3e} of {float(value.flatten()[at]):.3e}, "
                          f"bound {float(bound.flatten()[at]):.3e} at {at}")
