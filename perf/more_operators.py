"""Performance cases of the wide products of a language model: the vocabulary's cross entropy and the distillation
from a teacher's top logits, both straight from the head's input without keeping logits, and the gated feed-forward.

    own                    False: the plain form in elementary torch operations; True: this package's operators
    listed()               the cases
    draw(rng)              one more case of the same ranges
    prepare(case, seed)    what a program holds before the call, on the GPU
    run(state)             one pass
    work(case)             bytes and flops a pass cannot do without
    exact(case, seed)      the same outputs from the definitions in 64 bits

Kinds of case (`kind`):
    ce       softmax cross entropy of rows against a vocabulary
    distill  divergence of the rows' softmax from a teacher's over its K largest logits
    gated    act(x Wg^T) * (x Wu^T)

`train`: forward and backward, which returns the gradients too; otherwise the forward alone (scores of given tokens,
the feed-forward of a decoding step).
"""

import math
import os
import sys

import torch

own = False

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                   "pytorch-implementation-of-screening-attention_amd")
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100


def _ops():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    from multiscreen import ops
    return ops


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _ce(name, B, T, d, V, dtype, train, trained=True, pad=0.0):
    return {"name": name, "kind": "ce", "B": B, "T": T, "d": d, "V": V, "dtype": dtype, "train": train,
            "trained": trained, "pad": pad}


def _distill(name, B, T, d, V, K, dtype, temperature, train=True, empty=0.0):
    return {"name": name, "kind": "distill", "B": B, "T": T, "d": d, "V": V, "K": K, "dtype": dtype,
            "temperature": temperature, "train": train, "empty": empty}


def _gated(name, B, T, d, F, dtype, act, train):
    return {"name": name, "kind": "gated", "B": B, "T": T, "d": d, "F": F, "dtype": dtype, "act": act,
            "train": train}


def listed():
    return [
        # scores of one given token of each of 16 sequences under the LM's head: the weight's stream
        _ce("ce_score_16_bf16", 16, 1, 512, 50257, "bf16", False),
        # a training step's loss at the model's longest sequences
        _ce("ce_train_8k_bf16", 4, 2048, 512, 50257, "bf16", True),
        # the package's default type, sequences padded to the longest one
        _ce("ce_train_pad_f32", 8, 512, 512, 50257, "f32", True, True, 0.3),
        # a small vocabulary and odd sizes, before training
        _ce("ce_train_odd_f16", 3, 331, 200, 8003, "f16", True, False),
        # the largest: four sequences of 8192 tokens
        _ce("ce_train_32k_bf16", 4, 8192, 512, 50257, "bf16", True),
        # the drafting model (d 256) learns the large one's 64 largest logits
        _distill("distill_8k_bf16", 4, 2048, 256, 50257, 64, "bf16", 2.0),
        # few tokens, a row in ten without a teacher's record
        _distill("distill_small_f16", 2, 200, 256, 50257, 16, "f16", 1.0, True, 0.1),
        # the default type, an odd vocabulary
        _distill("distill_f32", 4, 401, 256, 32001, 8, "f32", 1.5),
        # the feed-forward of a decoding step of 16 sequences
        _gated("gated_token_bf16", 16, 1, 512, 2048, "bf16", "silu", False),
        # a training step
        _gated("gated_train_32k_bf16", 4, 8192, 512, 2048, "bf16", "silu", True),
        # the default type, two thirds of the plain feed-forward's width
        _gated("gated_train_f32", 4, 1000, 512, 1365, "f32", "gelu", True),
        # a wider model
        _gated("gated_train_f16", 2, 1100, 1024, 4096, "f16", "gelu", True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["ce", "ce", "ce", "distill", "distill", "gated", "gated"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    d = rng.choice([64, 96, 100, 128, 200, 256, 256, 333, 512, 512, 512, 768, 1024])
    B, train = rng.choice([1, 2, 4, 8, 16]), rng.random() < 0.8
    T = max(1, _log_int(rng, 1, 32768) // B)
    if kind == "gated":
        F = _log_int(rng, 100, 8192)
        T = max(1, min(T, 32768 * 512 * 2048 // (B * d * F)))
        return _gated("", B, T, d, F, dtype, rng.choice(["silu", "gelu"]), train)
    V = _log_int(rng, 300, 60000)
    T = max(1, min(T, 32768 * 512 * 50257 // (B * d * V), 32768 * 50257 // (B * V)))
    if kind == "distill":
        return _distill("", B, T, d, V, _log_int(rng, 1, 128), dtype, rng.choice([1.0, 1.5, 2.0, 4.0]), train,
                        rng.choice([0.0, 0.1, 0.5]))
    return _ce("", B, T, d, V, dtype, train, rng.random() < 0.7, rng.choice([0.0, 0.0, 0.2, 0.4]))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _head(case, g, trained):
    """The head's weight, a token for each row, and rows that make it likely where the model is trained."""
    B, T, d, V = (case[x] for x in ("B", "T", "d", "V"))
    # trained: logits of deviation 1.8, the row's own token 2 below the others together (a loss of 2.3 or so);
    # before: the initial deviation of 0.02
    weight = _randn(g, V, d) * (1.8 / math.sqrt(d) if trained else 0.02)
    token = torch.randint(0, V, (B, T), device=DEV, generator=g)
    hidden = _randn(g, B, T, d)
    if trained:
        hidden = hidden + max(0.0, math.log(V) - 0.4) / 1.8 ** 2 * weight[token]
    dt = TYPES[case["dtype"]]
    return hidden.to(dt), weight.to(dt), token


def prepare(case, seed):
    g = _gen(seed)
    B, T, d, dt = case["B"], case["T"], case["d"], TYPES[case["dtype"]]
    s = {"kind": case["kind"], "train": case["train"]}
    if case["kind"] == "gated":
        F = case["F"]
        s["x"] = _randn(g, B, T, d).to(dt)
        s["gate"], s["up"] = ((_randn(g, F, d) / math.sqrt(d)).to(dt) for _ in range(2))
        s["act"] = case["act"]
        if case["train"]:
            s["dh"] = (0.01 * _randn(g, B, T, F)).to(dt)
        return s
    if case["kind"] == "ce":
        s["hidden"], s["weight"], s["labels"] = _head(case, g, case["trained"])
        if case["pad"]:  # sequences end at different lengths
            low = 1.0 - 2.0 * case["pad"]
            length = (T * (low + (1.0 - low) * torch.rand(B, 1, device=DEV, generator=g))).ceil().clamp(min=1)
            s["labels"] = torch.where(torch.arange(T, device=DEV) < length, s["labels"], IGNORE)
        return s
    s["hidden"], s["weight"], token = _head(case, g, True)
    V, K = case["V"], case["K"]
    K = min(K, V)
    at = torch.arange(K, device=DEV)
    step = torch.randint(1, V // K + 1, (B, T, 1), device=DEV, generator=g)
    s["ids"] = (token.unsqueeze(-1) + at * step) % V  # the row's token first, no token twice
    logits = 12.0 - 2.0 * torch.log1p(at.float()) + 0.5 * _randn(g, B, T, K)
    s["logits"] = logits.to(dt)
    if case["empty"]:  # rows without a record, and rows that hold fewer than K
        few = torch.randint(1, K + 1, (B, T, 1), device=DEV, generator=g)
        none = torch.rand(B, T, 1, device=DEV, generator=g) < case["empty"]
        none[0, 0] = False
        s["ids"] = torch.where((at < few) & ~none, s["ids"], -1)
    s["temperature"] = case["temperature"]
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _rows(x):
    return x.reshape(-1, x.shape[-1]).float()


def _plain_head_gradients(s, x, w, p, scale):
    """Gradients of hidden and weight for the logits' gradient p * scale (rows)."""
    p = p * scale.unsqueeze(-1)
    return {"dhidden": torch.matmul(p, w).view(s["hidden"].shape).to(s["hidden"].dtype),
            "dweight": torch.matmul(p.t(), x).to(s["weight"].dtype)}


def _plain_ce(s):
    x, w, y = _rows(s["hidden"]), s["weight"].float(), s["labels"].reshape(-1)
    z = torch.matmul(x, w.t())
    top = z.amax(-1, keepdim=True)
    live = y != IGNORE
    at = torch.where(live, y, 0).unsqueeze(-1)
    picked = z.gather(1, at)
    z = torch.exp(z - top)
    total = z.sum(-1, keepdim=True)
    loss = torch.where(live, (torch.log(total) + top - picked).squeeze(-1), 0.0)
    if not s["train"]:
        return {"loss": loss.view(s["labels"].shape)}
    n = live.sum()
    z = z / total
    z.scatter_add_(1, at, torch.full_like(picked, -1.0))
    out = _plain_head_gradients(s, x, w, z, live / n)
    out["loss"] = (loss.double().sum() / n).float()
    return out


def _plain_distill(s):
    x, w, temp = _rows(s["hidden"]), s["weight"].float(), s["temperature"]
    ids = s["ids"].reshape(-1, s["ids"].shape[-1])
    held = ids >= 0
    t = torch.where(held, _rows(s["logits"]) / temp, -math.inf)
    live = held.any(-1)
    t = torch.where(live.unsqueeze(-1), t, 0.0)
    log_p = t - t.amax(-1, keepdim=True)
    log_p = log_p - torch.log(torch.exp(log_p).sum(-1, keepdim=True))
    p = torch.where(held, torch.exp(log_p), 0.0)
    z = torch.matmul(x, w.t()) / temp
    top = z.amax(-1, keepdim=True)
    at = ids.clamp(min=0)
    picked = z.gather(1, at)
    z = torch.exp(z - top)
    total = z.sum(-1, keepdim=True)
    log_q = picked - top - torch.log(total)
    loss = temp * temp * torch.where(held, p * (log_p - log_q), 0.0).sum(-1)
    loss = torch.where(live, loss, 0.0)
    if not s["train"]:
        return {"loss": loss.view(s["ids"].shape[:-1])}
    n = live.sum()
    z = z / total
    z.scatter_add_(1, at, -p)
    out = _plain_head_gradients(s, x, w, z, live * (temp / n))
    out["loss"] = (loss.double().sum() / n).float()
    return out


def _plain_gated(s):
    x, wg, wu = _rows(s["x"]), s["gate"].float(), s["up"].float()
    g, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
    if s["act"] == "silu":
        c = 1.0 / (1.0 + torch.exp(-g))
        slope = c * (1.0 + g * (1.0 - c))
    else:
        c = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        slope = c + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    a = g * c
    dt, shape = s["x"].dtype, s["x"].shape
    out = {"h": (a * u).view(*shape[:-1], -1).to(dt)}
    if s["train"]:
        dh = _rows(s["dh"])
        dg, du = dh * u * slope, dh * a
        out["dx"] = (torch.matmul(dg, wg) + torch.matmul(du, wu)).view(shape).to(dt)
        out["dgate"] = torch.matmul(dg.t(), x).to(dt)
        out["dup"] = torch.matmul(du.t(), x).to(dt)
    return out


def _own_ce(s, ops):
    if not s["train"]:
        return {"loss": ops.linear_cross_entropy(s["hidden"], s["weight"], s["labels"], reduction="none")}
    x, w = (s[k].detach().requires_grad_() for k in ("hidden", "weight"))
    loss = ops.linear_cross_entropy(x, w, s["labels"])
    dx, dw = torch.autograd.grad(loss, (x, w))
    return {"loss": loss.detach(), "dhidden": dx, "dweight": dw}


def _own_distill(s, ops):
    if not s["train"]:
        return {"loss": ops.linear_distillation(s["hidden"], s["weight"], s["logits"], s["ids"], s["temperature"],
                                                reduction="none")}
    x, w = (s[k].detach().requires_grad_() for k in ("hidden", "weight"))
    loss = ops.linear_distillation(x, w, s["logits"], s["ids"], s["temperature"])
    dx, dw = torch.autograd.grad(loss, (x, w))
    return {"loss": loss.detach(), "dhidden": dx, "dweight": dw}


def _own_gated(s, ops):
    if not s["train"]:
        return {"h": ops.gated_linear(s["x"], s["gate"], s["up"], s["act"])}
    x, wg, wu = (s[k].detach().requires_grad_() for k in ("x", "gate", "up"))
    h = ops.gated_linear(x, wg, wu, s["act"])
    dx, dg, du = torch.autograd.grad(h, (x, wg, wu), s["dh"])
    return {"h": h.detach(), "dx": dx, "dgate": dg, "dup": du}


def run(state):
    if own:
        return {"ce": _own_ce, "distill": _own_distill, "gated": _own_gated}[state["kind"]](state, _ops())
    with torch.no_grad():
        return {"ce": _plain_ce, "distill": _plain_distill, "gated": _plain_gated}[state["kind"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    """Each input read and each output written once; the products x W^T and, in training, g W and g^T x over the rows
    that count (the logits that a backward pass forms again are not counted)."""
    N, d, es = case["B"] * case["T"], case["d"], SIZE[case["dtype"]]
    times = 3 if case["train"] else 1
    ways = 2 if case["train"] else 1
    if case["kind"] == "gated":
        F = case["F"]
        return {"bytes": es * (ways * (N * d + 2 * F * d) + ways * N * F), "flops": times * 4 * N * d * F}
    V = case["V"]
    rows = N * (1.0 - case["pad"]) if case["kind"] == "ce" else N * (1.0 - case["empty"])
    extra = 8 * N if case["kind"] == "ce" else N * min(case["K"], V) * (8 + es)
    loss = 4 if case["train"] else 4 * N
    return {"bytes": es * ways * (N * d + V * d) + extra + loss, "flops": times * 2 * rows * V * d}


# ---------------------------------------------------------------------------
# From the definitions, in 64 bits
# ---------------------------------------------------------------------------
def _targets(s):
    """Per row: the tokens of its target distribution, their probabilities, whether it counts, the temperature."""
    if s["kind"] == "ce":
        y = s["labels"].flatten()
        return y.clamp(min=0)[:, None], torch.ones_like(y, dtype=torch.float64)[:, None], y != IGNORE, 1.0
    ids = s["ids"].flatten(0, -2)
    e = torch.exp((s["logits"].flatten(0, -2).double() - 12.0) / s["temperature"]) * (ids >= 0)
    mass = e.sum(1, keepdim=True)
    return ids.clamp(min=0), e / mass.clamp(min=1e-300), mass[:, 0] > 0, s["temperature"]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "gated":
        return _exact_gated(s)
    ids, p, live, temp = _targets(s)
    W = s["weight"].double()
    X = s["hidden"].flatten(0, -2).double()
    N = X.shape[0]
    share = 1.0 / int(live.sum())
    loss = torch.zeros(N, dtype=torch.float64, device=DEV)
    dX, dW = torch.zeros_like(X), torch.zeros_like(W)
    piece = max(1, (1 << 28) // W.shape[0])
    for a in range(0, N, piece):
        r = slice(a, min(N, a + piece))
        log_q = torch.log_softmax((X[r] @ W.T) / temp, -1)
        own_p = p[r]
        entropy = torch.special.xlogy(own_p, own_p).sum(1)
        cross = -(own_p * log_q.gather(1, ids[r])).sum(1)
        loss[r] = temp ** 2 * torch.where(live[r], entropy + cross, 0.0)
        if case["train"]:
            q = log_q.exp_()
            q.scatter_add_(1, ids[r], -own_p)
            q *= (live[r] * (temp * share))[:, None]
            dX[r] = q @ W
            dW += q.T @ X[r]
    if not case["train"]:
        return {"loss": loss.view(s["hidden"].shape[:-1])}
    return {"dhidden": dX.view(s["hidden"].shape), "dweight": dW, "loss": loss.sum() * share}


def _exact_gated(s):
    shape, wg, wu = s["x"].shape, s["gate"].double(), s["up"].double()
    x = s["x"].flatten(0, -2).double()
    g, u = x @ wg.T, x @ wu.T
    with torch.enable_grad():
        g.requires_grad_()
        a = g * torch.sigmoid(g) if s["act"] == "silu" else g * torch.special.ndtr(g)
        (slope,) = torch.autograd.grad(a.sum(), g)
    g, a = g.detach(), a.detach()
    out = {"h": (a * u).view(*shape[:-1], -1)}
    if s["train"]:
        dh = s["dh"].flatten(0, -2).double()
        dg, du = dh * u * slope, dh * a
        out |= {"dx": (dg @ wg + du @ wu).view(shape), "dgate": dg.T @ x, "dup": du.T @ x}
    return out
