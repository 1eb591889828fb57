"""Performance cases of the serving operators: a quantised key/value cache, the screening of a tree of drafted tokens
over a cache, and the verification of drafted tokens.

    own                    False: the plain form in elementary torch operations; True: this package's operators
    listed()               the cases
    draw(rng)              one more case of the same ranges
    prepare(case, seed)    what a program holds before the call, on the GPU
    run(state)             one pass
    work(case)             bytes and flops a pass cannot do without
    exact(case, seed)      the same outputs from the definitions in 64 bits

Kinds of case (`kind`):
    store   rows of k and v written to a cache (at each sequence's own position where `ragged`, only the accepted rows
            of a draft where `gather`), then read back
    tree    screening attention of M drafted nodes per sequence over the cache that holds them (M = 1: decoding)
    verify  drafted tokens against the target's probabilities: a chain drawn from a draft model's probabilities, a
            tree of proposed tokens, or a tree under greedy decoding

A tree has M nodes: node 0 is the last committed token, `parents[i] < i` is the node that node i continues and
parents[0] = -1.  Regimes are those of a model before training (`init`: hardly any pair passes the threshold) and
after it (`trained`: q and k around 18 centres per head, about 5% of the pairs pass at r = 2).
"""

import math
import os
import sys

import torch

own = False

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                   "pytorch-implementation-of-screening-attention_amd")
DEV = "cuda"
EPS = 1e-8
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
         "int8": torch.int8, "fp8": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "int8": 1, "fp8": 1}
TOP = {"int8": 127.0, "fp8": 448.0}  # the largest code
CENTRES, RHO = 18, 0.8


def _ops():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    from multiscreen import ops
    return ops


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _store(name, B, T, H, D, dtype, cache, cap, ragged, gather):
    return {"name": name, "kind": "store", "B": B, "T": T, "H": H, "D": D, "dtype": dtype, "cache": cache, "cap": cap,
            "ragged": ragged, "gather": gather}


def _tree(name, B, M, shape, H, D, dtype, cache, n, regime, r, w_lo, w_hi):
    return {"name": name, "kind": "tree", "B": B, "M": M, "shape": shape, "H": H, "D": D, "dtype": dtype,
            "cache": cache, "len": n, "cap": n + M + 31, "regime": regime, "r": r, "w_lo": float(w_lo),
            "w_hi": float(w_hi)}


def _verify(name, B, M, V, mode, dtype):
    return {"name": name, "kind": "verify", "B": B, "M": M, "V": V, "mode": mode, "dtype": dtype}


def listed():
    return [
        # the prompt of four sequences enters an int8 cache
        _store("store_prompt_bf16_int8", 4, 8192, 8, 64, "bf16", "int8", 8448, False, False),
        # one new token of each of 16 sequences of different lengths: the smallest write
        _store("store_token_f16_fp8", 16, 1, 8, 64, "f16", "fp8", 2048, True, False),
        # the accepted rows of a 48-node draft of each of 32 sequences, float32 rows of wide heads
        _store("store_accepted_f32_int8", 32, 48, 8, 128, "f32", "int8", 4096, True, True),
        # a 32-node tree at the initial windows (2 .. 256) over a 16-bit cache: the smallest screening call
        _tree("tree_windows_bf16", 16, 32, "tree", 8, 64, "bf16", "bf16", 8000, "trained", 1.135, 2, 256),
        # a 64-node tree, trained, windows as wide as a 30K context
        _tree("tree_wide_bf16_30k", 4, 64, "tree", 8, 64, "bf16", "bf16", 30000, "trained", 2.0, 30000, 30000),
        # a chain of 8 drafted tokens over an int8 cache, windows from narrow to the whole context
        _tree("chain_int8_16k", 16, 8, "chain", 8, 64, "bf16", "int8", 16000, "trained", 2.0, 256, 16000),
        # one token of 16 sequences over an int8 cache of 100K positions: the cache's stream bounds it
        _tree("token_int8_100k", 16, 1, "chain", 8, 64, "bf16", "int8", 100000, "init", 2.0, 100000, 100000),
        # an odd tree over an 8-bit floating-point cache of wide heads
        _tree("tree_fp8_d128_f16", 8, 21, "tree", 4, 128, "f16", "fp8", 5001, "trained", 2.0, 64, 5001),
        # the package's default type
        _tree("tree_f32_d32", 4, 40, "tree", 8, 32, "f32", "f32", 6000, "trained", 2.0, 64, 6000),
        # eight tokens drafted by a smaller model for each of 16 sequences, the LM's vocabulary
        _verify("verify_chain_f32", 16, 9, 50257, "chain", "f32"),
        # a 64-node tree of proposed tokens, sampled
        _verify("verify_tree_f16", 32, 64, 50257, "tree", "f16"),
        # the same tree under greedy decoding: every row's largest logit
        _verify("verify_greedy_bf16", 8, 64, 50257, "greedy", "bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "store", "tree", "tree", "tree", "verify", "verify"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "store":
        B, H, D = rng.choice([1, 3, 8, 16, 32]), rng.choice([4, 8, 12]), rng.choice([16, 32, 64, 64, 128])
        gather = rng.random() < 0.4
        T = rng.randint(1, 64) if gather else _log_int(rng, 1, max(2, 4 * 8192 * 8 * 64 // (B * H * D)))
        return _store("", B, T, H, D, dtype, rng.choice(["int8", "fp8"]), T + rng.randint(0, 600),
                      gather or rng.random() < 0.5, gather)
    if kind == "tree":
        B, H, D = rng.choice([1, 3, 4, 8, 16]), rng.choice([4, 8, 12]), rng.choice([16, 32, 64, 64, 128])
        M, n = _log_int(rng, 1, 64), _log_int(rng, 40, 100000)
        # no more keys than the largest listed case streams, and no more pairs than its plain form forms
        n = max(1, min(n, 16 * 8 * 100000 * 64 // (B * H * D) // 2, 4 * 8 * 64 * 30000 // (B * H * M)))
        w_hi = rng.choice([256.0, float(n), n * rng.uniform(0.2, 1.0)])
        regime = rng.choice(["init", "trained", "trained"])
        return _tree("", B, M, rng.choice(["chain", "tree"]), H, D, dtype, rng.choice([dtype, "int8", "fp8"]), n,
                     regime, rng.choice([1.135, 2.0]) if regime == "trained" else 2.0, min(2.0, w_hi),
                     max(2.0, w_hi))
    mode = rng.choice(["chain", "tree", "greedy"])
    B, V = rng.choice([1, 4, 16, 32]), _log_int(rng, 300, 60000)
    M = rng.randint(1, 12) if mode == "chain" else rng.randint(1, 64)
    B = max(1, min(B, 32 * 64 * 50257 // (4 * M * V)))
    return _verify("", B, M, V, mode, dtype)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _cache_store(B, H, cap, D, dtype):
    """Head-major storage of codes or values."""
    return torch.zeros(B, H, cap, D, dtype=dtype, device=DEV)


def _bthd(x):
    """The (B, T, H, ...) view of head-major storage, as the projections are laid out."""
    return x.transpose(1, 2)


def _parents(M, shape, B, g):
    """(B, M): each sequence's own tree; a node hangs on one of the eight nodes before it."""
    at = torch.arange(M, device=DEV).expand(B, M)
    if shape == "chain":
        return at - 1
    back = 1 + torch.randint(0, 8, (B, M), device=DEV, generator=g)
    return torch.where(at == 0, -1, (at - back).clamp(min=0))


def _prepare_store(case, seed):
    g = _gen(seed)
    B, T, H, D, cap = (case[x] for x in ("B", "T", "H", "D", "cap"))
    dt, ct = TYPES[case["dtype"]], TYPES[case["cache"]]
    # k and v as the last two thirds of one stacked projection; rows differ in length, as a model's do
    qkv = _randn(g, B, T, 3 * H * D) * torch.exp(0.5 * _randn(g, B, T, 1))
    qkv = qkv.to(dt)
    s = {"kind": "store", "dtype": dt, "cache": case["cache"], "T": T}
    s["k"], s["v"] = (x.view(B, T, H, D) for x in qkv.split(H * D, dim=-1)[1:])
    for x in ("k", "v"):
        s[x + "c"] = _bthd(_cache_store(B, H, cap, D, ct))
        s[x + "s"] = _bthd(torch.zeros(B, H, cap, device=DEV))
    room = cap - T
    s["start"] = torch.randint(0, room + 1, (B,), device=DEV, generator=g) if case["ragged"] else 0
    s["rows"] = s["count"] = None
    if case["gather"]:
        # an accepted path: increasing node numbers, a few of them
        s["rows"] = torch.rand(B, T, device=DEV, generator=g).argsort(-1)
        s["count"] = torch.randint(1, min(T, 12) + 1, (B,), device=DEV, generator=g)
        head = torch.arange(T, device=DEV) < s["count"].unsqueeze(1)
        s["rows"] = torch.where(head, s["rows"], T).sort(-1).values
        s["rows"] = torch.where(head, s["rows"], -1)
    return s


def _prepare_tree(case, seed):
    g = _gen(seed)
    B, M, H, D, n, cap = (case[x] for x in ("B", "M", "H", "D", "len", "cap"))
    dt, ct = TYPES[case["dtype"]], TYPES[case["cache"]]
    centres = _randn(g, H, CENTRES, D)
    heads = torch.arange(H, device=DEV).view(H, 1)

    def rows(T, mixed):
        """(H, T, D) rows of one sequence."""
        x = _randn(g, H, T, D)
        if mixed and case["regime"] == "trained":
            at = torch.randint(0, CENTRES, (H, T), device=DEV, generator=g)
            x = RHO * centres[heads, at] + math.sqrt(1.0 - RHO * RHO) * x
        return x

    s = {"kind": "tree", "hint": min(cap, math.ceil(case["w_hi"])), "M": M, "cache": case["cache"]}
    q = torch.stack([rows(M, True) for _ in range(B)])  # (B, H, M, D)
    s["q"] = q.transpose(1, 2).contiguous().to(dt)
    for x in ("k", "v"):
        store = _cache_store(B, H, cap, D, ct)
        scale = torch.zeros(B, H, cap, device=DEV) if case["cache"] in TOP else None
        for b in range(B):
            y = rows(cap, x == "k")
            if scale is not None:
                scale[b] = y.abs().amax(-1) / TOP[case["cache"]]
                y = y / scale[b].unsqueeze(-1)
                y = y.round() if case["cache"] == "int8" else y
            store[b] = y.to(ct)
        s[x + "c"] = _bthd(store)
        s[x + "s"] = None if scale is None else _bthd(scale)
    # sequences of the batch end at different lengths, the longest at n
    s["lengths"] = (n - torch.randint(0, 1 + n // 8, (B,), device=DEV, generator=g) * (torch.arange(B, device=DEV) > 0))
    s["parents"] = _parents(M, case["shape"], B, g)
    s["r"] = case["r"] + (0.1 * torch.rand(H, device=DEV, generator=g) - 0.05 if case["r"] > 1.5 else 0.0) \
        * torch.ones(H, device=DEV)
    s["w"] = torch.linspace(case["w_lo"], case["w_hi"], H, device=DEV)
    return s


def _prepare_verify(case, seed):
    g = _gen(seed)
    B, M, V, mode, dt = (case[x] for x in ("B", "M", "V", "mode", "dtype"))
    dt = TYPES[dt]
    logits = 3.0 * _randn(g, B, M, V)
    s = {"kind": "verify", "uniforms": None, "draft": None}
    s["parents"] = _parents(M, "chain" if mode == "chain" else "tree", B, g)
    tokens = torch.randint(0, V, (B, M), device=DEV, generator=g)
    if mode == "chain":
        # a draft model that mostly agrees with the target
        q = torch.softmax(logits[:, :M - 1] + 0.3 * _randn(g, B, M - 1, V), -1)
        if M > 1:
            tokens[:, 1:] = torch.multinomial(q.reshape(-1, V), 1, generator=g).view(B, M - 1)
        s["draft"] = q.to(dt)
    elif M > 1:
        # proposals: one of the likelier tokens after each node's parent
        k = min(V, 4)
        top = logits.topk(k, -1).indices
        pick = torch.randint(0, k, (B, M - 1), device=DEV, generator=g)
        at = s["parents"][:, 1:].unsqueeze(-1).expand(-1, -1, k)
        tokens[:, 1:] = top.gather(1, at).gather(2, pick.unsqueeze(-1)).squeeze(-1)
    s["tokens"] = tokens
    if mode == "greedy":
        s["target"] = logits.to(dt)
    else:
        s["target"] = torch.softmax(logits, -1).to(dt)
        s["uniforms"] = torch.rand(B, M, device=DEV, generator=g)
    return s


def prepare(case, seed):
    return {"store": _prepare_store, "tree": _prepare_tree, "verify": _prepare_verify}[case["kind"]](case, seed)


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _quantise(x, cache):
    """Codes (as the cache keeps them) and scales of rows x (..., D).  A code is the nearest one to
    TOP * x / max|x|, ties to the even one: taken in 64 bits, which decide every border."""
    top = x.float().abs().amax(-1)
    t = TOP[cache] * x.double() / top.double().unsqueeze(-1)
    t = torch.where(top.unsqueeze(-1) > 0, t, 0.0)
    if cache == "int8":
        code = t.round().to(torch.int8)
    else:  # 4 significant bits, spaced 2^-9 below 2^-6
        step = torch.ldexp(torch.ones_like(t), (torch.frexp(t).exponent - 4).clamp(min=-9))
        code = ((t / step).round() * step).float().to(torch.float8_e4m3fn)
    return code, top / TOP[cache]


def _plain_store(s):
    B, T = s["k"].shape[0], s["T"]
    at = torch.arange(T, device=DEV)
    pos = (s["start"].unsqueeze(1) if torch.is_tensor(s["start"]) else s["start"]) + at.expand(B, T)
    b = torch.arange(B, device=DEV).unsqueeze(1)
    out = []
    for x in ("k", "v"):
        rows, cache, scale = s[x], s[x + "c"].view(torch.uint8), s[x + "s"]
        keep = torch.ones(B, T, 1, 1, dtype=torch.bool, device=DEV)
        if s["rows"] is not None:
            rows = rows[b, s["rows"].clamp(min=0)]
            keep = (at < s["count"].unsqueeze(1)).view(B, T, 1, 1)
        code, sc = _quantise(rows, s["cache"])
        cache[b, pos] = torch.where(keep, code.view(torch.uint8), cache[b, pos])
        scale[b, pos] = torch.where(keep.squeeze(-1), sc, scale[b, pos])
        back = s[x + "c"].view(torch.uint8)[b, pos].view(TYPES[s["cache"]]).float() * scale[b, pos].unsqueeze(-1)
        out.append(back.to(s["dtype"]))
    return {"k": out[0], "v": out[1]}


def _unit(x):
    return x / torch.linalg.vector_norm(x, dim=-1, keepdim=True).clamp(min=EPS)


def _relations(parents):
    """(B, M, M) whether node j is node i or above it, and the nodes' depths (B, M)."""
    M = parents.shape[1]
    at = torch.arange(M, device=DEV)
    step = (parents.unsqueeze(-1) == at).double() + torch.eye(M, dtype=torch.float64, device=DEV)
    above = torch.linalg.matrix_power(step, max(M, 1)) > 0
    return above, above.sum(-1) - 1


def _plain_tree(s):
    q, M = s["q"].float(), s["M"]
    B, _, H, _ = q.shape
    above, depth = _relations(s["parents"])
    # the keys that the widest window can reach, then the drafted nodes
    W = s["hint"]
    j = s["lengths"].view(B, 1) - W + torch.arange(W + M, device=DEV)
    b = torch.arange(B, device=DEV).unsqueeze(1)

    def rows(x):
        y = s[x + "c"]
        at = j.clamp(min=0)
        y = y.view(torch.uint8)[b, at].view(y.dtype) if y.element_size() == 1 else y[b, at]
        y = y.float() if s[x + "s"] is None else y.float() * s[x + "s"][b, at].unsqueeze(-1)
        return _unit(y).transpose(1, 2)  # (B, H, W + M, D)

    sim = torch.matmul(_unit(q).transpose(1, 2), rows("k").transpose(2, 3).contiguous())
    r, w = s["r"].view(1, H, 1, 1), s["w"].view(1, H, 1, 1)
    pos = s["lengths"].view(B, 1) + depth
    kpos = torch.cat((j[:, :W], pos), 1)
    ok = torch.cat(((j[:, :W] >= 0).unsqueeze(1).expand(B, M, W), above), 2).unsqueeze(1)
    dist = (pos.unsqueeze(2) - kpos.unsqueeze(1)).unsqueeze(1).float()
    mask = torch.where(ok & (dist >= 0) & (dist < w), 0.5 * (torch.cos(math.pi * dist / w) + 1.0), 0.0)
    p = torch.relu(1.0 - r * (1.0 - sim)).square() * mask
    h = torch.matmul(p, rows("v"))
    n = torch.linalg.vector_norm(h, dim=-1, keepdim=True).clamp(min=EPS)
    return (h * (torch.tanh(n) / n)).transpose(1, 2).to(s["q"].dtype)


def _first_index(hit):
    """The lowest index of a true entry along the last axis (0 if there is none)."""
    V = hit.shape[-1]
    return torch.where(hit, torch.arange(V, device=DEV), V).amin(-1) % V


def _plain_verify(s):
    tokens, parents, target = s["tokens"], s["parents"], s["target"]
    B, M = tokens.shape
    at = torch.arange(M, device=DEV)
    b = torch.arange(B, device=DEV)
    above, depth = _relations(parents)
    up = parents.clamp(min=0)
    # the siblings before node i under the same parent
    before = (parents.unsqueeze(1) == parents.unsqueeze(2)) & (at < at.view(M, 1)) & (parents >= 0).unsqueeze(1)
    if s["uniforms"] is None:
        best = _first_index(target == target.amax(-1, keepdim=True))
        taken = tokens == best.gather(1, up)
    else:
        u = s["uniforms"].double()
        px = target[b.unsqueeze(1), up, tokens].double()
        if s["draft"] is not None:
            d = s["draft"]
            qx = d[b.unsqueeze(1), up.clamp(max=max(0, M - 2)), tokens].double() if M > 1 else px
            taken = u * qx < px
        else:
            # earlier siblings were refused: their tokens' shares are gone, and equal tokens count once
            same = tokens.unsqueeze(1) == tokens.unsqueeze(2)
            gone = (before & same).any(-1)  # an earlier sibling had this token
            share = torch.where(gone, 0.0, px)
            left = 1.0 - (before * share.unsqueeze(1)).sum(-1)
            taken = u * left < share
    taken = taken & ~(before & taken.unsqueeze(1)).any(-1)
    taken = torch.where(at == 0, True, taken & (parents >= 0))
    held = (above <= taken.unsqueeze(1)).all(-1) & above[:, :, 0]  # the node and all above it are taken
    count = held.sum(-1)
    path = torch.where(held, at, M).sort(-1).values
    path = torch.where(at < count.unsqueeze(1), path, -1)
    last = path.gather(1, (count - 1).unsqueeze(1)).squeeze(1)
    if s["uniforms"] is None:
        return {"path": path, "count": count, "token": best.gather(1, last.unsqueeze(1)).squeeze(1)}
    p = target[b, last].double()
    weight = p
    if s["draft"] is not None:
        if M > 1:
            rest = (p - s["draft"][b, last.clamp(max=M - 2)].double()).clamp(min=0)
            weight = torch.where(((last < M - 1) & (rest.sum(-1) > 0)).unsqueeze(1), rest, p)
    else:
        refused = parents == last.unsqueeze(1)  # no child of the last node was taken
        hit = torch.zeros_like(p).scatter_add_(1, tokens, refused.double())
        rest = torch.where(hit > 0, 0.0, p)
        weight = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p)
    below = weight.cumsum(-1)
    want = s["uniforms"][:, 0].double() * below[:, -1]
    over = (below > want.unsqueeze(1)) & (weight > 0)
    return {"path": path, "count": count, "token": _first_index(over)}


def _own(s):
    ops = _ops()
    if s["kind"] == "store":
        ops.cache_write(s["k"], s["v"], s["kc"], s["vc"], s["start"], s["ks"], s["vs"], s["rows"], s["count"])
        k, v = ops.cache_read(s["kc"], s["vc"], s["ks"], s["vs"], s["start"], s["T"], s["dtype"])
        return {"k": k, "v": v}
    if s["kind"] == "tree":
        return ops.tree_decode(s["q"], s["kc"], s["vc"], s["lengths"], s["parents"], s["r"], s["w"], EPS, s["ks"],
                               s["vs"], None, s["hint"])
    path, count, token = ops.verify_drafts(s["target"], s["tokens"], s["parents"], s["uniforms"], s["draft"])
    return {"path": path, "count": count, "token": token}


def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "tree": _plain_tree, "verify": _plain_verify}[state["kind"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    """Each input read and each output written once.  tree: the windows' key rows and the value rows that some node's
    weight reaches (of the pairs, 5% pass trained at r = 2, 17% at r = 1.135, none before training).  verify: the rows
    that decide (one row of target and draft a sequence; every row where each row's largest entry is asked for)."""
    if case["kind"] == "store":
        rows = case["B"] * case["T"] * case["H"] * 2
        if case["gather"]:
            rows *= min(case["T"], 12) / 2 / case["T"]
        D = case["D"]
        # written (row in, code and scale out) and read back (code and scale in, row out)
        return {"bytes": rows * 2 * (D * SIZE[case["dtype"]] + D + 4), "flops": rows * 6 * D}
    if case["kind"] == "tree":
        B, M, H, D, n = (case[x] for x in ("B", "M", "H", "D", "len"))
        w = [case["w_lo"] + (case["w_hi"] - case["w_lo"]) * h / max(1, H - 1) for h in range(H)]
        keys = B * sum(min(n, math.ceil(x)) + M for x in w)
        passing = 0.0 if case["regime"] == "init" else 0.17 if case["r"] < 1.5 else 0.05
        row = D * SIZE[case["cache"]] + (4 if case["cache"] in TOP else 0)
        return {"bytes": keys * row * (1 + (1 - (1 - passing) ** M)) + 2 * B * M * H * D * SIZE[case["dtype"]],
                "flops": 2 * D * keys * M * (1 + passing)}
    B, M, V, es = case["B"], case["M"], case["V"], SIZE[case["dtype"]]
    rows = B * M if case["mode"] == "greedy" else B * (2 if case["mode"] == "chain" else 1)
    return {"bytes": rows * V * es + B * M * 32, "flops": rows * V * 2}


# ---------------------------------------------------------------------------
# From the definitions, in 64 bits
# ---------------------------------------------------------------------------
def _exact_row_values(x, cache):
    """The values that a quantised row stands for: TOP codes to each side of zero, scaled to the largest entry."""
    big = x.abs().max(-1, keepdim=True).values
    unit = torch.where(big > 0, x / big, torch.zeros_like(x)) * TOP[cache]
    if cache == "int8":
        near = torch.round(unit)
    else:
        binade = torch.floor(torch.log2(unit.abs().clamp(min=2.0 ** -6)))
        grid = torch.pow(2.0, binade - 3)
        near = torch.round(unit / grid) * grid
    return near * big / TOP[cache]


def _exact_store(case, seed):
    s = _prepare_store(case, seed)
    B, T = case["B"], case["T"]
    out = {}
    for x in ("k", "v"):
        rows = s[x].double()
        if s["rows"] is None:
            out[x] = _exact_row_values(rows, case["cache"])
        else:  # rows past the accepted ones keep what the new cache holds, zeros
            out[x] = torch.zeros_like(rows)
            for b, n in enumerate(s["count"].tolist()):
                out[x][b, :n] = _exact_row_values(rows[b][s["rows"][b, :n]], case["cache"])
    return out


def _exact_tree(case, seed):
    s = _prepare_tree(case, seed)
    B, M, H, D = (case[x] for x in ("B", "M", "H", "D"))
    y = torch.zeros(B, M, H, D, dtype=torch.float64, device=DEV)
    w, r = s["w"].tolist(), s["r"].tolist()
    for b, n in enumerate(s["lengths"].tolist()):
        up = s["parents"][b].tolist()
        lines = []  # each node's way up, itself first
        for i in range(M):
            lines.append([i] + (lines[up[i]] if up[i] >= 0 else []))
        depth = torch.tensor([len(x) - 1 for x in lines], device=DEV)
        over = torch.zeros(M, M, dtype=torch.bool)
        for i in range(M):
            over[i, lines[i]] = True
        over = over.to(DEV)
        for h in range(H):
            lo = max(0, n - math.ceil(w[h]))

            def rows(x):
                t = s[x + "c"][b, lo:n + M, h].double()
                if s[x + "s"] is not None:
                    t = t * s[x + "s"][b, lo:n + M, h].double().unsqueeze(-1)
                return t / torch.sqrt((t * t).sum(-1, keepdim=True)).clamp(min=EPS)

            qh = s["q"][b, :, h].double()
            qh = qh / torch.sqrt((qh * qh).sum(-1, keepdim=True)).clamp(min=EPS)
            a = (1.0 - r[h] * (1.0 - qh @ rows("k").T)).clamp(min=0.0)
            place = torch.cat((torch.arange(lo, n, device=DEV), n + depth))
            d = ((n + depth).view(M, 1) - place.view(1, -1)).double()
            seen = torch.cat((torch.ones(M, n - lo, dtype=torch.bool, device=DEV), over), 1) & (d < w[h])
            m = torch.cos(0.5 * math.pi * d / w[h]) ** 2
            acc = torch.where(seen, a * a * m, torch.zeros_like(a)) @ rows("v")
            size = torch.sqrt((acc * acc).sum(-1, keepdim=True)).clamp(min=EPS)
            y[b, :, h] = acc * torch.tanh(size) / size
    return y


def _exact_verify(case, seed):
    import numpy as np
    s = _prepare_verify(case, seed)
    B, M, V = case["B"], case["M"], case["V"]
    target = s["target"].float().cpu().numpy()
    draft = None if s["draft"] is None else s["draft"].float().cpu().numpy()
    uni = None if s["uniforms"] is None else s["uniforms"].cpu().numpy().astype(np.float64)
    tokens, parents = s["tokens"].cpu().numpy(), s["parents"].cpu().numpy()
    path, count, token = np.full((B, M), -1), np.zeros(B, dtype=np.int64), np.zeros(B, dtype=np.int64)
    for b in range(B):
        node, walk = 0, [0]
        while True:
            row = target[b, node].astype(np.float64)
            children = [i for i in range(1, M) if parents[b, i] == node]
            found, left, weight = None, 1.0, row.copy()
            for c in children:
                x = tokens[b, c]
                if uni is None:
                    hit = int(np.argmax(row)) == x
                elif draft is not None:
                    hit = uni[b, c] * float(draft[b, node, x]) < row[x]
                else:
                    hit = uni[b, c] * left < weight[x]
                    if not hit:
                        left -= weight[x]
                        weight[x] = 0.0
                if hit:
                    found = c
                    break
            if found is None:
                break
            node = found
            walk.append(node)
        path[b, :len(walk)], count[b] = walk, len(walk)
        if uni is None:
            token[b] = int(np.argmax(row))
            continue
        if draft is not None and children:
            weight = np.maximum(row - draft[b, node].astype(np.float64), 0.0)
        if not weight.sum() > 0:
            weight = row
        sums = np.cumsum(weight)
        over = np.flatnonzero((sums > uni[b, 0] * sums[-1]) & (weight > 0))
        token[b] = over[0] if len(over) else 0
    return {k: torch.from_numpy(v).to(DEV) for k, v in (("path", path), ("count", count), ("token", token))}


def exact(case, seed):
    return {"store": _exact_store, "tree": _exact_tree, "verify": _exact_verify}[case["kind"]](case, seed)
