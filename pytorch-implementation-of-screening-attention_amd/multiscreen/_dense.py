"""Screening attention core for CPU tensors: explicit (Tq x Tk) matrices.

This is how the module runs when its tensors live on the host (the
reference's own unit tests are CPU-only, tests/test_attention.py).  GPU
tensors never come here: they always take the fused HIP kernels in ops.py.
Same inputs and output as ops.screening_core: raw (B,T,H,D) projections in,
TanhNorm'd (B,Tq,H,D) out, following attention.py:155-196.
"""

import math

import torch
import torch.nn.functional as F


def pair_mask(Tq, Tk, w, causal, device, q_offset=0):
    """(H, Tq, Tk) cosine soft mask with the window cut (attention.py:92-119, :174-183).

    Query row t sits at position q_offset + t (0 in the reference's forward,
    which aligns both index ranges at 0, attention.py:108-110)."""
    i = q_offset + torch.arange(Tq, device=device).view(Tq, 1)
    j = torch.arange(Tk, device=device).view(1, Tk)
    rel = (j - i).to(torch.float32).unsqueeze(0)          # j - i
    w = w.to(torch.float32).view(-1, 1, 1)
    m = 0.5 * (torch.cos(math.pi * rel / w) + 1.0)
    inside = (rel > -w) & (rel <= 0) if causal else (rel.abs() < w)
    return m * inside.to(m.dtype)


def screening_core_dense(q, k, v, r, w, causal=True, eps=1e-8, key_padding_mask=None,
                         dropout=None, q_offset=0):
    B, Tq, H, D = q.shape
    Tk = k.shape[1]
    qn = F.normalize(q.transpose(1, 2), dim=-1, eps=eps)
    kn = F.normalize(k.transpose(1, 2), dim=-1, eps=eps)
    vn = F.normalize(v.transpose(1, 2), dim=-1, eps=eps)
    s = qn @ kn.transpose(-2, -1)                            # (B,H,Tq,Tk)
    a = torch.relu(1.0 - r.view(1, H, 1, 1) * (1.0 - s))
    p = a * a * pair_mask(Tq, Tk, w, causal, q.device, q_offset).unsqueeze(0).to(a.dtype)
    if key_padding_mask is not None:
        p = p.masked_fill(key_padding_mask.view(B, 1, 1, Tk), 0.0)
    if dropout is not None:
        p = dropout(p)
    h = p @ vn.to(p.dtype)                                    # (B,H,Tq,D)
    n = torch.linalg.vector_norm(h, dim=-1, keepdim=True).clamp(min=eps)
    y = h * (torch.tanh(n) / n)
    return y.transpose(1, 2)                                  # (B,Tq,H,D)


# ---------------------------------------------------------------------------
# Serving on the host: the forms of ops.cache_write, ops.tree_decode and
# ops.verify_drafts that CPU tensors take.
# ---------------------------------------------------------------------------
CODE_TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def quantise_rows(x, dtype):
    """(codes, float32 scales) of rows x (..., D): the codes nearest to TOP x / max|x|,
    ties to the even code; decided in float64."""
    top = x.double().abs().amax(-1, keepdim=True)
    some = torch.isfinite(top) & (top > 0)
    t = torch.where(some, CODE_TOP[dtype] * x.double() / torch.where(some, top, 1.0), 0.0)
    if dtype == torch.int8:
        t = t.round()
    else:  # 4 significant bits, spaced 2^-9 below 2^-6
        step = torch.exp2(torch.frexp(t).exponent.double() - 4).clamp(min=2.0 ** -9)
        t = (t / step).round() * step
    scale = torch.where(torch.isfinite(top), top.float() / CODE_TOP[dtype], math.nan)
    return t.float().to(dtype), scale.squeeze(-1)


def tree_relations(parents):
    """(above, depth) of parents (B, M): above[b, i, j], whether node j is node i or one
    of its ancestors, and the nodes' depths.  A parent outside [0, i) makes a root."""
    B, M = parents.shape
    at = torch.arange(M, device=parents.device)
    up = torch.where((parents >= 0) & (parents < at), parents, -1)
    above = torch.eye(M, dtype=torch.bool, device=parents.device).expand(B, M, M)
    step = 1
    while step < M:  # `up` is the first node that `above` does not cover yet
        on = (up >= 0).unsqueeze(-1)
        to = up.clamp(min=0)
        above = above | (on & above.gather(1, to.unsqueeze(-1).expand(B, M, M)))
        up = torch.where(up >= 0, up.gather(1, to), -1)
        step *= 2
    return above, above.sum(-1) - 1


def tree_dense(q, k, v, lengths, parents, r, w, eps=1e-8):
    """Screening of a tree of drafted rows: q (B, M, H, D) over values k, v (B, cap, H, D) of
    a cache that holds sequence b's committed rows below lengths[b] and its nodes' rows from there on."""
    B, M, H, D = q.shape
    cap = k.shape[1]
    n = lengths.clamp(0, cap - M).view(-1, 1).expand(B, 1)
    above, depth = tree_relations(parents)
    j = torch.arange(cap).expand(B, cap)
    node = (j - n).clamp(0, M - 1)
    drafted = (j >= n) & (j < n + M)
    kpos = torch.where(drafted, n + depth.gather(1, node), j)
    dist = ((n + depth).unsqueeze(-1) - kpos.unsqueeze(1)).unsqueeze(1).float()          # (B, 1, M, cap)
    seen = torch.where(drafted.unsqueeze(1), above.gather(2, node.unsqueeze(1).expand(B, M, cap)), (j < n).unsqueeze(1))
    wh = w.float().view(1, H, 1, 1)
    m = torch.where(seen.unsqueeze(1) & (dist >= 0) & (dist < wh), 0.5 * (torch.cos(math.pi * dist / wh) + 1.0), 0.0)
    qn, kn, vn = (F.normalize(x.transpose(1, 2).float(), dim=-1, eps=eps) for x in (q, k, v))
    a = torch.relu(1.0 - r.float().view(1, H, 1, 1) * (1.0 - qn @ kn.transpose(-2, -1)))
    p = a * a * m
    p = torch.where(p > 0, p, 0.0)  # a NaN, of a q or k row that is not finite, is not live
    odd = ~torch.isfinite(v).all(-1).transpose(1, 2).unsqueeze(2)                         # (B, H, 1, cap)
    h = p @ torch.where(odd.transpose(2, 3), 0.0, vn)
    h = torch.where((odd & (p > 0)).any(-1, keepdim=True), math.nan, h)  # a live pair brings NaN to its node alone
    size = torch.linalg.vector_norm(h, dim=-1, keepdim=True).clamp(min=eps)
    return (h * (torch.tanh(size) / size)).transpose(1, 2).to(q.dtype)


def verify_dense(target, tokens, parents=None, uniforms=None, draft=None):
    """ops.verify_drafts on the host, sequence by sequence."""
    B, M, V = target.shape
    path, count, token = torch.full((B, M), -1), torch.ones(B, dtype=torch.int64), torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        up = list(range(-1, M - 1)) if parents is None else (parents[b] if parents.dim() == 2 else parents).tolist()
        node, length = 0, 0
        while True:
            path[b, length] = node
            length += 1
            row = target[b, node].double()
            best = -1
            if uniforms is None:  # a NaN is the largest entry
                top = row.isnan() if row.isnan().any() else row == row.amax()
                best = int(top.nonzero()[0])
            p = torch.where(row > 0, row, 0.0)  # entries that are negative or NaN count as 0
            rest, left, refused, taken = p.clone(), 1.0, False, -1
            for c in range(max(1, node + 1), M):
                x = int(tokens[b, c])
                if up[c] != node or not 0 <= x < V or (draft is not None and c != node + 1):
                    continue
                if uniforms is None:
                    hit = x == best
                elif draft is not None:
                    hit = float(uniforms[b, c]) * float(draft[b, node, x]) < float(row[x])
                else:
                    hit = float(uniforms[b, c]) * left < float(rest[x])
                if hit:
                    taken = c
                    break
                refused = True
                if draft is None and uniforms is not None:
                    left -= float(rest[x])
                    rest[x] = 0.0
            if taken < 0:
                break
            node = taken
        count[b] = length
        if uniforms is None:
            token[b] = best
            continue
        if draft is not None and refused:
            more = row - draft[b, node].double()
            rest = torch.where(more > 0, more, 0.0)
        rest = rest if float(rest.sum()) > 0 else p
        below = rest.cumsum(0)
        over = ((below > float(uniforms[b, 0]) * float(below[-1])) & (rest > 0)).nonzero()
        some = (rest > 0).nonzero()
        token[b] = int(over[0]) if len(over) else int(some[-1]) if len(some) else 0
    return path, count, token
