"""ops.verify_drafts against the rule followed step by step in float64, in
every mode and type, at vocabularies from one token up; borders that probability
and uniform hit exactly; rows without weight; the distribution of the tokens."""

import math

import pytest
import torch

from test_gpu_cache_rows import DEV, FLOATS, _name, _native_error, _ops
from test_gpu_tree_decode import tree_of


def rule(target, tokens, parents, uniforms, draft):
    """One sequence, python floats (64 bits): (walked nodes, next token)."""
    M, V = target.shape
    node, walk = 0, [0]
    while True:
        row = target[node].double().tolist()
        children = [i for i in range(1, M) if parents[i] == node and (draft is None or i == node + 1)]
        found, left, out = None, 1.0, set()
        for c in children:
            x = int(tokens[c])
            inside = 0 <= x < V
            if uniforms is None:
                hit = inside and x == largest(row)
            elif draft is not None:
                hit = inside and float(uniforms[c]) * float(draft[node, x]) < row[x]
            else:
                p = row[x] if inside and x not in out and row[x] > 0 else 0.0
                hit = float(uniforms[c]) * left < p
                if inside and not hit:
                    left -= p
                    out.add(x)
            if hit:
                found = c
                break
        if found is None:
            break
        node = found
        walk.append(node)
    if uniforms is None:
        return walk, largest(row)
    p = [x if x > 0 else 0.0 for x in row]
    weight = [0.0 if v in out else x for v, x in enumerate(p)]
    if draft is not None and any(0 <= int(tokens[c]) < V for c in children):
        weight = [max(x - y, 0.0) if x - y > 0 else 0.0 for x, y in zip(row, draft[node].double().tolist())]
    if not math.fsum(weight) > 0:
        weight = p
    want, run = float(uniforms[0]) * math.fsum(weight), 0.0
    last = 0
    for v, x in enumerate(weight):
        run += x
        if x > 0:
            last = v
            if run > want:
                return walk, v
    return walk, last


def largest(row):
    for v, x in enumerate(row):
        if x != x:
            return v
    return row.index(max(row))


def check(target, tokens, parents, uniforms, draft):
    ops = _ops()
    B, M, V = target.shape
    d = [x if x is None else x.to(DEV) for x in (target, tokens, parents, uniforms, draft)]
    path, count, token = (x.cpu() for x in ops.verify_drafts(*d))
    counts = []
    for b in range(B):
        par = [-1] + list(range(M - 1)) if parents is None else parents[b if parents.dim() == 2 else slice(None)].tolist()
        par = [p if 0 <= p < i else -1 for i, p in enumerate(par)]
        walk, tok = rule(target[b], tokens[b], par, None if uniforms is None else uniforms[b], None if draft is None else draft[b])
        assert path[b].tolist() == walk + [-1] * (M - len(walk)), b
        assert int(count[b]) == len(walk) and int(token[b]) == tok, (b, int(token[b]), tok)
        counts.append(len(walk))
    return counts


def proposals(target, parents, g):
    """Tokens among the three likeliest after each node's parent."""
    B, M, V = target.shape
    top = target.float().topk(min(3, V), -1).indices
    tokens = torch.randint(0, V, (B, M), generator=g)
    for i in range(1, M):
        p = parents[:, i].clamp(min=0)
        pick = torch.randint(0, top.shape[-1], (B,), generator=g)
        tokens[:, i] = top[torch.arange(B), p, pick]
    return tokens


@pytest.mark.gpu
@pytest.mark.parametrize("dt", FLOATS, ids=_name)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 63, 127, 1000, 8191, 20011])
def test_modes_types_and_vocabularies(V, dt):
    g = torch.Generator().manual_seed(V)
    B, seen = 4, {"greedy": [], "tree": [], "chain": []}
    for M, kind in ((1, "chain"), (2, "chain"), (6, "chain"), (13, "tree"), (64, "tree"), (20, "star")):
        logits = 2.5 * torch.randn(B, M, V, generator=g)
        p = torch.softmax(logits, -1).to(dt)
        parents = tree_of(M, kind, B, g)
        tokens = proposals(p, parents, g)
        u = torch.rand(B, M, generator=g)
        seen["greedy"] += check(logits.to(dt), tokens, parents, None, None)
        seen["tree"] += check(p, tokens, parents, u, None)
        if kind == "chain":
            q = torch.softmax(logits[:, :M - 1] + 0.5 * torch.randn(B, M - 1, V, generator=g), -1).to(dt)
            seen["chain"] += check(p, tokens, None, u, q)
            assert torch.equal(*[x[0] for x in (_ops().verify_drafts(p.to(DEV), tokens.to(DEV), y, u.to(DEV), q.to(DEV))
                                                for y in (None, parents.to(DEV)))])
    assert max(seen["greedy"] + seen["tree"]) > 1  # some draft was taken


@pytest.mark.gpu
@pytest.mark.parametrize("dt", FLOATS, ids=_name)
def test_borders(dt):
    """Cumulated weights, acceptance and ties that are hit exactly: refusal and the next token at equality, the first
    of equal entries."""
    V = 8
    p = torch.full((1, 2, V), 0.125)
    for u0 in (0.0, 0.125, 0.25, 0.5, 0.875, 1 - 2.0 ** -24):
        for u1 in (0.0, 0.125, 0.5, 1 - 2.0 ** -24):
            u = torch.tensor([[u0, u1]])
            for tok in (0, 3, 7):
                t = torch.tensor([[0, tok]])
                check(p.to(dt), t, None, u, None)
                q = torch.zeros(1, 1, V)
                q[0, 0, tok], q[0, 0, (tok + 1) % V] = 0.25, 0.75
                check(p.to(dt), t, None, u, q.to(dt))
                check(p.to(dt), t, None, u, p[:, :1].to(dt))  # draft and target agree: accepted for every u < 1
    tie = torch.zeros(1, 3, 5000)
    tie[0, 0, [7, 4099]] = 1.0
    tie[0, 1] = -0.0
    tie[0, 2, [4999, 3000, 3001]] = math.inf
    check(tie.to(dt), torch.tensor([[0, 7, 0]]), None, None, None)
    check(tie.to(dt), torch.tensor([[0, 4099, 0]]), None, None, None)
    check(-tie.to(dt), torch.tensor([[0, 0, 0]]), None, None, None)
    tie[0, 1, 17] = math.nan
    check(tie.to(dt), torch.tensor([[0, 7, 17]]), None, None, None)
    check(torch.full((1, 2, 300), -math.inf, dtype=dt), torch.tensor([[0, 0]]), None, None, None)


@pytest.mark.gpu
def test_rows_without_weight_and_odd_entries():
    V = 600
    zero = torch.zeros(1, 2, V)
    u = torch.tensor([[0.3, 0.9]])
    t = torch.tensor([[0, 5]])
    check(zero, t, None, u, None)                     # no weight: token 0
    one = zero.clone()
    one[0, 0, 5] = 1.0
    one[0, 1, 599] = 1.0
    check(one, t, None, u, None)                      # accepted for sure
    check(one, torch.tensor([[0, 6]]), None, u, None)
    q = zero[:, :1].clone()
    q[0, 0, 6] = 1.0
    check(one, torch.tensor([[0, 6]]), None, u, q)
    # every token with weight was refused (their sum stays below 1): p itself
    few = zero.clone()
    few[0, 0, 5], few[0, 0, 9] = 0.25, 0.25
    both = torch.tensor([[0, 5, 9]])
    few3 = torch.cat((few, few[:, :1]), 1)
    check(few3, both, torch.tensor([[-1, 0, 0]]), torch.tensor([[0.6, 0.9, 0.9]]), None)
    # draft above target everywhere
    check(few, t, None, u, (few[:, :1] * 2 + 0.5))
    odd = torch.softmax(torch.randn(1, 4, V, generator=torch.Generator().manual_seed(1)), -1)
    odd[0, :, 3], odd[0, :, 4] = math.nan, -0.5
    check(odd, torch.tensor([[0, 3, 4, 8]]), torch.tensor([[-1, 0, 0, 0]]), torch.tensor([[0.001, 0.0, 0.0, 0.9]]), None)
    # tokens outside the vocabulary, parents that are no earlier node, the same token twice
    tok = torch.tensor([[0, V, -1, 2 ** 40, 8, 8, 11]])
    par = torch.tensor([[5, 0, 0, 0, 0, 0, 9]])
    for u1 in (0.0, 0.99):
        check(torch.cat((odd, odd[:, :3]), 1), tok, par, torch.full((1, 7), u1), None)
        check(torch.cat((odd, odd[:, :3]), 1), tok, par, None, None)
    # a uniform of 1 or a NaN still gives a token of the vocabulary
    for bad in (1.0, math.nan, -1.0):
        out = _ops().verify_drafts(odd.to(DEV), torch.tensor([[0, 9, 9, 9]], device=DEV), None,
                                   torch.tensor([[bad, 0.9, 0.9, 0.9]], device=DEV))[2]
        assert 0 <= int(out) < V


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["tree", "chain"])
def test_tokens_are_distributed_as_the_target(mode):
    """The first token emitted (the accepted child or the next token) over 200000 sequences of one row: each share
    within 5 standard deviations of the target's probability."""
    B, V = 200000, 6
    g = torch.Generator(device=DEV).manual_seed(0)
    p = torch.tensor([0.05, 0.3, 0.2, 0.25, 0.15, 0.05], device=DEV)
    q = torch.tensor([0.4, 0.1, 0.1, 0.1, 0.2, 0.1], device=DEV)
    if mode == "chain":
        M, par, draft = 2, None, q.expand(B, 1, V).contiguous()
        tokens = torch.zeros(B, M, dtype=torch.int64, device=DEV)
        tokens[:, 1] = torch.multinomial(q, B, True, generator=g)
    else:
        M, draft = 4, None
        par = torch.tensor([-1, 0, 0, 0], device=DEV)
        tokens = torch.tensor([0, 2, 5, 2], device=DEV).expand(B, M)
    u = torch.rand(B, M, device=DEV, generator=g)
    path, count, token = _ops().verify_drafts(p.expand(B, M, V).contiguous(), tokens, par, u, draft)
    first = torch.where(count > 1, tokens.gather(1, path[:, 1:2].clamp(min=0)).squeeze(1), token)
    share = torch.bincount(first, minlength=V).double() / B
    sigma = (p.double() * (1 - p.double()) / B).sqrt()
    assert ((share - p.double()).abs() < 5 * sigma).all(), share.tolist()
    assert 0.2 < float((count > 1).double().mean()) < 0.9


@pytest.mark.gpu
@pytest.mark.parametrize("dt", FLOATS, ids=_name)
@pytest.mark.parametrize("pad", [-1, 37, 2 ** 40])
def test_a_padded_chain_is_the_shorter_chain(dt, pad):
    """Sequences with fewer drafts than the batch holds: behind them stand tokens outside the vocabulary, or parents that
    are none, with draft rows of any content."""
    V, B, M = 37, 64, 6
    g = torch.Generator().manual_seed(5)
    logits = 2 * torch.randn(B, M, V, generator=g)
    p = torch.softmax(logits, -1).to(dt)
    q = torch.softmax(logits[:, :M - 1] + 0.3 * torch.randn(B, M - 1, V, generator=g), -1).to(dt)
    tokens = torch.cat((torch.zeros(B, 1), torch.multinomial(q.float().flatten(0, 1), 1, generator=g).view(B, M - 1)), 1).long()
    u = torch.rand(B, M, generator=g)
    short = torch.arange(B) % M + 1  # nodes of each sequence
    behind = torch.arange(M) >= short.unsqueeze(1)
    padded = torch.where(behind, pad, tokens)
    parents = torch.where(behind, -1, torch.arange(-1, M - 1))
    for t, par in ((padded, None), (tokens, parents), (padded, parents)):
        check(p, t, par, u, q)
        out = [x.cpu() for x in _ops().verify_drafts(p.to(DEV), t.to(DEV), None if par is None else par.to(DEV), u.to(DEV), q.to(DEV))]
        for b in range(B):
            n = int(short[b])
            one = _ops().verify_drafts(*(x[b:b + 1, :m].contiguous().to(DEV) if x is not None else None
                                         for x, m in ((p, n), (tokens, n), (None, 0), (u, n), (q, n - 1))))
            assert out[0][b, :n].tolist() == one[0][0].tolist() and (out[0][b, n:] == -1).all()
            assert int(out[1][b]) == int(one[1]) and int(out[2][b]) == int(one[2]), b


@pytest.mark.gpu
def test_strides_and_offsets():
    """Rows at odd addresses, transposed batches, a vocabulary that is not the last stride."""
    g = torch.Generator().manual_seed(3)
    B, M, V = 3, 5, 1001
    p = torch.softmax(torch.randn(B, M, V, generator=g), -1)
    tokens = proposals(p, tree_of(M, "chain", B, g), g)
    u = torch.rand(B, M, generator=g)
    ops = _ops()
    for dt in FLOATS:
        x = p.to(dt).to(DEV)
        d = torch.softmax(p[:, :M - 1] * 30, -1).to(dt).to(DEV)
        for uu, dd in ((u.to(DEV), None), (u.to(DEV), d), (None, None)):
            base = ops.verify_drafts(x, tokens.to(DEV), None, uu, dd)
            wide = torch.zeros(B, M, V + 6, dtype=dt, device=DEV)
            wide[..., 3:3 + V] = x
            turned = x.transpose(0, 1).contiguous().transpose(0, 1)
            strided = torch.zeros(B, M, V, 2, dtype=dt, device=DEV)
            strided[..., 0] = x
            for y in (wide[..., 3:3 + V], turned, strided[..., 0]):
                assert all(torch.equal(a, b) for a, b in zip(base, ops.verify_drafts(y, tokens.to(DEV), None, uu, dd)))


@pytest.mark.gpu
def test_replays_in_a_graph():
    ops = _ops()
    g = torch.Generator().manual_seed(5)
    B, M, V = 4, 9, 3001
    x = torch.softmax(2 * torch.randn(B, M, V, generator=g), -1).to(DEV)
    tokens = proposals(x.cpu(), tree_of(M, "chain", B, g), g).to(DEV)
    u = torch.rand(B, M, device=DEV)
    q = torch.softmax(torch.randn(B, M - 1, V, device=DEV), -1)
    calls = [lambda: ops.verify_drafts(x, tokens, None, u, None), lambda: ops.verify_drafts(x, tokens, None, u, q),
             lambda: ops.verify_drafts(x, tokens)]
    for call in calls:
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for _ in range(4):
            x.copy_(torch.softmax(2 * torch.randn(B, M, V, device=DEV), -1))
            u.uniform_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, call()))


@pytest.mark.gpu
def test_refusals():
    ops = _ops()
    x = torch.zeros(2, 3, 9, device=DEV)
    t = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    u = torch.zeros(2, 3, device=DEV)
    d = torch.zeros(2, 2, 9, device=DEV)
    assert ops.verify_drafts(x[:0], t[:0])[0].shape == (0, 3)
    for error, args in ((TypeError, (x.double(), t)), (TypeError, (x[0], t)), (ValueError, (x, t.int())),
                        (ValueError, (x, t[:, :2])), (ValueError, (x, t, t[:, :2])), (ValueError, (x, t, t.int())),
                        (ValueError, (x, t, None, u.double())), (ValueError, (x, t, None, u[:, :2])),
                        (ValueError, (x, t, None, None, d)), (ValueError, (x, t, None, u, x)),
                        (ValueError, (x, t, None, u, d.half())), (RuntimeError, (x.cpu(), t)), (RuntimeError, (x, t.cpu())),
                        (ValueError, (torch.zeros(1, 65, 4, device=DEV), torch.zeros(1, 65, dtype=torch.int64, device=DEV))),
                        (ValueError, (x[:, :0], t[:, :0])), (_native_error(), (x[..., :0], t))):
        with pytest.raises(error):
            ops.verify_drafts(*args)


def test_c_entry_refuses_bad_arguments():
    """Argument checks run before any device work.  The pointers are no addresses, so this runs only where no
    kernel could start."""
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would start a kernel")
    from multiscreen import _native
    L = _native.lib()

    def verify(**kw):
        a = dict(t=16, d=0, tok=16, par=0, psb=0, u=16, B=2, M=4, V=100, dt=0, path=16, count=16, token=16, ws=0, wsb=0)
        a.update(kw)
        return L.msa_verify(_native.pack_verify_args(a["t"], 400, 100, a["d"], 300, 100, a["tok"], a["par"], a["psb"], a["u"], a["path"],
                                                     a["count"], a["token"], a["ws"], a["wsb"], a["B"], a["M"], a["V"], a["dt"]), None)

    for kw, code, msg in ((dict(dt=3), 1, "dtype"), (dict(M=65), 1, "nodes"), (dict(M=0), 1, "nodes"), (dict(V=0), 1, "vocabulary"),
                          (dict(V=1 << 31), 1, "vocabulary"), (dict(u=0, d=16), 1, "uniforms"), (dict(t=0), 1, "null"),
                          (dict(t=18), 1, "aligned"), (dict(path=0), 1, "null"), (dict(psb=-1), 1, "strides"),
                          (dict(u=0), 2, "verify workspace")):
        assert verify(**kw) == code, kw
        assert msg in L.msa_last_error().decode(), (kw, L.msa_last_error())
    assert verify(B=0) == 0
    assert L.msa_verify_workspace_bytes(2, 4, 100, 1) == 2 * 4 * 8 and L.msa_verify_workspace_bytes(2, 4, 100, 0) == 0
