"""ops.tree_decode against the definition in float64: every pairing of query
and cache type, head sizes, one to 64 nodes, chains and trees, windows from
less than a step to endless, sequences from empty to long, rows that are zero
or not finite, masked places that hold garbage, splits, graphs, refusals."""

import math

import pytest
import torch

from test_gpu_cache_rows import CODES, DEV, FLOATS, TOP, _name, _native_error, _ops, empty_cache

EPS = 1e-8


def tree_of(M, kind, B, g):
    """(B, M) parents: a chain, a star, two roots, or a random tree of each sequence's own."""
    i = torch.arange(M).expand(B, M)
    if kind == "chain":
        return i - 1
    if kind == "star":
        return torch.where(i == 0, -1, 0)
    if kind == "roots":
        return torch.where(i < 2, -1, i - 2)
    back = 1 + torch.randint(0, 6, (B, M), generator=g)
    return torch.where(i == 0, -1, (i - back).clamp(min=0))


def lines_of(parents):
    """Each node's way up (itself first) by walking."""
    out = []
    for i, p in enumerate(parents.tolist()):
        out.append([i] + (out[p] if 0 <= p < i else []))
    return out


def definition(q, k, v, n, parents, r, w, eps=EPS):
    """One sequence, float64: q (M, H, D), k and v (n + M, H, D) as the cache holds them."""
    M, H, D = q.shape
    lines = lines_of(parents)
    depth = torch.tensor([len(x) - 1 for x in lines])
    place = torch.cat((torch.arange(n), n + depth))
    seen = torch.zeros(M, n + M, dtype=torch.bool)
    seen[:, :n] = True
    for i, x in enumerate(lines):
        seen[i, [n + j for j in x]] = True
    d = (n + depth).view(M, 1) - place.view(1, -1)
    y = torch.zeros(M, H, D, dtype=torch.float64)

    def unit(x):
        return x / x.norm(dim=-1, keepdim=True).clamp(min=eps)

    for h in range(H):
        s = unit(q[:, h]) @ unit(k[:, h]).T
        a = (1.0 - float(r[h]) * (1.0 - s)).clamp(min=0.0)
        m = torch.cos(0.5 * math.pi * d / float(w[h])) ** 2
        weight = torch.where(seen & (d >= 0) & (d < float(w[h])), a * a * m, 0.0)
        weight = torch.where(weight > 0, weight, 0.0)  # a NaN key is not live
        rows = unit(v[:, h])
        live = weight.unsqueeze(-1) * rows
        x = torch.where(weight.unsqueeze(-1) > 0, live, 0.0).sum(1)
        size = x.norm(dim=-1, keepdim=True).clamp(min=eps)
        y[:, h] = x * torch.tanh(size) / size
    return y


class Case:
    """A cache of B sequences with their drafted rows, filled by torch alone."""

    def __init__(self, B, M, H, D, dt, ct, lengths, kind="tree", w=(2.0, 300.0), r=1.2, seed=0, room=5, centred=True):
        g = torch.Generator().manual_seed(seed)
        self.M, self.lengths = M, lengths
        cap = max(lengths) + M + room
        centres = torch.randn(H, 6, D, generator=g)

        def rows(T, mixed):
            x = torch.randn(B, T, H, D, generator=g)
            if mixed and centred:
                at = torch.randint(0, 6, (B, T, H), generator=g)
                x = 0.7 * centres[torch.arange(H), at] + 0.7 * x
            return x * torch.exp(0.5 * torch.randn(B, T, H, 1, generator=g))

        self.q = rows(M, True).to(dt)
        k, v = rows(cap, True), rows(cap, False)
        self.kc, self.vc, self.ks, self.vs = empty_cache(B, cap, H, D, ct, device="cpu", fill=0)
        for x, c, s in ((k, self.kc, self.ks), (v, self.vc, self.vs)):
            if s is None:
                c.copy_(x.to(dt))
            else:
                s.copy_(x.abs().amax(-1) / TOP[ct])
                c.copy_((x / s.unsqueeze(-1)).clamp(-TOP[ct], TOP[ct]).round() if ct == torch.int8 else x / s.unsqueeze(-1))
        self.r = torch.full((H,), r) + 0.05 * torch.rand(H, generator=g)
        self.w = torch.linspace(w[0], w[1], H)
        self.parents = tree_of(M, kind, B, g)

    def run(self, parents="own", hint=0, lengths=None, **kw):
        dev = [x if x is None else x.to(DEV) for x in (self.q, self.kc, self.vc, self.ks, self.vs, self.r, self.w)]
        # .to keeps the head-major layout
        p = self.parents if isinstance(parents, str) else parents
        n = torch.tensor(self.lengths if lengths is None else lengths, device=DEV)
        return _ops().tree_decode(dev[0], dev[1], dev[2], n, None if p is None else p.to(DEV), dev[5], dev[6], EPS,
                                  dev[3], dev[4], None, hint, **kw)

    def expected(self):
        k, v = self.kc.double(), self.vc.double()
        if self.ks is not None:
            k, v = k * self.ks.double().unsqueeze(-1), v * self.vs.double().unsqueeze(-1)
        return torch.stack([definition(self.q[b].double(), k[b, :n + self.M], v[b, :n + self.M], n, self.parents[b],
                                       self.r, self.w) for b, n in enumerate(self.lengths)])


# The result is a sum of weighted unit rows of norm up to 1 before it is rounded to q's type.
#  - rounding to the type: at most eps/2 of each element (float32's is below the rest)
#  - s: D products of 2-byte operands are exact in fp32 and their sum is off by at most (D + 3) 2^-24; the weight a^2
#    moves by 2 a r ds, so relative to the sum of weights by at most 2 r ds / a.  Weighted by a^2 the mean of 1/a is at
#    most the inverse of the rms a; the cases' live pairs have an rms a above 0.1, so 2 * 1.25 * 131 * 2^-24 / 0.1
#    = 2e-4 at D = 128 in the worst rounding; random roundings grow with sqrt(D): 2e-5.
#  - weights as two terms: 2^-17 (bf16) or 2^-23 (fp16) of a weight.
# Sums of M rows of mixed sign may cancel to a tenth of their terms: a factor 10 on the second and third.
def tolerance(dt):
    return torch.finfo(dt).eps / 2 + (2e-4 if dt != torch.float32 else 2e-5)


def check(case, got):
    ref = case.expected()
    got = got.double().cpu()
    dt = case.q.dtype
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    ref, got = ref.nan_to_num(0.0), got.nan_to_num(0.0)
    size = ref.abs().amax(dim=(1, 3), keepdim=True)  # per sequence and head
    err = (got - ref).abs() / size.clamp(min=1e-2 * float(ref.abs().max()) + 1e-30)
    assert float(err.max()) <= tolerance(dt), float(err.max())
    return float(err.max())


PAIRS = [(dt, ct) for dt in FLOATS for ct in [dt] + CODES]
PAIR_IDS = [f"{_name(a)}-{_name(b)}" for a, b in PAIRS]


@pytest.mark.gpu
@pytest.mark.parametrize("dt,ct", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_types_and_head_sizes(dt, ct, D):
    for M, kind, lengths in ((1, "chain", [77, 0]), (21, "tree", [300, 5]), (64, "tree", [95, 401])):
        case = Case(2, M, 3, D, dt, ct, lengths, kind, seed=D + M)
        assert case.expected().abs().max() > 0.05
        check(case, case.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dt,ct", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_small_trees(dt, ct, D):
    """Up to 16 nodes and one more, over short and split windows."""
    for M, kind, lengths in ((2, "chain", [31, 1]), (9, "roots", [64, 130]), (15, "tree", [0, 250]), (16, "tree", [40, 97]),
                             (17, "tree", [40, 97])):
        check_case = Case(2, M, 2, D, dt, ct, lengths, kind, w=(40.0, 200.0), seed=7 * D + M)
        check(check_case, check_case.run())
    case = Case(1, 12, 3, D, dt, ct, [3000], "tree", w=(500.0, 4000.0), r=1.3, seed=D)
    check(case, case.run())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "star", "roots", "tree"])
@pytest.mark.parametrize("M", [1, 2, 5, 31, 32, 33, 63, 64])
def test_trees(M, kind):
    for dt, ct in ((torch.bfloat16, torch.bfloat16), (torch.float32, torch.int8)):
        case = Case(2, M, 2, 64, dt, ct, [150, 31], kind, w=(3.0, 90.0), seed=M)
        got = case.run()
        check(case, got)
        if kind == "chain":
            assert torch.equal(got, case.run(parents=None))
        assert torch.equal(got, case.run())  # the same call gives the same bits


@pytest.mark.gpu
@pytest.mark.parametrize("n", [0, 1, 2, 30, 31, 32, 33, 63, 64, 65, 255, 256, 257, 1000])
def test_lengths_and_windows(n):
    """Units that start and end anywhere; windows below one step, at unit borders, longer than everything."""
    for w in ((0.5, 1.0), (1.0, 1.5), (2.0, 32.0), (33.0, 64.0), (100.0, math.inf)):
        case = Case(1, 7, 2, 32, torch.bfloat16, torch.bfloat16, [n], "tree", w=(1.0, 1.0), seed=n)
        case.w = torch.tensor(w)
        check(case, case.run())
        case = Case(1, 40, 2, 64, torch.float16, torch.int8, [n], "chain", w=(1.0, 1.0), seed=n)
        case.w = torch.tensor(w)
        check(case, case.run())


@pytest.mark.gpu
@pytest.mark.parametrize("H", [1, 63, 64, 65, 130])
def test_many_heads_share_the_blocks(H):
    """Windows from nothing to everything over more heads than a wave has lanes; heads without a key."""
    for M, n in ((3, [2000, 100]), (40, [1500])):
        case = Case(len(n), M, H, 32, torch.bfloat16, torch.int8, n, "tree", r=1.3, seed=H)
        case.w = torch.exp(torch.linspace(0.0, math.log(3000.0), H))[torch.randperm(H, generator=torch.Generator().manual_seed(H))]
        base = case.run()
        check(case, base)
        empty = case.w.clone()
        empty[:: 3] = math.nan
        case.w, full = empty, case.w
        got = case.run()
        assert (got[:, :, ::3] == 0).all()
        keep = [h for h in range(H) if h % 3]
        size = float(base.float().abs().max())
        # another split of the same sums: two roundings of bf16 apart
        assert float((got[:, :, keep].float() - base[:, :, keep].float()).abs().max() if keep else 0.0) <= 2 * 2.0 ** -8 * size


@pytest.mark.gpu
def test_split_over_blocks_and_hints():
    """Long windows split over blocks; a hint only changes the split."""
    for dt, ct, M in ((torch.bfloat16, torch.bfloat16, 9), (torch.bfloat16, torch.int8, 64), (torch.float32, torch.float32, 33),
                      (torch.float16, torch.float8_e4m3fn, 1)):
        case = Case(2, M, 3, 64, dt, ct, [5000, 3777], "tree", w=(100.0, 6000.0), r=1.3, seed=M)
        for hint in (0, 1, 256, 3000, 10 ** 6):
            check(case, case.run(hint=hint))


@pytest.mark.gpu
@pytest.mark.parametrize("ct", [torch.float32, torch.bfloat16, torch.float16] + CODES, ids=_name)
def test_masked_places_may_hold_anything(ct):
    """Rows past the drafted ones, of other branches and before every window hold NaN and infinities: nothing changes."""
    dt = torch.bfloat16 if ct in TOP else ct
    case = Case(2, 12, 2, 64, dt, ct, [200, 90], "star", w=(20.0, 40.0), seed=3)
    clean = case.run()
    check(case, clean)
    bad = torch.tensor([math.nan, math.inf, -math.inf])
    for b, n in enumerate(case.lengths):
        for pos in list(range(0, n - 60)) + list(range(n + 12, case.kc.shape[1])):
            for c, s in ((case.kc, case.ks), (case.vc, case.vs)):
                if s is None:
                    c[b, pos] = bad[pos % 3]
                else:
                    s[b, pos] = bad[pos % 3]
                    if ct == torch.float8_e4m3fn:
                        c[b, pos] = torch.full((2, 64), math.nan).to(ct)
    assert torch.equal(case.run(), clean)
    # node 5's rows: node 5 alone changes
    for c, s in ((case.kc, case.ks), (case.vc, case.vs)):
        for b, n in enumerate(case.lengths):
            if s is None:
                c[b, n + 5] = math.nan
            else:
                s[b, n + 5] = math.nan
    got = case.run()
    keep = [i for i in range(12) if i != 5]
    assert torch.equal(got[:, keep], clean[:, keep])


@pytest.mark.gpu
@pytest.mark.parametrize("ct", [torch.float32, torch.bfloat16, torch.float16] + CODES, ids=_name)
def test_rows_that_are_not_finite_or_zero(ct):
    """A live value row with a NaN or an infinity makes the nodes that see it NaN, a key row drops out; zero rows of
    q, k and v take part as zeros."""
    dt = torch.bfloat16 if ct in TOP else ct
    case = Case(2, 6, 2, 32, dt, ct, [40, 33], "chain", w=(60.0, 80.0), r=1.02, seed=8)
    case.kc[0, 7] = 0
    case.vc[0, 9] = 0
    case.q[0, 2] = 0
    if case.ks is not None:
        case.ks[1, 11] = math.nan
        case.vs[1, 35, 0] = math.nan  # drafted row 2 of sequence 1
        case.ks[0, 12], case.vs[0, 13] = 0.0, 0.0
    else:
        case.kc[1, 11, :, 3] = math.inf
        case.kc[1, 12, :, 3] = math.nan
        case.vc[1, 35, 0, 5] = math.nan
        case.vc[1, 36, 1, 5] = -math.inf
    ref = case.expected()
    # some node with a live pair to that row, and none that does not see it
    assert torch.isnan(ref[1, 2:, 0]).any() and not torch.isnan(ref[0]).any() and not torch.isnan(ref[1, :2]).any()
    check(case, case.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", FLOATS, ids=_name)
def test_rows_of_extreme_length(dt):
    """Rows far from length 1 in the cache and in q: only directions matter."""
    small = {torch.float32: 1e-7, torch.bfloat16: 1e-7, torch.float16: 2e-4}[dt]
    big = {torch.float32: 1e15, torch.bfloat16: 1e15, torch.float16: 5e3}[dt]
    for f in (small, big):
        for ct in [dt] + CODES:
            case = Case(1, 10, 2, 64, dt, ct, [70], "tree", w=(50.0, 90.0), seed=2)
            case.q = (case.q.float() * f).to(dt)
            for c, s in ((case.kc, case.ks), (case.vc, case.vs)):
                if s is None:
                    c.copy_((c.float() * f).to(dt))
                else:
                    s.mul_(f)
            check(case, case.run())


@pytest.mark.gpu
@pytest.mark.parametrize("ct", CODES, ids=_name)
def test_codes_that_do_not_reach_the_top(ct):
    """Rows of small codes (one scale for many rows, say) and zero codes under a scale: directions and zeros as ever."""
    case = Case(1, 8, 2, 64, torch.bfloat16, ct, [90], "tree", w=(50.0, 120.0), seed=5)
    for c in (case.kc, case.vc):
        x = c.float()
        x[:, ::3] = (x[:, ::3] / 40).round()
        x[:, 1::3] = torch.sign(x[:, 1::3]) * (torch.arange(64) == 5) * (1.0 if ct == torch.int8 else 2.0 ** -9)
        x[:, 8] = 0
        c.copy_(x.to(ct))
    check(case, case.run())


@pytest.mark.gpu
def test_empty_window_and_foreign_parents():
    case = Case(1, 9, 3, 32, torch.float32, torch.float32, [50], "chain", seed=4)
    case.w = torch.tensor([math.nan, -1.0, 30.0])
    got = case.run()
    assert (got[:, :, :2] == 0).all() and got[:, :, 2].abs().max() > 0
    # a parent that is no earlier node makes a root
    case.w = torch.tensor([5.0, 10.0, 30.0])
    odd = torch.tensor([[3, 0, 2, 100, -7, 4, 6, 2 ** 40, 7]])
    case.parents = torch.tensor([[-1, 0, -1, -1, -1, 4, -1, -1, 7]])
    check(case, case.run(parents=odd))


@pytest.mark.gpu
def test_lengths_are_clamped_and_shared():
    case = Case(2, 5, 2, 32, torch.bfloat16, torch.int8, [60, 60], "chain", room=0, seed=6)
    base = case.run()
    check(case, base)
    assert torch.equal(case.run(lengths=[60]), base)
    assert torch.equal(case.run(lengths=[61, 2 ** 40]), base)  # past the capacity
    assert torch.equal(case.run(lengths=[-5]), case.run(lengths=[0]))
    shared = case.parents[:1]
    assert torch.equal(case.run(parents=shared[0]), base)


@pytest.mark.gpu
def test_strided_inputs():
    """q as a slice of a stacked projection, caches in (B, T, H, D) order and as slices of longer ones."""
    case = Case(2, 6, 3, 64, torch.bfloat16, torch.int8, [40, 77], "tree", seed=7)
    base = case.run()
    ops = _ops()
    x = torch.randn(2, 6, 3 * 3 * 64, dtype=torch.bfloat16, device=DEV)
    x[:, :, 192:384] = case.q.reshape(2, 6, 192).to(DEV)
    q = x.split(192, dim=-1)[1].view(2, 6, 3, 64)

    def long(c):
        big = torch.zeros(2, c.shape[1] + 16, *c.shape[2:], device=DEV, dtype=torch.float32).to(c.dtype)
        big[:, 7:7 + c.shape[1]] = c.to(DEV)
        return big[:, 7:7 + c.shape[1]]

    got = ops.tree_decode(q, long(case.kc), long(case.vc), torch.tensor(case.lengths, device=DEV), case.parents.to(DEV),
                          case.r.to(DEV), case.w.to(DEV), EPS, long(case.ks), long(case.vs))
    assert torch.equal(got, base)


@pytest.mark.gpu
def test_a_cache_past_32_bit_offsets():
    """Keys whose byte and element offsets pass 2^32: the last window of a long cache of many heads."""
    ops = _ops()
    case = Case(1, 4, 9, 128, torch.bfloat16, torch.int8, [100], "chain", w=(50.0, 90.0), seed=9, room=0)
    cap, H, D = 2 ** 22 - 1, 9, 128
    shift = cap - 104
    kc, vc = (torch.zeros(1, H, cap, D, dtype=torch.int8, device=DEV).transpose(1, 2) for _ in range(2))
    ks, vs = (torch.zeros(1, H, cap, device=DEV).transpose(1, 2) for _ in range(2))
    for a, b in ((kc, case.kc), (vc, case.vc), (ks, case.ks), (vs, case.vs)):
        a[:, shift:] = b.to(DEV)
    got = ops.tree_decode(case.q.to(DEV), kc, vc, torch.tensor([shift + 100], device=DEV), None, case.r.to(DEV),
                          case.w.to(DEV), EPS, ks, vs, None, 90)
    check(case, got)


@pytest.mark.gpu
def test_one_node_is_the_decode_step():
    """M = 1 over a cache of the input type against ops.decode_step of the same position."""
    ops = _ops()
    for dt in FLOATS:
        case = Case(3, 1, 4, 64, dt, dt, [500, 500, 500], "chain", w=(2.0, 400.0), seed=1)
        got = case.run()[:, 0]
        ref = ops.decode_step(case.q[:, 0].to(DEV), case.kc.to(DEV), case.vc.to(DEV), 501, case.r.to(DEV), case.w.to(DEV))
        size = ref.float().abs().amax()
        # both are within `tolerance` of the definition
        assert float((got.float() - ref.float()).abs().max() / size) <= 2 * tolerance(dt)


@pytest.mark.gpu
def test_other_stream_and_graph_replays():
    case = Case(2, 8, 2, 64, torch.bfloat16, torch.int8, [3000, 2500], "tree", w=(100.0, 4000.0), seed=12)
    ops = _ops()
    dev = [x.to(DEV) for x in (case.q, case.kc, case.vc, case.ks, case.vs, case.r, case.w)]
    n, par = torch.tensor(case.lengths, device=DEV), case.parents.to(DEV)

    def step():
        return ops.tree_decode(dev[0], dev[1], dev[2], n, par, dev[5], dev[6], EPS, dev[3], dev[4])

    base = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(base, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for shift in (0, -400, -37, 0, 3):
        n.copy_(torch.tensor(case.lengths) + shift)
        dev[0].normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step()), shift


@pytest.mark.gpu
def test_calls_at_the_same_time():
    """Split calls on two streams, each with its own scratch, interleaved with writes to other caches."""
    ops = _ops()
    cases = [Case(2, 20, 4, 64, torch.bfloat16, torch.int8, [4000, 3500], "tree", w=(100.0, 4000.0), seed=20),
             Case(1, 5, 6, 64, torch.bfloat16, torch.bfloat16, [6000], "chain", w=(50.0, 6000.0), seed=21)]
    args = [[x if x is None else x.to(DEV) for x in (c.q, c.kc, c.vc, c.ks, c.vs, c.r, c.w, torch.tensor(c.lengths), c.parents)]
            for c in cases]

    def call(d):
        return ops.tree_decode(d[0], d[1], d[2], d[7], d[8], d[5], d[6], EPS, d[3], d[4])

    base = [call(d) for d in args]
    for c, y in zip(cases, base):
        check(c, y)
    streams = [torch.cuda.Stream() for _ in args]
    spare = empty_cache(1, 64, 6, 64, torch.int8)
    x = torch.randn(1, 64, 6, 64, device=DEV, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (d, st) in enumerate(zip(args, streams)):
            with torch.cuda.stream(st):
                got[i].append(call(d))
        ops.cache_write(x, x, spare[0], spare[1], 0, spare[2], spare[3])
    torch.cuda.synchronize()
    assert all(torch.equal(y, b) for ys, b in zip(got, base) for y in ys)


@pytest.mark.gpu
def test_empty_batch_and_refusals():
    ops = _ops()
    case = Case(2, 4, 2, 32, torch.bfloat16, torch.int8, [20, 9], "chain", seed=1)
    d = [x.to(DEV) for x in (case.q, case.kc, case.vc, case.ks, case.vs, case.r, case.w)]
    n, par = torch.tensor([20, 9], device=DEV), case.parents.to(DEV)
    assert ops.tree_decode(d[0][:0], d[1][:0], d[2][:0], n[:0], None, d[5], d[6], EPS, d[3][:0], d[4][:0]).shape[0] == 0
    assert ops.tree_decode(d[0][:, :0], d[1], d[2], n, None, d[5], d[6], EPS, d[3], d[4]).shape[1] == 0

    def call(q=d[0], kc=d[1], vc=d[2], n=n, par=par, r=d[5], w=d[6], eps=EPS, ks=d[3], vs=d[4]):
        return ops.tree_decode(q, kc, vc, n, par, r, w, eps, ks, vs)

    big = torch.zeros(2, 65, 2, 32, dtype=torch.bfloat16, device=DEV)
    for error, kw in ((ValueError, dict(q=big)), (ValueError, dict(ks=None)), (ValueError, dict(ks=d[3].double())),
                      (TypeError, dict(kc=d[1].float(), vc=d[2].float(), ks=None, vs=None)), (RuntimeError, dict(q=case.q)),
                      (ValueError, dict(n=n.int())), (ValueError, dict(n=n[:0])), (ValueError, dict(par=par[:, :3])),
                      (ValueError, dict(par=par.int())), (ValueError, dict(r=d[5][:1])), (ValueError, dict(q=d[0][:1])),
                      (_native_error(), dict(eps=0.0)), (TypeError, dict(q=d[0].double())), (RuntimeError, dict(n=n.cpu())),
                      (ValueError, dict(kc=d[1][:, :5]))):
        with pytest.raises(error):
            call(**kw)
    with pytest.raises(IndexError):
        call(q=big[:, :64], par=None)


def test_c_entry_refuses_bad_arguments():
    """Argument checks run before any device work.  The pointers are no addresses, so this runs only where no
    kernel could start."""
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would start a kernel")
    from multiscreen import _native
    L = _native.lib()

    def tree(**kw):
        a = dict(q=16, qs=(512, 128, 64), c=16, cs=(25600000, 64, 12800000), cap=200000, ct=3, s=16, ss=(400000, 1, 200000), B=2, N=4,
                 H=2, D=64, dt=1, n=16, nn=2, par=0, psb=0, hint=0, r=16, w=16, eps=1e-8, y=16, ws=16, wsb=1 << 30)
        a.update(kw)
        c, s = (a["c"], *a["cs"]), (a["s"], *a["ss"])
        return L.msa_tree_decode(_native.pack_tree_args(a["q"], *a["qs"], *c, *c, *s, *s, a["n"], a["par"], a["r"], a["w"], a["y"],
                                                        a["ws"], a["wsb"], a["nn"], a["psb"], a["B"], a["N"], a["H"], a["D"], a["dt"],
                                                        a["cap"], a["ct"], a["hint"], a["eps"]), None)

    for kw, code, msg in ((dict(N=65), 1, "at most 64"), (dict(N=4, cap=3), 1, "do not hold"), (dict(D=48), 1, "head_dim"),
                          (dict(ct=0), 1, "cache_dtype"), (dict(q=0), 1, "q is null"), (dict(qs=(512, 4, 64)), 1, "strides"),
                          (dict(n=0), 1, "lengths"), (dict(nn=3), 1, "lengths"), (dict(r=0), 1, "r and w"),
                          (dict(eps=0.0), 1, "eps"), (dict(y=8), 1, "aligned"), (dict(s=0), 1, "scales"),
                          (dict(wsb=16), 2, "tree workspace"), (dict(ws=0), 2, "tree workspace"), (dict(psb=-1), 1, "parents"),
                          (dict(H=32768, B=1, cap=2 ** 22), 1, "2^35"), (dict(N=2 ** 33), 1, "size")):
        assert tree(**kw) == code, kw
        assert msg in L.msa_last_error().decode(), (kw, L.msa_last_error())
    assert tree(B=0) == 0 and tree(N=0) == 0
    # short spans take one block a head; sums of several blocks a head are N D floats each
    assert L.msa_tree_workspace_bytes(2, 2, 4, 64, 1, 3, 500, 200) == 0
    need = L.msa_tree_workspace_bytes(2, 2, 4, 64, 1, 3, 200000, 0)
    assert need > 256 and (need - 256) % (2 * 4 * 64 * 4) == 0  # and the heads' table
    assert L.msa_tree_workspace_bytes(2, 2, 65, 64, 1, 3, 500, 200) == 0
