"""ops.linear_cross_entropy and ops.linear_distillation on the GPU: values and gradients against 64 bits within bounds
counted in roundings, rows that do not count, odd sizes and strides, every reduction, graphs, streams, equal calls."""

import math

import pytest
import torch

import wide_reference as R
from multiscreen import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _data(N, d, V, dtype, seed=0, scale=1.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(N, d, device=DEV, generator=g).to(dtype)
    w = (torch.randn(V, d, device=DEV, generator=g) * scale / math.sqrt(d)).to(dtype)
    y = torch.randint(0, V, (N,), device=DEV, generator=g)
    return x, w, y, g


def _teacher(N, V, K, g, dtype=torch.float32):
    ids = torch.randint(0, V, (N, K), device=DEV, generator=g)
    return (3.0 * torch.randn(N, K, device=DEV, generator=g)).to(dtype), ids


def _grads(loss, x, w, dloss=None):
    return torch.autograd.grad(loss, (x, w), dloss)


def _leaf(*t):
    return [x.detach().requires_grad_() for x in t]


def _check_head(x, w, ids, p, live, temperature, coef, loss, dx, dw, reduction):
    want = R.head(x.detach(), w.detach(), ids, p, live, temperature, coef)
    value, bound = want["loss"]
    if reduction == "none":
        R.check("loss", loss, value, bound)
    else:
        n = live.sum() if reduction == "mean" else 1
        R.check("loss", loss, value.sum() / n, bound.sum() / n + 4 * R.U32 * value.abs().sum() / n)
    R.check("dhidden", dx, *want["dhidden"])
    R.check("dweight", dw, *want["dweight"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,d,V", [(1, 1, 1), (1, 64, 300), (5, 32, 7), (127, 33, 255), (128, 64, 256), (129, 96, 257),
                                   (300, 100, 1003), (64, 512, 5000), (700, 200, 2000), (33, 1000, 511), (16, 512, 50257),
                                   (2500, 48, 900)])
def test_cross_entropy(N, d, V, dtype):
    x, w, y, g = _data(N, d, V, dtype)
    y[torch.rand(N, device=DEV, generator=g) < 0.2] = -100
    y[0] = 0
    x, w = _leaf(x, w)
    loss = ops.linear_cross_entropy(x, w, y)
    assert loss.dtype == torch.float32 and loss.shape == ()
    dx, dw = _grads(loss, x, w)
    ids, p, live = R.targets_of_labels(y)
    _check_head(x, w, ids, p, live, 1.0, torch.full((N,), 1.0 / int(live.sum()), device=DEV).double(), loss, dx, dw, "mean")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_cross_entropy_reductions(dtype, reduction):
    N, d, V = 210, 64, 777
    x, w, y, g = _data(N, d, V, dtype, 1)
    y[::5] = -1
    x, w = _leaf(x, w)
    loss = ops.linear_cross_entropy(x.view(3, 70, d), w, y.view(3, 70), ignore_index=-1, reduction=reduction)
    coef = torch.randn(N, device=DEV, generator=g) * 3e-4 if reduction == "none" else torch.tensor(2.5, device=DEV)
    assert loss.shape == ((3, 70) if reduction == "none" else ())
    dx, dw = _grads(loss, x, w, coef.view(loss.shape))
    ids, p, live = R.targets_of_labels(y, -1)
    _check_head(x, w, ids, p, live, 1.0, coef.double().expand(N), loss, dx, dw, reduction)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,d,V,K,T", [(1, 64, 300, 1, 1.0), (6, 32, 9, 9, 2.0), (130, 100, 1000, 16, 1.5),
                                       (200, 256, 3001, 64, 2.0), (129, 64, 400, 256, 4.0), (40, 333, 700, 65, 0.5)])
def test_distillation(N, d, V, K, T, dtype):
    x, w, _, g = _data(N, d, V, dtype, 2)
    t, ids = _teacher(N, V, K, g, dtype)
    if K > 2:
        ids[:, K - 1] = ids[:, 0]  # a token named twice
        ids[torch.rand(N, K, device=DEV, generator=g) < 0.1] = -1
        t[torch.rand(N, K, device=DEV, generator=g) < 0.1] = -math.inf
    if N > 4:
        ids[1] = -1
        t[2] = -math.inf
    x, w = _leaf(x, w)
    loss = ops.linear_distillation(x, w, t, ids, T)
    dx, dw = _grads(loss, x, w)
    i, p, live = R.targets_of_teacher(t, ids, T)
    _check_head(x, w, i, p, live, T, torch.full((N,), 1.0 / int(live.sum()), device=DEV).double(), loss, dx, dw, "mean")


@pytest.mark.parametrize("teacher", TYPES)
def test_distillation_per_row(teacher):
    N, d, V, K, T = 90, 64, 500, 20, 1.5
    x, w, _, g = _data(N, d, V, torch.bfloat16, 3)
    t, ids = _teacher(N, V, K, g, teacher)
    ids[7] = -1
    x, w = _leaf(x, w)
    loss = ops.linear_distillation(x.view(2, 45, d), w, t.view(2, 45, K), ids.view(2, 45, K), T, reduction="none")
    coef = torch.rand(2, 45, device=DEV, generator=g)
    dx, dw = _grads(loss, x, w, coef)
    i, p, live = R.targets_of_teacher(t, ids, T)
    assert float(loss.detach().flatten()[7]) == 0.0 and not dx[7].any()
    _check_head(x, w, i, p, live, T, coef.flatten().double(), loss, dx, dw, "none")


def test_distillation_of_labels_is_cross_entropy():
    x, w, y, _ = _data(150, 64, 333, torch.bfloat16, 4)
    one = ops.linear_cross_entropy(x, w, y, reduction="none")
    same = ops.linear_distillation(x, w, torch.full((150, 1), 2.0, device=DEV), y.unsqueeze(1), reduction="none")
    assert torch.equal(one, same)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_do_not_count_may_hold_anything(dtype):
    N, d, V = 260, 96, 600
    x, w, y, g = _data(N, d, V, dtype, 5)
    gone = torch.rand(N, device=DEV, generator=g) < 0.4
    y[gone] = -100
    clean = x.clone()
    clean[gone] = 0
    x[gone] = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).max], device=DEV, dtype=dtype).repeat(d // 4)
    out = []
    for v in (x, clean):
        a, b = _leaf(v, w)
        loss = ops.linear_cross_entropy(a, b, y)
        out.append((loss.detach(), *_grads(loss, a, b)))
    for a, b in zip(*out):
        assert torch.equal(a, b)
    assert not out[0][1][gone].any() and bool(out[0][1][~gone].any())
    t, ids = _teacher(N, V, 5, g)
    ids[gone] = -1
    t[gone] = math.nan
    out = []
    for v in (x, clean):
        a, b = _leaf(v, w)
        loss = ops.linear_distillation(a, b, t, ids, 2.0)
        out.append((loss.detach(), *_grads(loss, a, b)))
    for a, b in zip(*out):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())


def test_entries_that_are_none_may_name_any_token():
    N, d, V = 70, 64, 300
    x, w, _, g = _data(N, d, V, torch.bfloat16, 21)
    t, ids = _teacher(N, V, 6, g)
    t[:, 2] = -math.inf
    t[5] = -math.inf  # no entry at all
    ids[:, 2] = -7
    ids[5] = -7
    far = ids.clone()
    far[::2, 2] = V + 5
    far[5] = V
    out = []
    for i in (ids, far):
        a, b = _leaf(x, w)
        loss = ops.linear_distillation(a, b, t, i, 1.5)
        out.append((loss.detach(), *_grads(loss, a, b)))
    for a, b in zip(*out):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())


def test_no_row_counts():
    x, w, _, _ = _data(20, 64, 100, torch.bfloat16)
    y = torch.full((20,), -100, device=DEV)
    assert math.isnan(float(ops.linear_cross_entropy(x, w, y)))
    a, b = _leaf(x, w)
    loss = ops.linear_cross_entropy(a, b, y, reduction="sum")
    dx, dw = _grads(loss, a, b)
    assert float(loss.detach()) == 0.0 and not dx.any() and not dw.any()
    dx, dw = _grads(ops.linear_cross_entropy(a, b, y), a, b)  # a mean of none is NaN, its gradients are zeros
    assert not dx.any() and not dw.any()
    rows = ops.linear_cross_entropy(x, w, y, reduction="none")
    assert not rows.any()
    none = ops.linear_distillation(x, w, torch.zeros(20, 3, device=DEV), torch.full((20, 3), -1, device=DEV), reduction="sum")
    assert float(none) == 0.0


def test_no_rows():
    x, w, _, _ = _data(4, 65, 7, torch.bfloat16)
    a, b = _leaf(x[:0], w)
    y = torch.zeros(0, dtype=torch.int64, device=DEV)
    loss = ops.linear_cross_entropy(a, b, y, reduction="sum")
    dx, dw = _grads(loss, a, b)
    assert float(loss.detach()) == 0.0 and dx.shape == (0, 65) and not dw.any()
    assert math.isnan(float(ops.linear_cross_entropy(a, b, y).detach()))
    assert ops.linear_cross_entropy(a, b, y, reduction="none").shape == (0,)


def test_labels_outside_the_vocabulary_are_nan():
    x, w, y, _ = _data(40, 64, 100, torch.bfloat16)
    y[3], y[9] = 100, -7
    a, b = _leaf(x, w)
    loss = ops.linear_cross_entropy(a, b, y, reduction="none")
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[3] = bad[9] = True
    assert torch.equal(torch.isnan(loss), bad)
    dx, = torch.autograd.grad(loss.sum(), a)
    assert torch.equal(torch.isnan(dx).all(1), bad) and bool(torch.isfinite(dx[~bad]).all())
    t, ids = torch.zeros(40, 2, device=DEV), y.clamp(min=0).unsqueeze(1).repeat(1, 2)
    assert torch.equal(torch.isnan(ops.linear_distillation(x, w, t, ids, reduction="none")), bad & (y == 100))


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_of_a_row_stays_in_it(dtype):
    x, w, y, _ = _data(140, 64, 300, dtype, 6)
    x[5, 3] = math.nan
    x[77, 0] = math.inf
    loss = ops.linear_cross_entropy(x, w, y, reduction="none")
    bad = torch.zeros(140, dtype=torch.bool, device=DEV)
    bad[5] = bad[77] = True
    assert torch.equal(torch.isnan(loss), bad)
    clean = ops.linear_cross_entropy(torch.where(bad.unsqueeze(1), 0.0, x).to(dtype), w, y, reduction="none")
    assert torch.equal(loss[~bad], clean[~bad])


@pytest.mark.parametrize("dtype", TYPES)
def test_large_logits(dtype):
    # logits of hundreds: the largest takes all; a row of equal logits
    x, w, y, _ = _data(64, 64, 200, dtype, 7, scale=60.0)
    x[0] = 0
    a, b = _leaf(x, w)
    loss = ops.linear_cross_entropy(a, b, y)
    dx, dw = _grads(loss, a, b)
    ids, p, live = R.targets_of_labels(y)
    _check_head(a, b, ids, p, live, 1.0, torch.full((64,), 1 / 64, device=DEV).double(), loss, dx, dw, "mean")


@pytest.mark.parametrize("dtype", TYPES)
def test_views_and_strides(dtype):
    # rows of a wider tensor, columns from an odd place, labels of a transposed tensor, a weight with gaps
    big = torch.randn(60, 3, 300, device=DEV).to(dtype)
    x = big[:, 1, 7:7 + 96]
    store = (torch.randn(500, 130, device=DEV) * 0.2).to(dtype)
    w = store[:, 3:99]
    y = torch.randint(0, 500, (2, 60), device=DEV).t()[:, 0]
    a, b = _leaf(x, w)
    loss = ops.linear_cross_entropy(a, b, y)
    got = _grads(loss, a, b)
    c, e = _leaf(x.contiguous(), w.contiguous())
    want = ops.linear_cross_entropy(c, e, y.contiguous())
    for p, q in zip((loss, *got), (want, *_grads(want, c, e))):
        assert torch.equal(p, q)
    # one row for all (stride 0) and a transposed weight
    one = x[:1].expand(60, 96)
    assert torch.equal(ops.linear_cross_entropy(one, w, y, reduction="none"),
                       ops.linear_cross_entropy(one.contiguous(), w.t().contiguous().t(), y, reduction="none"))


def test_gradients_of_broadcast_and_shared_inputs():
    x, w, y, _ = _data(40, 64, 64, torch.float32, 8)
    h, = _leaf(x[:1])
    loss = ops.linear_cross_entropy(h.expand(40, 64), w, y)
    dh, = torch.autograd.grad(loss, h)
    g, = _leaf(x[:1].repeat(40, 1))
    dg, = torch.autograd.grad(ops.linear_cross_entropy(g, w, y), g)
    torch.testing.assert_close(dh, dg.sum(0, keepdim=True), rtol=40 * R.U32, atol=1e-6)
    # the weight is the rows too
    s, = _leaf(w)
    both, = torch.autograd.grad(ops.linear_cross_entropy(s, s, y.repeat(2)[:64]), s)
    a, b = _leaf(w, w)
    parts = _grads(ops.linear_cross_entropy(a, b, y.repeat(2)[:64]), a, b)
    assert torch.equal(both, parts[0] + parts[1])


def test_only_what_is_asked_for():
    x, w, y, _ = _data(130, 64, 300, torch.bfloat16, 9)
    a, b = _leaf(x, w)
    both = _grads(ops.linear_cross_entropy(a, b, y), a, b)
    c, = _leaf(x)
    assert torch.equal(both[0], torch.autograd.grad(ops.linear_cross_entropy(c, w, y), c)[0])
    e, = _leaf(w)
    assert torch.equal(both[1], torch.autograd.grad(ops.linear_cross_entropy(x, e, y), e)[0])
    assert not ops.linear_cross_entropy(x, w, y).requires_grad


def test_gradient_against_differences():
    N, d, V = 12, 16, 50
    x, w, y, g = _data(N, d, V, torch.float32, 10)
    t, ids = _teacher(N, V, 4, g)
    for fn in (lambda a, b: ops.linear_cross_entropy(a, b, y, reduction="sum"),
               lambda a, b: ops.linear_distillation(a, b, t, ids, 2.0, reduction="sum")):
        a, b = _leaf(x, w)
        dx, dw = _grads(fn(a, b), a, b)
        for leaf, grad in ((0, dx), (1, dw)):
            v = torch.randn(grad.shape, device=DEV, generator=g)
            v = v / v.norm()
            e = 2.0 ** -6  # central differences: e^2 / 6 times third derivatives of about 1, and 2^-24 loss / e
            step = [x, w]
            step[leaf] = step[leaf] + e * v
            up = fn(*step)
            step[leaf] = step[leaf] - 2 * e * v
            slope = float(up - fn(*step)) / (2 * e)
            assert abs(slope - float((grad * v).sum())) < 2e-3 * max(1.0, float(grad.norm()))


def test_equal_calls_give_equal_bits_and_calls_at_the_same_time():
    x, w, y, _ = _data(900, 256, 3000, torch.bfloat16, 11)

    def once():
        a, b = _leaf(x, w)
        loss = ops.linear_cross_entropy(a, b, y)
        return (loss.detach(), *_grads(loss, a, b))

    first = once()
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in side:
            with torch.cuda.stream(s):
                got.append(once())
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(first, r):
            assert torch.equal(a, b)


def test_backward_twice_and_no_second_order():
    x, w, y, _ = _data(50, 64, 200, torch.float32, 12)
    a, b = _leaf(x, w)
    loss = ops.linear_cross_entropy(a, b, y)
    first = torch.autograd.grad(loss, (a, b), retain_graph=True)
    again = torch.autograd.grad(loss, (a, b), retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    dx, = torch.autograd.grad(loss, a, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_captured_forward_and_backward():
    x, w, y, g = _data(300, 64, 1000, torch.bfloat16, 13)
    t, ids = _teacher(300, 1000, 8, g)
    a, b = _leaf(x, w)

    def body():
        loss = ops.linear_cross_entropy(a, b, y) + ops.linear_distillation(a, b, t, ids, 2.0)
        return (loss.detach(), *_grads(loss, a, b))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body()
    for seed in range(3):
        nx, nw, ny, _ = _data(300, 64, 1000, torch.bfloat16, 20 + seed)
        with torch.no_grad():
            a.copy_(nx)
            b.copy_(nw)
            y.copy_(ny)
            y[: 50 * seed] = -100
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        for p, q in zip(got, body()):
            assert torch.equal(p, q)


def test_two_captured_calls_at_once():
    sides, graphs, outs, wants = [torch.cuda.Stream() for _ in range(2)], [], [], []
    kept = []  # a graph reads its inputs where they were: they have to live as long
    for seed in range(2):
        x, w, y, _ = _data(700, 64, 3000, torch.float32 if seed else torch.bfloat16, 30 + seed)
        a, b = _leaf(x, w)

        def body():
            loss = ops.linear_cross_entropy(a, b, y)
            return (loss.detach(), *_grads(loss, a, b))

        wants.append(body())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = body()
        graphs.append(graph)
        outs.append(out)
        kept.append((a, b, y))
    for _ in range(3):
        for side, graph, out in zip(sides, graphs, outs):
            with torch.cuda.stream(side):
                for t in out:
                    t.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, wants):
            assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_pieces_of_the_vocabulary():
    # rows enough for several pieces (1 GB of 2 N bytes a column): 300000 rows take at most 1536 columns a piece
    N, d, V = 300000, 32, 2000
    x, w, y, _ = _data(N, d, V, torch.bfloat16, 14)
    a, b = _leaf(x, w)
    loss = ops.linear_cross_entropy(a, b, y)
    dx, dw = _grads(loss, a, b)
    ids, p, live = R.targets_of_labels(y)
    _check_head(a, b, ids, p, live, 1.0, torch.full((N,), 1.0 / N, device=DEV).double(), loss, dx, dw, "mean")


@pytest.mark.parametrize("dtype,N,d,V", [(torch.bfloat16, 4001, 300, 20001), (torch.float16, 4001, 300, 20001),
                                         (torch.float32, 1999, 520, 12001)])
@pytest.mark.parametrize("gone", [0.02, 0.6])
def test_blocks_that_share_both_products(dtype, N, d, V, gone):
    # sizes at which each CU's block takes ranges of dW and then one of dx; with most rows taken out as well
    x, w, y, g = _data(N, d, V, dtype, 17)
    y[torch.rand(N, device=DEV, generator=g) < gone] = -100
    x, w = _leaf(x, w)
    loss = ops.linear_cross_entropy(x, w, y)
    dx, dw = _grads(loss, x, w)
    ids, p, live = R.targets_of_labels(y)
    _check_head(x, w, ids, p, live, 1.0, torch.full((N,), 1.0 / int(live.sum()), device=DEV).double(), loss, dx, dw, "mean")


def test_rows_past_32_bits():
    # 4.4 GB of rows, of their copies and of dx: the reference takes them in parts, whose bounds add up
    N, d, V = 2 ** 21 + 77, 1040, 70
    x, w, y, g = _data(N, d, V, torch.bfloat16, 18)
    y[::5] = -100
    x, w = _leaf(x, w)
    loss = ops.linear_cross_entropy(x, w, y, reduction="none")
    coef = torch.rand(N, device=DEV, generator=g)
    dx, dw = _grads(loss, x, w, coef)
    value = bound = 0.0
    for at in range(0, N, 2 ** 18):
        rows = slice(at, at + 2 ** 18)
        ids, p, live = R.targets_of_labels(y[rows])
        want = R.head(x.detach()[rows], w.detach(), ids, p, live, 1.0, coef[rows].double(), N)
        R.check("loss", loss[rows], *want["loss"])
        R.check("dhidden", dx[rows], *want["dhidden"])
        value, bound = value + want["dweight"][0], bound + want["dweight"][1]
    # fp32 sums over all rows, not over a part's
    ids, p, live = R.targets_of_labels(y)
    reach = sum(x.detach()[at: at + 2 ** 18].double().abs().sum(0) for at in range(0, N, 2 ** 18))
    R.check("dweight", dw, value, bound + R.product_slack(N, torch.bfloat16) * reach)


def test_autocast():
    x, w, y, _ = _data(100, 64, 300, torch.float32, 15)
    a, b = _leaf(x, w)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = ops.linear_cross_entropy(a, b, y)
    dx, dw = _grads(loss, a, b)
    assert dx.dtype == dw.dtype == torch.float32
    want = ops.linear_cross_entropy(x.bfloat16(), w.bfloat16(), y)
    assert torch.equal(loss, want)


def test_refusals():
    x, w, y, _ = _data(10, 64, 50, torch.bfloat16)
    t, ids = torch.zeros(10, 3, device=DEV), torch.zeros(10, 3, dtype=torch.int64, device=DEV)
    ce, kd = ops.linear_cross_entropy, ops.linear_distillation
    for error, call in [
            (RuntimeError, lambda: ce(x.cpu(), w, y)), (RuntimeError, lambda: ce(x, w.cpu(), y)), (RuntimeError, lambda: ce(x, w, y.cpu())),
            (TypeError, lambda: ce(x, w.float(), y)), (TypeError, lambda: ce(x.double(), w.double(), y)),
            (ValueError, lambda: ce(x, w[:, :32], y)), (ValueError, lambda: ce(x, w, y[:9])), (ValueError, lambda: ce(x, w, y.int())),
            (ValueError, lambda: ce(x, w[:0], y)), (ValueError, lambda: ce(x, w, y, reduction="batch")),
            (ValueError, lambda: kd(x, w, t, ids[:9])), (ValueError, lambda: kd(x, w, t, ids.int())), (TypeError, lambda: kd(x, w, t.double(), ids)),
            (TypeError, lambda: kd(x, w, t[:, :2], ids)), (ValueError, lambda: kd(x, w, t[:, :0], ids[:, :0])),
            (ValueError, lambda: kd(x, w, t.repeat(1, 100), ids.repeat(1, 100))), (ValueError, lambda: kd(x, w, t, ids, 0.0)),
            (ValueError, lambda: kd(x, w, t, ids, math.inf))]:
        with pytest.raises(error):
            call()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [1, 16, 32, 33, 200, 1025])
def test_scores_without_a_gradient_are_the_training_passs(N, dtype):
    # a forward pass alone takes the rows as they are, where it can; others and masked rows go through a copy
    x, w, y, g = _data(N, 128, 999, dtype, 16)
    y[torch.rand(N, device=DEV, generator=g) < 0.2] = -100
    a, b = _leaf(x, w)
    want = ops.linear_cross_entropy(a, b, y, reduction="none").detach()
    assert torch.equal(ops.linear_cross_entropy(x, w, y, reduction="none"), want)
    odd = torch.empty(N * 128 + 1, device=DEV, dtype=dtype)[1:].view(N, 128)
    odd.copy_(x)
    assert torch.equal(ops.linear_cross_entropy(odd, w, y, reduction="none"), want)
    ids, p, live = R.targets_of_labels(y)
    value, bound = R.head(x, w, ids, p, live, 1.0, torch.ones(N, device=DEV).double())["loss"]
    R.check("loss", want, value, bound)
    x[y == -100] = math.nan
    assert torch.equal(ops.linear_cross_entropy(x, w, y, reduction="none"), want)
