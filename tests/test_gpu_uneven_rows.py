"""fp32 losses and gated feed-forwards whose rows, columns, weights or gradients lie far from each other: what a large
entry has no part in comes out as if it were not there, within the bounds of even data."""

import math

import pytest
import torch

import wide_reference as R
from multiscreen import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
FAR = [12, 30, 40, 60, 80]  # powers of two; up to the first fp16 terms with one scale for all would do


def _leaf(*t):
    return [x.detach().requires_grad_() for x in t]


def _head(N, d, V, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(N, d, device=DEV, generator=g)
    w = torch.randn(V, d, device=DEV, generator=g) * 1.5 / math.sqrt(d)
    return x, w, torch.randint(0, V, (N,), device=DEV, generator=g), g


def _check(got, want, rows=None, features=None):
    # want: of these rows and features alone
    for name, value in got.items():
        pick = features if name in ("dweight", "dgate", "dup") else rows
        R.check(name, value if pick is None else value[pick], *want[name])


def _grads(fn, x, w, coef):
    x, w = _leaf(x, w)
    loss = fn(x, w)
    return dict(zip(("loss", "dhidden", "dweight"), (loss.detach(), *torch.autograd.grad(loss, (x, w), coef))))


@pytest.mark.parametrize("up", FAR)
@pytest.mark.parametrize("N,d,V", [(8, 64, 300), (150, 100, 1003), (700, 512, 2000), (3, 520, 64)])
def test_a_row_far_above_the_others(N, d, V, up):
    # in columns in which the weight is as far below, so that the row's logits are ordinary
    x, w, y, g = _head(N, d, V)
    x[1, :8] *= 2.0 ** up
    w[:, :8] *= 2.0 ** -up
    coef = torch.rand(N, device=DEV, generator=g) + 0.5
    got = _grads(lambda a, b: ops.linear_cross_entropy(a, b, y, reduction="none"), x, w, coef)
    ids, p, live = R.targets_of_labels(y)
    want = R.head(x, w, ids, p, live, 1.0, coef.double())
    _check(got, want)
    others = torch.arange(N, device=DEV) != 1
    own = R.head(x[others], w, ids[others], p[others], live[others], 1.0, coef[others].double())
    for name in ("loss", "dhidden"):
        R.check(name, got[name][others], *own[name])


@pytest.mark.parametrize("up", FAR)
def test_a_token_far_above_the_others(up):
    # the rows that count have no part in it
    N, d, V = 190, 96, 500
    x, w, y, g = _head(N, d, V, 1)
    y[y == 7] = 8
    w[7] *= 2.0 ** up
    y[x.double() @ w.double()[7] > -300] = -100
    assert int((y >= 0).sum()) > 20
    coef = torch.rand(N, device=DEV, generator=g) + 0.5
    got = _grads(lambda a, b: ops.linear_cross_entropy(a, b, y, reduction="none"), x, w, coef)
    keep = torch.arange(V, device=DEV) != 7
    ids, p, live = R.targets_of_labels(torch.where(y > 7, y - 1, y))
    want = R.head(x, w[keep], ids, p, live, 1.0, coef.double())
    _check(got, want, features=keep)


@pytest.mark.parametrize("up", FAR)
def test_columns_that_make_up_for_each_other(up):
    # a column of the rows far above the others and the weight's as far below: every logit is ordinary
    N, d, V = 130, 64, 400
    x, w, y, g = _head(N, d, V, 2)
    x[:, 5] *= 2.0 ** up
    w[:, 5] *= 2.0 ** -up
    coef = torch.rand(N, device=DEV, generator=g)
    got = _grads(lambda a, b: ops.linear_cross_entropy(a, b, y, reduction="none"), x, w, coef)
    ids, p, live = R.targets_of_labels(y)
    _check(got, R.head(x, w, ids, p, live, 1.0, coef.double()))


@pytest.mark.parametrize("up", FAR)
def test_a_coefficient_far_above_the_others(up):
    N, d, V, K, T = 210, 64, 777, 5, 1.5
    x, w, y, g = _head(N, d, V, 3)
    t, ids = torch.randn(N, K, device=DEV, generator=g), torch.randint(0, V, (N, K), device=DEV, generator=g)
    coef = torch.rand(N, device=DEV, generator=g) + 0.5
    coef[3] = 2.0 ** up
    others = torch.arange(N, device=DEV) != 3
    got = _grads(lambda a, b: ops.linear_cross_entropy(a, b, y, reduction="none"), x, w, coef)
    i, p, live = R.targets_of_labels(y)
    want = R.head(x[others], w, i[others], p[others], live[others], 1.0, coef[others].double(), N)
    R.check("dhidden", got["dhidden"][others], *want["dhidden"])
    got = _grads(lambda a, b: ops.linear_distillation(a, b, t, ids, T, reduction="none"), x, w, coef)
    i, p, live = R.targets_of_teacher(t, ids, T)
    want = R.head(x[others], w, i[others], p[others], live[others], T, coef[others].double(), N)
    R.check("dhidden", got["dhidden"][others], *want["dhidden"])


def test_wide_calls_with_everything_else():
    # the wide format through a mean, rows that do not count, pieces and shares, distillation, strides, and the few rows' kernel
    for N, d, V in ((20, 64, 999), (1999, 520, 12001)):
        x, w, y, g = _head(N, d, V, 4)
        x[2] = 0
        x[5] *= 2.0 ** -50
        y[::7] = -100
        x[0] = torch.finfo(torch.float32).max
        got = _grads(lambda a, b: ops.linear_cross_entropy(a, b, y), x, w, None)
        ids, p, live = R.targets_of_labels(y)
        want = R.head(x, w, ids, p, live, 1.0, torch.full((N,), 1.0 / int(live.sum()), device=DEV).double())
        value, bound = want["loss"]
        n = live.sum()
        R.check("loss", got["loss"], value.sum() / n, bound.sum() / n + 4 * R.U32 * value.abs().sum() / n)
        R.check("dhidden", got["dhidden"], *want["dhidden"])
        R.check("dweight", got["dweight"], *want["dweight"])
        t, ids = torch.randn(N, 6, device=DEV, generator=g), torch.randint(0, V, (N, 6), device=DEV, generator=g)
        ids[::7] = -1
        coef = torch.rand(N, device=DEV, generator=g)
        big = torch.empty(V, d + 3, device=DEV)
        big[:, 1:-2] = w
        got = _grads(lambda a, b: ops.linear_distillation(a, b, t, ids, 2.0, reduction="none"), x, big[:, 1:-2], coef)
        i, p, live = R.targets_of_teacher(t, ids, 2.0)
        _check(got, R.head(x, w, i, p, live, 2.0, coef.double()))


def test_a_large_row_that_does_not_count_leaves_the_others_bits():
    x, w, y, _ = _head(140, 64, 300, 5)
    y[3] = -100
    clean = _grads(lambda a, b: ops.linear_cross_entropy(a, b, y), x, w, None)
    x[3] *= 2.0 ** 60
    for k, v in _grads(lambda a, b: ops.linear_cross_entropy(a, b, y), x, w, None).items():
        assert torch.equal(v, clean[k])


def _gated(N, d, F, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(N, d, device=DEV, generator=g)
    wg, wu = (torch.randn(F, d, device=DEV, generator=g) / math.sqrt(d) for _ in range(2))
    return x, wg, wu, 0.01 * torch.randn(N, F, device=DEV, generator=g)


def _run(x, wg, wu, dh, act):
    x, wg, wu = _leaf(x, wg, wu)
    h = ops.gated_linear(x, wg, wu, act)
    return dict(zip(("h", "dx", "dgate", "dup"), (h.detach(), *torch.autograd.grad(h, (x, wg, wu), dh))))


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("up", [12, 30, 40])
@pytest.mark.parametrize("N,d,F", [(16, 64, 100), (150, 64, 200), (1100, 520, 3001)])
def test_gated_row_far_above_the_others(N, d, F, up, act):
    # a padded position with large values, whose gradient is zero
    x, wg, wu, dh = _gated(N, d, F)
    others = torch.arange(N, device=DEV) != 1
    x[1] *= 2.0 ** up
    dh[1] = 0
    got = _run(x, wg, wu, dh, act)
    _check(got, R.gated(x[others], wg, wu, act, dh[others]), rows=others)
    assert not got["dx"][1].any()


@pytest.mark.parametrize("up", [12, 30, 40])
def test_gated_feature_far_above_the_others(up):
    x, wg, wu, dh = _gated(150, 64, 200, 1)
    others = torch.arange(200, device=DEV) != 9
    wg[9] *= 2.0 ** up
    wu[9] *= 2.0 ** up
    dh[:, 9] = 0
    got = _run(x, wg, wu, dh, "silu")
    got["h"] = got["h"][:, others]
    _check(got, R.gated(x, wg[others], wu[others], "silu", dh[:, others]), features=others)


@pytest.mark.parametrize("up", [12, 30, 40, 60])
def test_gated_gradient_far_above_the_others(up):
    x, wg, wu, dh = _gated(150, 64, 200, 2)
    row = dh.clone()
    row[4] *= 2.0 ** up
    others = torch.arange(150, device=DEV) != 4
    got = _run(x, wg, wu, row, "silu")
    want = R.gated(x[others], wg, wu, "silu", dh[others])
    for name in ("h", "dx"):
        R.check(name, got[name][others], *want[name])
    column = dh.clone()
    column[:, 4] *= 2.0 ** up
    others = torch.arange(200, device=DEV) != 4
    got = _run(x, wg, wu, column, "silu")
    want = R.gated(x, wg[others], wu[others], "silu", dh[:, others])
    for name in ("dgate", "dup"):
        R.check(name, got[name][others], *want[name])


def test_a_captured_call_finds_the_format_of_each_replays_data():
    N, d, V = 300, 64, 1000
    x, w, y, _ = _head(N, d, V, 6)
    a, b = _leaf(x, w)
    xg, wg, wu, dh = _gated(N, d, 200, 7)

    def body():
        loss = ops.linear_cross_entropy(a, b, y)
        return {"loss": loss.detach(), **dict(zip(("dhidden", "dweight"), torch.autograd.grad(loss, (a, b)))), **_run(xg, wg, wu, dh, "silu")}

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body()
    for up in (0, 40, 0, 25):
        with torch.no_grad():
            a.copy_(x)
            a[3] *= 2.0 ** -up
            xg[3] *= 2.0 ** -up
        graph.replay()
        torch.cuda.synchronize()
        got = {k: v.clone() for k, v in out.items()}
        want = body()
        for k in want:
            assert torch.equal(got[k], want[k]), (up, k)
        with torch.no_grad():
            xg[3] *= 2.0 ** up
