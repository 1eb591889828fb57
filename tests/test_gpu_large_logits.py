"""Losses of rows whose logits are large: the largest takes all, its own gradient is what is left of 1, and nothing leaves
the type's range on the way."""

import math

import pytest
import torch

from multiscreen import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rows(up, dtype, N=64, d=64, V=300, weight=1.0):
    """Row n has logit a_n = (1.3 to 1.9) 2^up at token n % d and zero elsewhere, exactly: 8 bits each."""
    g = torch.Generator(device=DEV).manual_seed(up)
    size = ((1.3 + 0.6 * torch.rand(N, device=DEV, generator=g)) * 2.0 ** up / weight).bfloat16().to(dtype)
    x = torch.zeros(N, d, device=DEV, dtype=dtype)
    x[torch.arange(N), torch.arange(N) % d] = size
    w = torch.zeros(V, d, device=DEV, dtype=dtype)
    w[torch.arange(d), torch.arange(d)] = weight
    return x, w, size.double() * weight


def _grads(x, w, y, N):
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ops.linear_cross_entropy(a, b, y, reduction="none")
    return (loss.detach(), *torch.autograd.grad(loss, (a, b), torch.ones(N, device=DEV)))


@pytest.mark.parametrize("dtype,up", [(t, u) for t in TYPES for u in (5, 8, 12, 15, 20, 24, 31, 60, 100) if t != torch.float16 or u <= 24])
@pytest.mark.parametrize("N", [17, 64, 400])
def test_the_largest_logit_takes_all(dtype, up, N):
    weight = 2.0 ** 12 if dtype == torch.float16 and up > 12 else 1.0
    x, w, size = _rows(up, dtype, N, weight=weight)
    at = torch.arange(N, device=DEV) % 64
    hit = torch.arange(N, device=DEV) % 3 == 0
    y = torch.where(hit, at, 200)
    loss, dx, dw = _grads(x, w, y, N)
    # the others' share, below 300 e^-41, is no number beside 1; a sum and its logarithm are off by a few roundings of 1
    one = 8 * 2.0 ** -24
    want = torch.where(hit, 0.0, size)
    assert bool(((loss.double() - want).abs() <= one * (1 + want)).all())
    # dx = W_at - W_y where the label is another, W_200 = 0; zeros where it is the largest
    expect = torch.zeros(N, 64, device=DEV, dtype=torch.float64)
    expect[torch.arange(N), at] = torch.where(hit, 0.0, weight).double()
    assert bool(((dx.double() - expect).abs() <= 2 * torch.finfo(dtype).eps * expect + 2 * one * weight).all())
    # dW_v = sum_n (q_nv - [v = y_n]) x_n: a row's x is in its own column
    expect = torch.zeros(300, 64, device=DEV, dtype=torch.float64)
    x_at = x.double()[torch.arange(N), at]
    expect.index_put_((at, at), torch.where(hit, 0.0, x_at), accumulate=True)
    expect.index_put_((y, at), torch.where(hit, 0.0, -x_at), accumulate=True)
    met = torch.zeros(300, 64, device=DEV, dtype=torch.float64)
    met[at, at] = met[y, at] = 1
    slack = 2 * torch.finfo(dtype).eps * expect.abs() + x_at.max() * N * (2 * one * met + 300 * math.exp(-41))
    assert bool(((dw.double() - expect).abs() <= slack).all())


@pytest.mark.parametrize("dtype,up", [(t, u) for t in TYPES for u in (6, 14, 22, 60) if t != torch.float16 or u <= 14])
def test_equal_largest_logits_share(dtype, up):
    N = 40
    x, w, size = _rows(up, dtype, N)
    w[100:164] = w[:64]  # every token twice
    at = torch.arange(N, device=DEV) % 64
    loss, dx, _ = _grads(x, w, at, N)
    assert bool(((loss.double() - math.log(2)).abs() <= 8 * 2.0 ** -24).all())
    assert bool((dx.double().abs() <= 1e-6).all())  # half of W_at twice, less W_at
    t = torch.tensor([0.0, 0.0], device=DEV).expand(N, 2)
    both = ops.linear_distillation(x, w, t, torch.stack([at, at + 100], 1), 1.0, reduction="none")
    assert bool((both.abs() <= 8 * 2.0 ** -24).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_row_of_large_logits_leaves_the_others(dtype):
    N, d, V = 150, 64, 700
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(N, d, device=DEV, generator=g).to(dtype)
    w = (torch.randn(V, d, device=DEV, generator=g) * 0.2).to(dtype)
    y = torch.randint(0, V, (N,), device=DEV, generator=g)
    others = torch.arange(N, device=DEV) != 70
    want = _grads(x[others], w, y[others], N - 1)
    for up in (10, 33, 60):
        far = x.clone()
        far[70] = (far[70].float() * 2.0 ** up).to(dtype)
        loss, dx, dw = _grads(far, w, y, N)
        # the others' logits are formed alike, or in fp32's other terms: off by twice a product's error at most
        X, W = x[others].double(), w.double()
        off = 2 * (3 * 2.0 ** -22 + d * 2.0 ** -24) * (X.abs() @ W.abs().T).amax(-1, keepdim=True) + 8 * 2.0 ** -24
        q = torch.softmax(X @ W.T, -1)
        step = torch.finfo(dtype).eps
        assert bool(((loss[others] - want[0]).abs() <= 2 * off[:, 0] + 8 * 2.0 ** -24 * want[0]).all())
        reach = (2 * q * off) @ W.abs() + 2 * off * W.abs().max()  # the target's own q among them
        assert bool(((dx[others].double() - want[1].double()).abs() <= reach + 2 * step * want[1].double().abs()).all())
        assert bool(torch.isfinite(loss).all() and torch.isfinite(dx).all() and torch.isfinite(dw).all())
        row = torch.softmax(far[70].double() @ W.T, 0)
        away = row < 1e-60
        away[y[70]] = False
        assert int(away.sum()) > V // 2
        g = q.scatter_add(1, y[others].unsqueeze(1), -torch.ones(N - 1, 1, device=DEV).double()).abs()
        reach = (2 * off * (q + g)).T @ X.abs() + N * 2.0 ** -24 * (g.T @ X.abs()) + 2.0 ** -39 * X.abs().sum(0)
        assert bool(((dw.double() - want[2].double()).abs() <= 2 * reach + 2 * step * want[2].double().abs())[away].all())


@pytest.mark.parametrize("up", [4, 6, 10, 20, 30])
@pytest.mark.parametrize("N", [30, 700])
def test_the_largest_logit_of_all_bits(up, N):
    # as above, with rows that fp32's two terms hold to 22 bits only: the target's logit is the one in the sum
    x, w, _ = _rows(up, torch.float32, N)
    g = torch.Generator(device=DEV).manual_seed(up)
    x = x * (1.0 + 2.0 ** -9 * torch.rand(N, 1, device=DEV, generator=g))
    at = torch.arange(N, device=DEV) % 64
    loss, dx, _ = _grads(x, w, at, N)
    a = x.double()[torch.arange(N), at]
    rest = 299 * torch.exp(-a)  # beside the largest
    one = 8 * 2.0 ** -24
    off = a * 2.0 ** -21  # of a logit
    assert bool((loss >= 0).all())
    assert bool(((loss.double() - torch.log1p(rest)).abs() <= one + 2 * off.clamp(max=1) * rest).all())
    # dx = -(1 - q) W_at + sum of the others' q W
    left = rest / (1 + rest)
    expect = (torch.exp(-a) / (1 + rest)).unsqueeze(1).repeat(1, 64)
    expect[torch.arange(N), at] = -left
    assert bool(((dx.double() - expect).abs() <= one + (2 * off.clamp(max=1) * left + 2.0 ** -21 * left).unsqueeze(1)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,d,V,top", [(8, 512, 300, 120.0), (150, 512, 1000, 30.0), (600, 512, 3000, 60.0), (20, 333, 4001, 100.0), (700, 100, 500, 16.0)])
def test_confident_rows(N, d, V, top, dtype):
    # each row's own token is `top` above the others: what is left of 1 is the loss and the gradient
    g = torch.Generator(device=DEV).manual_seed(N)
    w = (torch.randn(V, d, device=DEV, generator=g) / math.sqrt(d)).to(dtype)
    y = torch.randint(0, V, (N,), device=DEV, generator=g)
    x = (top * w.double()[y] + 0.2 * torch.randn(N, d, device=DEV, generator=g)).to(dtype)
    loss, dx, dw = _grads(x, w, y, N)
    X, W = x.double(), w.double()
    z = X @ W.T
    z = z - z.gather(1, y.unsqueeze(1))
    q = torch.exp(z)
    q[torch.arange(N), y] = 0
    rest = q.sum(1)
    q = q / (1 + rest).unsqueeze(1)
    # Differences of two logits of one product: both of their errors, and per term e^-z of the sum one of 2^-23 (exp2) and two
    # of 2^-24 z (the difference and its factor; z < 64 where a term counts beside the largest): 130 2^-24.  A sum of 1 + rest: 64
    # additions in a lane, 2 of lanes and waves, 12 of tiles at most 4 x 256 of them, and 8 of its logarithm: 96, each
    # at most 2^-24 of it.
    off = 2 * (d * 2.0 ** -24 + (3 * 2.0 ** -22 if dtype == torch.float32 else 0)) * (X.abs() @ W.abs().T).amax(1)
    off = torch.expm1(off) + 130 * 2.0 ** -24
    one = 96 * 2.0 ** -24 * (1 + rest)
    assert bool((loss >= 0).all())
    assert bool(((loss.double() - torch.log1p(rest)).abs() <= one + off * rest).all())
    ug = torch.finfo(dtype).eps / 2 if N > 256 and dtype != torch.float32 else 2.0 ** -16
    G, B = q.clone(), q * (2 * off.unsqueeze(1) + ug) + 2.0 ** -39
    G[torch.arange(N), y] = -rest / (1 + rest)
    B[torch.arange(N), y] = one + 2 * off * rest + ug * rest
    u = torch.finfo(dtype).eps
    for got, a, b, m in ((dx, G, B, W), (dw, G.T, B.T, X)):
        want, reach = a @ m, b @ m.abs() + a.shape[1] * 2.0 ** -24 * (a.abs() @ m.abs())
        tiny = torch.finfo(dtype).smallest_normal * u
        assert bool(((got.double() - want).abs() <= reach + u * (want.abs() + reach) + tiny).all())
