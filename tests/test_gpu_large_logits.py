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
