"""Sums over rows, and over weights, that lie past 32 bits of bytes: only few of them have a gradient, so that each one's
part in the sum is far larger than the bound."""

import math

import pytest
import torch

import wide_reference as R
from multiscreen import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 1040
FAR = 2 ** 32 // (2 * D)  # the first row past 4 GB
N = 2 ** 21 + 77          # 4.4 GB of bf16 rows
FEW = [5, 1000, 2 ** 20 + 3, FAR - 1, FAR, FAR + 1, N - 130, N - 1]


def _sensitive(value, bound):
    # a sum without one of its parts, or of zeros, is outside of the bound nearly everywhere
    assert float((8 * bound < value.abs()).double().mean()) > 0.9


def test_weight_gradient_of_rows_past_32_bits():
    V = 70
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(N, D, device=DEV, generator=g, dtype=torch.bfloat16).requires_grad_()
    w = (torch.randn(V, D, device=DEV, generator=g) * 1.5 / math.sqrt(D)).bfloat16().requires_grad_()
    y = torch.randint(0, V, (N,), device=DEV, generator=g)
    few = torch.tensor(FEW, device=DEV)
    for rows in (few, few[4:5], few[7:8]):
        coef = torch.zeros(N, device=DEV)
        coef[rows] = 1.0 + 0.5 * torch.rand(len(rows), device=DEV, generator=g)
        loss = ops.linear_cross_entropy(x, w, y, reduction="none")
        dx, dw = torch.autograd.grad(loss, (x, w), coef)
        ids, p, live = R.targets_of_labels(y[rows])
        want = R.head(x.detach()[rows], w.detach(), ids, p, live, 1.0, coef[rows].double(), N)
        R.check("dweight", dw, *want["dweight"])
        R.check("dhidden", dx[rows], *want["dhidden"])
        _sensitive(*want["dhidden"])
        _sensitive(want["dweight"][0][y[rows]], want["dweight"][1][y[rows]])
        dx[rows] = 0
        assert not dx.any()
        del dx


def test_row_gradient_of_weights_past_32_bits():
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(4, D, device=DEV, generator=g, dtype=torch.bfloat16).requires_grad_()
    wg, wu = ((torch.randn(N, D, device=DEV, generator=g, dtype=torch.bfloat16) / math.sqrt(D)).requires_grad_() for _ in range(2))
    few = torch.tensor(FEW, device=DEV)
    for features in (few, few[4:5], few[7:8]):
        dh = torch.zeros(4, N, device=DEV, dtype=torch.bfloat16)
        dh[:, features] = (1.0 + 0.5 * torch.rand(4, len(features), device=DEV, generator=g)).bfloat16()
        h = ops.gated_linear(x, wg, wu)
        dx, dgate, dup = torch.autograd.grad(h, (x, wg, wu), dh)
        want = R.gated(x.detach(), wg.detach()[features], wu.detach()[features], "silu", dh[:, features])
        R.check("dx", dx, *want["dx"])
        _sensitive(*want["dx"])
        R.check("h", h.detach()[:, features], *want["h"])
        for name, got in (("dgate", dgate), ("dup", dup)):
            R.check(name, got[features], *want[name])
            _sensitive(*want[name])
            got[features] = 0
            assert not got.any()
        del h, dgate, dup
