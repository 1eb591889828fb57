"""Sizes on both sides of the rules that choose between tiles: small ones for few rows or few features, halves, whole ones."""

import math

import pytest
import torch

import wide_reference as R
from multiscreen import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,d,F", [(256, 64, 2048), (257, 64, 2048), (64, 96, 8192), (65, 96, 8193), (32, 64, 16384), (1, 64, 16385),
                                   (31, 40, 16390), (700, 100, 1000), (2500, 64, 1365), (513, 32, 3001), (1025, 33, 515)])
def test_gated_forward(N, d, F, dtype):
    g = torch.Generator(device=DEV).manual_seed(N)
    x = torch.randn(N, d, device=DEV, generator=g).to(dtype)
    wg, wu = ((torch.randn(F, d, device=DEV, generator=g) / math.sqrt(d)).to(dtype) for _ in range(2))
    for act in ("silu", "gelu"):
        R.check("h", ops.gated_linear(x, wg, wu, act), *R.gated(x, wg, wu, act)["h"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [1, 31, 32, 33])
@pytest.mark.parametrize("V", [49152, 49153, 50000])
def test_scores(N, V, dtype):
    g = torch.Generator(device=DEV).manual_seed(N)
    x = torch.randn(N, 64, device=DEV, generator=g).to(dtype)
    w = (torch.randn(V, 64, device=DEV, generator=g) * 0.2).to(dtype)
    y = torch.randint(0, V, (N,), device=DEV, generator=g)
    y[0] = V - 1
    ids, p, live = R.targets_of_labels(y)
    value, bound = R.head(x, w, ids, p, live, 1.0, torch.ones(N, device=DEV).double())["loss"]
    R.check("loss", ops.linear_cross_entropy(x, w, y, reduction="none"), value, bound)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    assert torch.equal(ops.linear_cross_entropy(a, b, y, reduction="none").detach(), ops.linear_cross_entropy(x, w, y, reduction="none"))
