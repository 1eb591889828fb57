"""The CPU form of ops.verify_drafts against the rule followed step by step: borders,
ties, and entries that are no probabilities."""

import math

import pytest
import torch

from multiscreen._dense import verify_dense
from test_gpu_cache_rows import FLOATS, _name
from test_gpu_verify_drafts import check as check_kernel, rule


def check(target, tokens, parents, uniforms, draft):
    B, M, _ = target.shape
    path, count, token = verify_dense(target, tokens, parents, uniforms, draft)
    for b in range(B):
        par = [-1] + list(range(M - 1)) if parents is None else parents[b].tolist()
        par = [p if 0 <= p < i else -1 for i, p in enumerate(par)]
        walk, tok = rule(target[b], tokens[b], par, None if uniforms is None else uniforms[b], None if draft is None else draft[b])
        assert path[b].tolist() == walk + [-1] * (M - len(walk)) and int(count[b]) == len(walk)
        assert int(token[b]) == tok, (int(token[b]), tok)


@pytest.mark.parametrize("dt", FLOATS, ids=_name)
def test_greedy_ties_nan_and_infinities(dt):
    tie = torch.zeros(1, 3, 500)
    tie[0, 0, [7, 409]] = 1.0
    tie[0, 1] = -0.0
    tie[0, 2, [499, 300, 301]] = math.inf
    for first in (7, 409, 0):
        check(tie.to(dt), torch.tensor([[0, first, 0]]), None, None, None)
        check(-tie.to(dt), torch.tensor([[0, first, 0]]), None, None, None)
    tie[0, 1, [17, 30]] = math.nan
    check(tie.to(dt), torch.tensor([[0, 7, 17]]), None, None, None)   # a NaN is the largest, the first of them
    check(tie.to(dt), torch.tensor([[0, 7, 30]]), None, None, None)
    check(torch.full((1, 2, 300), -math.inf, dtype=dt), torch.tensor([[0, 0]]), None, None, None)
    check(torch.full((1, 2, 300), math.nan, dtype=dt), torch.tensor([[0, 0]]), None, None, None)


@pytest.mark.parametrize("dt", FLOATS, ids=_name)
def test_borders(dt):
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


@pytest.mark.parametrize("check", [check, pytest.param(check_kernel, marks=pytest.mark.gpu)], ids=["cpu", "cuda"])
def test_odd_entries(check):
    """NaN, negative and infinite entries of the target's and the draft's rows count as the operator has it."""
    V = 60
    g = torch.Generator().manual_seed(1)
    odd = torch.softmax(torch.randn(1, 4, V, generator=g), -1)
    odd[0, :, 3], odd[0, :, 4] = math.nan, -0.5
    par = torch.tensor([[-1, 0, 0, 0]])
    for u in ([0.001, 0.0, 0.0, 0.9], [0.9, 0.5, 0.9, 0.99]):
        check(odd, torch.tensor([[0, 3, 4, 8]]), par, torch.tensor([u]), None)
    draft = torch.softmax(torch.randn(1, 3, V, generator=g), -1)
    for column, value in ((8, math.nan), (40, math.nan), (40, math.inf), (8, math.inf)):
        q = draft.clone()
        q[0, :, column] = value
        for u0 in (0.0, 0.3, 0.99):
            check(odd, torch.tensor([[0, 8, 9, 10]]), None, torch.tensor([[u0, 0.99, 0.99, 0.99]]), q)
    high = odd.clone()
    high[0, :, 20] = math.inf
    for u0 in (0.0, 0.3, 0.99):
        check(high, torch.tensor([[0, 8, 9, 10]]), par, torch.tensor([[u0, 0.99, 0.99, 0.99]]), None)
        check(high, torch.tensor([[0, 20, 9, 10]]), None, torch.tensor([[u0, 0.99, 0.99, 0.99]]), draft)
    zero = torch.zeros(1, 2, V)
    u = torch.tensor([[0.3, 0.9]])
    check(zero, torch.tensor([[0, 5]]), None, u, None)
    check(zero, torch.tensor([[0, 5]]), None, u, zero[:, :1])
    few = zero.clone()
    few[0, 0, 5] = 0.25
    check(few, torch.tensor([[0, 5]]), None, u, few[:, :1] * 2 + 0.5)  # the draft above the target everywhere
