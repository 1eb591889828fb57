"""The CPU form of ops.verify_drafts against the rule followed step by step: borders,
ties, and entries that are no probabilities."""

import math

import pytest
import torch

from multiscreen._dense import verify_dense
from test_gpu_cache_rows import FLOATS, _name
from test_gpu_verify_drafts import rule


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
