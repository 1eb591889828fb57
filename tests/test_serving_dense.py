"""The CPU forms of the serving operators beside the rules that the GPU forms
keep: rows that are not finite, masked places, odd entries of probability rows."""

import math

import pytest
import torch

from multiscreen._dense import tree_dense
from test_gpu_cache_rows import CODES, FLOATS, TOP, _name
from test_gpu_tree_decode import Case, check

TYPES = FLOATS + CODES


def dense(case):
    k, v = case.kc, case.vc
    if case.ks is not None:
        k, v = k.float() * case.ks.unsqueeze(-1), v.float() * case.vs.unsqueeze(-1)
    return tree_dense(case.q, k, v, torch.tensor(case.lengths), case.parents, case.r, case.w)


@pytest.mark.parametrize("ct", TYPES, ids=_name)
def test_dense_rows_that_are_not_finite_or_zero(ct):
    """A live value row with a NaN or an infinity makes the nodes that see it NaN and no others, a key row drops out;
    zero rows take part as zeros."""
    dt = torch.bfloat16 if ct in TOP else ct
    for kind in ("chain", "star"):
        case = Case(2, 6, 2, 32, dt, ct, [40, 33], kind, w=(60.0, 80.0), r=1.02, seed=8)
        check(case, dense(case))
        case.kc[0, 7] = 0
        case.vc[0, 9] = 0
        case.q[0, 2] = 0
        if case.ks is not None:
            case.ks[1, 11] = math.nan
            case.vs[1, 35, 0] = math.nan  # drafted row 2 of sequence 1
        else:
            case.kc[1, 11, :, 3] = math.inf
            case.kc[1, 12, :, 3] = math.nan
            case.vc[1, 35, 0, 5] = math.nan
            case.vc[1, 36, 1, 5] = -math.inf
        ref = case.expected()
        assert not torch.isnan(ref[0]).any() and not torch.isnan(ref[1, :2]).any()
        assert kind == "star" or torch.isnan(ref[1, 2:, 0]).any()
        check(case, dense(case))


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_dense_value_rows_of_one_branch(value):
    """Each node sees its own row, by the key that is its query: node 2's values are node 2's alone."""
    case = Case(1, 4, 2, 32, torch.float32, torch.float32, [30], "star", w=(20.0, 40.0), seed=6)
    case.kc[0, 30:34] = case.q[0]
    case.vc[0, 32, :, 7] = value
    ref = case.expected()
    assert torch.isnan(ref[0, 2]).all() and not torch.isnan(ref[0, [0, 1, 3]]).any()
    check(case, dense(case))


@pytest.mark.parametrize("ct", TYPES, ids=_name)
def test_dense_masked_places_may_hold_anything(ct):
    dt = torch.bfloat16 if ct in TOP else ct
    case = Case(2, 12, 2, 64, dt, ct, [200, 90], "star", w=(20.0, 40.0), seed=3)
    bad = torch.tensor([math.nan, math.inf, -math.inf])
    for b, n in enumerate(case.lengths):
        for pos in list(range(0, n - 60)) + list(range(n + 12, case.kc.shape[1])):
            for c, s in ((case.kc, case.ks), (case.vc, case.vs)):
                if s is None:
                    c[b, pos] = bad[pos % 3]
                else:
                    s[b, pos] = bad[pos % 3]
    got = dense(case)
    assert torch.isfinite(got).all()
    check(case, got)


def test_dense_queries_that_are_not_finite_see_nothing():
    case = Case(1, 4, 2, 32, torch.float32, torch.float32, [30], "star", w=(20.0, 40.0), seed=4)
    base = dense(case)
    case.q[0, 2, 0, 3], case.q[0, 3, 1, 5] = math.nan, math.inf
    got = dense(case)
    assert (got[0, 2, 0] == 0).all() and (got[0, 3, 1] == 0).all()
    assert torch.equal(got[0, :2], base[0, :2]) and torch.equal(got[0, 2, 1], base[0, 2, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("ct", TYPES, ids=_name)
def test_queries_that_are_not_finite_see_nothing(ct):
    """The kernels alike: one block a head and split windows, few nodes and many."""
    for dt in FLOATS if ct in TOP else [ct]:
        for M, n, w in ((4, 30, 40.0), (40, 90, 60.0), (7, 3000, 3500.0)):
            case = Case(1, M, 2, 64, dt, ct, [n], "star", w=(0.5 * w, w), r=1.3, seed=M)
            base = case.run()
            case.q[0, 2, 0, 3], case.q[0, 3, 1, 5] = math.nan, math.inf
            got = case.run()
            assert (got[0, 2, 0] == 0).all() and (got[0, 3, 1] == 0).all()
            got[0, 2, 0], got[0, 3, 1] = base[0, 2, 0], base[0, 3, 1]
            assert torch.equal(got, base) and torch.isfinite(base).all()
