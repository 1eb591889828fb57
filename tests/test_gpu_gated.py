"""ops.gated_linear on the GPU: values and gradients against 64 bits within bounds counted in roundings."""

import math

import pytest
import torch

import wide_reference as R
from multiscreen import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _data(N, d, F, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(N, d, device=DEV, generator=g).to(dtype)
    wg, wu = ((torch.randn(F, d, device=DEV, generator=g) / math.sqrt(d)).to(dtype) for _ in range(2))
    dh = (0.01 * torch.randn(N, F, device=DEV, generator=g)).to(dtype)
    return x, wg, wu, dh


def _leaf(*t):
    return [x.detach().requires_grad_() for x in t]


def _run(x, wg, wu, dh, act):
    x, wg, wu = _leaf(x, wg, wu)
    h = ops.gated_linear(x, wg, wu, act)
    return dict(zip(("h", "dx", "dgate", "dup"), (h.detach(), *torch.autograd.grad(h, (x, wg, wu), dh))))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("N,d,F", [(1, 1, 1), (1, 64, 100), (16, 512, 2048), (127, 33, 129), (128, 64, 128), (129, 96, 255),
                                   (300, 100, 301), (200, 256, 1365), (33, 1000, 64), (2500, 64, 96)])
def test_gated(N, d, F, act, dtype):
    x, wg, wu, dh = _data(N, d, F, dtype)
    got = _run(x, wg, wu, dh, act)
    for name, (value, bound) in R.gated(x, wg, wu, act, dh).items():
        R.check(name, got[name], value, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_far_arguments(act, dtype):
    # gates from -60 to 60: the lower tail goes to zero, the upper one is linear
    x, wg, wu, dh = _data(64, 32, 200, dtype, 1)
    wg = (wg.float() * 15).to(dtype)
    got = _run(x, wg, wu, dh, act)
    for name, (value, bound) in R.gated(x, wg, wu, act, dh).items():
        R.check(name, got[name], value, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_of_gradients(dtype):
    # upstream gradients of very different size: loss scaling, and tiny ones
    x, wg, wu, dh = _data(150, 64, 200, dtype, 2)
    for s in (2.0 ** -14, 2.0 ** 10):
        d = (dh.float() * s).to(dtype)
        got = _run(x, wg, wu, d, "silu")
        for name, (value, bound) in R.gated(x, wg, wu, "silu", d).items():
            R.check(name, got[name], value, bound)


@pytest.mark.parametrize("up", [66, -66])
def test_operands_whose_squares_leave_the_range(up):
    # x and the weights far from 1 in opposite directions, in fp32: the products are ordinary, the rows' squares are not, and
    # the bound of a row's norm is its largest entry times sqrt(d)
    x, wg, wu, dh = _data(150, 64, 200, torch.float32, 5)
    x, wg, wu, dh = x * 2.0 ** up, wg * 2.0 ** -up, wu * 2.0 ** -up, dh * 2.0 ** -20
    got = _run(x, wg, wu, dh, "silu")
    w = torch.cat([wg, wu])
    spread = math.prod(8.0 * float(t.abs().amax()) / float(t.double().norm(dim=1).amax()) for t in (x, w))
    for name, (value, bound) in R.gated(x, wg, wu, "silu", dh, spread).items():
        R.check(name, got[name], value, bound)


def test_zero_gradient_and_no_rows():
    for dtype in TYPES:
        x, wg, wu, dh = _data(70, 64, 100, dtype)
        got = _run(x, wg, wu, torch.zeros_like(dh), "silu")
        assert not got["dx"].any() and not got["dgate"].any() and not got["dup"].any()
        got = _run(x[:0], wg, wu, dh[:0], "gelu")
        assert got["h"].shape == (0, 100) and got["dx"].shape == (0, 64) and not got["dgate"].any() and not got["dup"].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_of_a_row_stays_in_it(dtype):
    x, wg, wu, dh = _data(140, 64, 200, dtype, 3)
    clean = _run(x, wg, wu, dh, "silu")
    x[5, 3] = math.nan
    got = _run(x, wg, wu, dh, "silu")
    keep = torch.arange(140, device=DEV) != 5
    assert bool(torch.isnan(got["h"][5]).all()) and bool(torch.isnan(got["dx"][5]).all())
    assert torch.equal(got["h"][keep], clean["h"][keep])
    assert bool(torch.isfinite(got["dx"][keep]).all())
    assert bool(torch.isnan(got["dgate"]).all())  # as of any sum over the rows


@pytest.mark.parametrize("dtype", TYPES)
def test_views_and_strides(dtype):
    big = torch.randn(60, 3, 300, device=DEV).to(dtype)
    x = big[:, 1, 7:7 + 96]
    both = (torch.randn(2, 200, 130, device=DEV) * 0.1).to(dtype)
    wg, wu = both[0, :, 3:99], both[1, :, 8:104]
    dh = torch.randn(200, 60, device=DEV).to(dtype).t()
    got = _run(x, wg, wu, dh, "silu")
    want = _run(x.contiguous(), wg.contiguous(), wu.contiguous(), dh.contiguous(), "silu")
    for k in got:
        assert torch.equal(got[k], want[k])
    # gate and up as halves of one weight, a broadcast gradient
    w = (torch.randn(400, 96, device=DEV) * 0.1).to(dtype)
    got = _run(x, w[:200], w[200:], torch.ones(1, 1, device=DEV, dtype=dtype).expand(60, 200), "gelu")
    want = _run(x, w[:200].clone(), w[200:].clone(), torch.ones(60, 200, device=DEV, dtype=dtype), "gelu")
    for k in got:
        assert torch.equal(got[k], want[k])


def test_only_what_is_asked_for_and_shared_weights():
    x, wg, wu, dh = _data(130, 64, 200, torch.bfloat16, 4)
    full = _run(x, wg, wu, dh, "silu")
    for k, name in ((0, "dx"), (1, "dgate"), (2, "dup")):
        t = [x, wg, wu]
        t[k], = _leaf(t[k])
        g, = torch.autograd.grad(ops.gated_linear(*t), t[k], dh)
        assert torch.equal(g, full[name])
    w, = _leaf(wg)
    g, = torch.autograd.grad(ops.gated_linear(x, w, w), w, dh)
    a, b = _leaf(wg, wg)
    parts = torch.autograd.grad(ops.gated_linear(x, a, b), (a, b), dh)
    assert torch.equal(g, parts[0] + parts[1])


def test_gradient_against_differences():
    x, wg, wu, dh = (t.float() for t in _data(10, 16, 24, torch.float32, 5))
    dh = dh * 100
    got = _run(x, wg, wu, dh, "gelu")
    gen = torch.Generator(device=DEV).manual_seed(1)
    for k, name in ((0, "dx"), (1, "dgate"), (2, "dup")):
        v = torch.randn(got[name].shape, device=DEV, generator=gen)
        v = v / v.norm()
        e, t = 2.0 ** -6, [x, wg, wu]
        ends = []
        for sign in (1, -1):
            u = list(t)
            u[k] = u[k] + sign * e * v
            ends.append(float((ops.gated_linear(*u, "gelu").double() * dh.double()).sum()))
        slope = (ends[0] - ends[1]) / (2 * e)
        assert abs(slope - float((got[name] * v).sum())) < 2e-3 * max(1.0, float(got[name].norm()))


def test_pieces_of_the_features():
    # 4 N F bytes of dg and du above 1 GB: several pieces
    N, d, F = 140000, 32, 2100
    x, wg, wu, dh = _data(N, d, F, torch.bfloat16, 6)
    got = _run(x, wg, wu, dh, "silu")
    for name, (value, bound) in R.gated(x, wg, wu, "silu", dh).items():
        R.check(name, got[name], value, bound)


@pytest.mark.parametrize("dtype,N", [(torch.bfloat16, 1999), (torch.float16, 1999), (torch.float32, 1100)])
def test_blocks_that_share_both_products(dtype, N):
    # sizes at which each CU's block takes ranges of dWg and dWu and then one of dx
    x, wg, wu, dh = _data(N, 520, 7001, dtype, 9)
    got = _run(x, wg, wu, dh, "silu")
    for name, (value, bound) in R.gated(x, wg, wu, "silu", dh).items():
        R.check(name, got[name], value, bound)


def test_weights_past_32_bits():
    # 4.4 GB of each weight, of its copy and of its gradient: the reference takes the features in parts
    N, d, F = 4, 1040, 2 ** 21 + 77
    x, wg, wu, dh = _data(N, d, F, torch.bfloat16, 10)
    got = _run(x, wg, wu, dh, "silu")
    value = bound = reach = 0.0
    for at in range(0, F, 2 ** 18):
        c = slice(at, at + 2 ** 18)
        want = R.gated(x, wg[c], wu[c], "silu", dh[:, c])
        R.check("h", got["h"][:, c], *want["h"])
        R.check("dgate", got["dgate"][c], *want["dgate"])
        R.check("dup", got["dup"][c], *want["dup"])
        value, bound = value + want["dx"][0], bound + want["dx"][1]
        # of the sums over all features: |dg| and |du| are at most 1.15 |dh| max|x| max|w|
        top = 1.15 * float(x.double().norm(dim=1).amax()) * float(torch.cat([wg[c], wu[c]]).float().norm(dim=1).amax())
        reach = reach + top * (dh[:, c].double().abs() @ (wg[c].double().abs() + wu[c].double().abs()))
    R.check("dx", got["dx"], value, bound + R.product_slack(2 * F, torch.bfloat16) * reach)


def test_equal_calls_streams_and_graph():
    x, wg, wu, dh = _data(500, 128, 700, torch.float16, 7)
    first = _run(x, wg, wu, dh, "silu")
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in side:
            with torch.cuda.stream(s):
                got.append(_run(x, wg, wu, dh, "silu"))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(x, wg, wu, dh, "silu")
    for seed in range(3):
        graph.replay()
        torch.cuda.synchronize()
        got.append({k: v.clone() for k, v in out.items()})
        _run(x, wg, wu, dh, "silu")
    for r in got:
        for k in first:
            assert torch.equal(first[k], r[k]), k


def test_autocast():
    x, wg, wu, dh = _data(40, 64, 100, torch.float32, 8)
    a, b, c = _leaf(x, wg, wu)
    with torch.autocast("cuda", dtype=torch.float16):
        h = ops.gated_linear(a, b, c)
    assert h.dtype == torch.float16
    assert all(g.dtype == torch.float32 for g in torch.autograd.grad(h, (a, b, c), dh.half()))
    assert torch.equal(h, ops.gated_linear(x.half(), wg.half(), wu.half()))


def test_refusals():
    x, wg, wu, _ = _data(10, 64, 50, torch.bfloat16)
    f = ops.gated_linear
    for error, call in [(RuntimeError, lambda: f(x.cpu(), wg, wu)), (RuntimeError, lambda: f(x, wg.cpu(), wu)),
                        (TypeError, lambda: f(x, wg.float(), wu)), (TypeError, lambda: f(x.double(), wg.double(), wu.double())),
                        (ValueError, lambda: f(x, wg[:, :32], wu[:, :32])), (ValueError, lambda: f(x, wg, wu[:40])),
                        (ValueError, lambda: f(x, wg[:0], wu[:0])), (ValueError, lambda: f(x, wg, wu, "relu"))]:
        with pytest.raises(error):
            call()
