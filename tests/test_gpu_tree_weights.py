"""The bits of ops.tree_decode's pair weights: beside a result in bf16 an error
of a weight shows only where it moves a value over a border between two results,
so each element is held to half a step of its own size and little more."""

import pytest
import torch

from test_gpu_cache_rows import CODES, TOP, _name
from test_gpu_tree_decode import Case


def lone_pairs(M, D, ct, dt, seed):
    """Nodes that see their own row only (a window of one step), by a key near the query."""
    B, H, n = 24, 6, 40
    case = Case(B, M, H, D, dt, ct, [n] * B, "chain", w=(1.0, 1.0), r=1.2, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = case.q.float()
    k = q + 0.3 * q.norm(dim=-1, keepdim=True) * D ** -0.5 * torch.randn(q.shape, generator=g)
    at = slice(n, n + M)
    if case.ks is None:
        case.kc[:, at] = k.to(dt)
    else:
        scale = k.abs().amax(-1) / TOP[ct]
        code = k / scale.unsqueeze(-1)
        case.ks[:, at] = scale
        case.kc[:, at] = (code.round() if ct == torch.int8 else code).to(ct)
    return case


# One pair a node: y = tanh(a^2) v^, a = 1 - r (1 - s) with r < 1.25 and a > 0.5.
#  - s: the sum of D <= 128 exact products, off by at most (D + 3) 2^-24 = 7.8e-6, and the two inverse lengths, 2^-22
#    each: ds < 8.3e-6.  a^2 moves by 2 r ds / a < 4.2e-5 of itself in the worst rounding of every addition; random
#    roundings grow with sqrt(D) to a tenth of that.
#  - the weight as two terms: 2^-22 (fp16); the value's length, the row's length, tanh and the product: 2^-22 each
# so an element is off by less than 5e-5 of itself before it is rounded to bf16, by half a step.  One fp16 term alone
# would add up to 2^-12 = 2.4e-4.
@pytest.mark.gpu
@pytest.mark.parametrize("ct", CODES, ids=_name)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("M", [1, 12, 20, 40])
def test_a_bf16_result_is_the_nearest(M, D, ct):
    case = lone_pairs(M, D, ct, torch.bfloat16, seed=D + M)
    ref = case.expected()
    q, k = case.q.double(), case.kc.double()[:, 40:40 + M]
    s = (q * k).sum(-1) / (q.norm(dim=-1) * k.norm(dim=-1))
    assert float((1 - case.r * (1 - s)).min()) > 0.5
    got = case.run().double().cpu()
    half = torch.exp2(torch.frexp(ref).exponent.double() - 9)  # half a bf16 step at ref
    over = ((got - ref).abs() - half) / ref.abs().clamp(min=1e-30)
    assert float(over.max()) < 5e-5, float(over.max())
