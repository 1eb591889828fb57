"""generate_speculative takes the prompts that generate and generate_greedy take."""

import pytest
import torch

from test_serving import CODES, DEVICES, prompt_of
from test_serving_attention import VOCAB, apart, blind, lm_of


@pytest.mark.parametrize("dev", DEVICES)
def test_an_empty_batch(dev):
    lm = lm_of(dev)
    none = prompt_of(0, 5, VOCAB, dev)
    for t in (0, 1.0):
        got = lm.generate_speculative(none, lm, 4, temperature=t)
        assert got.shape == (0, 9) and got.dtype == lm.generate(none, 4).dtype


@pytest.mark.parametrize("dev", DEVICES)
def test_prompts_of_32_bit_tokens(dev):
    lm, small = lm_of(dev), lm_of(dev, seed=5, layers=1)
    prompt = prompt_of(2, 9, VOCAB, dev)
    got = lm.generate_speculative(prompt.int(), small, 12, 3, temperature=0)
    assert got.dtype == lm.generate(prompt.int(), 2).dtype == torch.int64
    assert torch.equal(got, lm.generate_greedy(prompt, 12))
    torch.manual_seed(3)
    a = lm.generate_speculative(prompt.int(), small, 12, 3)
    torch.manual_seed(3)
    assert torch.equal(a, lm.generate_speculative(prompt, small, 12, 3))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("ct", [None] + CODES)
def test_up_to_the_last_position(dev, ct):
    """The last token needs no position of its own: positions + 1 tokens are the most that generate gives."""
    lm, small = lm_of(dev, cap=30), lm_of(dev, seed=5, layers=1, cap=30)
    prompt = prompt_of(3, 12, VOCAB, dev)
    for new in (17, 18, 19):
        want = lm.generate_greedy(prompt, new, cache_dtype=ct)
        for drafter, drafts in ((small, 5), (lm, 7)):
            assert torch.equal(lm.generate_speculative(prompt, drafter, new, drafts, temperature=0, cache_dtype=ct), want)
    with pytest.raises(IndexError):
        lm.generate_speculative(prompt, small, 20)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("ct", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_caches_of_another_floating_type(dev, dt, ct):
    """A token decoded over rows of ct is a tree of one node over them."""
    lm, T = lm_of(dev).to(dt), 20
    prompt, token = prompt_of(2, T, VOCAB, dev), prompt_of(2, 1, VOCAB, dev, seed=2)
    one, two, full = (lm.new_cache(2, 32, t, dev) for t in (ct, ct, dt))
    for c in (one, two, full):
        lm.prefill(prompt, c)
    got, ref = lm.decode_step(token, one, T), lm.tree_step(token, two, torch.tensor([T], device=dev))[0][:, 0]
    # roundings of the narrower type through two layers: 2^-8 of every activation, some ten of them a layer
    coarse = torch.bfloat16 in (dt, ct)
    assert apart(got, ref) < (0.1 if coarse else 2e-2) and apart(got, lm.decode_step(token, full, T)) < (0.1 if coarse else 2e-2)
    assert apart(blind(lm).decode_step(token, full, T), got) > 0.4
    assert all(c.k.dtype == ct for c in one)
    assert lm.generate_greedy(prompt, 4, cache_dtype=ct).shape == lm.generate(prompt, 4, cache_dtype=ct).shape == (2, T + 4)
