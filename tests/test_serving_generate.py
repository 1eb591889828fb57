"""generate_speculative takes the prompts that generate and generate_greedy take."""

import pytest
import torch

from test_serving import CODES, DEVICES, prompt_of
from test_serving_attention import VOCAB, lm_of


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
