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
