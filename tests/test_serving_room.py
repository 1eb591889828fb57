"""Steps over trees whose rows do not fit their cache: refused where the host
holds the lengths, NaN for those sequences (and no others) where the device does."""

import pytest
import torch

from multiscreen import ScreeningAttention
from multiscreen.attention import KVCache
from test_serving import CODES, DEVICES, lm_of, prompt_of

TYPES = [torch.float32] + CODES


def step(lm, caches, tokens, lengths):
    return lm.tree_step(tokens, caches, torch.tensor(lengths, device=tokens.device))[0]


@pytest.mark.parametrize("ct", TYPES)
def test_the_host_refuses_lengths_without_room(ct):
    lm, T, M = lm_of("cpu"), 20, 4
    prompt, tokens = prompt_of(2, T, 53, "cpu"), prompt_of(2, M, 53, "cpu", seed=2)
    caches = lm.new_cache(2, T + M - 1, ct, "cpu")
    lm.prefill(prompt, caches)
    before = caches[0].read(0, T, torch.float32)[0]
    for lengths in ([T], [3, T], [-1, 3], [2 ** 40]):
        with pytest.raises(IndexError):
            step(lm, caches, tokens, lengths)
    assert torch.equal(caches[0].read(0, T, torch.float32)[0], before)  # nothing was written
    assert torch.isfinite(step(lm, caches, tokens, [T - 1])).all()
    with pytest.raises(IndexError):  # more nodes than positions
        step(lm, caches, prompt_of(2, T + M, 53, "cpu"), [0])


@pytest.mark.parametrize("ct", TYPES)
def test_a_layer_on_the_host(ct):
    torch.manual_seed(0)
    attn, x = ScreeningAttention(32, 2), torch.randn(2, 3, 32)
    cache = KVCache(2, 10, 2, 16, ct, "cpu")
    with torch.no_grad():
        assert torch.isfinite(attn.tree_step(x, cache, torch.tensor([7, 0]))[0]).all()
        for lengths in ([8, 0], [-1, 0], [8]):
            with pytest.raises(IndexError):
                attn.tree_step(x, cache, torch.tensor(lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("ct", TYPES)
def test_the_device_gives_nan_without_room(ct):
    lm, T, M, cap = lm_of("cuda"), 20, 4, 24
    prompt, tokens = prompt_of(3, T, 53, "cuda"), prompt_of(3, M, 53, "cuda", seed=2)

    def run(lengths):
        caches = lm.new_cache(3, cap, ct, "cuda")
        lm.prefill(prompt, caches)
        return step(lm, caches, tokens, lengths), caches

    base, _ = run([T, T, T])
    assert torch.isfinite(base).all()
    for far in (T + 1, cap, 2 ** 40, -1, -2 ** 40):
        got, caches = run([T, far, T])
        assert torch.isnan(got[1]).all(), far
        assert torch.equal(got[::2], base[::2])
        assert all(torch.isfinite(x).all() for c in caches for x in c.read(0, cap, torch.float32))
    assert torch.isnan(run([T + 1])[0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("ct", TYPES)
def test_a_layer_on_the_device(ct):
    lm = lm_of("cuda")
    x = torch.randn(2, 3, 64, device="cuda")
    for part in (lm.blocks[0], lm.blocks[0].attn):
        cache = KVCache(2, 10, 4, 16, ct, "cuda")
        with torch.no_grad():
            base = part.tree_step(x, cache, torch.tensor([7, 7], device="cuda"))[0]
            got = part.tree_step(x, cache, torch.tensor([8, 7], device="cuda"))[0]
        assert torch.isfinite(base).all() and torch.isnan(got[0]).all() and torch.equal(got[1], base[1])


@pytest.mark.gpu
def test_room_is_found_at_each_replay():
    """A captured step follows its lengths past the end of the cache and back."""
    lm, T, M, cap = lm_of("cuda"), 20, 4, 26
    prompt, tokens = prompt_of(2, T, 53, "cuda"), prompt_of(2, M, 53, "cuda", seed=2)
    caches = lm.new_cache(2, cap, torch.int8, "cuda")
    lm.prefill(prompt, caches)
    lengths = torch.full((2,), T, dtype=torch.int64, device="cuda")
    lm.tree_step(tokens, caches, lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = lm.tree_step(tokens, caches, lengths)
    for n in ([T, T], [T + 3, T + 2], [T, T + 9], [T + 2, T]):
        lengths.copy_(torch.tensor(n))
        graph.replay()
        torch.cuda.synchronize()
        ref, _ = lm.tree_step(tokens, caches, lengths)
        assert [bool(torch.isnan(out[b]).all()) for b in range(2)] == [x + M > cap for x in n]
        assert torch.equal(out.nan_to_num(0.5), ref.nan_to_num(0.5))
