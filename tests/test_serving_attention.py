"""The serving paths of a model whose logits are its attention's: every comparison
here fails for a stale, shifted or missing cache row, which the fixture and the
planted mistakes show.  On the CPU (the dense forms) and on the GPU."""

import copy
import math

import pytest
import torch

from multiscreen import MultiscreenLM
from test_gpu_tree_decode import lines_of
from test_serving import CODES, DEVICES, prompt_of

VOCAB = 53


def lm_of(dev, seed=8, layers=2, cap=256):
    """out_proj scaled up, so that attention outweighs the embedding; r = 1.2, windows 3 .. 100."""
    torch.manual_seed(seed)
    lm = MultiscreenLM(vocab_size=VOCAB, d_model=64, num_heads=4, num_layers=layers, max_seq_len=cap)
    with torch.no_grad():
        for blk in lm.blocks:
            blk.attn.s_r.fill_(math.log(0.2))
            blk.attn.s_v.copy_(torch.log(torch.linspace(2.0, 99.0, 4)))
            blk.attn.out_proj.weight.mul_(16)
    return lm.to(dev).eval()


def blind(lm):
    """The model without attention."""
    lm = copy.deepcopy(lm)
    with torch.no_grad():
        for blk in lm.blocks:
            blk.attn.out_proj.weight.zero_()
    return lm


def apart(a, b):
    a, b = a.detach().float(), b.detach().float()
    return float((a - b).abs().max() / b.abs().max())


# fp32 sums in another order.  A row of codes may also have a neighbouring code where a projection's rounding crosses a
# border: 1/127 (int8) or 1/16 (e4m3) of one element of one row, among some twenty live rows.
def bound(ct):
    return 1e-4 if ct == torch.float32 else 2e-2


def fed(lm, ct, seqs, cap):
    """Caches of sequences decoded token by token from empty prompts' ends: (prompt, further tokens) of each."""
    caches, logits = [], []
    for prompt, line in seqs:
        one = lm.new_cache(1, cap, ct, prompt.device)
        out = lm.prefill(prompt.unsqueeze(0), one)
        for t, tok in enumerate(line.tolist()):
            out = lm.decode_step(torch.tensor([[tok]], device=prompt.device), one, len(prompt) + t)
        caches.append(one)
        logits.append(out[0])
    return caches, torch.stack(logits)


def order(c):
    """Codes as integers in the order of their values, neighbours one apart."""
    if c.dtype == torch.int8:
        return c.int()
    b = c.contiguous().view(torch.uint8).int()
    return torch.where(b >= 128, -(b - 128), b)


@pytest.mark.parametrize("dev", DEVICES)
def test_the_model_is_its_attention(dev):
    lm = lm_of(dev)
    prompt = prompt_of(3, 12, VOCAB, dev)
    assert apart(blind(lm)(prompt)["logits"], lm(prompt)["logits"]) > 0.5
    for ct in [None] + CODES:
        a, b = (m.generate_greedy(prompt, 17, cache_dtype=ct)[:, 12:] for m in (lm, blind(lm)))
        assert float((a == b).float().mean()) < 0.25 and min(len(set(x)) for x in a.tolist()) >= 5


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("ct", [torch.float32] + CODES)
def test_tree_step_and_accept(dev, ct):
    lm, B, T, M, cap = lm_of(dev), 2, 20, 8, 32
    prompt, tokens = prompt_of(B, T, VOCAB, dev), prompt_of(B, M, VOCAB, dev, seed=2)
    parents = torch.tensor([[-1, 0, 0, 1, 1, 3, 2, 6], [-1, 0, 1, 2, 0, 4, 4, 1]], device=dev)
    at = torch.full((B,), T, device=dev)
    caches = lm.new_cache(B, cap, ct, dev)
    lm.prefill(prompt, caches)
    logits, kvs = lm.tree_step(tokens, caches, at, parents)
    for b in range(B):
        lines = [list(reversed(x)) for x in lines_of(parents[b].cpu())]
        _, ref = fed(lm, ct, [(prompt[b], tokens[b, x]) for x in lines], cap)
        assert apart(logits[b], ref) < bound(ct)
        # a node's parent missing from its line is far outside the bound
        for i, x in enumerate(lines):
            if len(x) > 2:
                assert apart(logits[b, i], fed(lm, ct, [(prompt[b], tokens[b, x[:1] + x[2:]])], cap)[1][0]) > 5 * bound(ct)

    # nodes 0, 1, 3, 5 and 0, 4, 6 are accepted: the caches then are those of the sequences decoded token by token
    path = torch.tensor([[0, 1, 3, 5] + [-1] * 4, [0, 4, 6] + [-1] * 5], device=dev)
    count = torch.tensor([4, 3], device=dev)
    lengths = lm.accept(caches, kvs, path, count, at)
    assert lengths.tolist() == [T + 4, T + 3]
    line = [tokens[b, path[b, :count[b]]] for b in range(B)]
    ref, _ = fed(lm, ct, [(prompt[b], line[b]) for b in range(B)], cap)
    wrong, _ = fed(lm, ct, [(prompt[b], line[b].flip(0)) for b in range(B)], cap)
    for layer in range(2):
        for b in range(B):
            n = int(lengths[b])
            for x in ("k", "v"):
                got, want, other = (getattr(c[layer], x)[i] for c, i in ((caches, b), (ref[b], 0), (wrong[b], 0)))
                if ct == torch.float32:
                    assert apart(got[:n], want[:n]) < 1e-5 and apart(got[:n], other[:n]) > 1e-2
                    continue
                off = (order(got[:n]) - order(want[:n])).abs()
                assert int(off.max()) <= 1 and float((off > 0).float().mean()) < 0.05
                assert int((order(got[:n]) - order(other[:n])).abs().max()) > 5
                s, w = (getattr(c[layer], x + "_scale")[i, :n] for c, i in ((caches, b), (ref[b], 0)))
                assert apart(s, w) < 1e-3

    # the step after it
    nxt = prompt_of(B, 1, VOCAB, dev, seed=3)
    got, _ = lm.tree_step(nxt, caches, lengths)
    _, ref = fed(lm, ct, [(prompt[b], torch.cat((line[b], nxt[b]))) for b in range(B)], cap)
    assert apart(got[:, 0], ref) < bound(ct)
    _, wrong = fed(lm, ct, [(prompt[b], torch.cat((line[b].flip(0), nxt[b]))) for b in range(B)], cap)
    assert min(apart(got[b, 0], wrong[b]) for b in range(B)) > 5 * bound(ct)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("ct", [None] + CODES)
def test_speculative_greedy_is_greedy(dev, ct):
    lm = lm_of(dev)
    prompt = prompt_of(3, 12, VOCAB, dev)
    want = lm.generate_greedy(prompt, 17, cache_dtype=ct)
    for drafter, drafts in ((lm_of(dev, seed=5, layers=1), 3), (lm, 4), (blind(lm), 9)):
        for new in (1, 2, 17):
            got = lm.generate_speculative(prompt, drafter, new, drafts, temperature=0, cache_dtype=ct)
            assert torch.equal(got, want[:, :12 + new])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("ct", [None] + CODES)
def test_sequences_that_accept_different_numbers(dev, ct):
    """One sequence's drafts are right, another's never, the third's every second step."""
    lm = lm_of(dev)
    prompt = prompt_of(3, 12, VOCAB, dev)
    want = lm.generate_greedy(prompt, 17, cache_dtype=ct)

    class Half(MultiscreenLM):
        steps = 0

        def tree_step(self, tokens, caches, lengths, parents=None, rws=None):
            logits, kvs = lm.tree_step(tokens, caches, lengths, parents, rws)
            self.steps += 1
            logits[1] = logits[1].roll(1, -1)
            if self.steps % 2:
                logits[2] = logits[2].roll(1, -1)
            return logits, kvs

        def new_cache(self, *a):
            return lm.new_cache(*a)

        def prefill(self, ids, caches):
            return lm.prefill(ids, caches)

    half = Half(VOCAB, 64, 4, 2, max_seq_len=256).to(dev)
    assert torch.equal(lm.generate_speculative(prompt, half, 17, 5, temperature=0, cache_dtype=ct), want)


@pytest.mark.gpu
@pytest.mark.parametrize("ct", [None] + CODES)
def test_under_autocast(ct):
    """fp32 weights under fp16 autocast: a tree's logits are those of its lines decoded one by one, both near the
    fp32 model's; those without attention are not."""
    lm, B, T, M = lm_of("cuda"), 2, 20, 6
    prompt, tokens = prompt_of(B, T, VOCAB, "cuda"), prompt_of(B, M, VOCAB, "cuda", seed=2)
    parents = torch.tensor([-1, 0, 0, 1, 3, 2], device="cuda")
    at = torch.full((B,), T, device="cuda")
    caches = lm.new_cache(B, 32, ct or torch.float32, "cuda")
    lm.prefill(prompt, caches)
    full, _ = lm.tree_step(tokens, caches, at, parents)
    with torch.autocast("cuda", dtype=torch.float16):
        dt = lm._cache_dtype(prompt.device, ct)
        assert dt == (ct or torch.float16)
        caches = lm.new_cache(B, 32, dt, "cuda")
        lm.prefill(prompt, caches)
        got, _ = lm.tree_step(tokens, caches, at, parents)
        lines = [list(reversed(x)) for x in lines_of(parents.cpu())]
        ref = torch.stack([fed(lm, dt, [(prompt[b], tokens[b, x]) for x in lines], 32)[1] for b in range(B)])
        dark = blind(lm)
        none, _ = dark.tree_step(tokens, dark.new_cache(B, 32, dt, "cuda"), at, parents)
    # fp16 roundings (2^-11 of every activation, some ten of them a layer) through two layers
    assert apart(got, ref) < 3e-2 and apart(got, full) < 3e-2 and apart(none, full) > 0.3
