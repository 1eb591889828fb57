"""Generation over caches of 8-bit rows, steps over trees of drafted tokens and
speculative generation, on the CPU (the dense forms) and on the GPU (the
kernels run together as a program uses them)."""

import math

import pytest
import torch

from multiscreen import MultiscreenLM, ScreeningAttention
from multiscreen._dense import quantise_rows, tree_relations, verify_dense
from multiscreen.attention import KVCache
from test_gpu_cache_rows import quantised
from test_gpu_tree_decode import definition, lines_of, tree_of
from test_gpu_verify_drafts import rule

CODES = [torch.int8, torch.float8_e4m3fn]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def lm_of(dev, dtype=torch.float32, seed=0, layers=2, d=64, vocab=53, cap=256):
    torch.manual_seed(seed)
    lm = MultiscreenLM(vocab_size=vocab, d_model=d, num_heads=4, num_layers=layers, max_seq_len=cap)
    with torch.no_grad():
        for blk in lm.blocks:  # live pairs at init: r = 1.2, windows 3 .. 100
            blk.attn.s_r.fill_(math.log(0.2))
            blk.attn.s_v.copy_(torch.log(torch.linspace(2.0, 99.0, 4)))
        lm.token_emb.weight.mul_(20)  # logits far enough apart for greedy choices
    return lm.to(dev, dtype).eval()


def prompt_of(B, T, vocab, dev, seed=1):
    return torch.randint(0, vocab, (B, T), generator=torch.Generator().manual_seed(seed)).to(dev)


# ---------------------------------------------------------------------------
# The dense forms
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("ct", CODES)
def test_dense_codes(ct):
    x = torch.randn(5, 3, 32, generator=torch.Generator().manual_seed(0))
    x[0, 0], x[1, 1, 4], x[2, 2, 5] = 0.0, math.inf, math.nan
    code, scale = quantise_rows(x, ct)
    want, wscale = quantised(x, ct)
    assert torch.equal(code.float().double(), want)
    assert torch.equal(scale.nan_to_num(-1.0), wscale.nan_to_num(-1.0))


def test_dense_relations():
    g = torch.Generator().manual_seed(0)
    for M in (1, 2, 3, 17, 64):
        for kind in ("chain", "tree", "roots"):
            p = tree_of(M, kind, 2, g)
            above, depth = tree_relations(p)
            for b in range(2):
                for i, line in enumerate(lines_of(p[b])):
                    assert above[b, i].nonzero().flatten().tolist() == sorted(line) and int(depth[b, i]) == len(line) - 1


@pytest.mark.parametrize("ct", [None] + CODES)
def test_dense_tree_step(ct):
    """ScreeningAttention.tree_step on the CPU against the float64 definition over what the cache holds."""
    torch.manual_seed(0)
    B, M, n = 2, 9, [14, 3]
    attn = ScreeningAttention(32, 2)
    with torch.no_grad():
        attn.s_r.fill_(math.log(0.2))
    cache = KVCache(B, 30, 2, 16, ct or torch.float32, "cpu")
    with torch.no_grad():
        cache.store(torch.randn(B, 14, 2, 16), torch.randn(B, 14, 2, 16), 0)
        parents = tree_of(M, "tree", B, torch.Generator().manual_seed(1))
        x = torch.randn(B, M, 32)
        y, (k, v) = attn.tree_step(x, cache, torch.tensor(n), parents)
        q = attn.project(x, attn.q_proj)
        kc, vc = cache.read(0, 30, torch.float32)
        ref = torch.stack([definition(q[b].double(), kc[b, :n[b] + M].double(), vc[b, :n[b] + M].double(), n[b], parents[b],
                                      attn.sharpness(), attn.window()) for b in range(B)])
        ref = ref.view(B, M, 32) @ attn.out_proj.weight.double().T
    assert float((y.double() - ref).abs().max() / ref.abs().max()) < 2e-5  # fp32 sums of 32 terms through a threshold
    if ct is None:
        assert torch.equal(cache.k[0, 14:23], k[0])


def test_dense_verify():
    g = torch.Generator().manual_seed(0)
    for M, kind in ((1, "chain"), (5, "chain"), (12, "tree")):
        p = torch.softmax(2 * torch.randn(3, M, 11, generator=g), -1)
        par = tree_of(M, kind, 3, g)
        tok = torch.randint(0, 11, (3, M), generator=g)
        u = torch.rand(3, M, generator=g)
        q = torch.softmax(torch.randn(3, max(M - 1, 0), 11, generator=g), -1)
        for uu, qq in ((None, None), (u, None)) + (((u, q),) if kind == "chain" else ()):
            path, count, token = verify_dense(p, tok, par, uu, qq)
            for b in range(3):
                walk, t = rule(p[b], tok[b], par[b].tolist(), None if uu is None else uu[b], None if qq is None else qq[b])
                assert path[b].tolist() == walk + [-1] * (M - len(walk)) and int(count[b]) == len(walk) and int(token[b]) == t


def test_dense_verify_of_a_padded_chain():
    """Behind a sequence's drafts stand tokens outside the vocabulary: the result is the shorter chain's."""
    g = torch.Generator().manual_seed(1)
    p, q = (torch.softmax(2 * torch.randn(64, n, 11, generator=g), -1) for n in (4, 3))
    tok, u = torch.randint(0, 11, (64, 4), generator=g), torch.rand(64, 4, generator=g)
    for b in range(64):
        n = b % 4 + 1
        line = torch.where(torch.arange(4) < n, tok[b], -1)
        path, count, token = verify_dense(p[b:b + 1], line[None], None, u[b:b + 1], q[b:b + 1])
        short = verify_dense(p[b:b + 1, :n], tok[b:b + 1, :n], None, u[b:b + 1, :n], q[b:b + 1, :n - 1])
        assert (int(count), int(token)) == (int(short[1]), int(short[2]))
        assert path[0].tolist() == short[0][0].tolist() + [-1] * (4 - n)
        assert rule(p[b], line, [-1, 0, 1, 2], u[b], q[b])[1] == int(token)


# ---------------------------------------------------------------------------
# The model, on both
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("ct", [torch.float32] + CODES)
def test_a_tree_step_is_its_paths_decoded_token_by_token(dev, ct):
    lm = lm_of(dev)
    B, T, M = 2, 20, 8
    prompt = prompt_of(B, T, 53, dev)
    parents = torch.tensor([[-1, 0, 0, 1, 1, 3, 2, 6], [-1, 0, 1, 2, 0, 4, 4, 1]], device=dev)
    tokens = prompt_of(B, M, 53, dev, seed=2)
    caches = lm.new_cache(B, T + M, ct, dev)
    lm.prefill(prompt, caches)
    logits, kvs = lm.tree_step(tokens, caches, torch.full((B,), T, device=dev), parents)
    for b in range(B):
        for i, line in enumerate(lines_of(parents[b].cpu())):
            one = lm.new_cache(1, T + M, ct, dev)
            lm.prefill(prompt[b:b + 1], one)
            for t, node in enumerate(reversed(line)):
                ref = lm.decode_step(tokens[b:b + 1, node:node + 1], one, T + t)
            # fp32 throughout; an 8-bit row moves to the next code where a projection's rounding crosses its border
            assert float((logits[b, i] - ref[0]).abs().max() / ref.abs().max()) < (1e-4 if ct == torch.float32 else 5e-2)
    # keep node 5's way (0, 1, 3, 5) and node 6's (0, 4, 6): the caches then hold those sequences
    path = torch.tensor([[0, 1, 3, 5] + [-1] * 4, [0, 4, 6] + [-1] * 5], device=dev)
    count = torch.tensor([4, 3], device=dev)
    before = caches[0].read(0, T, torch.float32)[0]
    lengths = lm.accept(caches, kvs, path, count, torch.full((B,), T, device=dev))
    assert lengths.tolist() == [T + 4, T + 3]
    assert torch.equal(caches[0].read(0, T, torch.float32)[0], before)
    nxt = prompt_of(B, 1, 53, dev, seed=3)
    got, _ = lm.tree_step(nxt, caches, lengths)
    for b in range(B):
        n = int(count[b])
        one = lm.new_cache(1, T + M, ct, dev)
        seq = torch.cat((prompt[b], tokens[b, path[b, :n]], nxt[b])).unsqueeze(0)
        ref = lm.prefill(seq, one) if ct == torch.float32 else None
        if ref is not None:
            assert float((got[b, 0] - ref[0]).abs().max() / ref.abs().max()) < 1e-4


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("ct", [None] + CODES)
def test_speculative_greedy_is_greedy(dev, ct):
    lm, small = lm_of(dev), lm_of(dev, seed=5, layers=1)
    prompt = prompt_of(3, 12, 53, dev)
    for drafter, drafts in ((small, 3), (lm, 4), (small, 1), (lm_of(dev, seed=7), 9)):
        for new in (1, 2, 17):
            want = lm.generate_greedy(prompt, new, cache_dtype=ct)
            assert torch.equal(lm.generate_speculative(prompt, drafter, new, drafts, temperature=0, cache_dtype=ct), want)


@pytest.mark.parametrize("dev", DEVICES)
def test_sequences_of_a_batch_accept_different_numbers(dev):
    """Half the sequences' drafts are right, the others' mostly not: those that are done wait for the others."""
    lm = lm_of(dev)
    prompt = prompt_of(6, 8, 53, dev)
    want = lm.generate_greedy(prompt, 30)

    class Half(MultiscreenLM):
        def tree_step(self, tokens, caches, lengths, parents=None, rws=None):
            logits, kvs = lm.tree_step(tokens, caches, lengths, parents, rws)
            logits[3:] = logits[3:].roll(1, -1)
            return logits, kvs

        def new_cache(self, *a):
            return lm.new_cache(*a)

        def prefill(self, ids, caches):
            return lm.prefill(ids, caches)

    half = Half(53, 64, 4, 2, max_seq_len=256).to(dev)
    assert torch.equal(lm.generate_speculative(prompt, half, 30, 7, temperature=0), want)


@pytest.mark.parametrize("dev", DEVICES)
def test_speculative_sampling(dev):
    lm, small = lm_of(dev), lm_of(dev, seed=5, layers=1)
    prompt = prompt_of(2, 9, 53, dev)
    torch.manual_seed(3)
    a = lm.generate_speculative(prompt, small, 20, 4, 0.8, 10)
    torch.manual_seed(3)
    b = lm.generate_speculative(prompt, small, 20, 4, 0.8, 10)
    assert a.shape == (2, 29) and torch.equal(a, b) and torch.equal(a[:, :9], prompt)
    assert int(a.min()) >= 0 and int(a.max()) < 53
    # every sampled token is one of its row's ten likeliest
    logits = lm(a)["logits"][:, 8:-1]
    rank = (logits > logits.gather(2, a[:, 9:].unsqueeze(-1))).sum(-1)
    assert int(rank.max()) < 10
    assert torch.equal(lm.generate_speculative(prompt, small, 0), prompt)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("ct", CODES)
def test_generate_over_codes(dev, ct):
    lm = lm_of(dev)
    prompt = prompt_of(2, 10, 53, dev)
    greedy = lm.generate_greedy(prompt, 12, cache_dtype=ct)
    assert torch.equal(lm.generate(prompt, 12, top_k=1, cache_dtype=ct), greedy)
    caches = lm.new_cache(2, 22, ct, dev)
    assert caches[0].k.dtype == ct
    x = lm.embed(prompt)
    # the cache's bytes: codes and a scale for each row of 16
    assert caches[0]._k.numel() * caches[0]._k.element_size() + caches[0].k_scale.numel() * 4 == 2 * 22 * 4 * (16 + 4)


def test_refusals():
    lm, other = lm_of("cpu"), lm_of("cpu", vocab=54)
    prompt = prompt_of(1, 4, 53, "cpu")
    for kw in (dict(num_drafts=0), dict(num_drafts=64)):
        with pytest.raises(ValueError):
            lm.generate_speculative(prompt, lm, 5, **kw)
    with pytest.raises(ValueError):
        lm.generate_speculative(prompt, other, 5)
    with pytest.raises(IndexError):
        lm.generate_speculative(prompt, lm, 300)
    attn = ScreeningAttention(32, 2, causal=False)
    with pytest.raises(RuntimeError):
        attn.tree_step(torch.zeros(1, 2, 32), KVCache(1, 8, 2, 16, torch.float32, "cpu"), torch.tensor([0]))
    cache = KVCache(1, 8, 2, 16, torch.int8, "cpu")
    with pytest.raises(IndexError):
        cache.store(torch.zeros(1, 9, 2, 16), torch.zeros(1, 9, 2, 16), 0)
    with pytest.raises(IndexError):
        cache.read(0, 9, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ct", CODES)
def test_replayed_decode_over_codes(dtype, ct):
    """GraphDecoder's replays over an 8-bit cache against eager steps, with eager work between them."""
    from multiscreen.model import GraphDecoder
    lm = lm_of("cuda", dtype)
    B, T, steps = 3, 15, 10
    prompt = prompt_of(B, T, 53, "cuda")
    eager, held = (lm.new_cache(B, T + steps + 1, ct, "cuda") for _ in range(2))
    tok = lm.prefill(prompt, eager).argmax(-1, keepdim=True)
    lm.prefill(prompt, held)
    dec = GraphDecoder(lm, held, tok, T, steps)
    for s in range(steps):
        ref = lm.decode_step(tok, eager, T + s)
        tok = ref.argmax(-1, keepdim=True)
        dec.step()
        torch.cuda.synchronize()
        assert torch.equal(dec.logits, ref) and torch.equal(dec.token, tok), s
    assert torch.equal(held[1].k.view(torch.uint8), eager[1].k.view(torch.uint8))


@pytest.mark.gpu
def test_under_autocast():
    """fp32 weights under fp16 autocast: the caches take fp16 rows, or codes of them."""
    lm = lm_of("cuda")
    prompt = prompt_of(2, 12, 53, "cuda")
    with torch.autocast("cuda", dtype=torch.float16):
        for ct in [None] + CODES:
            out = lm.generate(prompt, 6, top_k=1, cache_dtype=ct)
            spec = lm.generate_speculative(prompt, lm, 6, 3, 0.7, cache_dtype=ct)
            assert out.shape == spec.shape == (2, 18)


def test_packed_arguments_have_the_headers_fields():
    """Every field of the argument structs is 8 bytes wide, so a count of the header's fields is the packed size."""
    import re
    from conftest import ROOT
    from multiscreen import _native
    text = re.sub(r"/\*.*?\*/", "", open(f"{ROOT}/include/msa.h").read(), flags=re.S)
    for name, pack, values in (("msa_cache_args", _native.pack_cache_args, [0] * 37),
                               ("msa_tree_args", _native.pack_tree_args, [0] * 37 + [1.0]),
                               ("msa_verify_args", _native.pack_verify_args, [0] * 19)):
        body = re.search(r"typedef struct \{([^{}]*)\} " + name, text).group(1)
        fields = sum(len(part.split(",")) * (4 if part.split()[0] == "msa_tensor" else 1)
                     for part in body.split(";") if part.strip())
        assert len(pack(*values)) == 8 * fields, name
