"""The wide layers where they are used together: a MultiscreenLM with gated feed-forwards trained by loss() and by
distillation_loss() from a larger one, then decoding, on the GPU."""

import pytest
import torch

from multiscreen import MultiscreenBlock, MultiscreenDecoderLayer, MultiscreenLM

pytestmark = pytest.mark.gpu
V = 500


def _lm(seed=0, **kw):
    torch.manual_seed(seed)
    return MultiscreenLM(V, **{"d_model": 64, "num_heads": 2, "num_layers": 2, "max_seq_len": 128, **kw})


def _close(a, b, tol):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert float((a - b).norm()) <= tol * float(b.norm()) + 1e-12, float((a - b).norm() / b.norm())


@pytest.mark.parametrize("ffn", ["gelu", "swiglu", "geglu"])
def test_loss_and_gradients_are_the_cpus(ffn):
    cpu = _lm(ffn=ffn)
    gpu = _lm(ffn=ffn).cuda()
    ids, y = torch.randint(0, V, (3, 40)), torch.randint(0, V, (3, 40))
    y[1, 25:] = -100
    pad = torch.zeros(3, 40, dtype=torch.bool)
    pad[1, 25:] = True
    a = cpu.loss(ids, y, pad)
    b = gpu.loss(ids.cuda(), y.cuda(), pad.cuda())
    _close(b, a, 1e-5)
    _close(gpu(ids.cuda(), pad.cuda(), y.cuda())["loss"], b, 1e-5)
    a.backward()
    b.backward()
    for (name, p), q in zip(cpu.named_parameters(), gpu.parameters()):
        if p.grad is not None and float(p.grad.norm()) > 0:
            _close(q.grad, p.grad, 2e-4)  # fp32 through two layers of fused attention


def test_distillation_step_and_decoding():
    teacher, draft = _lm(1, d_model=128, num_heads=4).cuda().bfloat16(), _lm(2, ffn="swiglu").cuda().bfloat16()
    ids = torch.randint(0, V, (4, 50), device="cuda")
    t, at = teacher.top_logits(ids, 16)
    before = [p.detach().clone() for p in draft.parameters()]
    opt = torch.optim.SGD(draft.parameters(), lr=0.1)
    loss = draft.distillation_loss(ids, t, at, 2.0) + draft.loss(ids, ids)
    opt.zero_grad()
    loss.backward()
    opt.step()
    assert bool(torch.isfinite(loss)) and any(not torch.equal(p, q) for p, q in zip(before, draft.parameters()))
    rows = draft.distillation_loss(ids, t, at, 2.0, reduction="none")
    assert rows.shape == (4, 50) and rows.dtype == torch.float32
    out = teacher.generate_speculative(ids[:, :10], draft, 12, num_drafts=3, temperature=0)
    assert out.shape == (4, 22)
    greedy = draft.generate_greedy(ids[:, :10], 8)
    assert greedy.shape == (4, 18)


def test_scores_of_single_tokens_are_the_full_forwards():
    lm = _lm(3, ffn="geglu").cuda().eval()
    ids = torch.randint(0, V, (5, 20), device="cuda")
    with torch.no_grad():
        scores = lm.loss(ids, ids.roll(-1, 1), reduction="none")
        logp = torch.log_softmax(lm(ids)["logits"].double(), -1).gather(-1, ids.roll(-1, 1).unsqueeze(-1)).squeeze(-1)
    _close(scores, -logp, 1e-5)


def test_cached_decoding_with_gated_feed_forward():
    lm = _lm(4, ffn="swiglu").cuda().eval()
    ids = torch.randint(0, V, (2, 12), device="cuda")
    out = lm.generate_greedy(ids, 10)
    again = lm.generate(ids, 10, top_k=1)
    assert out.shape == again.shape == (2, 22)
    with torch.no_grad():
        caches = lm.new_cache(2, 40, torch.float32, "cuda")
        lm.prefill(out[:, :12], caches)
        step = lm.decode_step(out[:, 12:13], caches, 12)
        full = lm(out[:, :13])["logits"][:, -1]
        nodes, _ = lm.tree_step(out[:, 12:15], lm_caches(lm, out[:, :12]), torch.tensor([12], device="cuda"))
        whole = lm(out[:, :15])["logits"][:, 12:]
    _close(step, full, 1e-4)
    _close(nodes, whole, 1e-4)


def lm_caches(lm, prompt):
    caches = lm.new_cache(prompt.shape[0], 40, torch.float32, "cuda")
    lm.prefill(prompt, caches)
    return caches


def test_training_under_autocast_and_dropout():
    lm = _lm(5, ffn="swiglu", dropout=0.1).cuda()
    ids = torch.randint(0, V, (2, 30), device="cuda")
    with torch.autocast("cuda", dtype=torch.float16):
        loss = lm.loss(ids, ids)
    (loss * 1024).backward()
    assert loss.dtype == torch.float32
    assert all(p.grad is None or bool(torch.isfinite(p.grad).all()) for p in lm.parameters())
    assert lm.blocks[0].ffn.gate.weight.grad is not None and lm.token_emb.weight.grad.dtype == torch.float32


def test_blocks_and_decoder_layers():
    torch.manual_seed(6)
    x = torch.randn(2, 33, 64)
    for make in (lambda: MultiscreenBlock(64, 2, 100, ffn="swiglu"), lambda: MultiscreenBlock(64, 2, ffn="geglu")):
        block = make()
        _close(block.cuda()(x.cuda()), block.cpu()(x), 1e-4)
    layer = MultiscreenDecoderLayer(64, 2, ffn="geglu")
    _close(layer.cuda()(x.cuda(), x.cuda()), layer.cpu()(x, x), 1e-4)
