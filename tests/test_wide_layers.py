"""The wide layers on the CPU: dense forms of the vocabulary losses and of the gated feed-forward, the model's methods
over them, and what the C entry points refuse."""

import math

import pytest
import torch
import torch.nn.functional as F

from multiscreen import GatedFFN, MultiscreenBlock, MultiscreenDecoderLayer, MultiscreenLM, _native
from multiscreen import _dense


def _lm(**kw):
    torch.manual_seed(0)
    return MultiscreenLM(61, d_model=32, num_heads=2, num_layers=2, max_seq_len=64, **kw)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy_is_torchs(reduction):
    torch.manual_seed(1)
    x, w = torch.randn(3, 7, 16), torch.randn(29, 16)
    y = torch.randint(0, 29, (3, 7))
    y[1, 2:] = -100
    got = _dense.linear_cross_entropy_dense(x, w, y, -100, reduction)
    want = F.cross_entropy((x @ w.T).view(-1, 29), y.flatten(), ignore_index=-100, reduction=reduction)
    torch.testing.assert_close(got.flatten(), want.flatten())
    with pytest.raises(IndexError):
        _dense.linear_cross_entropy_dense(x, w, y.clamp(max=28) + 1, -100)
    with pytest.raises(ValueError):
        _dense.linear_cross_entropy_dense(x, w, y, -100, "batch")


def test_a_mean_of_no_rows_has_gradients_of_zeros():
    x, w = torch.randn(5, 8, requires_grad=True), torch.randn(11, 8, requires_grad=True)
    loss = _dense.linear_cross_entropy_dense(x, w, torch.full((5,), -100))
    loss.backward()
    assert bool(torch.isnan(loss)) and not x.grad.any() and not w.grad.any()


def test_distillation_over_the_whole_vocabulary_is_kl():
    torch.manual_seed(2)
    x, w, t = torch.randn(9, 16), torch.randn(13, 16), torch.randn(9, 13)
    ids = torch.arange(13).expand(9, 13)
    for T in (1.0, 2.5):
        got = _dense.linear_distillation_dense(x, w, t, ids, T)
        want = T * T * F.kl_div(torch.log_softmax(x @ w.T / T, -1), torch.softmax(t / T, -1), reduction="batchmean")
        torch.testing.assert_close(got, want)


def test_distillation_entries_that_are_none():
    torch.manual_seed(3)
    x, w, t = torch.randn(6, 16), torch.randn(13, 16), torch.randn(6, 4)
    ids = torch.randint(0, 13, (6, 4))
    ids[0] = -1
    t[1] = -math.inf
    ids[2, 1], t[3, 2] = -1, -math.inf
    x[0] = math.nan
    x.requires_grad_()
    rows = _dense.linear_distillation_dense(x, w, t, ids, 1.0, "none")
    assert rows[0] == 0 and rows[1] == 0 and bool(torch.isfinite(rows).all())
    keep = [0, 2, 3]
    torch.testing.assert_close(rows[2], _dense.linear_distillation_dense(x[2:3], w, t[2:3, keep], ids[2:3, keep], 1.0))
    rows.sum().backward()
    assert not x.grad[:2].any() and bool(torch.isfinite(x.grad).all())
    ids[4, 0] = 13
    with pytest.raises(IndexError):
        _dense.linear_distillation_dense(x, w, t, ids)
    with pytest.raises(ValueError):
        _dense.linear_distillation_dense(x, w, t, ids, 0.0)


def test_gated_dense():
    torch.manual_seed(4)
    x, g, u = torch.randn(5, 8), torch.randn(12, 8), torch.randn(12, 8)
    torch.testing.assert_close(_dense.gated_linear_dense(x, g, u), F.silu(x @ g.T) * (x @ u.T))
    torch.testing.assert_close(_dense.gated_linear_dense(x, g, u, "gelu"), F.gelu(x @ g.T) * (x @ u.T))
    with pytest.raises(ValueError):
        _dense.gated_linear_dense(x, g, u, "relu")


@pytest.mark.parametrize("ffn", ["gelu", "swiglu", "geglu"])
def test_loss_is_forwards(ffn):
    lm = _lm(ffn=ffn)
    ids, y = torch.randint(0, 61, (2, 9)), torch.randint(0, 61, (2, 9))
    y[1, 6:] = -100
    pad = torch.zeros(2, 9, dtype=torch.bool)
    pad[1, 6:] = True
    want = lm(ids, key_padding_mask=pad, labels=y)
    got = lm.loss(ids, y, pad)
    torch.testing.assert_close(got, want["loss"])
    a = torch.autograd.grad(got, list(lm.parameters()), allow_unused=True)
    b = torch.autograd.grad(want["loss"], list(lm.parameters()), allow_unused=True)
    for p, q in zip(a, b):
        assert (p is None) == (q is None)
        if p is not None:
            torch.testing.assert_close(p, q, rtol=1e-4, atol=1e-6)
    scores = lm.loss(ids, y, pad, reduction="none")
    assert scores.shape == (2, 9) and not scores[1, 6:].any()


def test_distilling_a_draft():
    teacher, draft = _lm(), _lm(ffn="swiglu")
    ids = torch.randint(0, 61, (2, 9))
    t, at = teacher.top_logits(ids, 5)
    want, where = teacher(ids)["logits"].topk(5, -1)
    assert torch.equal(t, want) and torch.equal(at, where) and not t.requires_grad
    loss = draft.distillation_loss(ids, t, at, 2.0)
    assert float(loss.detach()) > 0
    loss.backward()
    assert all(bool(torch.isfinite(p.grad).all()) for p in draft.parameters() if p.grad is not None)
    # a model has no divergence from itself once the entries are the whole vocabulary
    t, at = teacher.top_logits(ids, 61)
    assert abs(float(teacher.distillation_loss(ids, t, at).detach())) < 1e-6
    empty = teacher.top_logits(ids[:0], 3)
    assert empty[0].shape == empty[1].shape == (0, 9, 3)


def test_feed_forward_kinds():
    block = MultiscreenBlock(32, 2, ffn="geglu")
    assert isinstance(block.ffn, GatedFFN) and block.ffn.gate.weight.shape == (128, 32)
    assert isinstance(MultiscreenDecoderLayer(32, 2, 48, ffn="swiglu").ffn, GatedFFN)
    with pytest.raises(ValueError):
        MultiscreenBlock(32, 2, ffn="relu")
    x = torch.randn(2, 5, 32)
    f = block.ffn
    torch.testing.assert_close(f(x), F.linear(F.gelu(f.gate(x)) * f.up(x), f.down.weight))
    names = set(MultiscreenBlock(32, 2).state_dict())
    assert "ffn.0.weight" in names and "ffn.3.weight" in names  # the reference's, as they were


def test_generation_with_gated_feed_forward():
    lm = _lm(ffn="swiglu").eval()
    ids = torch.randint(0, 61, (2, 5))
    out = lm.generate_greedy(ids, 6)
    for n in range(5, 11):  # each token is the full forward's
        with torch.no_grad():
            assert torch.equal(lm(out[:, :n])["logits"][:, -1].argmax(-1), out[:, n])


@pytest.mark.parametrize("place", [0, 1])
def test_forward_mode_derivatives_are_refused_or_right(place):
    # the kernels have none: refused before any check of devices, also where no weight requires a gradient
    import torch.autograd.forward_ad as ad

    from multiscreen import ops
    torch.manual_seed(5)
    x, w, y = torch.randn(6, 8), torch.randn(11, 8), torch.randint(0, 11, (6,))
    t, ids = torch.randn(6, 3), torch.randint(0, 11, (6, 3))
    with ad.dual_level():
        args = [x, w]
        args[place] = ad.make_dual(args[place], torch.randn(args[place].shape))
        for call in (lambda: ops.linear_cross_entropy(*args, y), lambda: ops.linear_distillation(*args, t, ids),
                     lambda: ops.linear_distillation(x, w, ad.make_dual(t, t), ids), lambda: ops.gated_linear(*args, w),
                     lambda: ops.gated_linear(x, w, ad.make_dual(w, w))):
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        # the CPU's forms have them
        got = ad.unpack_dual(_dense.linear_cross_entropy_dense(*args, y)).tangent
        want = ad.unpack_dual(F.cross_entropy(args[0] @ args[1].T, y)).tangent
        torch.testing.assert_close(got, want)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_teacher_logits_at_the_ends_of_the_type(dtype, device):
    # a finite logit is an entry whatever the temperature makes of it
    from multiscreen import ops
    fn = ops.linear_distillation if device == "cuda" else _dense.linear_distillation_dense
    torch.manual_seed(6)
    x, w, ids = torch.randn(5, 32, device=device), torch.randn(40, 32, device=device), torch.arange(10, 14, device=device).repeat(5, 1)
    t = torch.randn(5, 4, device=device).to(dtype)
    info = torch.finfo(dtype)
    t[1] = info.min                       # all as low as can be: as equal logits
    t[2, 1:] = info.min                   # all on the first
    t[3] = info.max
    t[4] = -math.inf                      # none
    log_q = torch.log_softmax(x.double() @ w.double().T / 0.5, -1)[:, 10:14]
    p = torch.softmax(t.double() / 0.5, -1)
    p[1] = p[3] = 0.25
    want = 0.25 * (torch.special.xlogy(p, p) - p * log_q).sum(-1)
    want[4] = 0
    got = fn(x, w, t, ids, 0.5, reduction="none")
    torch.testing.assert_close(got.double(), want, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(fn(x, w, t, ids, 0.5).double(), want.sum() / 4, rtol=1e-5, atol=1e-5)


class _Adapted(torch.nn.Module):
    """A low-rank adapter around a Linear, with the weight that the Linear has."""

    def __init__(self, base, scale=0.5):
        super().__init__()
        self.base = base
        self.a = torch.nn.Parameter(scale * torch.randn(3, base.in_features) / math.sqrt(base.in_features))
        self.b = torch.nn.Parameter(scale * torch.randn(base.out_features, 3))

    @property
    def weight(self):
        return self.base.weight

    def forward(self, x):
        return self.base(x) + x @ self.a.T @ self.b.T


def _adapt(kind, owner, name):
    m = getattr(owner, name)
    if kind == "adapter":
        setattr(owner, name, _Adapted(m))
    elif kind == "bias":
        new = torch.nn.Linear(m.in_features, m.out_features)
        new.weight = m.weight
        setattr(owner, name, new)
    elif kind == "hook":
        m.register_forward_hook(lambda mod, args, out: out * 0.5)
    elif kind == "pre-hook":
        m.register_forward_pre_hook(lambda mod, args: (args[0] * 0.5,))
    elif kind == "own forward":
        m.forward = lambda x: 0.5 * F.linear(x, m.weight)


KINDS = ["adapter", "bias", "hook", "pre-hook", "own forward"]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("ffn", ["swiglu", "geglu"])
def test_an_adapted_feed_forward_is_called(kind, ffn, device):
    for name in ("gate", "up"):
        block = MultiscreenBlock(32, 2, 40, ffn=ffn)
        f = block.ffn.to(device)
        _adapt(kind, f, name)
        f.to(device)
        x = torch.randn(2, 5, 32, device=device)
        want = f.down((F.silu if ffn == "swiglu" else F.gelu)(f.gate(x)) * f.up(x))
        torch.testing.assert_close(f(x), want, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("kind", KINDS)
def test_an_adapted_head_is_called(kind, device):
    lm = _lm().to(device)
    _adapt(kind, lm, "lm_head")
    lm.to(device)
    ids, y = torch.randint(0, 61, (2, 9), device=device), torch.randint(0, 61, (2, 9), device=device)
    y[1, 6:] = -100
    want = lm(ids, labels=y)
    torch.testing.assert_close(lm.loss(ids, y), want["loss"], rtol=1e-5, atol=1e-6)
    assert not lm.loss(ids, y, reduction="none")[1, 6:].any()
    t, at = lm.top_logits(ids, 61)  # of its own logits a model has no divergence
    assert abs(float(lm.distillation_loss(ids, t, at).detach())) < 1e-6
    for got, loss in ((lm.loss(ids, y), want["loss"]),):
        a, b = (torch.autograd.grad(v, list(lm.parameters()), allow_unused=True) for v in (got, loss))
        for p, q in zip(a, b):
            assert (p is None) == (q is None)
            if p is not None:
                torch.testing.assert_close(p, q, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_hooks_of_the_backward_pass_see_it(device):
    lm = _lm(ffn="swiglu").to(device)
    seen = []
    for m in (lm.lm_head, lm.blocks[0].ffn.gate, lm.blocks[1].ffn.up):
        m.register_full_backward_hook(lambda mod, gi, go: seen.append(mod))
    ids = torch.randint(0, 61, (2, 9), device=device)
    lm.loss(ids, ids).backward()
    assert len(seen) == 3


# ---------------------------------------------------------------------------
# The C entry points refuse on the host, before any GPU call.
# ---------------------------------------------------------------------------
def _head(fn="msa_head_fwd", **kw):
    L = _native.lib()
    a = dict(x=1 << 20, x_ld=64, w=1 << 21, w_ld=64, ids=1 << 22, ids_ld=1, t=0, t_ld=0, state=1 << 23, sb=1 << 30, loss=1 << 24,
             dloss=1 << 24, dx=1 << 25, dw=1 << 26, ws=1 << 27, wsb=1 << 40, N=10, d=64, V=50, K=1, dt=1, tdt=0, red=1, ignore=-100, T=1.0)
    a.update(kw)
    packed = _native.pack_head_args(*[a[k] for k in ("x", "x_ld", "w", "w_ld", "ids", "ids_ld", "t", "t_ld", "state", "sb", "loss", "dloss",
                                                     "dx", "dw", "ws", "wsb", "N", "d", "V", "K", "dt", "tdt", "red", "ignore", "T")])
    if fn == "bytes":
        return L.msa_head_workspace_bytes(packed, 1), ""
    return getattr(L, fn)(packed, None), L.msa_last_error().decode()


@pytest.mark.parametrize("fn", ["msa_head_fwd", "msa_head_bwd"])
@pytest.mark.parametrize("kw,code,msg", [
    (dict(dt=3), 1, "dtype"), (dict(N=-1), 1, "rows"), (dict(N=(1 << 23) + 1), 1, "rows"), (dict(d=0), 1, "columns"),
    (dict(d=65537), 1, "columns"), (dict(V=0), 1, "weight rows"), (dict(V=(1 << 23) + 1), 1, "weight rows"),
    (dict(N=1 << 23, V=1 << 20), 1, "too many"), (dict(N=1 << 23, d=65536, V=100), 1, "too many"), (dict(K=2), 1, "K must be"),
    (dict(t=1 << 22, t_ld=300, K=257, ids_ld=300), 1, "K must be"), (dict(t=1 << 22, tdt=3), 1, "teacher_dtype"),
    (dict(red=3), 1, "reduction"), (dict(T=0.0), 1, "temperature"),
    (dict(T=math.nan), 1, "temperature"), (dict(T=math.inf), 1, "temperature"), (dict(x=0), 1, "hidden is null"), (dict(x=(1 << 20) + 1), 1, "hidden"),
    (dict(w=0), 1, "weight is null"), (dict(ids=0), 1, "ids is null"), (dict(x_ld=-64), 1, "stride"),
    (dict(sb=10), 2, "state"), (dict(ws=0), 2, "workspace"), (dict(wsb=10), 2, "workspace"), (dict(ws=(1 << 27) + 8), 1, "aligned"),
    (dict(loss=0, dloss=0), 1, "null"), (dict(dx=(1 << 25) + 2), 1, "aligned")])
def test_head_refusals(fn, kw, code, msg):
    rc, said = _head(fn, **kw)
    assert rc == code and msg in said


def test_head_backward_needs_the_forwards_state():
    rc, said = _head("msa_head_bwd", state=0)
    assert rc == 2 and "state" in said


def test_head_sizes():
    # operand rows 128 x 64 and the state's rows, at the least
    assert _head("bytes")[0] >= 128 * 64 * 2 and _head("bytes", V=0)[0] == 0
    assert _native.lib().msa_head_state_bytes(10, 4) >= 10 * 4 * 4 and _native.lib().msa_head_state_bytes(10, 257) == 0
    # the gradient of the logits is there in pieces of at most 1 GB: 131072 rows of 50257 logits would be 13.2 GB
    assert _head("bytes", N=131072, V=50257, d=64)[0] < 1300 << 20


def _gated(fn="msa_gated_fwd", **kw):
    L = _native.lib()
    a = dict(x=1 << 20, x_ld=64, g=1 << 21, g_ld=64, u=1 << 22, u_ld=64, h=1 << 23, dh=1 << 24, dh_ld=50, dx=1 << 25, dg=1 << 26, du=1 << 27,
             ws=1 << 28, wsb=1 << 40, N=10, d=64, F=50, dt=1, act=0)
    a.update(kw)
    packed = _native.pack_gated_args(*[a[k] for k in ("x", "x_ld", "g", "g_ld", "u", "u_ld", "h", "dh", "dh_ld", "dx", "dg", "du", "ws", "wsb",
                                                      "N", "d", "F", "dt", "act")])
    return getattr(L, fn)(packed, None), L.msa_last_error().decode()


@pytest.mark.parametrize("fn", ["msa_gated_fwd", "msa_gated_bwd"])
@pytest.mark.parametrize("kw,code,msg", [
    (dict(dt=4), 1, "dtype"), (dict(N=-1), 1, "rows"), (dict(d=0), 1, "columns"), (dict(F=0), 1, "weight rows"), (dict(F=(1 << 23) + 1), 1, "weight rows"),
    (dict(N=1 << 23, F=1 << 20), 1, "too many"), (dict(act=2), 1, "act"), (dict(x=0), 1, "x is null"), (dict(g=0), 1, "gate is null"),
    (dict(u=3), 1, "up is not aligned"), (dict(x_ld=-1), 1, "stride"), (dict(wsb=10, dt=0), 2, "workspace"), (dict(ws=8), 1, "aligned"),
    (dict(dx=8), 1, "aligned")])
def test_gated_refusals(fn, kw, code, msg):
    rc, said = _gated(fn, **kw)
    assert rc == code and msg in said


def test_gated_refusals_of_one_direction():
    rc, said = _gated("msa_gated_fwd", h=0)
    assert rc == 1 and "h is null" in said
    rc, said = _gated("msa_gated_bwd", dh=0)
    assert rc == 1 and "dh is null" in said
    rc, said = _gated("msa_gated_bwd", dg=0)
    assert rc == 1 and "together" in said


def test_structs_match_the_header():
    import os
    import re

    from conftest import ROOT
    text = open(os.path.join(ROOT, "include", "msa.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, pack, values in (("msa_head_args", _native.pack_head_args, [0] * 24 + [1.0]),
                               ("msa_gated_args", _native.pack_gated_args, [0] * 19)):
        body = re.search(r"typedef struct \{([^}]*)\} " + name, text).group(1)
        fields = [f for line in body.split(";") for f in line.split(",") if f.strip()]
        assert len(pack(*values)) == 8 * len(fields) == 8 * len(values)
    assert f"MSA_HEAD_MAX_K {_native.HEAD_MAX_K}" in text


@pytest.mark.gpu
def test_autocast_leaves_float64_alone():
    # as torch's own: refused with a type of its own, not narrowed to 8 bits
    from multiscreen import ops
    x, w, y = torch.randn(4, 32, device="cuda"), torch.randn(9, 32, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        for call in (lambda: ops.linear_cross_entropy(x.double(), w.double(), y), lambda: ops.gated_linear(x.double(), w.double(), w.double()),
                     lambda: ops.linear_distillation(x.double(), w, x[:, :2], y.unsqueeze(1).repeat(1, 2))):
            with pytest.raises(TypeError):
                call()
        assert ops.linear_cross_entropy(x, w.half(), y).dtype == torch.float32
