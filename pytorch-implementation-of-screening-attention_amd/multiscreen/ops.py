"""Operator boundary of the fused Screening Attention core on MI355X.

`screening_core(q, k, v, r, w, causal, eps, key_padding_mask)` takes the raw
per-head projections as (B, T, H, D) views -- the `proj(x).view(B,T,H,D)`
tensors of multiscreen/attention.py:150-153, before their transpose -- and
returns TanhNorm(sum_j alpha_ij m_ij v^_j) as a (B, Tq, H, D) tensor, i.e. the
whole span attention.py:155-196 (normalise, similarity, trim-and-square,
softmask, key padding, aggregation, TanhNorm) as one HIP forward and one HIP
backward through libmsa.so.  The backward also returns the gradients of the
per-head r and w that the reference fused path drops
(attention_triton.py:44).

It is the counterpart of the reference's `_ScreeningFunc`
(attention_triton.py:24-48), whose inputs are already normalised and whose
output is pre-TanhNorm; here normalisation and TanhNorm are inside the
kernels, so their backward is too.

GPU tensors only: a CPU tensor, or a missing libmsa.so, raises.
"""

import torch

from . import _native

_DTYPES = {torch.float32: _native.MSA_F32, torch.bfloat16: _native.MSA_BF16, torch.float16: _native.MSA_F16}


def _stream_ptr(device):
    return torch.cuda.current_stream(device).cuda_stream


def _as_bthd(x, name, esize):
    """Returns x (B,T,H,D) with unit D stride and 16-byte-friendly strides."""
    if x.dim() != 4:
        raise ValueError(f"{name} must be 4-D (B, T, H, D), got {tuple(x.shape)}")
    mult = 16 // esize
    ok = (x.stride(3) == 1 and all(s % mult == 0 for s in x.stride()[:3])
          and x.data_ptr() % 16 == 0)
    return x if ok else x.contiguous()


def _args_bthd(x):
    return (x.data_ptr(), x.stride(0), x.stride(1), x.stride(2))


def tile_bits_words(B, H, Tq, Tk):
    return int(_native.lib().msa_tile_bits_words(B, H, Tq, Tk))


def _kpm_u8(key_padding_mask, B, Tk, dev):
    if key_padding_mask is None:
        return None
    if key_padding_mask.shape != (B, Tk):
        raise ValueError(f"key_padding_mask must have shape ({B}, {Tk})")
    return key_padding_mask.to(device=dev, dtype=torch.uint8).contiguous()


def _dropout_args(dropout_p, seed):
    p = float(dropout_p)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout probability must be in [0, 1), got {p}")
    return p, int(seed) & (2 ** 64 - 1)


def fwd_raw(q, k, v, r, w, causal=True, eps=1e-8, key_padding_mask=None, dropout_p=0.0, seed=0):
    """One msa_fwd call.  Returns (y, hnorm, tile_bits).

    q (B,Tq,H,D), k/v (B,Tk,H,D) in float32, bfloat16 or float16 on one GPU; r, w (H,).
    dropout_p / seed: attention dropout with the counter-based keep mask that
    include/msa.h defines (p = 0: none).
    """
    L = _native.lib()
    if not q.is_cuda:
        raise RuntimeError("screening_core runs on the GPU only (got a CPU tensor)")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q/k/v must share dtype float32, bfloat16 or float16, got {q.dtype}, {k.dtype}, {v.dtype}")
    dt = _DTYPES[q.dtype]
    es = q.element_size()
    q, k, v = _as_bthd(q, "q", es), _as_bthd(k, "k", es), _as_bthd(v, "v", es)
    B, Tq, H, D = q.shape
    Tk = k.shape[1]
    if k.shape != (B, Tk, H, D) or v.shape != k.shape:
        raise ValueError(f"k/v shape {tuple(k.shape)}/{tuple(v.shape)} do not match q {tuple(q.shape)}")
    if r.shape != (H,) or w.shape != (H,):
        raise ValueError(f"r and w must have shape ({H},)")
    dev = q.device
    r32 = r.detach().to(device=dev, dtype=torch.float32).contiguous()
    w32 = w.detach().to(device=dev, dtype=torch.float32).contiguous()
    kpm = _kpm_u8(key_padding_mask, B, Tk, dev)
    p, seed = _dropout_args(dropout_p, seed)
    y = torch.empty((B, Tq, H, D), dtype=q.dtype, device=dev)
    hnorm = torch.empty((B, H, Tq), dtype=torch.float32, device=dev)
    nwords = tile_bits_words(B, H, Tq, Tk)
    bits = torch.empty((max(nwords, 1),), dtype=torch.int32, device=dev)
    wsb = int(L.msa_fwd_workspace_bytes(B, H, Tq, Tk, D, dt))
    ws = torch.empty((max(wsb, 16),), dtype=torch.uint8, device=dev)
    rc = L.msa_fwd(*_args_bthd(q), *_args_bthd(k), *_args_bthd(v),
                   B, H, Tq, Tk, D, dt, r32.data_ptr(), w32.data_ptr(),
                   kpm.data_ptr() if kpm is not None else None, int(bool(causal)), float(eps), p, seed,
                   y.data_ptr(), hnorm.data_ptr(), bits.data_ptr(), nwords,
                   ws.data_ptr(), wsb, _stream_ptr(dev))
    _native.check(rc, "msa_fwd")
    return y, hnorm, bits


def bwd_raw(q, k, v, r, w, causal, eps, y, hnorm, bits, dy, key_padding_mask=None, dropout_p=0.0, seed=0):
    """One msa_bwd call.  Returns (dq, dk, dv, dr, dw); dq/dk/dv in (B,T,H,D).
    dropout_p / seed must be the forward's."""
    L = _native.lib()
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q/k/v must share dtype float32, bfloat16 or float16, got {q.dtype}, {k.dtype}, {v.dtype}")
    dt = _DTYPES[q.dtype]
    es = q.element_size()
    q, k, v = _as_bthd(q, "q", es), _as_bthd(k, "k", es), _as_bthd(v, "v", es)
    B, Tq, H, D = q.shape
    Tk = k.shape[1]
    dev = q.device
    dq = torch.empty((B, Tq, H, D), dtype=q.dtype, device=dev)
    dk = torch.empty((B, Tk, H, D), dtype=q.dtype, device=dev)
    dv = torch.empty((B, Tk, H, D), dtype=q.dtype, device=dev)
    dr = torch.empty((H,), dtype=torch.float32, device=dev)
    dw = torch.empty((H,), dtype=torch.float32, device=dev)
    if B == 0 or Tq == 0 or Tk == 0:
        return dq.zero_(), dk.zero_(), dv.zero_(), dr.zero_(), dw.zero_()
    dy = dy.to(q.dtype).contiguous()
    r32 = r.detach().to(device=dev, dtype=torch.float32).contiguous()
    w32 = w.detach().to(device=dev, dtype=torch.float32).contiguous()
    kpm = _kpm_u8(key_padding_mask, B, Tk, dev)
    p, seed = _dropout_args(dropout_p, seed)
    wsb = int(L.msa_bwd_workspace_bytes(B, H, Tq, Tk, D, dt))
    ws = torch.empty((max(wsb, 16),), dtype=torch.uint8, device=dev)
    rc = L.msa_bwd(*_args_bthd(q), *_args_bthd(k), *_args_bthd(v),
                   B, H, Tq, Tk, D, dt, r32.data_ptr(), w32.data_ptr(),
                   kpm.data_ptr() if kpm is not None else None, int(bool(causal)), float(eps), p, seed,
                   y.data_ptr(), hnorm.data_ptr(), dy.data_ptr(), bits.data_ptr(),
                   tile_bits_words(B, H, Tq, Tk),
                   dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dr.data_ptr(), dw.data_ptr(),
                   ws.data_ptr(), wsb, _stream_ptr(dev))
    _native.check(rc, "msa_bwd")
    return dq, dk, dv, dr, dw


class ScreeningCoreFunction(torch.autograd.Function):
    """Autograd wrapper: forward = msa_fwd, backward = msa_bwd."""

    @staticmethod
    def forward(ctx, q, k, v, r, w, causal, eps, key_padding_mask, dropout_p=0.0, seed=0):
        y, hnorm, bits = fwd_raw(q, k, v, r, w, causal, eps, key_padding_mask, dropout_p, seed)
        if any(ctx.needs_input_grad[:5]):
            ctx.save_for_backward(q, k, v, r, w, y, hnorm, bits, key_padding_mask)
        ctx.causal = causal
        ctx.eps = eps
        ctx.dropout = (dropout_p, seed)
        return y

    @staticmethod
    def backward(ctx, dy):
        q, k, v, r, w, y, hnorm, bits, kpm = ctx.saved_tensors
        dq, dk, dv, dr, dw = bwd_raw(q, k, v, r, w, ctx.causal, ctx.eps, y, hnorm, bits, dy, kpm, *ctx.dropout)
        return dq, dk, dv, dr.to(r.dtype), dw.to(w.dtype), None, None, None, None, None


def screening_core(q, k, v, r, w, causal=True, eps=1e-8, key_padding_mask=None, dropout_p=0.0, seed=0):
    """Fused screening attention core; see the module docstring.  dropout_p > 0
    applies attention dropout (attention.py:190) with the keep mask of `seed`."""
    return ScreeningCoreFunction.apply(q, k, v, r, w, causal, eps, key_padding_mask, dropout_p, seed)


def _decode_args(q, kcache, vcache, r, w):
    if not q.is_cuda:
        raise RuntimeError("decode_step runs on the GPU only (got a CPU tensor)")
    if q.dtype not in _DTYPES or kcache.dtype != q.dtype or vcache.dtype != q.dtype:
        raise TypeError(f"decode_step needs q and the caches in one of float32 / bfloat16 / float16, got "
                        f"{q.dtype}, {kcache.dtype}, {vcache.dtype}")
    B, H, D = q.shape
    if q.stride(2) != 1:
        q = q.contiguous()
    es = q.element_size()
    kcache, vcache = _as_bthd(kcache, "kcache", es), _as_bthd(vcache, "vcache", es)
    if kcache.shape != vcache.shape or kcache.shape[0] != B or kcache.shape[2:] != (H, D):
        raise ValueError(f"cache shapes {tuple(kcache.shape)}/{tuple(vcache.shape)} do not match q {tuple(q.shape)}")
    dev = q.device
    r32 = r.detach().to(device=dev, dtype=torch.float32).contiguous()
    w32 = w.detach().to(device=dev, dtype=torch.float32).contiguous()
    return q, kcache, vcache, r32, w32


def _scratch(workspace, need, device):
    """The caller's workspace if it holds `need` bytes in one piece, else one of this call's own."""
    if workspace is None or not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty((need,), dtype=torch.uint8, device=device)
    return workspace


def _decode_workspace(L, workspace, B, H, D, length, dev):
    return _scratch(workspace, max(int(L.msa_decode_workspace_bytes(B, H, D, int(length))), 16), dev)


def decode_step(q, kcache, vcache, cache_len, r, w, eps=1e-8, workspace=None, window_hint=0):
    """Screening attention of one new query per (b, h) against a KV cache.

    q (B, H, D); kcache/vcache (B, Tcap, H, D) holding the raw k/v projections
    of positions [0, cache_len), the last being the query's own token.
    window_hint: 0, or a bound on ceil(w) over the heads (sizes the launch only).
    Returns y (B, H, D) = TanhNorm(h) of that token.
    """
    L = _native.lib()
    q, kcache, vcache, r32, w32 = _decode_args(q, kcache, vcache, r, w)
    B, H, D = q.shape
    dev = q.device
    y = torch.empty((B, H, D), dtype=q.dtype, device=dev)
    workspace = _decode_workspace(L, workspace, B, H, D, cache_len, dev)
    rc = L.msa_decode(q.data_ptr(), q.stride(0), q.stride(1),
                      *_args_bthd(kcache), *_args_bthd(vcache),
                      B, H, D, _DTYPES[q.dtype], int(cache_len), int(kcache.shape[1]), int(window_hint),
                      r32.data_ptr(), w32.data_ptr(),
                      float(eps),
                      y.data_ptr(), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                      _stream_ptr(dev))
    _native.check(rc, "msa_decode")
    return y


def decode_step_at(q, kcache, vcache, last_pos, r, w, eps=1e-8, workspace=None, window_hint=0):
    """decode_step with the query's position in device memory: last_pos is a
    CUDA int64 tensor of one element, the position of the newest key, so the
    cache holds positions [0, last_pos] (the length is clamped to the
    capacity).  Launches depend only on the shapes, so a captured call stays
    valid as last_pos advances on the device."""
    L = _native.lib()
    q, kcache, vcache, r32, w32 = _decode_args(q, kcache, vcache, r, w)
    if not (last_pos.is_cuda and last_pos.dtype == torch.int64 and last_pos.numel() == 1):
        raise TypeError("last_pos must be a CUDA int64 tensor of one element")
    B, H, D = q.shape
    dev = q.device
    cap = int(kcache.shape[1])
    y = torch.empty((B, H, D), dtype=q.dtype, device=dev)
    workspace = _decode_workspace(L, workspace, B, H, D, cap, dev)
    rc = L.msa_decode_at(q.data_ptr(), q.stride(0), q.stride(1),
                         *_args_bthd(kcache), *_args_bthd(vcache),
                         B, H, D, _DTYPES[q.dtype], last_pos.data_ptr(), cap, int(window_hint),
                         r32.data_ptr(), w32.data_ptr(),
                         float(eps),
                         y.data_ptr(), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                         _stream_ptr(dev))
    _native.check(rc, "msa_decode_at")
    return y


# ---------------------------------------------------------------------------
# Caches of 8-bit codes, several new tokens at once, and drafted tokens.  These
# calls are short (a decode step's rows, a few hundred keys), so their checks
# look at each tensor once and build messages only for a call that is refused.
# ---------------------------------------------------------------------------
_CACHE_DTYPES = {**_DTYPES, torch.int8: _native.MSA_I8, torch.float8_e4m3fn: _native.MSA_FP8}
CODE_DTYPES = (torch.int8, torch.float8_e4m3fn)


def _launch(what, fn, index, args):
    """Calls fn(args, stream) for tensors of GPU `index`, whichever device is current."""
    if torch.cuda.current_device() == index:
        rc = fn(args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        _native.check(rc, what)


def _one_gpu(what, index, *tensors):
    """Raises unless every tensor given is on GPU `index`."""
    if index < 0:
        raise RuntimeError(f"{what} runs on the GPU only (got a CPU tensor)")
    for x in tensors:
        if x is not None and x.get_device() != index:
            raise RuntimeError(f"{what} runs on one GPU: got a tensor on {x.device} beside cuda:{index}")


def _index(x, name, *shapes):
    """An int64 tensor of one of the shapes, contiguous."""
    if x.dtype != torch.int64 or x.shape not in shapes:
        raise ValueError(f"{name} must be int64 of shape {' or '.join(map(str, shapes))}, got {x.dtype} {tuple(x.shape)}")
    return x.contiguous()


def _float32(x):
    """r or w as the kernels take it."""
    if x.dtype != torch.float32 or not x.is_contiguous():
        x = x.detach().to(torch.float32).contiguous()
    return x


def _rows_bthd(x, name):
    """x (B, T, H, D) as the kernels read it, its pointer and its first three strides."""
    if x.dim() == 4:
        sb, st, sh, sd = x.stride()
        p = x.data_ptr()
        if sd == 1 and not ((sb | st | sh) * x.element_size() | p) & 15:
            return x, (p, sb, st, sh)
    x = _as_bthd(x, name, x.element_size())
    return x, _args_bthd(x)


def _cache_args(what, kcache, vcache, kscale, vscale, dtype):
    """The type and the C arguments of a cache pair (B, cap, H, D) and its scales (B, cap, H), checked against
    the rows' type."""
    shape = kcache.shape
    if len(shape) != 4 or vcache.shape != shape or vcache.dtype != kcache.dtype:
        raise ValueError(f"{what}: the caches must be (B, cap, H, D) of one shape and type, got {kcache.dtype} "
                         f"{tuple(kcache.shape)}, {vcache.dtype} {tuple(vcache.shape)}")
    ct = _CACHE_DTYPES.get(kcache.dtype, -1)
    codes = ct >= _native.MSA_I8
    if not codes and kcache.dtype != dtype:
        raise TypeError(f"{what}: a cache of {kcache.dtype} does not hold rows of {dtype}")
    kb, kt, kh, kd = kcache.stride()
    vb, vt, vh, vd = vcache.stride()
    kp, vp = kcache.data_ptr(), vcache.data_ptr()
    if kd != 1 or vd != 1 or ((kb | kt | kh | vb | vt | vh) * (1 if codes else kcache.element_size()) | kp | vp) & 15:
        raise ValueError(f"{what}: the caches need unit stride over D and 16-byte aligned rows, got strides "
                         f"{kcache.stride()}, {vcache.stride()}")
    if not codes:
        if kscale is not None or vscale is not None:
            raise ValueError(f"{what}: a cache of {kcache.dtype} takes no scales")
        return ct, (kp, kb, kt, kh, vp, vb, vt, vh, 0, 0, 0, 0, 0, 0, 0, 0)
    rows = shape[:3]
    if kscale is None or vscale is None or kscale.shape != rows or vscale.shape != rows \
            or kscale.dtype != torch.float32 or vscale.dtype != torch.float32:
        raise ValueError(f"{what}: a cache of {kcache.dtype} needs kscale and vscale, float32 {tuple(rows)}")
    return ct, (kp, kb, kt, kh, vp, vb, vt, vh, kscale.data_ptr(), *kscale.stride(), vscale.data_ptr(), *vscale.stride())


def _start_args(start, B):
    """(pointer or 0, count, host value, tensor to keep) of an int or int64 device tensor."""
    if not isinstance(start, torch.Tensor):
        return 0, 0, int(start), None
    start = _index(start, "start", (1,), (B,))
    return start.data_ptr(), start.shape[0], 0, start


def cache_write(k, v, kcache, vcache, start, kscale=None, vscale=None, rows=None, count=None):
    """Writes rows k, v (B, T, H, D) to positions start, start + 1, ... of a cache.

    kcache, vcache (B, cap, H, D): of k's type (copied), or torch.int8 /
    torch.float8_e4m3fn codes with kscale, vscale float32 (B, cap, H): a row is
    kept as the codes nearest to TOP x / max|x| (TOP = 127 or 448, ties to the
    even code) and the scale max|x| / TOP.  Rows of zeros have scale 0; rows with
    an infinity or a NaN read back as NaN.
    start: an int (then all rows must fit, unless `count` is given), or an int64
    CUDA tensor of 1 or B elements; rows that would lie outside the cache are
    not written.
    rows (B, T') int64, count (B) int64: row rows[b, t] of k and v goes to
    position start + t, for t < count[b] only: the accepted path of
    verify_drafts.  Rows outside k are not written.
    The caches' rows and scales must not share memory (refused).  k and v must not
    overlap the caches, as the order of the rows is open.  The rest of the cache
    is left as it was.  No gradient flows through it.
    """
    index = k.get_device()
    _one_gpu("cache_write", index, v, kcache, vcache, kscale, vscale, rows, count,
             start if isinstance(start, torch.Tensor) else None)
    dtype = k.dtype
    if dtype not in _DTYPES or v.dtype != dtype or k.shape != v.shape:
        raise TypeError(f"cache_write: k and v must share shape and dtype float32, bfloat16 or float16, got {k.dtype} "
                        f"{tuple(k.shape)}, {v.dtype} {tuple(v.shape)}")
    k, kargs = _rows_bthd(k, "k")
    v, vargs = _rows_bthd(v, "v")
    B, Tx, H, D = k.shape
    ct, cache = _cache_args("cache_write", kcache, vcache, kscale, vscale, dtype)
    Bc, cap, Hc, Dc = kcache.shape
    if Bc != B or Hc != H or Dc != D:
        raise ValueError(f"cache_write: cache {tuple(kcache.shape)} does not match rows {tuple(k.shape)}")
    T, rp, cp = Tx, 0, 0
    if rows is not None:
        T = rows.shape[-1]
        rows = _index(rows, "rows", (B, T))
        rp = rows.data_ptr()
    if count is not None:
        count = _index(count, "count", (B,))
        cp = count.data_ptr()
    sp, n, host, start = _start_args(start, B)
    if not sp and (host < 0 or host + (T if count is None else 0) > cap):
        raise IndexError(f"KV cache capacity {cap} exceeded at position {host + T}")
    _launch("msa_cache_write", _native.lib().msa_cache_write, index,
            _native.pack_cache_args(*kargs, *vargs, *cache, rp, cp, sp, n, host, B, T, Tx, H, D, _DTYPES[dtype], cap, ct))


def cache_read(kcache, vcache, kscale, vscale, start, length, dtype):
    """The rows at positions start .. start + length - 1 of a cache (as
    cache_write takes it) in `dtype`: the float32 product code * scale, rounded to
    dtype; (k, v), each contiguous (B, length, H, D).  With a device `start`, positions outside the
    cache read as zeros."""
    index = kcache.get_device()
    _one_gpu("cache_read", index, vcache, kscale, vscale, start if isinstance(start, torch.Tensor) else None)
    if dtype not in _DTYPES:
        raise TypeError(f"cache_read: dtype must be float32, bfloat16 or float16, got {dtype}")
    ct, cache = _cache_args("cache_read", kcache, vcache, kscale, vscale, dtype)
    B, cap, H, D = kcache.shape
    length = int(length)
    sp, n, host, start = _start_args(start, B)
    if length < 0 or (not sp and (host < 0 or host + length > cap)):
        raise IndexError(f"positions {host} .. {host + length} are outside the KV cache's capacity {cap}")
    k = torch.empty((B, length, H, D), dtype=dtype, device=kcache.device)
    v = torch.empty_like(k)
    st = H * D
    sb = length * st
    _launch("msa_cache_read", _native.lib().msa_cache_read, index,
            _native.pack_cache_args(k.data_ptr(), sb, st, D, v.data_ptr(), sb, st, D, *cache, 0, 0, sp, n, host, B, length,
                                    length, H, D, _DTYPES[dtype], cap, ct))
    return k, v


def _parents_arg(parents, B, N):
    """(pointer or 0, stride over sequences, tensor to keep) of parents (N,) or (B, N), or None: a chain."""
    if parents is None:
        return 0, 0, None
    parents = _index(parents, "parents", (B, N), (N,))
    return parents.data_ptr(), N if parents.dim() == 2 else 0, parents


def tree_decode(q, kcache, vcache, lengths, parents, r, w, eps=1e-8, kscale=None, vscale=None, workspace=None,
                window_hint=0):
    """Screening attention of a tree of N <= 64 drafted tokens per sequence
    over a cache (N = 1: of one new token).

    q (B, N, H, D) raw query projections.  kcache, vcache (B, cap, H, D), with
    kscale, vscale (B, cap, H) where they hold codes (as cache_write leaves
    them): sequence b's committed rows at positions [0, n_b), its nodes' own
    rows at n_b .. n_b + N - 1.  lengths: int64 CUDA tensor of 1 or B elements,
    the n_b (clamped to [0, cap - N]).
    parents: int64 (N,) or (B, N), parents[i] < i the node that node i
    continues, any other value for a root; None for a chain.  Node i stands at
    position n_b + depth_i and sees the committed keys of its window, itself
    and its ancestors.
    window_hint: 0, or a bound on ceil(w) over the heads (sizes the launch).
    workspace: scratch of this call on q's GPU; where it is None, too small or not
    contiguous the call allocates its own.
    Returns y (B, N, H, D) = TanhNorm(h), in q's dtype; no gradient.
    """
    index = q.get_device()
    _one_gpu("tree_decode", index, kcache, vcache, kscale, vscale, lengths, parents, r, w, workspace)
    dtype = q.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"tree_decode: q must be float32, bfloat16 or float16, got {q.dtype}")
    q, qargs = _rows_bthd(q, "q")
    B, N, H, D = q.shape
    if N > _native.TREE_MAX:
        raise ValueError(f"tree_decode: a tree holds at most {_native.TREE_MAX} nodes, got {N}")
    ct, cache = _cache_args("tree_decode", kcache, vcache, kscale, vscale, dtype)
    Bc, cap, Hc, Dc = kcache.shape
    if Bc != B or Hc != H or Dc != D:
        raise ValueError(f"tree_decode: cache {tuple(kcache.shape)} does not match q {tuple(q.shape)}")
    if N > cap:
        raise IndexError(f"KV cache capacity {cap} is below {N} nodes")
    if r.shape != (H,) or w.shape != (H,):
        raise ValueError(f"r and w must have shape ({H},)")
    lengths = _index(lengths, "lengths", (B,), (1,))
    par, par_sb, parents = _parents_arg(parents, B, N)
    r, w = _float32(r), _float32(w)
    hint = max(0, int(window_hint))
    L = _native.lib()
    y = torch.empty((B, N, H, D), dtype=dtype, device=q.device) if not q.is_contiguous() else torch.empty_like(q)
    qt = _DTYPES[dtype]
    need = L.msa_tree_workspace_bytes(B, H, N, D, qt, ct, cap, hint)
    if need:
        workspace = _scratch(workspace, need, q.device)
    _launch("msa_tree_decode", L.msa_tree_decode, index,
            _native.pack_tree_args(*qargs, *cache, lengths.data_ptr(), par, r.data_ptr(), w.data_ptr(), y.data_ptr(),
                                   workspace.data_ptr() if need else 0, need, lengths.shape[0], par_sb, B, N, H, D, qt,
                                   cap, ct, hint, float(eps)))
    return y


def verify_drafts(target, tokens, parents=None, uniforms=None, draft=None):
    """Which drafted tokens the target model accepts, and its next token.

    A tree of M <= 64 nodes per sequence; node 0 is the last committed token,
    node i >= 1 continues node parents[i] in [0, i) (any other value: it is never
    reached).  parents int64 (M,) or (B, M), or None for a chain; tokens int64
    (B, M).
    target (B, M, V) float32, bfloat16 or float16: row i is the target's
    distribution after node i: probabilities, or any scores where uniforms is
    None.
    uniforms float32 (B, M) in [0, 1), or None for greedy decoding.
    draft (B, M - 1, V) probabilities in target's dtype, or None: row i is what
    token i + 1 was drawn from; the drafts are then a chain, which ends before
    the first token outside [0, V) (so -1 pads a sequence with fewer drafts).

    From node 0 the walk goes on to the first child, in index order, that is
    accepted: with `draft` if u_i q(x) < p(x), without if u_i (1 - the p of the
    siblings refused before it) < p(x), greedily if x is the row's largest entry.
    Behind the last node the next token is drawn with u_0 from what is left of p
    (max(p - q, 0), or p without the refused tokens), so that the tokens are
    distributed as the target's own samples.  Sums are in 64 bits.
    Returns int64 path (B, M), the nodes walked, node 0 first, -1 behind them;
    count (B), how many; token (B), the next token.  The count[b] rows path[b]
    are what cache_write takes as `rows` and `count`.
    """
    index = target.get_device()
    _one_gpu("verify_drafts", index, tokens, parents, uniforms, draft)
    dtype = target.dtype
    if target.dim() != 3 or dtype not in _DTYPES:
        raise TypeError(f"verify_drafts: target must be (B, M, V) float32, bfloat16 or float16, got {target.dtype} "
                        f"{tuple(target.shape)}")
    B, M, V = target.shape
    if not 1 <= M <= _native.TREE_MAX:
        raise ValueError(f"verify_drafts: a tree holds 1 to {_native.TREE_MAX} nodes, got {M}")
    tokens = _index(tokens, "tokens", (B, M))
    par, par_sb, parents = _parents_arg(parents, B, M)
    up = dp = 0
    d_sb = d_sn = 0
    if uniforms is not None:
        if uniforms.dtype != torch.float32 or uniforms.shape != (B, M):
            raise ValueError(f"uniforms must be float32 ({B}, {M}), got {uniforms.dtype} {tuple(uniforms.shape)}")
        uniforms = uniforms.contiguous()
        up = uniforms.data_ptr()
    if draft is not None:
        if uniforms is None:
            raise ValueError("verify_drafts: draft probabilities need uniforms")
        if draft.dtype != dtype or draft.shape != (B, M - 1, V):
            raise ValueError(f"draft must be {dtype} ({B}, {M - 1}, {V}), got {draft.dtype} {tuple(draft.shape)}")
        draft = draft if draft.stride(2) == 1 else draft.contiguous()
        d_sb, d_sn, _ = draft.stride()
        dp = draft.data_ptr() if M > 1 else 0  # a chain of one node has no draft rows: nothing can be refused
    target = target if target.stride(2) == 1 else target.contiguous()
    t_sb, t_sn, _ = target.stride()
    L = _native.lib()
    path = torch.empty_like(tokens)
    count = torch.empty((B,), dtype=torch.int64, device=target.device)
    token = torch.empty_like(count)
    need, workspace = 0, None
    if uniforms is None:
        need = L.msa_verify_workspace_bytes(B, M, V, 1)
        workspace = torch.empty((need,), dtype=torch.uint8, device=target.device)
    _launch("msa_verify", L.msa_verify, index,
            _native.pack_verify_args(target.data_ptr(), t_sb, t_sn, dp, d_sb, d_sn, tokens.data_ptr(), par, par_sb, up,
                                     path.data_ptr(), count.data_ptr(), token.data_ptr(),
                                     workspace.data_ptr() if need else 0, need, B, M, V, _DTYPES[dtype]))
    return path, count, token
