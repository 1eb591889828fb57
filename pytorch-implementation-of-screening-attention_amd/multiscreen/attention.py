"""Multi-head Screening Attention with the MI355X fused core.

Public interface, parameter names and initialisation are those of the
reference module (multiscreen/attention.py:23-200), so reference state_dicts
load unchanged:

    ScreeningAttention(d_model, num_heads, dropout=0.0, causal=True, eps=1e-8)
    .forward(query, key, value, key_padding_mask=None) -> (B, T_q, d_model)

    q_proj, k_proj, v_proj, out_proj : Linear(d, d, bias=False), created in
                                       that order (attention.py:52-55)
    s_v = linspace(0, ln 255, H)     : w = exp(s_v) + 1   (attention.py:63-64)
    s_r = zeros(H)                   : r = exp(s_r) + 1   (attention.py:65)

The projections and out_proj stay torch GEMMs.  Everything between them --
unit normalisation, similarity, trim-and-square, the cosine window, key
padding, the un-normalised aggregation and TanhNorm (attention.py:155-196) --
is one fused HIP forward and one fused HIP backward (ops.screening_core) for
GPU tensors; CPU tensors use the explicit-matrix form in _dense.py.
"""

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from .norm import TanhNorm
from . import ops
from ._dense import CODE_TOP, quantise_rows, screening_core_dense, tree_dense


class ScreeningAttention(nn.Module):
    """Multi-head Screening Attention (reference: attention.py:23-42).

    Args:
        d_model:    Total model dimension.
        num_heads:  Number of attention heads.
        dropout:    Dropout probability on attention weights.
        causal:     If True, apply causal masking (autoregressive decoding).
        eps:        Small value for numerical stability.
    """

    def __init__(self, d_model: int, num_heads: int, dropout: float = 0.0, causal: bool = True,
                 eps: float = 1e-8):
        super().__init__()
        assert d_model % num_heads == 0, "d_model must be divisible by num_heads"
        self.d_model = d_model
        self.num_heads = num_heads
        self.head_dim = d_model // num_heads
        self.causal = causal
        self.eps = eps

        self.q_proj = nn.Linear(d_model, d_model, bias=False)
        self.k_proj = nn.Linear(d_model, d_model, bias=False)
        self.v_proj = nn.Linear(d_model, d_model, bias=False)
        self.out_proj = nn.Linear(d_model, d_model, bias=False)

        # w = exp(s_v) + 1 (window), r = exp(s_r) + 1 (acceptance sharpness)
        self.s_v = nn.Parameter(torch.linspace(0, math.log(255), num_heads))
        self.s_r = nn.Parameter(torch.zeros(num_heads))

        self.attn_dropout = nn.Dropout(dropout)
        # attribute name kept from the reference (attention.py:69)
        self.tahn_norm = TanhNorm(eps=eps)

    def window(self) -> torch.Tensor:
        return torch.exp(self.s_v) + 1.0

    def sharpness(self) -> torch.Tensor:
        return torch.exp(self.s_r) + 1.0

    def project(self, x: torch.Tensor, proj: nn.Linear) -> torch.Tensor:
        """proj(x) viewed as (B, T, H, D) -- no copy (attention.py:150-151)."""
        return proj(x).view(x.shape[0], x.shape[1], self.num_heads, self.head_dim)

    @staticmethod
    def _plain(projs) -> bool:
        """True when every projection is a bias-free nn.Linear with no forward
        hooks (its own or global): only then does one GEMM over the stacked
        weights give exactly what calling the modules gives.  Anything else
        (hooks such as weight_norm or LoRA wrappers, subclasses, a bias) takes
        the per-module calls of attention.py:150-153."""
        from torch.nn.modules import module as _m
        if _m._global_forward_hooks or _m._global_forward_pre_hooks:
            return False
        return all(type(p) is nn.Linear and p.bias is None and not p._forward_hooks
                   and not p._forward_pre_hooks for p in projs)

    def project_qkv(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor):
        """q, k, v projections as (B, T, H, D) views (attention.py:147-153) from
        as few GEMMs as the inputs allow: one over the stacked q/k/v weights
        for self-attention (query is key is value), one for q and one over the
        stacked k/v weights when key is value (cross-attention over a memory),
        else three.  The views' time stride is then 3*d_model (or 2*d_model);
        the fused kernels read them in place.  The stacked weight is formed on
        every call (a copy of 2-3 d x d weights), so weight updates of any kind,
        in place or through .data, are always seen."""
        B, Tq, _ = query.shape
        Tk = key.shape[1]
        H, D, d = self.num_heads, self.head_dim, self.d_model
        if query is key and key is value and self._plain((self.q_proj, self.k_proj, self.v_proj)):
            wqkv = torch.cat((self.q_proj.weight, self.k_proj.weight, self.v_proj.weight))
            q, k, v = F.linear(query, wqkv).split(d, dim=-1)
            return q.view(B, Tq, H, D), k.view(B, Tq, H, D), v.view(B, Tq, H, D)
        q = self.project(query, self.q_proj)
        if key is value and self._plain((self.k_proj, self.v_proj)):
            k, v = F.linear(key, torch.cat((self.k_proj.weight, self.v_proj.weight))).split(d, dim=-1)
            return q, k.view(B, Tk, H, D), v.view(B, Tk, H, D)
        return q, self.project(key, self.k_proj), self.project(value, self.v_proj)

    def core(self, q, k, v, key_padding_mask=None):
        """(B,T,H,D) raw projections -> TanhNorm'd (B,Tq,H,D) head outputs."""
        w, r = self.window(), self.sharpness()
        dropping = self.training and self.attn_dropout.p > 0.0
        if q.is_cuda:
            if dropping:
                # keep mask from a counter-based hash of this seed (drawn from
                # torch's default generator, so torch.manual_seed reproduces it)
                seed = int(torch.randint(0, 2 ** 62, (1,)).item())
                return ops.screening_core(q, k, v, r, w, self.causal, self.eps, key_padding_mask,
                                          self.attn_dropout.p, seed)
            return ops.screening_core(q, k, v, r, w, self.causal, self.eps, key_padding_mask)
        return screening_core_dense(q, k, v, r, w, self.causal, self.eps, key_padding_mask,
                                    self.attn_dropout if dropping else None)

    def forward(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                key_padding_mask: torch.Tensor | None = None) -> torch.Tensor:
        """
        Args:
            query:            (B, T_q, d_model)
            key:              (B, T_k, d_model)
            value:            (B, T_k, d_model)
            key_padding_mask: (B, T_k) bool mask; True = position to ignore.
        Returns:
            out: (B, T_q, d_model)
        """
        B, T_q, _ = query.shape
        q, k, v = self.project_qkv(query, key, value)
        y = self.core(q, k, v, key_padding_mask)
        return self.out_proj(y.reshape(B, T_q, self.d_model))

    # ------------------------------------------------------------------
    # KV-cache inference (no reference counterpart: the reference's
    # MultiscreenLM.generate re-runs forward() on the whole prefix for every
    # token, model.py:111-141).  The cache holds the raw k/v projections
    # (viewed as (B, T_cap, H, D)); decode(pos) computes exactly row `pos` of
    # forward().
    # ------------------------------------------------------------------
    def prefill(self, x: torch.Tensor, cache) -> torch.Tensor:
        """Causal self-attention forward over x (B,T,d) at positions 0..T-1;
        also writes its k/v projections into cache[:, :T]."""
        B, T, _ = x.shape
        q, k, v = self.project_qkv(x, x, x)
        cache.store(k, v, 0)
        y = self.core(q, k, v)
        return self.out_proj(y.reshape(B, T, self.d_model))

    def decode(self, x: torch.Tensor, cache, pos, rw=None) -> torch.Tensor:
        """x (B,1,d) is the token at position `pos`; returns its attention output (B,1,d).

        pos: an int, or (on GPU) a CUDA int64 tensor of one element holding the
        position, so that the step can be captured once and replayed as the
        position advances on the device.  rw: optional (r, w) fp32 tensors
        computed beforehand (exp(s_r)+1, exp(s_v)+1), for callers decoding
        many tokens with fixed parameters."""
        if not self.causal:
            raise RuntimeError("KV-cache decode is defined for causal self-attention only")
        B = x.shape[0]
        if cache.k_scale is not None:  # 8-bit rows: a tree of one node
            if not torch.is_tensor(pos):
                if not 0 <= pos < cache.k.shape[1]:
                    raise IndexError(f"KV cache capacity {cache.k.shape[1]} exceeded at position {pos + 1}")
                pos = torch.full((1,), pos, dtype=torch.int64, device=x.device)
            return self.tree_step(x, cache, pos, None, rw, checked=True)[0]
        q, k, v = self.project_qkv(x, x, x)
        r, w = rw if rw is not None else (self.sharpness(), self.window())
        if torch.is_tensor(pos):
            if not x.is_cuda:
                raise RuntimeError("a device position needs the GPU decode path")
            cache.store_at(k, v, pos)
            y = ops.decode_step_at(q[:, 0].to(cache.k.dtype), cache.k, cache.v, pos, r, w, self.eps,
                                   cache.workspace, cache.window_hint).to(x.dtype)
            return self.out_proj(y.reshape(B, 1, self.d_model))
        cache.store(k, v, pos)
        if x.is_cuda:
            y = ops.decode_step(q[:, 0].to(cache.k.dtype), cache.k, cache.v, pos + 1, r, w, self.eps,
                                cache.workspace, cache.window_hint).to(x.dtype)
        else:
            rows = (q, cache.k[:, :pos + 1], cache.v[:, :pos + 1])
            ct = cache.k.dtype
            if ct != q.dtype and not torch.is_autocast_enabled("cpu"):
                # the cache's type is the query's and the result's too, as on the GPU
                rows = tuple(t.to(ct).to(torch.promote_types(q.dtype, ct)) for t in rows)
            y = screening_core_dense(*rows, r, w, True, self.eps, q_offset=pos)[:, 0]
            if rows[0] is not q:
                y = y.to(ct).to(x.dtype)
        return self.out_proj(y.reshape(B, 1, self.d_model))

    def tree_step(self, x: torch.Tensor, cache, lengths: torch.Tensor, parents=None, rw=None, checked=False):
        """x (B, M, d): the M <= 64 nodes of a tree of drafted tokens that follows sequence b's
        lengths[b] cached positions (lengths int64, 1 or B elements; parents as in
        ops.tree_decode, None for a chain).  Writes the nodes' k and v behind the committed rows and
        returns the attention output (B, M, d), node i seeing the sequence and its own ancestors,
        and (k, v), from which KVCache.store_rows keeps an accepted path.
        A sequence needs 0 <= lengths[b] <= capacity - M: on the CPU others raise IndexError; on the
        GPU, where the host does not see them, their output is NaN (checked=True: the caller sees to
        it, and theirs is meaningless)."""
        if not self.causal:
            raise RuntimeError("KV-cache decode is defined for causal self-attention only")
        B, M, _ = x.shape
        if not x.is_cuda and not bool(cache.has_room(lengths, M).all()):
            raise IndexError(f"KV cache capacity {cache.k.shape[1]} exceeded by {M} nodes behind positions {lengths.tolist()}")
        q, k, v = self.project_qkv(x, x, x)
        if cache.k_scale is None:
            q, k, v = (t.to(cache.k.dtype) for t in (q, k, v))
        cache.store_rows(k, v, lengths)
        r, w = rw if rw is not None else (self.sharpness(), self.window())
        if x.is_cuda:
            y = ops.tree_decode(q, cache.k, cache.v, lengths, parents, r, w, self.eps, cache.k_scale, cache.v_scale,
                                None, cache.window_hint)
        else:
            up = torch.arange(-1, M - 1) if parents is None else parents
            kc, vc = cache.read(0, cache.k.shape[1], q.dtype)
            y = tree_dense(q, kc, vc, lengths, up.expand(B, M), r, w, self.eps)
        y = self.out_proj(y.to(x.dtype).reshape(B, M, self.d_model))
        if x.is_cuda and not checked:
            y = torch.where(cache.has_room(lengths, M).view(-1, 1, 1), y, math.nan)
        return y, (k, v)


class KVCache:
    """Raw k/v projections of one attention layer.

    Stored head-major, (B, H, capacity, D), so that one head's window is one
    contiguous stream for the decode kernel; `k` and `v` are the (B, capacity,
    H, D) views of that storage, the layout of the projections, in the model's
    dtype (float32, bfloat16 or float16).

    With dtype torch.int8 or torch.float8_e4m3fn the cache holds 8-bit codes and
    `k_scale`, `v_scale` (B, capacity, H) a float32 scale per row, as
    ops.cache_write leaves them: a half or a quarter of the bytes to keep and
    to read per token."""

    def __init__(self, batch, capacity, num_heads, head_dim, dtype, device, window_hint=0):
        # 0, or a bound on ceil(w) over the layer's heads: sizes the decode
        # launch to the windows instead of the cache (results do not depend on it)
        self.window_hint = int(window_hint)
        self._k = torch.zeros((batch, num_heads, capacity, head_dim), dtype=dtype, device=device)
        self._v = torch.zeros_like(self._k)
        self.k = self._k.permute(0, 2, 1, 3)
        self.v = self._v.permute(0, 2, 1, 3)
        self.k_scale = self.v_scale = None
        if dtype in CODE_TOP:
            self.k_scale, self.v_scale = (torch.zeros((batch, num_heads, capacity), device=device).transpose(1, 2)
                                          for _ in range(2))
        self.workspace = None
        if self.k.is_cuda and self.k_scale is None:
            from . import _native
            nbytes = int(_native.lib().msa_decode_workspace_bytes(batch, num_heads, head_dim, capacity))
            self.workspace = torch.empty((max(nbytes, 16),), dtype=torch.uint8, device=device)

    def has_room(self, lengths, rows):
        """Of each element of lengths (int64): whether `rows` positions from there on lie in the cache."""
        return lengths == lengths.clamp(0, self.k.shape[1] - rows)

    def store(self, k, v, pos):
        T = k.shape[1]
        if pos + T > self.k.shape[1]:
            raise IndexError(f"KV cache capacity {self.k.shape[1]} exceeded at position {pos + T}")
        if self.k_scale is not None:
            if self.k.is_cuda:
                ops.cache_write(k, v, self.k, self.v, pos, self.k_scale, self.v_scale)
            else:
                self.store_rows(k, v, torch.tensor([pos]))
            return
        self.k[:, pos:pos + T] = k.to(self.k.dtype)
        self.v[:, pos:pos + T] = v.to(self.v.dtype)

    def store_at(self, k, v, pos):
        """k, v (B,1,H,D) at the position held by the device int64 tensor pos
        (one element).  The caller keeps pos below the capacity."""
        if self.k_scale is not None:
            self.store_rows(k, v, pos)
            return
        self._k.index_copy_(2, pos, k.permute(0, 2, 1, 3).to(self._k.dtype))
        self._v.index_copy_(2, pos, v.permute(0, 2, 1, 3).to(self._v.dtype))

    def store_rows(self, k, v, start, rows=None, count=None):
        """k, v (B, T, H, D) at positions start[b], start[b] + 1, ... (start int64, 1 or B
        elements); with rows (B, T') and count (B), row rows[b, t] of k and v at start[b] + t for t <
        count[b] (an accepted path of ops.verify_drafts).  Positions outside the cache are not
        written."""
        if self.k_scale is None:
            k, v = k.to(self.k.dtype), v.to(self.v.dtype)
        if self.k.is_cuda:
            ops.cache_write(k, v, self.k, self.v, start, self.k_scale, self.v_scale, rows, count)
            return
        B, T = k.shape[:2] if rows is None else rows.shape
        src = torch.arange(T).expand(B, T) if rows is None else rows
        at = start.view(-1, 1) + torch.arange(T).expand(B, T)
        keep = (at >= 0) & (at < self.k.shape[1]) & (src >= 0) & (src < k.shape[1])
        if count is not None:
            keep &= torch.arange(T) < count.view(-1, 1)
        b, t = keep.nonzero(as_tuple=True)
        for x, c, s in ((k, self.k, self.k_scale), (v, self.v, self.v_scale)):
            x = x[b, src[b, t]]
            if s is not None:
                x, s[b, at[b, t]] = quantise_rows(x, c.dtype)
                x, c = x.view(torch.uint8), c.view(torch.uint8)
            c[b, at[b, t]] = x

    def read(self, start, length, dtype):
        """Rows start .. start + length - 1 as (k, v) of `dtype`, (B, length, H, D)."""
        if self.k_scale is not None and self.k.is_cuda:
            return ops.cache_read(self.k, self.v, self.k_scale, self.v_scale, start, length, dtype)
        if not 0 <= start <= start + length <= self.k.shape[1]:
            raise IndexError(f"positions {start} .. {start + length} are outside the KV cache's capacity {self.k.shape[1]}")
        part = slice(start, start + length)
        if self.k_scale is None:
            return self.k[:, part].to(dtype), self.v[:, part].to(dtype)
        return tuple((c[:, part].float() * s[:, part].unsqueeze(-1)).to(dtype)
                     for c, s in ((self.k, self.k_scale), (self.v, self.v_scale)))
