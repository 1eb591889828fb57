"""Pre-norm Multiscreen blocks (reference: multiscreen/layers.py:15-144).

Same constructors, submodule names and forward signatures as the reference,
so state_dicts are interchangeable:

    MultiscreenBlock(d_model, num_heads, ffn_dim=None, dropout=0.0, causal=True, ffn="gelu")
        x = x + attn(norm1(x));  x = x + ffn(norm2(x))
    MultiscreenDecoderLayer(d_model, num_heads, ffn_dim=None, dropout=0.0, ffn="gelu")
        x = x + self_attn(norm1(x));  x = x + cross_attn(norm2(x), memory)
        x = x + ffn(norm3(x))

ffn="gelu" is the reference's feed-forward; "swiglu" and "geglu" are gated ones
(GatedFFN), beyond the reference.

MultiscreenBlock additionally exposes prefill, decode and tree steps over a KV
cache, used by MultiscreenLM.generate and generate_speculative.
"""

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops
from ._dense import gated_linear_dense
from .attention import ScreeningAttention

_GATED = {"swiglu": "silu", "geglu": "gelu"}


def plain_linears(*modules) -> bool:
    """Whether using the modules' weights is what calling them does: bias-free nn.Linear without hooks of either
    direction or a forward of their own.  Replaced, adapted or observed modules are called."""
    from torch.nn.modules import module as _m
    return ScreeningAttention._plain(modules) and not (_m._global_backward_hooks or _m._global_backward_pre_hooks) and not any(
        m._backward_hooks or m._backward_pre_hooks or "forward" in m.__dict__ for m in modules)


class GatedFFN(nn.Module):
    """down(dropout(act(gate(x)) * up(x))), dropout behind it: both products, the
    activation and their product are one kernel on the GPU (ops.gated_linear), unless
    gate or up is not a plain nn.Linear (plain_linears)."""

    def __init__(self, d_model: int, ffn_dim: int, dropout: float = 0.0, activation: str = "silu"):
        super().__init__()
        self.gate = nn.Linear(d_model, ffn_dim, bias=False)
        self.up = nn.Linear(d_model, ffn_dim, bias=False)
        self.down = nn.Linear(ffn_dim, d_model, bias=False)
        self.dropout = nn.Dropout(dropout)
        self.activation = activation

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if plain_linears(self.gate, self.up):
            gated = ops.gated_linear if x.is_cuda else gated_linear_dense
            h = gated(x, self.gate.weight, self.up.weight, self.activation)
        else:
            act = F.silu if self.activation == "silu" else F.gelu
            h = act(self.gate(x)) * self.up(x)
        return self.dropout(self.down(self.dropout(h)))


def _ffn(d_model, ffn_dim, dropout, kind="gelu"):
    if kind in _GATED:
        return GatedFFN(d_model, ffn_dim, dropout, _GATED[kind])
    if kind != "gelu":
        raise ValueError(f"ffn must be 'gelu', 'swiglu' or 'geglu', got {kind!r}")
    return nn.Sequential(
        nn.Linear(d_model, ffn_dim, bias=False),
        nn.GELU(),
        nn.Dropout(dropout),
        nn.Linear(ffn_dim, d_model, bias=False),
        nn.Dropout(dropout),
    )


class MultiscreenBlock(nn.Module):
    def __init__(self, d_model: int, num_heads: int, ffn_dim: int | None = None,
                 dropout: float = 0.0, causal: bool = True, ffn: str = "gelu"):
        super().__init__()
        ffn_dim = ffn_dim or 4 * d_model
        self.norm1 = nn.RMSNorm(d_model)
        self.norm2 = nn.RMSNorm(d_model)
        self.attn = ScreeningAttention(d_model=d_model, num_heads=num_heads, dropout=dropout,
                                       causal=causal)
        self.ffn = _ffn(d_model, ffn_dim, dropout, ffn)

    def forward(self, x: torch.Tensor, key_padding_mask: torch.Tensor | None = None) -> torch.Tensor:
        normed = self.norm1(x)
        x = x + self.attn(normed, normed, normed, key_padding_mask=key_padding_mask)
        return x + self.ffn(self.norm2(x))

    def prefill(self, x: torch.Tensor, cache) -> torch.Tensor:
        """forward() over a prompt starting at position 0, storing its raw k/v in `cache`."""
        normed = self.norm1(x)
        x = x + self.attn.prefill(normed, cache)
        return x + self.ffn(self.norm2(x))

    def decode(self, x: torch.Tensor, cache, pos, rw=None) -> torch.Tensor:
        """One token x (B,1,d) at position `pos` (int or device tensor), attending to the cache."""
        normed = self.norm1(x)
        x = x + self.attn.decode(normed, cache, pos, rw)
        return x + self.ffn(self.norm2(x))

    def tree_step(self, x: torch.Tensor, cache, lengths, parents=None, rw=None, checked=False):
        """The nodes x (B, M, d) of a tree of drafted tokens (ScreeningAttention.tree_step); returns
        their outputs and the layer's (k, v)."""
        y, kv = self.attn.tree_step(self.norm1(x), cache, lengths, parents, rw, checked)
        x = x + y
        return x + self.ffn(self.norm2(x)), kv


class MultiscreenDecoderLayer(nn.Module):
    def __init__(self, d_model: int, num_heads: int, ffn_dim: int | None = None,
                 dropout: float = 0.0, ffn: str = "gelu"):
        super().__init__()
        ffn_dim = ffn_dim or 4 * d_model
        self.norm1 = nn.RMSNorm(d_model)
        self.norm2 = nn.RMSNorm(d_model)
        self.norm3 = nn.RMSNorm(d_model)
        self.self_attn = ScreeningAttention(d_model=d_model, num_heads=num_heads, dropout=dropout,
                                            causal=True)
        self.cross_attn = ScreeningAttention(d_model=d_model, num_heads=num_heads, dropout=dropout,
                                             causal=False)
        self.ffn = _ffn(d_model, ffn_dim, dropout, ffn)

    def forward(self, x: torch.Tensor, memory: torch.Tensor,
                tgt_key_padding_mask: torch.Tensor | None = None,
                memory_key_padding_mask: torch.Tensor | None = None) -> torch.Tensor:
        normed = self.norm1(x)
        x = x + self.self_attn(normed, normed, normed, key_padding_mask=tgt_key_padding_mask)
        normed = self.norm2(x)
        x = x + self.cross_attn(normed, memory, memory, key_padding_mask=memory_key_padding_mask)
        return x + self.ffn(self.norm3(x))
