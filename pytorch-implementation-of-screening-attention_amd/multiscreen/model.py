"""MultiscreenLM: causal language model built from Multiscreen blocks.

Reference: multiscreen/model.py:12-141.  Same constructor, submodule names
(token_emb, pos_emb, emb_dropout, blocks, norm, lm_head), tied weights,
initialisation (_init_weights, model.py:64-69), forward() contract (logits and
an un-shifted cross-entropy with ignore_index=-100, model.py:101-106) and
generate() signature and sampling (temperature, optional top-k, multinomial,
model.py:111-141).

generate() differs only in cost: instead of re-running forward() over the
whole prefix for every new token, it prefills a per-layer KV cache once and
then runs one single-query decode step per token (the HIP decode kernel on
GPU), which computes the same last-position logits.

Beyond the reference: caches of 8-bit rows (cache_dtype=torch.int8 or
torch.float8_e4m3fn), steps over several tokens or a tree of drafts at once
(tree_step, accept) and generation with a smaller model that drafts
(generate_speculative).
"""

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops
from ._dense import tree_relations, verify_dense
from .attention import KVCache
from .layers import MultiscreenBlock


class MultiscreenLM(nn.Module):
    def __init__(self, vocab_size: int, d_model: int = 512, num_heads: int = 8, num_layers: int = 6,
                 ffn_dim: int | None = None, max_seq_len: int = 2048, dropout: float = 0.0,
                 tie_weights: bool = True):
        super().__init__()
        self.d_model = d_model
        self.token_emb = nn.Embedding(vocab_size, d_model)
        self.pos_emb = nn.Embedding(max_seq_len, d_model)
        self.emb_dropout = nn.Dropout(dropout)
        self.blocks = nn.ModuleList([
            MultiscreenBlock(d_model=d_model, num_heads=num_heads, ffn_dim=ffn_dim, dropout=dropout,
                             causal=True)
            for _ in range(num_layers)
        ])
        self.norm = nn.RMSNorm(d_model)
        self.lm_head = nn.Linear(d_model, vocab_size, bias=False)
        if tie_weights:
            self.lm_head.weight = self.token_emb.weight
        self._init_weights()

    def _init_weights(self):
        nn.init.normal_(self.token_emb.weight, std=0.02)
        nn.init.normal_(self.pos_emb.weight, std=0.02)
        for module in self.modules():
            if isinstance(module, nn.Linear):
                nn.init.normal_(module.weight, std=0.02)

    def embed(self, input_ids: torch.Tensor, start=0) -> torch.Tensor:
        """Token + position embeddings from position `start` (an int, or for one
        token a device int64 tensor of one element)."""
        T = input_ids.shape[1]
        if torch.is_tensor(start):
            positions = start.view(1, 1)
        else:
            positions = torch.arange(start, start + T, device=input_ids.device).unsqueeze(0)
        return self.emb_dropout(self.token_emb(input_ids) + self.pos_emb(positions))

    def forward(self, input_ids: torch.Tensor, key_padding_mask: torch.Tensor | None = None,
                labels: torch.Tensor | None = None) -> dict[str, torch.Tensor]:
        """
        Args:
            input_ids:        (B, T) integer token ids.
            key_padding_mask: (B, T) bool -- True = padding position.
            labels:           (B, T) token ids; -100 is ignored.
        Returns:
            {'logits': (B, T, vocab)} plus 'loss' when labels are given.
        """
        x = self.embed(input_ids)
        for block in self.blocks:
            x = block(x, key_padding_mask=key_padding_mask)
        logits = self.lm_head(self.norm(x))
        result = {"logits": logits}
        if labels is not None:
            result["loss"] = F.cross_entropy(logits.view(-1, logits.size(-1)), labels.view(-1),
                                             ignore_index=-100)
        return result

    def new_cache(self, batch: int, capacity: int, dtype: torch.dtype, device) -> list:
        """One KVCache per block.  Each carries its layer's widest window
        (ceil(max_h w_h), read once here) so that decode launches only the
        blocks the windows need.  dtype torch.int8 or torch.float8_e4m3fn: 8-bit
        rows with a scale each (KVCache)."""
        caches = []
        for block in self.blocks:
            attn = block.attn
            with torch.no_grad():
                wmax = float(attn.window().max())
            hint = min(capacity, math.ceil(wmax)) if math.isfinite(wmax) else 0
            caches.append(KVCache(batch, capacity, attn.num_heads, attn.head_dim, dtype, device, hint))
        return caches

    def _head(self, x: torch.Tensor) -> torch.Tensor:
        return self.lm_head(self.norm(x))

    @torch.no_grad()
    def prefill(self, input_ids: torch.Tensor, caches: list) -> torch.Tensor:
        """Runs the prompt once, filling `caches`; returns last-position logits (B, vocab)."""
        x = self.embed(input_ids)
        for block, cache in zip(self.blocks, caches):
            x = block.prefill(x, cache)
        return self._head(x[:, -1:])[:, 0]

    @torch.no_grad()
    def decode_step(self, token: torch.Tensor, caches: list, pos, rws=None) -> torch.Tensor:
        """token (B,1) at position `pos`; returns its logits (B, vocab).

        pos: an int, or on GPU a CUDA int64 tensor of one element (see
        GraphDecoder).  rws: optional per-layer (r, w) fp32 tensors."""
        x = self.embed(token, start=pos)
        for i, (block, cache) in enumerate(zip(self.blocks, caches)):
            x = block.decode(x, cache, pos, None if rws is None else rws[i])
        return self._head(x)[:, 0]

    @torch.no_grad()
    def tree_step(self, tokens: torch.Tensor, caches: list, lengths: torch.Tensor, parents=None, rws=None):
        """One step over a tree of M <= 64 tokens per sequence: tokens (B, M), node 0 the last
        committed token at position lengths[b] (int64, 1 or B elements), the others drafted
        continuations (parents as in ops.tree_decode; None: a chain).  Writes the nodes' rows into
        the caches from position lengths[b] on.  Positions past the last position embedding take
        the last one.  0 <= lengths[b] <= capacity - M: others raise IndexError on the CPU; on the GPU
        the logits of their sequences are NaN.
        Returns the logits (B, M, vocab) and per layer (k, v), for accept()."""
        B, M = tokens.shape
        if parents is None:
            depth = torch.arange(M, device=tokens.device)
        else:
            parents = parents.expand(B, M)
            depth = tree_relations(parents)[1]
        pos = (lengths.view(-1, 1) + depth).clamp(0, self.pos_emb.num_embeddings - 1)
        x = self.emb_dropout(self.token_emb(tokens) + self.pos_emb(pos))
        kvs = []
        for i, (block, cache) in enumerate(zip(self.blocks, caches)):
            x, kv = block.tree_step(x, cache, lengths, parents, None if rws is None else rws[i], checked=True)
            kvs.append(kv)
        if x.is_cuda and caches:  # once, for all layers
            x = torch.where(caches[0].has_room(lengths, M).view(-1, 1, 1), x, math.nan)
        return self._head(x), kvs

    @torch.no_grad()
    def accept(self, caches: list, kvs: list, path: torch.Tensor, count: torch.Tensor, lengths: torch.Tensor):
        """Keeps an accepted path of a tree_step (path, count of ops.verify_drafts): its rows move
        to positions lengths[b], lengths[b] + 1, ... of every layer's cache.  Returns lengths + count.
        (A chain's path is where it belongs already: lengths + count is all it needs.)"""
        for cache, (k, v) in zip(caches, kvs):
            cache.store_rows(k, v, lengths, path, count)
        return lengths + count

    @torch.no_grad()
    def generate_speculative(self, input_ids: torch.Tensor, draft: "MultiscreenLM", max_new_tokens: int = 100,
                             num_drafts: int = 4, temperature: float = 1.0, top_k: int | None = None,
                             cache_dtype: torch.dtype | None = None) -> torch.Tensor:
        """generate() with `draft`, a smaller model of the same vocabulary: it drafts num_drafts tokens
        one by one, this model scores them in one step (tree_step), and ops.verify_drafts keeps those
        that leave the tokens distributed as generate()'s own.  temperature 0 is greedy: the tokens
        of generate_greedy, up to the rounding of logits that nearly tie.  The steps are eager: a
        round takes as long as num_drafts + 1 of generate()'s steps of the two models.

        cache_dtype: as in generate().  Returns (B, T + max_new_tokens) token ids.
        """
        self.eval()
        draft.eval()
        B, T = input_ids.shape
        if not 1 <= num_drafts <= 63:
            raise ValueError(f"num_drafts must be in 1 .. 63, got {num_drafts}")
        if max_new_tokens <= 0:
            return input_ids
        if B == 0:
            return input_ids.new_zeros(0, T + max_new_tokens, dtype=torch.int64)
        end = T + max_new_tokens
        for m in (self, draft):
            if end - 1 > m.pos_emb.num_embeddings:  # the last token is not read again
                raise IndexError(f"{end - 1} positions exceed the model's {m.pos_emb.num_embeddings}")
        if draft.lm_head.out_features != self.lm_head.out_features:
            raise ValueError("the draft model's vocabulary differs")
        dev = input_ids.device
        # room for the drafts behind the last position of a sequence that is done
        both = [(m, m.new_cache(B, end + num_drafts + 1, m._cache_dtype(dev, cache_dtype), dev)) for m in (self, draft)]
        logits = [m.prefill(input_ids, caches) for m, caches in both][0]
        out = torch.cat((input_ids.long(), input_ids.new_zeros(B, max_new_tokens + num_drafts + 1, dtype=torch.int64)), 1)
        lengths = torch.full((B,), T, dtype=torch.int64, device=dev)
        token = self._pick(_probabilities(logits, temperature, top_k))
        out[:, T] = token.squeeze(1)
        at = torch.arange(num_drafts + 1, device=dev)
        verify = ops.verify_drafts if input_ids.is_cuda else verify_dense
        for _ in range(max_new_tokens - 1):
            # the draft's rows of the last two tokens (it has not seen the last accepted one), then on from there
            nodes, probs = [token], []
            step = torch.cat((out.gather(1, lengths.unsqueeze(1) - 1), token), 1)
            for i in range(num_drafts):
                logits, _ = draft.tree_step(step, both[1][1], lengths - 1 if i == 0 else lengths + i)
                probs.append(_probabilities(logits[:, -1], temperature, top_k))
                step = self._pick(probs[-1])
                nodes.append(step)
            nodes = torch.cat(nodes, 1)
            logits, _ = self.tree_step(nodes, both[0][1], lengths)
            if temperature == 0:
                _, count, token = verify(logits, nodes)
            else:
                _, count, token = verify(_probabilities(logits, temperature, top_k), nodes, None,
                                         torch.rand(B, num_drafts + 1, device=dev), torch.stack(probs, 1))
            # the accepted drafts and the token after them; a sequence that is done stays at its last position
            count = torch.where(lengths + 1 < end, count, 0)
            place = lengths.unsqueeze(1) + at
            out.scatter_(1, place, torch.where(at < count.unsqueeze(1), nodes, out.gather(1, place)))
            place = (lengths + count).unsqueeze(1)
            out.scatter_(1, place, torch.where(count.unsqueeze(1) > 0, token.unsqueeze(1), out.gather(1, place)))
            lengths = (lengths + count).clamp(max=end - 1)
            token = out.gather(1, lengths.unsqueeze(1))
            if int(lengths.min()) + 1 >= end:
                break
        return out[:, :end]

    @staticmethod
    def _pick(probs: torch.Tensor) -> torch.Tensor:
        """A token (B, 1) of what _probabilities gives for one row per sequence."""
        return torch.multinomial(probs, num_samples=1) if probs.dtype.is_floating_point else probs

    def _cache_dtype(self, device, cache_dtype=None) -> torch.dtype:
        """The type generate() keeps its rows in: cache_dtype, else the model's (autocast's under it)."""
        if cache_dtype is not None:
            return cache_dtype
        if device.type == "cuda" and torch.is_autocast_enabled("cuda"):
            return torch.get_autocast_dtype("cuda")
        return self.blocks[0].attn.q_proj.weight.dtype

    @torch.no_grad()
    def generate_greedy(self, input_ids: torch.Tensor, max_new_tokens: int = 100,
                        cache_dtype: torch.dtype | None = None) -> torch.Tensor:
        """Greedy decoding (the argmax token; among equal logits the first).

        On GPU the per-token decode step runs as one replayed HIP graph
        (GraphDecoder); on CPU it is the eager loop.  Returns
        (B, T + max_new_tokens) token ids.  generate(top_k=1) samples the same
        distribution but breaks exact ties at random, as the reference does.
        cache_dtype: as in generate()."""
        self.eval()
        B, T = input_ids.shape
        if max_new_tokens <= 0:
            return input_ids
        dtype = cache_dtype or self.blocks[0].attn.q_proj.weight.dtype
        caches = self.new_cache(B, T + max_new_tokens, dtype, input_ids.device)
        logits = self.prefill(input_ids, caches)
        first = logits.argmax(-1, keepdim=True)
        if not input_ids.is_cuda or max_new_tokens == 1:
            out, tok = [input_ids, first], first
            for step in range(1, max_new_tokens):
                tok = self.decode_step(tok, caches, T + step - 1).argmax(-1, keepdim=True)
                out.append(tok)
            return torch.cat(out, dim=1)
        dec = GraphDecoder(self, caches, first, T, max_new_tokens - 1)
        for _ in range(max_new_tokens - 1):
            dec.step()
        return torch.cat([input_ids, first, dec.tokens], dim=1)

    @torch.no_grad()
    def generate(self, input_ids: torch.Tensor, max_new_tokens: int = 100, temperature: float = 1.0,
                 top_k: int | None = None, cache_dtype: torch.dtype | None = None) -> torch.Tensor:
        """Temperature / top-k sampling (top_k=1 is greedy).

        cache_dtype: type of the cached rows; None: the model's own; torch.int8 or
        torch.float8_e4m3fn: 8-bit codes (KVCache).
        Returns (B, T + max_new_tokens) token ids.
        """
        self.eval()
        B, T = input_ids.shape
        if max_new_tokens <= 0:
            return input_ids
        caches = self.new_cache(B, T + max_new_tokens, self._cache_dtype(input_ids.device, cache_dtype), input_ids.device)
        logits = self.prefill(input_ids, caches)
        out = [input_ids]
        pos = T
        for step in range(max_new_tokens):
            logits = logits / temperature
            if top_k is not None:
                values, _ = torch.topk(logits, top_k)
                logits[logits < values[:, -1:]] = float("-inf")
            probs = F.softmax(logits, dim=-1)
            next_token = torch.multinomial(probs, num_samples=1)
            out.append(next_token)
            if step + 1 < max_new_tokens:
                logits = self.decode_step(next_token, caches, pos)
                pos += 1
        return torch.cat(out, dim=1)


def _probabilities(logits, temperature, top_k):
    """Sampling probabilities (float32) of logits (..., vocab) as generate() forms them; at temperature 0
    the first largest entry's index (..., 1)."""
    if temperature == 0:
        return logits.argmax(-1, keepdim=True)
    logits = logits / temperature
    if top_k is not None:
        values, _ = torch.topk(logits, top_k)
        logits = logits.masked_fill(logits < values[..., -1:], float("-inf"))
    return F.softmax(logits.float(), dim=-1)


class GraphDecoder:
    """Greedy decode steps of a MultiscreenLM, captured once as a HIP graph and
    replayed per token.

    One step embeds the token in `token` at the position in `pos` (device
    tensors), runs every layer's cache write and single-query decode
    (msa_decode_at reads the position on the device), the final norm and head,
    writes the argmax into `token` and into `tokens[:, n]` (n a device
    counter) and advances `pos` and n.  Every launch depends only on shapes,
    so the captured graph replays unchanged as the sequence grows; r and w of
    every layer are read once here (the model does not change while it
    decodes).  The first step runs eagerly before the capture: it warms the
    allocator and the kernels up, and the step the capture records overwrites
    its cache writes with the same values.
    """

    def __init__(self, lm, caches, token, pos: int, steps: int):
        if not token.is_cuda:
            raise RuntimeError("GraphDecoder needs the model and caches on the GPU")
        cap = caches[0].k.shape[1]
        if pos + steps > cap:
            raise IndexError(f"KV cache capacity {cap} is below {pos + steps} positions")
        dev = token.device
        self.lm, self.caches, self.steps, self.done = lm, caches, steps, 0
        self.token = token.detach().clone()
        self.pos = torch.tensor([pos], dtype=torch.int64, device=dev)
        self.n = torch.zeros(1, dtype=torch.int64, device=dev)
        self.tokens = torch.zeros((token.shape[0], max(steps, 1)), dtype=token.dtype, device=dev)
        with torch.no_grad():
            self.rws = [(b.attn.sharpness().detach().float().contiguous(),
                         b.attn.window().detach().float().contiguous()) for b in lm.blocks]
        # warm-up: one eager step on a side stream, then the state put back
        tok0, pos0 = self.token.clone(), self.pos.clone()
        side = torch.cuda.Stream(device=dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            self._body()
        torch.cuda.current_stream(dev).wait_stream(side)
        self.token.copy_(tok0)
        self.pos.copy_(pos0)
        self.n.zero_()
        torch.cuda.synchronize(dev)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.logits = self._body()

    @torch.no_grad()
    def _body(self):
        logits = self.lm.decode_step(self.token, self.caches, self.pos, self.rws)
        nxt = logits.argmax(-1, keepdim=True)
        self.token.copy_(nxt)
        self.tokens.index_copy_(1, self.n, nxt)
        self.pos.add_(1)
        self.n.add_(1)
        return logits

    def step(self):
        """Decodes one token; returns the (B, 1) token tensor (overwritten by the
        next step) -- its logits are in self.logits."""
        if self.done >= self.steps:
            raise IndexError("GraphDecoder: all planned steps are done")
        self.graph.replay()
        self.done += 1
        return self.token
