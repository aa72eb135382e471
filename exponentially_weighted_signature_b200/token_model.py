"""A token model on the package's operators: the embedding, residual blocks whose mixer is a decayed linear attention or
an EWS block, and the vocabulary loss on the tied table. One module for training (``loss``), prompts (``prompt``) and
single tokens (``step``), so that the operators run together as they are meant to.

The reference's stacked model takes tokens through an embedding (ews/block.py:473-600, ``tokens=True``); the decayed
attention blocks keep a matrix state a head that a served request carries from token to token, which the EWS blocks'
prefix scan does not, so ``prompt`` and ``step`` need a model of attention blocks alone.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn.functional as F
from torch import nn

from .block import EWSBlock, RMSNorm
from .token_ops import decayed_attention, decayed_attention_step, token_embedding, vocab_loss


class DecayBlock(nn.Module):
    """Pre-norm residual block: RMSNorm -> q, k, v -> decayed attention -> projection -> residual -> RMSNorm -> MLP ->
    residual. The heads' rates are constants, 2^-1 to 2^-9 a token (windows of 2 to 512 tokens)."""

    def __init__(self, hidden_dim: int, heads: int, kv_heads: Optional[int] = None, head_dim: Optional[int] = None, *,
                 ff_mult: int = 4, norm_eps: float = 1e-6):
        super().__init__()
        self.heads, self.kv_heads = int(heads), int(kv_heads or heads)
        self.head_dim = int(head_dim or hidden_dim // heads)
        self.norm1, self.norm2 = RMSNorm(hidden_dim, eps=norm_eps), RMSNorm(hidden_dim, eps=norm_eps)
        self.qkv = nn.Linear(hidden_dim, (self.heads + 2 * self.kv_heads) * self.head_dim, bias=False)
        self.out = nn.Linear(self.heads * self.head_dim, hidden_dim, bias=False)
        self.ff1 = nn.Linear(hidden_dim, ff_mult * hidden_dim)
        self.ff2 = nn.Linear(ff_mult * hidden_dim, hidden_dim)
        self.register_buffer("rate", self._rates().to(self.qkv.weight.device), persistent=False)

    def _rates(self):
        return torch.exp2(-torch.linspace(1.0, 9.0, self.heads, device="cpu"))

    def _apply(self, fn, recurse=True):
        """A change of type, or memory without contents, is for the weights: the rates keep their float32 values and only
        follow to the device (a model's decays are the same in every type; on the meta device they have no values yet)."""
        rate = self.rate
        super()._apply(fn, recurse)
        device = self.rate.device
        self.rate = (self._rates() if rate.is_meta else rate).to(device)
        return self

    def _heads(self, x):
        y = self.qkv(self.norm1(x)).unflatten(-1, (-1, self.head_dim))
        return y.split([self.heads, self.kv_heads, self.kv_heads], -2)

    def _close(self, x, o):
        x = x + self.out(o.flatten(-2))
        return x + self.ff2(F.gelu(self.ff1(self.norm2(x))))

    def forward(self, x, lengths=None, state=None, return_state=False):
        q, k, v = self._heads(x)
        got = decayed_attention(q, k, v, self.rate, initial_state=state, lengths=lengths, return_state=return_state)
        return (self._close(x, got[0]), got[1]) if return_state else self._close(x, got)

    def step(self, x, state, slots=None):
        q, k, v = self._heads(x)
        return self._close(x, decayed_attention_step(q, k, v, self.rate, state, slots=slots))


class TokenModel(nn.Module):
    """Embedding (scaled by sqrt(hidden)), blocks, RMSNorm, and logits on the embedding's table.

    ``mixers``: one entry a block, "decay" (DecayBlock) or "ews" (EWSBlock with ``ews_kwargs``; float32). ``seed`` is for the
    table and the EWS blocks' generators; linear layers draw from torch's global generator, as in ``StackedEWS``."""

    def __init__(self, vocab: int, hidden_dim: int = 128, heads: int = 4, mixers=("decay", "decay"), *,
                 kv_heads: Optional[int] = None, head_dim: Optional[int] = None, ews_kwargs: Optional[dict] = None, seed: int = 0):
        super().__init__()
        g = torch.Generator().manual_seed(int(seed))
        self.vocab, self.hidden_dim = int(vocab), int(hidden_dim)
        self.table = nn.Parameter(torch.randn(self.vocab, self.hidden_dim, generator=g) / math.sqrt(self.hidden_dim))
        blocks = []
        for kind in mixers:
            if kind == "decay":
                blocks.append(DecayBlock(hidden_dim, heads, kv_heads, head_dim))
            elif kind == "ews":
                blocks.append(EWSBlock(hidden_dim, generator=g, **(ews_kwargs or {})))
            else:
                raise ValueError(f"a mixer is 'decay' or 'ews', got {kind!r}")
        self.blocks = nn.ModuleList(blocks)
        self.norm = RMSNorm(hidden_dim)

    def _served(self):
        for block in self.blocks:
            if not isinstance(block, DecayBlock):
                raise NotImplementedError("prompt and step need a model of decayed attention blocks alone")

    def hidden(self, ids, lengths=None):
        """(B, T) ids -> the normalised hidden rows (B, T, hidden)."""
        x = token_embedding(ids, self.table, scale=math.sqrt(self.hidden_dim))
        for block in self.blocks:
            x = block(x, lengths) if isinstance(block, DecayBlock) else block(x)
        return self.norm(x)

    def loss(self, ids, targets, lengths=None, ignore_index: int = -100):
        """Mean loss over the positions that have a target."""
        losses = vocab_loss(self.hidden(ids, lengths), self.table, targets, ignore_index=ignore_index)
        return losses.sum() / (targets != ignore_index).sum().clamp(min=1)

    def states(self, slots: int):
        """Zero states for ``slots`` requests, one pool a block."""
        self._served()
        return [torch.zeros(slots, b.heads, b.head_dim, b.head_dim, device=self.table.device) for b in self.blocks]

    @torch.no_grad()
    def prompt(self, ids, lengths=None):
        """Logits after each sample's last token, and the blocks' states there (lengths of at least one)."""
        self._served()
        x, states = token_embedding(ids, self.table, scale=math.sqrt(self.hidden_dim)), []
        for block in self.blocks:
            x, s = block(x, lengths, return_state=True)
            states.append(s)
        last = x[:, -1] if lengths is None else x[torch.arange(len(x), device=x.device), lengths.long() - 1]
        return self.norm(last) @ self.table.T, states

    @torch.no_grad()
    def step(self, ids, states, slots=None):
        """One token (B,) a row on the states (updated in place), each row's in ``slots`` (-1: idle): logits (B, vocab)."""
        self._served()
        x = token_embedding(ids, self.table, scale=math.sqrt(self.hidden_dim))
        for block, s in zip(self.blocks, states):
            x = block.step(x, s, slots)
        return self.norm(x) @ self.table.T
