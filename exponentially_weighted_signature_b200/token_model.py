"""A token model on the package's operators: the embedding, residual blocks whose mixer is a decayed linear attention, a gated
linear recurrence or an EWS block, and the vocabulary loss on the tied table. One module for training (``loss``, from a
teacher ``distill``), prompts (``prompt``) and single tokens (``step``), so that the operators run together as they are meant to.

The reference's stacked model takes tokens through an embedding (ews/block.py:473-600, ``tokens=True``); the decayed
attention blocks keep a matrix state a head, the gated blocks one number a channel, that a served request carries from token to
token, which the EWS blocks' prefix scan does not, so ``prompt`` and ``step`` need a model without EWS blocks.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn.functional as F
from torch import nn

from .block import EWSBlock, RMSNorm
from .gated_ops import gated_linear
from .recur_ops import gated_recurrence, gated_recurrence_step
from .token_ops import decayed_attention, decayed_attention_step, distill_loss, token_embedding, vocab_loss


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

    def states(self, slots: int):
        return torch.zeros(slots, self.heads, self.head_dim, self.head_dim, device=self.out.weight.device)


class GatedBlock(nn.Module):
    """Pre-norm residual block: RMSNorm -> input, decay gate, input gate -> gated recurrence -> projection -> residual -> RMSNorm ->
    gated linear layer -> projection -> residual. The channels' rates are learned (their logarithms, float32 in the recurrence),
    at first 1 to 2^-8: half-open gates forget over 2 to 512 tokens. ``width``: the recurrence's channels (hidden_dim);
    ``ff_dim``: the channel stage's (8/3 hidden_dim, in steps of 8: as many weights as an MLP of four times the width)."""

    def __init__(self, hidden_dim: int, width: Optional[int] = None, ff_dim: Optional[int] = None, *, activation: str = "silu",
                 norm_eps: float = 1e-6):
        super().__init__()
        self.width, self.activation = int(width or hidden_dim), activation
        ff = int(ff_dim or -(-hidden_dim // 3) * 8)
        self.norm1, self.norm2 = RMSNorm(hidden_dim, eps=norm_eps), RMSNorm(hidden_dim, eps=norm_eps)
        self.inputs = nn.Linear(hidden_dim, 3 * self.width, bias=False)
        self.out = nn.Linear(self.width, hidden_dim, bias=False)
        self.log_rate = nn.Parameter(-math.log(2.0) * torch.linspace(0.0, 8.0, self.width))
        self.ff_gate, self.ff_up = nn.Linear(hidden_dim, ff, bias=False), nn.Linear(hidden_dim, ff, bias=False)
        self.ff_down = nn.Linear(ff, hidden_dim, bias=False)

    def _mixer(self, x):
        """The recurrence's x, decay, gate and rate."""
        return (*self.inputs(self.norm1(x)).split(self.width, -1), torch.exp(self.log_rate.float()))

    def _close(self, x, h):
        x = x + self.out(h)
        return x + self.ff_down(gated_linear(self.norm2(x), self.ff_gate.weight, self.ff_up.weight, activation=self.activation))

    def forward(self, x, lengths=None, state=None, return_state=False):
        got = gated_recurrence(*self._mixer(x), initial_state=state, lengths=lengths, return_state=return_state)
        return (self._close(x, got[0]), got[1]) if return_state else self._close(x, got)

    def step(self, x, state, slots=None):
        return self._close(x, gated_recurrence_step(*self._mixer(x), state, slots=slots))

    def states(self, slots: int):
        return torch.zeros(slots, self.width, device=self.out.weight.device)


class TokenModel(nn.Module):
    """Embedding (scaled by sqrt(hidden)), blocks, RMSNorm, and logits on the embedding's table.

    ``mixers``: one entry a block, "decay" (DecayBlock), "gated" (GatedBlock with ``gated_kwargs``) or "ews" (EWSBlock with
    ``ews_kwargs``; float32). ``seed`` is for the table and the EWS blocks' generators; linear layers draw from torch's global
    generator, as in ``StackedEWS``."""

    def __init__(self, vocab: int, hidden_dim: int = 128, heads: int = 4, mixers=("decay", "decay"), *,
                 kv_heads: Optional[int] = None, head_dim: Optional[int] = None, ews_kwargs: Optional[dict] = None,
                 gated_kwargs: Optional[dict] = None, seed: int = 0):
        super().__init__()
        g = torch.Generator().manual_seed(int(seed))
        self.vocab, self.hidden_dim = int(vocab), int(hidden_dim)
        self.table = nn.Parameter(torch.randn(self.vocab, self.hidden_dim, generator=g) / math.sqrt(self.hidden_dim))
        blocks = []
        for kind in mixers:
            if kind == "decay":
                blocks.append(DecayBlock(hidden_dim, heads, kv_heads, head_dim))
            elif kind == "gated":
                blocks.append(GatedBlock(hidden_dim, **(gated_kwargs or {})))
            elif kind == "ews":
                blocks.append(EWSBlock(hidden_dim, generator=g, **(ews_kwargs or {})))
            else:
                raise ValueError(f"a mixer is 'decay', 'gated' or 'ews', got {kind!r}")
        self.blocks = nn.ModuleList(blocks)
        self.norm = RMSNorm(hidden_dim)

    def _served(self):
        for block in self.blocks:
            if not isinstance(block, (DecayBlock, GatedBlock)):
                raise NotImplementedError("prompt and step need a model of decayed attention and gated blocks alone")

    def hidden(self, ids, lengths=None):
        """(B, T) ids -> the normalised hidden rows (B, T, hidden)."""
        x = token_embedding(ids, self.table, scale=math.sqrt(self.hidden_dim))
        for block in self.blocks:
            x = block(x, lengths) if isinstance(block, (DecayBlock, GatedBlock)) else block(x)
        return self.norm(x)

    def loss(self, ids, targets, lengths=None, ignore_index: int = -100):
        """Mean loss over the positions that have a target."""
        losses = vocab_loss(self.hidden(ids, lengths), self.table, targets, ignore_index=ignore_index)
        return losses.sum() / (targets != ignore_index).sum().clamp(min=1)

    def distill(self, ids, teacher_ids, teacher_logits, lengths=None, temperature: float = 1.0):
        """temperature^2 times the mean divergence from a teacher's top logits (B, T, K) over the positions that have any; an entry
        with a negative id is absent."""
        losses = distill_loss(self.hidden(ids, lengths), self.table, teacher_ids, teacher_logits, temperature=temperature)
        there = ((teacher_ids >= 0) & (teacher_logits != -math.inf)).any(-1).sum()
        return temperature**2 * losses.sum() / there.clamp(min=1)

    def states(self, slots: int):
        """Zero states for ``slots`` requests, one pool a block."""
        self._served()
        return [b.states(slots) for b in self.blocks]

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
