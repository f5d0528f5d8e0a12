"""Attention over behaviour sequences, on the output of ``SequenceEmbeddingFeatures``.  The reference hands un-pooled sequences out
(tensornet/layers/sequence_embedding_features.py:35-234) and leaves what reads them to TensorFlow."""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from ..ops import functional as F
from .dense import _glorot_aug
from .normalization_layer import LayerNormalization


class SequenceAttention(nn.Module):
    """One attention block in front of whose projections the rows are normalised.

    * ``layer(x, lengths)``: ``x + attention(norm(x)) W_o`` of ``[B, T, dim]`` sequences, ``lengths[b]`` rows each (None: all).  Rows
      behind a length, which have to be finite, come back as they were.
    * ``layer(x, lengths, target)``: what targets ``[B, dim]`` or ``[B, n, dim]`` (candidate items, say) gather from the
      sequence, ``target + attention(norm(target), norm(x)) W_o``, each by itself: all stand at the sequence's last row.

    Projections are bf16 products with biases, attention is :func:`tensornet_b200.ops.functional.attention`: ``heads`` of
    ``head_dim`` columns (``dim // heads``, a multiple of 8), ``kv_heads`` of them for keys and values.  ``causal``: a row sees
    itself and the rows before it; ``prefix`` (int32 ``[B]``, call without targets) rows are seen by all the same.  ``cap`` bounds the scores,
    ``distance_bias`` lets them fall with the distance, by ``2^(-8 (h + 1) / heads)`` per row in head ``h``."""

    def __init__(self, dim: int, heads: int = 4, kv_heads: Optional[int] = None, head_dim: Optional[int] = None, causal: bool = False,
                 cap: Optional[float] = None, distance_bias: bool = False, epsilon: float = 1e-5, name: Optional[str] = None):
        super().__init__()
        self.dim, self.heads, self.kv_heads = int(dim), int(heads), int(kv_heads or heads)
        self.head_dim = int(head_dim or self.dim // self.heads)
        if self.head_dim % 8 or not 8 <= self.head_dim <= 128:
            raise ValueError(f"SequenceAttention: 8 to 128 columns per head, a multiple of 8, not {self.head_dim}")
        if self.heads < 1 or self.heads % self.kv_heads:
            raise ValueError(f"SequenceAttention: {self.heads} heads are no multiple of {self.kv_heads} kv_heads")
        self.causal, self.cap, self.distance_bias, self.epsilon = bool(causal), cap, bool(distance_bias), float(epsilon)
        self.layer_name = name or "sequence_attention"
        self.norm = LayerNormalization(self.dim, epsilon=epsilon, name=self.layer_name + "_norm")
        wide, kv = self.heads * self.head_dim, self.kv_heads * self.head_dim
        self.query = nn.Parameter(_glorot_aug(wide, self.dim))
        self.key_value = nn.Parameter(_glorot_aug(2 * kv, self.dim))
        self.output = nn.Parameter(_glorot_aug(self.dim, wide))
        slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / self.heads) for h in range(self.heads)]) if distance_bias else None
        self.register_buffer("slopes", slopes, persistent=False)

    def get_config(self) -> dict:
        return {"dim": self.dim, "heads": self.heads, "kv_heads": self.kv_heads, "head_dim": self.head_dim, "causal": self.causal,
                "cap": self.cap, "distance_bias": self.distance_bias, "epsilon": self.epsilon, "name": self.layer_name}

    @staticmethod
    def _heads_of(rows: torch.Tensor, lead, n: int, columns: int, first: int = 0) -> torch.Tensor:
        return rows[:, first * columns:(first + n) * columns].unflatten(0, lead).unflatten(-1, (n, columns))

    def forward(self, x: torch.Tensor, lengths: Optional[torch.Tensor] = None, target: Optional[torch.Tensor] = None,
                prefix: Optional[torch.Tensor] = None) -> torch.Tensor:
        if x.dim() != 3 or x.shape[-1] != self.dim:
            raise ValueError(f"{self.layer_name}: sequences [B, T, {self.dim}], not {tuple(x.shape)}")
        if target is not None and (target.dim() not in (2, 3) or target.shape[0] != x.shape[0] or target.shape[-1] != self.dim):
            raise ValueError(f"{self.layer_name}: targets [{x.shape[0]}, (n,) {self.dim}], not {tuple(target.shape)}")
        if target is not None and prefix is not None:
            raise ValueError(f"{self.layer_name}: targets see all of their sequence, a prefix goes with the sequence's own rows")
        lead, D = x.shape[:2], self.head_dim
        asks = x if target is None else target.unsqueeze(1) if target.dim() == 2 else target
        if asks.numel() == 0 or (target is None and x.numel() == 0):
            return x if target is None else target
        if lengths is not None:
            lengths = lengths.to(x.device, torch.int32)

        def projected(rows, weight):
            return F.mlp(rows, [weight], self.dim, relu_last=False)

        rows = F.concat_cast([self.norm(x).reshape(-1, self.dim)]) if x.numel() else None
        asking = rows if target is None else F.concat_cast([self.norm(asks).reshape(-1, self.dim)])
        q = self._heads_of(projected(asking, self.query), asks.shape[:2], self.heads, D)
        if rows is None:
            k = v = q.new_zeros((*lead, self.kv_heads, D))
        else:
            kv = projected(rows, self.key_value)
            k, v = [self._heads_of(kv, lead, self.kv_heads, D, i * self.kv_heads) for i in range(2)]
        out = F.attention(q, k, v, lengths=lengths if target is None else None, kv_lengths=lengths, causal=self.causal and target is None,
                          prefix=prefix, cap=self.cap, slopes=self.slopes, newest=target is not None)
        y = F.mlp(F.concat_cast([out.reshape(-1, self.heads * D)]), [self.output], self.heads * D, relu_last=False)
        y = y[:, :self.dim].float().view(asks.shape)
        if target is None and lengths is not None:
            y = y * (torch.arange(lead[1], device=x.device) < lengths.unsqueeze(1)).unsqueeze(-1)
        return asks + y if target is None else (asks + y).view(target.shape)
