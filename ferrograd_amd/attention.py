"""A self-attention layer over the hand-written kernels (no reference
counterpart), for sequences held as matrices of one row per token."""
from __future__ import annotations

from . import Dropout, FerrogradError, Linear, Tensor


class SelfAttention:
    """Linear projections to queries, keys and values; the norm of each of their
    heads with the rotation of its position (Tensor.norm_rotate, with a weight
    for the queries' and one for the keys'); attention (Tensor.attention); a
    Linear projection back, and dropout while train() is on (as it is at first).

    `kv_heads` key heads (default: `heads`) are shared by the query heads in
    equal groups. `head_dim` (default: features / heads) is even and at most
    128."""

    def __init__(self, features: int, heads: int, kv_heads: int | None = None, head_dim: int | None = None, device=None,
                 causal: bool = True, dropout: float = 0.0, seed: int = 42, eps: float = 1e-6, base: float = 10000.0):
        if heads < 1:
            raise FerrogradError(f"SelfAttention: there must be at least one head, got {heads}")
        if head_dim is None:
            if features % heads:
                raise FerrogradError(f"SelfAttention: {features} features do not split into {heads} heads")
            head_dim = features // heads
        if head_dim % 2 or not 2 <= head_dim <= 128:
            raise FerrogradError(f"SelfAttention: the head size must be even and at most 128, got {head_dim}")
        self.heads, self.kv_heads = heads, heads if kv_heads is None else kv_heads
        if self.kv_heads < 1 or heads % self.kv_heads:
            raise FerrogradError(f"SelfAttention: {heads} heads do not share {self.kv_heads} key heads evenly")
        self.causal, self.eps, self.base = causal, eps, base
        self.query = Linear(features, heads * head_dim, device, bias=False)
        self.key = Linear(features, self.kv_heads * head_dim, device, bias=False)
        self.value = Linear(features, self.kv_heads * head_dim, device, bias=False)
        self.out = Linear(heads * head_dim, features, device, bias=False)
        self.query_norm = Tensor.ones([head_dim], device).with_requires_grad(True)
        self.key_norm = Tensor.ones([head_dim], device).with_requires_grad(True)
        self.dropout = Dropout(dropout, seed)

    def forward(self, x: Tensor, positions: Tensor, batch: int = 1, lengths: Tensor | None = None) -> Tensor:
        """x [batch * length, features] with each row's position (int32 [batch *
        length]); `lengths` (int32 [batch]) hides each sequence's padding."""
        q = self.query(x).norm_rotate(self.query_norm, positions, self.heads, self.eps, self.base)
        k = self.key(x).norm_rotate(self.key_norm, positions, self.kv_heads, self.eps, self.base)
        y = q.attention(k, self.value(x), self.heads, self.kv_heads, batch, self.causal, lengths)
        return self.dropout(self.out(y))

    __call__ = forward

    def train(self, on: bool = True) -> "SelfAttention":
        """Turn dropout on or off."""
        self.dropout.training = on
        return self

    def parameters(self) -> list:
        return [p for layer in (self.query, self.key, self.value, self.out) for p in layer.parameters()] + [
            self.query_norm, self.key_norm]
