"""KAN transformer: its feed-forward block (reference kanforge/torch/transformer.py:25-52)
and the stack of attention, norms and feed-forward blocks around it.

``KANFFN(dim, hidden, kind, ...)`` maps dim -> hidden -> dim with two KAN
layers and dropout after each:

* ``kind="grkan"``: KAT's two group-rational layers, the first rational
  starting as the identity and the second as ``activation`` (their linear
  maps run on the GR-KAN tensor-core kernels for bf16, on the three-TF32
  GEMM for float32); ``kan_kwargs`` do not apply to them, as in the reference;
* ``kind="kan"``: two KANLinear layers of ``basis`` with ``kan_kwargs``.

``KANTransformer`` runs whole packed sequences (training, and the prompts of a
``KVCache``) and single tokens over that cache.
"""

from __future__ import annotations

import math

import torch
from torch import nn

from .attention import ATTENTION_MAX_DIM, PackedSequences, RelativeBias, attention, attention_decode
from .layers import GRKAN, KANLinear
from .norm import ResidualNorm

FFN_KINDS = ("grkan", "kan")


def _ffn_layers(kind: str, dim: int, hidden: int, basis, groups: int, activation: str, kan_kwargs: dict):
    if kind == "grkan":
        return (GRKAN(dim, hidden, groups=groups, init="identity"), GRKAN(hidden, dim, groups=groups, init=activation))
    if kind == "kan":
        return KANLinear(dim, hidden, basis, **kan_kwargs), KANLinear(hidden, dim, basis, **kan_kwargs)
    raise ValueError("kind must be 'grkan' or 'kan'")


class KANFFN(nn.Module):
    """dim -> hidden (default 4 dim) -> dim with KAN layers; attributes ``fc1``,
    ``fc2`` and ``drop`` as in the reference, so state dicts carry over."""

    def __init__(self, dim: int, hidden: int | None = None, kind: str = "grkan", basis="bspline", groups: int = 8,
                 activation: str = "gelu", dropout: float = 0.0, **kan_kwargs):
        super().__init__()
        self.fc1, self.fc2 = _ffn_layers(kind, dim, hidden or 4 * dim, basis, groups, activation, kan_kwargs)
        self.drop = nn.Dropout(dropout)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        h = self.drop(self.fc1(x))
        return self.drop(self.fc2(h))


class KVCache:
    """Keys and values of every layer of a ``KANTransformer`` for a batch of
    sequences, (depth, batch, capacity, kv_heads, head width) each, and how many
    slots of each sequence are filled (``lengths``, int32 on the device).

    Steps in a CUDA graph are counted on the device alone: a replay past the
    capacity leaves ``lengths`` above it, touches the sequence's last slot and no
    other memory, and ``KANTransformer.decode`` answers NaN for that sequence."""

    def __init__(self, depth: int, batch: int, capacity: int, kv_heads: int, head_dim: int, *, device=None, dtype=None):
        if min(depth, batch, capacity) < 1:
            raise ValueError("a cache needs at least one layer, sequence and slot")
        self.k = torch.empty(depth, batch, capacity, kv_heads, head_dim, device=device, dtype=dtype)
        self.v = torch.empty_like(self.k)
        self.lengths = torch.zeros(batch, device=device, dtype=torch.int32)
        self.batch, self.capacity = batch, capacity
        self.longest = 0  # of ``lengths``, known on the host
        self._rows = torch.arange(batch, device=device)
        self._last = torch.full((batch,), capacity - 1, device=device)

    def begin(self, lens: list[int]) -> tuple[torch.Tensor, torch.Tensor]:
        """Starts the sequences anew with prompts of these lengths: (sequence, slot) of each packed row."""
        if len(lens) != self.batch or min(lens) < 0 or max(lens) > self.capacity:
            raise ValueError(f"{len(lens)} prompts of up to {max(lens, default=0)} tokens do not fit a cache of {self.batch} "
                             f"sequences with {self.capacity} slots")
        self.longest = max(lens)
        seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
        slot = torch.cat([torch.arange(n) for n in lens])
        self.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        return seq.to(self.k.device), slot.to(self.k.device)

    def step(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Room for one more token of every sequence: its (sequence, slot) rows."""
        if self.longest >= self.capacity:
            raise ValueError(f"the cache is full: {self.capacity} slots")
        if not (self.lengths.is_cuda and torch.cuda.is_current_stream_capturing()):
            self.longest += 1
        slot = torch.minimum(self.lengths, self._last)  # within the cache, whatever the host missed
        self.lengths += 1
        return self._rows, slot


class KANTransformerBlock(nn.Module):
    """Attention and a KANFFN, each joined to the residual stream by the norm that
    also makes the next one's input (``ResidualNorm``)."""

    def __init__(self, dim: int, heads: int, kv_heads: int | None = None, hidden: int | None = None, *, norm: str = "layer",
                 branch_norm: bool = False, gate_init: float | None = None, **ffn_kwargs):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or dim % heads or dim // heads % 8 or dim // heads > ATTENTION_MAX_DIM:
            raise ValueError(f"dim / heads must be a multiple of 8 up to {ATTENTION_MAX_DIM} (got {dim} and {heads})")
        if kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"{heads} query heads do not divide over {kv_heads} key heads")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, dim // heads
        self.qkv = nn.Linear(dim, (heads + 2 * kv_heads) * self.head_dim, bias=False)
        self.proj = nn.Linear(dim, dim, bias=False)
        self.ffn = KANFFN(dim, hidden, **ffn_kwargs)
        self.attention_norm = ResidualNorm(dim, norm, branch_norm=branch_norm, gate_init=gate_init)
        self.ffn_norm = ResidualNorm(dim, norm, branch_norm=branch_norm, gate_init=gate_init)

    def forward(self, x: torch.Tensor, h: torch.Tensor, attend) -> tuple[torch.Tensor, torch.Tensor]:
        """(x, h) after the block: the stream and its norm; ``attend(q, k, v)`` is (tokens, heads, head width)."""
        q, k, v = self.qkv(h).unflatten(-1, (-1, self.head_dim)).split([self.heads, self.kv_heads, self.kv_heads], dim=-2)
        x, h = self.attention_norm(x, self.proj(attend(q, k, v).flatten(-2)))
        return self.ffn_norm(x, self.ffn(h))


class KANTransformer(nn.Module):
    """A stack of ``depth`` KANTransformerBlocks over (tokens, dim) rows of packed
    sequences; all layers share one ``RelativeBias`` unless ``num_buckets`` is 0.
    Further arguments are KANTransformerBlock's and its KANFFN's.

    ``model(x, seqs)`` gives the normed rows of every token, with gradients;
    ``model.prefill(x, lens, cache)`` gives the same for the prompts of a batch
    and fills the cache, after which ``model.decode(x, cache)`` takes one new
    token of every sequence, (batch, dim).
    """

    def __init__(self, dim: int, depth: int, heads: int, kv_heads: int | None = None, hidden: int | None = None, *,
                 norm: str = "layer", causal: bool = True, num_buckets: int = 32, max_distance: int = 128, **block_kwargs):
        super().__init__()
        if depth < 1:
            raise ValueError("depth must be positive")
        self.causal = causal
        self.start = ResidualNorm(dim, norm)
        self.blocks = nn.ModuleList(
            KANTransformerBlock(dim, heads, kv_heads, hidden, norm=norm, **block_kwargs) for _ in range(depth))
        self.bias = RelativeBias(heads, num_buckets, max_distance, bidirectional=not causal) if num_buckets else None

    def _run(self, x: torch.Tensor, attend) -> torch.Tensor:
        x, h = self.start(x)
        for i, block in enumerate(self.blocks):
            x, h = block(x, h, lambda q, k, v, i=i: attend(i, q, k, v))
        return h

    def forward(self, x: torch.Tensor, seqs: PackedSequences) -> torch.Tensor:
        return self._run(x, lambda i, q, k, v: attention(q, k, v, seqs, causal=self.causal, bias=self.bias))

    def new_cache(self, batch: int, capacity: int) -> KVCache:
        block, weight = self.blocks[0], self.start.weight
        return KVCache(len(self.blocks), batch, capacity, block.kv_heads, block.head_dim, device=weight.device, dtype=weight.dtype)

    def _serve(self, x: torch.Tensor, rows: int, cache: KVCache) -> None:
        """The refusals, before the cache is touched."""
        if not self.causal:
            raise ValueError("a model that sees later tokens has no cache")
        block = self.blocks[0]
        if cache.k.shape != (len(self.blocks), cache.batch, cache.capacity, block.kv_heads, block.head_dim):
            raise ValueError(f"a cache of shape {tuple(cache.k.shape)} is not this model's: {len(self.blocks)} layers, "
                             f"{block.kv_heads} key heads of {block.head_dim}")
        if cache.k.device != x.device:
            raise ValueError(f"the cache lies on {cache.k.device}, the tokens on {x.device}")
        if x.shape != (rows, self.start.dim):
            raise ValueError(f"x must be ({rows}, {self.start.dim}), not {tuple(x.shape)}")

    @torch.no_grad()
    def prefill(self, x: torch.Tensor, lens: list[int], cache: KVCache) -> torch.Tensor:
        self._serve(x, sum(lens), cache)
        at, seqs = cache.begin(lens), PackedSequences(lens, device=x.device)

        def attend(i, q, k, v):
            cache.k[i][at], cache.v[i][at] = k, v
            return attention(q, k, v, seqs, bias=self.bias)

        return self._run(x, attend)

    @torch.no_grad()
    def decode(self, x: torch.Tensor, cache: KVCache) -> torch.Tensor:
        self._serve(x, cache.batch, cache)
        at = cache.step()

        def attend(i, q, k, v):
            cache.k[i][at], cache.v[i][at] = k, v
            return attention_decode(q, cache.k[i], cache.v[i], cache.lengths, bias=self.bias)

        h = self._run(x, attend)
        return torch.where((cache.lengths > cache.capacity)[:, None], math.nan, h)
