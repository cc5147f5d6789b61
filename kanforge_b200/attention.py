"""Attention of a KAN transformer: packed sequences, a learned relative position
bias, and the single-token form over a cache.

``attention`` runs whole prompts of different lengths packed into one batch,
causal or both ways, with query heads that share key heads, forward and
backward (``kf_attention_fwd`` / ``kf_attention_bwd``); ``RelativeBias`` adds
its bucketed bias to the scores inside those kernels, so that no (query, key)
matrix ever exists; ``attention_decode`` answers with one token per sequence
(``kf_attention_decode``).
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .kernels import _check_cuda, _launch, _unwatched

ATTENTION_MAX_DIM = 128
BIAS_MAX_DISTANCE, BIAS_MAX_BUCKETS = 512, 256

_DTYPE_CODE = {torch.float32: _lib.KF_DTYPE_F32, torch.bfloat16: _lib.KF_DTYPE_BF16}


class PackedSequences:
    """The lengths of sequences packed one after another, as the kernels read them.

    ``q_lens`` are the query rows of each sequence and ``kv_lens`` (default: the
    same) its key and value rows; a sequence's queries stand at the last of its
    positions.  Zero lengths are allowed.  Build it once for a batch layout and
    pass it to every layer's call, on any stream; the tables lie on ``device``.
    A CUDA graph that holds such a call needs it kept, as it does the tensors.
    """

    def __init__(self, q_lens, kv_lens=None, device="cuda"):
        self.q_lens = [int(n) for n in q_lens]
        self.kv_lens = list(self.q_lens) if kv_lens is None else [int(n) for n in kv_lens]
        if len(self.q_lens) != len(self.kv_lens):
            raise ValueError(f"{len(self.q_lens)} query lengths and {len(self.kv_lens)} key lengths")
        if any(n < 0 for n in self.q_lens + self.kv_lens):
            raise ValueError("lengths must not be negative")
        self.total_q, self.total_kv = sum(self.q_lens), sum(self.kv_lens)
        if max(self.total_q, self.total_kv) >= 2**31:
            raise ValueError("a batch holds fewer than 2**31 rows")
        rows, q0, k0 = [], 0, 0
        for lq, lk in zip(self.q_lens, self.kv_lens):
            rows.append((q0, lq, k0, lk))
            q0, k0 = q0 + lq, k0 + lk
        self._rows = torch.tensor(rows, dtype=torch.int32).reshape(-1, 4)
        self.table = self._rows.to(torch.device(device))
        self.device = self.table.device
        self._tiles: dict = {}
        self._plans: dict = {}  # by a call's shapes, strides and types

    def tiles(self, side: str, rows: int, causal: bool, pack: int = 1) -> torch.Tensor:
        """(n, 2) int32 (sequence, tile): every ``rows`` rows of the query ("q") or
        key ("k") side, ``pack`` rows to a token, those with the most work first."""
        found = []
        for s, (lq, lk) in enumerate(zip(self.q_lens, self.kv_lens)):
            off = lk - lq
            for t in range(-(-(lq if side == "q" else lk) * pack // rows)):
                if not causal:
                    cost = lk if side == "q" else lq
                elif side == "q":
                    cost = max(0, min(lk, -(-(t + 1) * rows // pack) + off))
                else:
                    cost = max(0, lq - max(0, t * rows - off))
                found.append((-cost, s, t))
        found.sort()
        return torch.tensor([f[1:] for f in found], dtype=torch.int32).reshape(-1, 2)

    def _entries(self, side: str, rows: int, causal: bool, pack: int) -> torch.Tensor:
        """``tiles`` as the kernels read them: (n, 8) int32 on the device, the rows of
        the tile's sequence and its index."""
        key = (side, rows, causal, pack)
        if key not in self._tiles:
            tiles = self.tiles(side, rows, causal, pack)
            out = torch.zeros(tiles.shape[0], 8, dtype=torch.int32)
            out[:, :4] = self._rows[tiles[:, 0].long()]
            out[:, 4] = tiles[:, 1]
            self._tiles[key] = out.to(self.device)
        return self._tiles[key]

    def __len__(self) -> int:
        return len(self.q_lens)

    def __getstate__(self) -> dict:  # for copies and pickles: plans hold addresses
        return {**self.__dict__, "_tiles": {}, "_plans": {}}


def relative_buckets(num_buckets: int, max_distance: int, bidirectional: bool) -> list[int]:
    """Bucket of every distance position - key from -max_distance to max_distance.

    One way (causal), keys after the query share bucket 0; both ways, keys after
    the query take the upper half of the buckets.  Of the n buckets of a
    direction the first e = n // 2 hold one distance each and the others grow
    geometrically: bucket e + floor(log(d / e) / log(max_distance / e) * (n - e)),
    at most n - 1.  The floor is exact (integers are compared)."""
    n = num_buckets // 2 if bidirectional else num_buckets
    exact = n // 2
    steps = n - exact

    def one_way(d: int) -> int:
        if d < exact:
            return d
        b = 0
        while b + 1 < steps and d**steps >= exact ** (steps - b - 1) * max_distance ** (b + 1):
            b += 1
        return exact + b

    out = []
    for d in range(-max_distance, max_distance + 1):
        if bidirectional:
            out.append(one_way(abs(d)) + (n if d < 0 else 0))
        else:
            out.append(one_way(max(0, d)))
    return out


class RelativeBias(nn.Module):
    """A learned bias per (bucket of the distance query - key, head), added to the
    attention scores; distances from ``max_distance`` on share a bucket (see
    ``relative_buckets``).  ``weight`` is (num_buckets, heads)."""

    def __init__(self, heads: int, num_buckets: int = 32, max_distance: int = 128, bidirectional: bool = True, *,
                 device=None, dtype=None):
        super().__init__()
        n = num_buckets // 2 if bidirectional else num_buckets
        if n < 2 or num_buckets > BIAS_MAX_BUCKETS or (bidirectional and num_buckets % 2):
            raise ValueError(f"num_buckets must be 2 to {BIAS_MAX_BUCKETS} (an even number from 4 when bidirectional)")
        if not n // 2 < max_distance <= BIAS_MAX_DISTANCE:
            raise ValueError(f"max_distance must exceed {n // 2} and be at most {BIAS_MAX_DISTANCE}")
        if heads < 1:
            raise ValueError("heads must be positive")
        self.heads, self.num_buckets, self.max_distance, self.bidirectional = heads, num_buckets, max_distance, bidirectional
        self.weight = nn.Parameter(torch.zeros(num_buckets, heads, device=device, dtype=dtype))
        self.register_buffer("buckets", None, persistent=False)
        self._fill_buckets()

    def _fill_buckets(self) -> torch.Tensor:
        buckets = relative_buckets(self.num_buckets, self.max_distance, self.bidirectional)
        self.buckets = torch.tensor(buckets, dtype=torch.int32, device=self.weight.device)
        return self.buckets

    def _apply(self, fn, recurse=True):
        # the buckets follow from the arguments: a move that gives them other memory or another type makes them anew
        # (to_empty() gives memory without contents, and from the meta device there is nothing to copy)
        before = self._buffers["buckets"]
        if before.is_meta:
            self._buffers["buckets"] = None
        try:
            super()._apply(fn, recurse)
        finally:
            if self._buffers["buckets"] is not before:
                self._fill_buckets()
        return self

    def _tables(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The weight and, where it lies, the buckets."""
        weight, buckets = self.weight, self.buckets
        if buckets.device != weight.device or buckets.dtype != torch.int32 or buckets.shape != (2 * self.max_distance + 1,):
            buckets = self._fill_buckets()  # the weight was put there by itself
        return weight, buckets

    def forward(self, distance: torch.Tensor) -> torch.Tensor:
        """(..., heads): the bias of integer distances query - key."""
        weight, buckets = self._tables()
        at = distance.clamp(-self.max_distance, self.max_distance) + self.max_distance
        return weight[buckets[at].long()]


def _vectors(t: torch.Tensor) -> torch.Tensor:
    """t, or a contiguous copy when its rows cannot be read in 16-byte vectors
    (contiguous tensors can: the head width is a multiple of 8)."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous() and t.numel():  # without elements, whatever the strides
            return t
        per = 16 // t.element_size()
        if t.stride(-1) == 1 and all(s % per == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
            return t
    return t.detach().clone(memory_format=torch.contiguous_format)


def _check_heads(q, k, v, bias, scale) -> tuple[int, int, int]:
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        _check_cuda(q, k, v)
    dtype, device = q.dtype, q.device
    heads, dim = q.shape[-2:]
    kv_heads = k.shape[-2]
    if dtype not in _DTYPE_CODE:
        raise TypeError(f"attention takes float32 or bfloat16, not {dtype}")
    if k.dtype != dtype or v.dtype != dtype:
        raise TypeError(f"q, k and v must have one type (got {dtype}, {k.dtype}, {v.dtype})")
    if k.shape != v.shape or k.shape[-1] != dim:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    if dim % 8 or not 8 <= dim <= ATTENTION_MAX_DIM:
        raise ValueError(f"the head width must be a multiple of 8 up to {ATTENTION_MAX_DIM}, not {dim}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads do not divide over {kv_heads} key heads")
    if heads > 65535:
        raise ValueError("at most 65535 heads")
    if k.device != device or v.device != device:
        raise ValueError(f"tensors lie on {device}, {k.device} and {v.device}")
    if scale is not None and not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive, not {scale}")
    if bias is not None:
        _check_bias(bias, heads, device)
    return heads, kv_heads, dim


def _check_bias(bias: RelativeBias, heads: int, device) -> None:
    weight = bias._tables()[0]
    if bias.heads != heads:
        raise ValueError(f"the bias has {bias.heads} heads, the queries {heads}")
    if weight.shape != (bias.num_buckets, heads):
        raise ValueError(f"the bias's weight must be ({bias.num_buckets}, {heads}), not {tuple(weight.shape)}")
    if weight.device != device:
        raise ValueError(f"the bias lies on {weight.device}, the queries on {device}")
    if weight.dtype not in _DTYPE_CODE:
        raise TypeError(f"the bias must be float32 or bfloat16, not {weight.dtype}")


def _raw_stream(t: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.get_device())


class _Plan:
    """What a call's shapes decide: the descriptor, the tiles of the forward's
    queries, the backward's queries and its keys, the backward's workspace."""

    __slots__ = ("desc", "ref", "tables", "tiles", "workspace", "streams")

    def __init__(self, seqs, q, k, v, causal, scale, table):
        dtype, buckets, span = table or (None, 0, 0)
        self.desc = _lib.AttentionDesc(
            q.shape[0], k.shape[0], q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
            q.shape[1], k.shape[1], q.shape[2], _DTYPE_CODE[q.dtype], int(causal),
            span, buckets, _DTYPE_CODE.get(dtype, 0), max(seqs.kv_lens, default=0), scale, 1)
        self.ref = ctypes.byref(self.desc)
        self.tables, self.tiles, self.streams = [], [], set()
        for what, side in enumerate("qqk"):
            rows, pack = ctypes.c_int32(), ctypes.c_int32()
            _lib.call("kf_attention_tiling", self.ref, what, ctypes.byref(rows), ctypes.byref(pack))
            t = seqs._entries(side, rows.value, causal, pack.value)
            self.tables.append(t)
            self.tiles.append((t.data_ptr(), t.shape[0]))
        self.workspace = max(1, int(_lib.load().kf_attention_bwd_workspace(self.tiles[1][1], self.ref)))


def _plan_stream(plan: _Plan, t: torch.Tensor) -> int:
    """The current stream of t's device, which from now on may read the plan's tables: they were
    allocated on the stream of the first call, and when the sequences go their memory must not
    be given away while another stream still reads it."""
    raw = _raw_stream(t)
    if raw not in plan.streams:
        plan.streams.add(raw)
        for table in plan.tables:
            if table.is_cuda:
                table.record_stream(torch.cuda.current_stream(table.device))
    return raw


def _plan(seqs, q, k, v, causal, scale, table) -> _Plan:
    """``table``: type, buckets and largest distance of the bias, or None."""
    key = (q.dtype, q.shape, q.stride(), k.shape, k.stride(), v.stride(), causal, scale, table)
    plan = seqs._plans.get(key)
    if plan is None:
        plan = seqs._plans[key] = _Plan(seqs, q, k, v, causal, scale, table)
    return plan


def _forward(q, k, v, table, seqs, causal, scale, bias, train: bool):
    """(o, rest, lse, plan): the output, and for the backward what the rounding of a
    bf16 output leaves out (delta = dout . o keeps float32's digits) and the
    logarithms of the sums, with what their rounding leaves out."""
    q, k, v = _vectors(q), _vectors(k), _vectors(v)
    plan = _plan(seqs, q, k, v, causal, scale,
                 None if bias is None else (bias.weight.dtype, bias.num_buckets, bias.max_distance))
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    rest = lse = None
    if train:
        lse = torch.empty(2, q.shape[1], q.shape[0], device=q.device, dtype=torch.float32)
        if q.dtype == torch.bfloat16:
            rest = torch.empty_like(o)
    tiles, n = plan.tiles[0]
    if n:
        table = None if table is None else table.detach().contiguous()
        _launch("kf_attention_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), tiles, n,
                None if table is None else table.data_ptr(), None if table is None else bias.buckets.data_ptr(),
                o.data_ptr(), None if rest is None else rest.data_ptr(), None if lse is None else lse.data_ptr(),
                plan.ref, _plan_stream(plan, q))
    return o, rest, lse, plan


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, seqs, causal, scale, bias):
        o, rest, lse, plan = _forward(q, k, v, table, seqs, causal, scale, bias, train=True)
        ctx.save_for_backward(q, k, v, table, o, rest, lse)
        ctx.seqs, ctx.buckets = seqs, None if bias is None else bias.buckets
        ctx.options = causal, scale, None if bias is None else (table.dtype, bias.num_buckets, bias.max_distance)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, table, o, rest, lse = ctx.saved_tensors
        need = ctx.needs_input_grad
        q, k, v = _vectors(q), _vectors(k), _vectors(v)
        plan = _plan(ctx.seqs, q, k, v, *ctx.options)  # saved tensors may come back with other strides
        o, rest, lse = (t if t is None or t.is_contiguous() else t.contiguous() for t in (o, rest, lse))
        if dout.dtype != q.dtype or not dout.is_contiguous() or dout.data_ptr() % 16:
            dout = dout.to(q.dtype).clone(memory_format=torch.contiguous_format)
        dq = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        dk, dv = torch.empty((2, *k.shape), device=q.device, dtype=q.dtype).unbind(0)
        want = table is not None and need[3]
        tab = None if table is None else table.detach().contiguous()
        dtable = torch.empty_like(tab) if want else None
        (q_tiles, n_q), (k_tiles, n_k) = plan.tiles[1:]
        if n_q or n_k or want:
            ws = torch.empty(plan.workspace, device=q.device, dtype=torch.float32)
            _launch("kf_attention_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                    None if rest is None else rest.data_ptr(), dout.data_ptr(), lse.data_ptr(),
                    q_tiles, n_q, k_tiles, n_k, None if tab is None else tab.data_ptr(),
                    None if tab is None else ctx.buckets.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                    None if dtable is None else dtable.data_ptr(), ws.data_ptr(), plan.ref, _plan_stream(plan, q),
                    kernels=2 + (q.dtype == torch.float32) + 2 * want)
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dtable, None, None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seqs: PackedSequences, *, causal: bool = True,
              scale: float | None = None, bias: RelativeBias | None = None) -> torch.Tensor:
    """softmax(scale q k^T + bias) v over each packed sequence: (Tq, heads, dim).

    ``q`` is (Tq, heads, dim), ``k`` and ``v`` (Tk, kv_heads, dim), float32 or
    bfloat16, strided as they come (views of one projection's output are read
    in place); query head h uses key head h // (heads / kv_heads).  ``scale``
    defaults to 1/sqrt(dim).  ``causal`` queries see the keys up to their own
    position; a query that sees no key gives 0 and passes no gradient.  Rows
    of other sequences never enter a result, whatever they hold; a non-finite
    value of a later key of the same sequence may reach a causal query near it.
    Gradients reach q, k, v and ``bias.weight``; every sum runs in a fixed order.
    """
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v must be (tokens, heads, dim)")
    dim = _check_heads(q, k, v, bias, scale)[2]
    if not isinstance(seqs, PackedSequences):
        raise TypeError("seqs must be a PackedSequences")
    if q.shape[0] != seqs.total_q or k.shape[0] != seqs.total_kv:
        raise ValueError(f"the sequences hold {seqs.total_q} query and {seqs.total_kv} key rows, the tensors {q.shape[0]} "
                         f"and {k.shape[0]}")
    if seqs.device != q.device:
        raise ValueError(f"the sequences lie on {seqs.device}, the queries on {q.device}")
    table = None if bias is None else bias.weight
    args = (q, k, v, table, seqs, bool(causal), 1.0 / math.sqrt(dim) if scale is None else float(scale), bias)
    if not _unwatched() or torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                                        (table is not None and table.requires_grad)):
        return _Attention.apply(*args)
    return _forward(*args, train=False)[0]


_DECODE_PLANS_MAX = 512
_decode_plans: dict = {}  # descriptors by what the arguments' checks and the launch look at


def _decode_plan(q, k, v, lengths, scale, bias, weight):
    """The call's descriptor; arguments like those of an earlier call have been checked then."""
    key = (q.dtype, k.dtype, v.dtype, lengths.dtype, q.device, k.device, v.device, lengths.device, q.shape, k.shape, v.shape,
           lengths.shape, q.stride(), k.stride(), v.stride(), scale,
           None if bias is None else (weight.dtype, weight.device, weight.shape, bias.num_buckets, bias.max_distance))
    ref = _decode_plans.get(key)
    if ref is None:
        if q.dim() != 3 or k.dim() != 4 or v.dim() != 4:
            raise ValueError("q must be (batch, heads, dim), the caches (batch, capacity, kv_heads, dim)")
        _check_heads(q, k, v, bias, scale)
        batch, capacity, kv_heads, dim = k.shape
        if q.shape[0] != batch or batch > 65535:
            raise ValueError(f"q holds {q.shape[0]} sequences, the caches {batch} (at most 65535)")
        if lengths.shape != (batch,) or lengths.dtype != torch.int32 or lengths.device != q.device:
            raise ValueError(f"lengths must be ({batch},) int32 on {q.device}")
        desc = _lib.DecodeDesc(q.stride(0), q.stride(1), *k.stride()[:3], *v.stride()[:3], batch, capacity, q.shape[1],
                               kv_heads, dim, _DTYPE_CODE[q.dtype], 0 if bias is None else bias.max_distance,
                               0 if bias is None else _DTYPE_CODE[weight.dtype],
                               1.0 / math.sqrt(dim) if scale is None else float(scale),
                               0 if bias is None else bias.num_buckets)
        if len(_decode_plans) >= _DECODE_PLANS_MAX:
            _decode_plans.clear()
        ref = _decode_plans[key] = ctypes.byref(desc)
    return ref


def attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, *,
                     scale: float | None = None, bias: RelativeBias | None = None) -> torch.Tensor:
    """One new token per sequence over its cache: (batch, heads, dim).

    ``q`` is (batch, heads, dim), the caches (batch, capacity, kv_heads, dim) and
    ``lengths`` (batch,) int32 on the device: how many slots of each cache are
    filled, the new token's own last.  Slots past the length are never read; a
    length of 0 gives 0, one above the capacity counts as the capacity.
    Inference only: tensors that require a gradient raise.
    """
    weight, buckets = (None, None) if bias is None else bias._tables()
    plan = _decode_plan(q, k_cache, v_cache, lengths, scale, bias, weight)
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad or
                                    (bias is not None and weight.requires_grad)):
        raise RuntimeError("attention_decode has no backward: call it under torch.no_grad(), or use attention")
    if not _unwatched():
        return _Decode.apply(q, k_cache, v_cache, lengths, weight, buckets, scale, bias)
    return _decode(q, k_cache, v_cache, lengths, weight, buckets, scale, bias, plan)


class _Decode(torch.autograd.Function):
    """``_decode`` where something watches the call; it has no derivative."""

    @staticmethod
    def forward(ctx, q, k_cache, v_cache, lengths, weight, buckets, scale, bias):
        return _decode(q, k_cache, v_cache, lengths, weight, buckets, scale, bias,
                       _decode_plan(q, k_cache, v_cache, lengths, scale, bias, weight))


def _decode(q, k_cache, v_cache, lengths, weight, buckets, scale, bias, plan):
    aligned = _vectors(q), _vectors(k_cache), _vectors(v_cache)
    if aligned[0] is not q or aligned[1] is not k_cache or aligned[2] is not v_cache:  # copies have strides of their own
        q, k_cache, v_cache = aligned
        plan = _decode_plan(q, k_cache, v_cache, lengths, scale, bias, weight)
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    if o.numel() == 0:
        return o
    lengths = lengths.contiguous()
    table = None if bias is None else weight.detach().contiguous()
    _launch("kf_attention_decode", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), lengths.data_ptr(),
            None if table is None else table.data_ptr(), None if bias is None else buckets.data_ptr(), o.data_ptr(),
            plan, _raw_stream(q))
    return o
