"""The norms around a transformer block, fused with its gate and residual scale.

``residual_norm`` joins two blocks in one pass over the rows:

    u = N_b(branch) * branch_weight + branch_bias     (or the branch itself)
    y = residual_scale * x + gate * u                 (the residual stream)
    h = N(y) * weight + bias                          (the next block's input)

with N a layer norm or a root-mean-square norm.  The kernels are
``kf_residual_norm_fwd`` / ``kf_residual_norm_bwd`` (csrc/norm.cu).
"""

from __future__ import annotations

import ctypes

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .kernels import _check_cuda, _launch, _unwatched

NORM_KINDS = ("layer", "rms")
NORM_MAX_WIDTH = 8192

_DTYPE_CODE = {torch.float32: _lib.KF_DTYPE_F32, torch.bfloat16: _lib.KF_DTYPE_BF16}


_descs: dict = {}  # descriptors by their values
_DESCS_MAX = 512


def _desc(*values):
    ref = _descs.get(values)
    if ref is None:
        if len(_descs) >= _DESCS_MAX:
            _descs.clear()
        ref = _descs[values] = ctypes.byref(_lib.ResidualNormDesc(*values))
    return ref


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _raw_stream(t: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.get_device())


class _Call:
    """The operands of one residual norm as the kernels take them."""

    __slots__ = ("x", "branch", "gate", "w", "s", "bw", "bs", "desc", "rows", "width", "gate_token")

    def __init__(self, x, branch, weight, bias, branch_weight, branch_bias, gate, kind, residual_scale, eps):
        self.width = width = x.shape[-1]
        self.x = x.contiguous()
        self.rows = x.numel() // width
        self.branch = None if branch is None else branch.contiguous()
        self.gate_token = token = gate is not None and gate.dim() > 1
        params = (weight, bias, branch_weight, branch_bias, None if token else gate)
        # parameters of one type are read as they are; mixed or other types as float32
        dtype = weight.dtype
        if dtype not in _DTYPE_CODE or any(p is not None and p.dtype != dtype for p in params):
            dtype = torch.float32
        self.w, self.s, self.bw, self.bs, self.gate = (
            p if p is None or (p.dtype == dtype and p.is_contiguous()) else p.detach().to(dtype).contiguous() for p in params)
        if token:
            self.gate = gate.contiguous()
        out = x.dtype if branch is None else branch.dtype
        self.desc = _desc(width, int(kind == "layer"), int(branch_weight is not None), int(token), _DTYPE_CODE[x.dtype],
                          _DTYPE_CODE[out], _DTYPE_CODE[dtype], residual_scale, eps)

    def forward(self, with_stats: bool):
        """(y, h, stats); y is None where there is no branch (it is x)."""
        x, branch = self.x, self.branch
        y = None if branch is None else torch.empty_like(x)
        h = torch.empty_like(x if branch is None else branch)
        stats = torch.empty(self.rows, 4, device=x.device, dtype=torch.float32) if with_stats else None
        if self.rows:
            _launch("kf_residual_norm_fwd", x.data_ptr(), _ptr(branch), _ptr(self.gate), self.w.data_ptr(), _ptr(self.s),
                    _ptr(self.bw), _ptr(self.bs), _ptr(y), h.data_ptr(), _ptr(stats), self.rows, self.desc, _raw_stream(x))
        return y, h, stats


_workspaces: dict = {}  # floats of the backward's workspace by (rows, width)


def _workspace(rows: int, width: int) -> int:
    n = _workspaces.get((rows, width))
    if n is None:
        if len(_workspaces) >= _DESCS_MAX:
            _workspaces.clear()
        n = _workspaces[rows, width] = int(_lib.load().kf_residual_norm_workspace(rows, width))
    return n


def _like(g, like):
    if g.dtype != like.dtype:
        g = g.to(like.dtype)
    return g if g.is_contiguous() else g.contiguous()


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, weight, bias, branch_weight, branch_bias, gate, kind, residual_scale, eps):
        call = _Call(x, branch, weight, bias, branch_weight, branch_bias, gate, kind, residual_scale, eps)
        y, h, stats = call.forward(with_stats=True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, branch, weight, bias, branch_weight, branch_bias, gate, stats)
        ctx.options = (kind, residual_scale, eps)
        return h if branch is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x, branch, weight, bias, branch_weight, branch_bias, gate, stats = ctx.saved_tensors
        dy, dh = (None, grads[0]) if branch is None else grads
        if dy is None and dh is None:
            return (None,) * 10
        need = ctx.needs_input_grad
        call = _Call(x, branch, weight, bias, branch_weight, branch_bias, gate, *ctx.options)
        x2, w, stats = call.x, call.w, stats.contiguous()  # hooks may give saved tensors back with other strides
        if dy is not None:
            dy = _like(dy, x2)
        if dh is not None:
            dh = _like(dh, x2 if branch is None else call.branch)
        dx = torch.empty_like(x2)
        dbranch = None if branch is None else torch.empty_like(call.branch)
        # the parameters' gradients that are asked for, rows of one tensor
        dgate = torch.empty_like(call.gate) if call.gate_token else None
        asked = [need[2], need[3], need[4], need[5], need[6] and not call.gate_token]
        out = torch.empty(sum(asked), call.width, device=w.device, dtype=w.dtype).unbind(0)
        rows = iter(out)
        dw, ds, dbw, dbs, dchannel = (next(rows) if a else None for a in asked)
        if not call.gate_token:
            dgate = dchannel
        ws = torch.empty(_workspace(call.rows, call.width), device=w.device, dtype=torch.float32)
        _launch("kf_residual_norm_bwd", x2.data_ptr(), _ptr(call.branch), _ptr(call.gate), w.data_ptr(), _ptr(call.bw),
                _ptr(call.bs), stats.data_ptr(), _ptr(dy), _ptr(dh), dx.data_ptr(), _ptr(dbranch), _ptr(dgate), _ptr(dw),
                _ptr(ds), _ptr(dbw), _ptr(dbs), ws.data_ptr(), call.rows, call.desc, _raw_stream(w),
                kernels=2 if call.rows else 1)
        cast = lambda g, p: g if g is None or g.dtype == p.dtype else g.to(p.dtype)  # noqa: E731
        return (dx if need[0] else None, dbranch if need[1] else None, cast(dw, weight), cast(ds, bias),
                cast(dbw, branch_weight), cast(dbs, branch_bias), cast(dgate, gate) if need[6] else None, None, None, None)


def residual_norm(x: torch.Tensor, branch: torch.Tensor | None, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                  kind: str = "layer", gate: torch.Tensor | None = None, branch_norm: bool = False,
                  branch_weight: torch.Tensor | None = None, branch_bias: torch.Tensor | None = None,
                  residual_scale: float = 1.0, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, h) of the formulas at the head of this module, on (..., width) tensors.

    ``x`` is the residual stream and ``branch`` a block's output, both float32
    or bfloat16 (a float32 stream may take a bfloat16 branch); ``y`` has the
    type of ``x``, ``h`` that of the branch.  ``gate`` is (width,), one factor
    per channel, or broadcasts to the branch's shape.  ``branch=None`` norms
    ``x`` alone, the start of a stack: y is x.  Sums and statistics are
    float32; ``h`` comes from y before its rounding.  Gradients reach every
    tensor argument; the sums over rows run in a fixed order.
    """
    if kind not in NORM_KINDS:
        raise ValueError(f"kind must be one of {NORM_KINDS}")
    if eps < 0:
        raise ValueError("eps must not be negative")
    device, grad = x.device, torch.is_grad_enabled()
    wanted = False
    for t in (x, branch, weight, bias, branch_weight, branch_bias, gate):
        if t is not None:
            if not t.is_cuda:
                _check_cuda(t)
            if t.device != device:
                raise ValueError(f"tensors lie on {device} and {t.device}")
            wanted = wanted or t.requires_grad
    if x.dim() < 1 or not 1 <= x.shape[-1] <= NORM_MAX_WIDTH:
        raise ValueError(f"rows must have 1 to {NORM_MAX_WIDTH} elements (got a tensor of shape {tuple(x.shape)})")
    width = x.shape[-1]
    if x.dtype not in _DTYPE_CODE or (branch is not None and branch.dtype not in _DTYPE_CODE):
        raise TypeError(f"x and branch must be float32 or bfloat16, not {x.dtype} and {None if branch is None else branch.dtype}")
    for t in (weight, bias, branch_weight, branch_bias):
        if t is not None and t.shape != (width,):
            raise ValueError(f"norm parameters must have shape ({width},), not {tuple(t.shape)}")
    if branch is None:
        if gate is not None or branch_norm or residual_scale != 1.0:
            raise ValueError("a gate, a branch norm or a residual scale needs a branch")
    else:
        if branch.shape != x.shape:
            raise ValueError(f"x {tuple(x.shape)} and branch {tuple(branch.shape)} differ in shape")
        if x.dtype == torch.bfloat16 and branch.dtype == torch.float32:
            raise TypeError("a bfloat16 residual stream takes no float32 branch")
    if branch_norm != (branch_weight is not None) or (branch_bias is not None and not branch_norm):
        raise ValueError("branch_norm, branch_weight and branch_bias belong together")
    if gate is not None and gate.shape != (width,):
        gate = gate.expand(branch.shape).to(branch.dtype)  # their gradients: autograd's
        if gate.dim() < 2:
            gate = gate.reshape(1, width)
    args = (x, branch, weight, bias, branch_weight, branch_bias, gate, kind, float(residual_scale), float(eps))
    if grad and wanted or not _unwatched():
        out = _ResidualNorm.apply(*args)
        return (x, out) if branch is None else out
    y, h, _ = _Call(*args).forward(with_stats=False)
    return (x if branch is None else y), h


class ResidualNorm(nn.Module):
    """``residual_norm`` with its parameters: ``weight`` (and ``bias`` for a layer
    norm), ``branch_weight`` (``branch_bias``) with ``branch_norm``, and ``gate``
    (one factor per channel, starting at ``gate_init``) unless that is None."""

    def __init__(self, dim: int, kind: str = "layer", *, branch_norm: bool = False, gate_init: float | None = None,
                 residual_scale: float = 1.0, eps: float = 1e-6, device=None, dtype=None):
        super().__init__()
        if kind not in NORM_KINDS:
            raise ValueError(f"kind must be one of {NORM_KINDS}")
        if not 1 <= dim <= NORM_MAX_WIDTH:
            raise ValueError(f"dim must be 1 to {NORM_MAX_WIDTH}")
        self.dim, self.kind, self.branch_norm = dim, kind, branch_norm
        self.residual_scale, self.eps = residual_scale, eps
        make = lambda on, v: nn.Parameter(torch.full((dim,), v, device=device, dtype=dtype)) if on else None  # noqa: E731
        self.weight, self.bias = make(True, 1.0), make(kind == "layer", 0.0)
        self.branch_weight = make(branch_norm, 1.0)
        self.branch_bias = make(branch_norm and kind == "layer", 0.0)
        self.gate = make(gate_init is not None, gate_init)

    def forward(self, x: torch.Tensor, branch: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        return residual_norm(x, branch, self.weight, self.bias, kind=self.kind, gate=self.gate,
                             branch_norm=self.branch_norm, branch_weight=self.branch_weight,
                             branch_bias=self.branch_bias, residual_scale=self.residual_scale, eps=self.eps)
