"""Layer norm with an optional residual add, forward and backward.

``layer_norm`` normalises the last dimension through ``gdn2_layer_norm_fwd`` /
``gdn2_layer_norm_bwd``; ``LayerNorm`` is the module around it.  Statistics,
and the sums of the weight's and the bias's gradients, are fp32.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


class LayerNormFunction(torch.autograd.Function):
    """``(y, s)`` of ``s = x + residual``, ``y = LN(s)``; ``y`` alone without a residual."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual, grad):
        D = x.shape[-1]
        xs = x.contiguous()
        rows = xs.numel() // D
        rs = None if residual is None else residual.contiguous()
        w = None if weight is None else weight.contiguous()
        b = None if bias is None else bias.contiguous()
        y = torch.empty_like(xs)
        s = None if rs is None else torch.empty_like(rs)
        save = grad and any(ctx.needs_input_grad)  # needs_input_grad alone is also set under no_grad
        stats = torch.empty(2, rows, device=x.device, dtype=torch.float32) if save else None
        ptr = _lib.ptr
        wt = w if w is not None else b
        args = _lib.LayerNormArgs(
            rows, D, eps, _DTYPES[x.dtype], _DTYPES[x.dtype if rs is None else rs.dtype],
            _DTYPES[torch.float32 if wt is None else wt.dtype], xs.data_ptr(), ptr(rs), ptr(w), ptr(b), y.data_ptr(),
            ptr(s), ptr(stats), None if stats is None else stats.data_ptr() + 4 * rows)
        with _lib.on_device(x.device):
            _lib.check(_lib.load().gdn2_layer_norm_fwd(args, _lib.stream_ptr(x.device)), "gdn2_layer_norm_fwd")
        if save:
            ctx.save_for_backward(xs if s is None else s, w, stats)
            ctx.meta = (rows, D, eps, x.dtype, None if rs is None else rs.dtype, None if wt is None else wt.dtype,
                        None if bias is None else bias.shape, ctx.needs_input_grad)
            ctx.set_materialize_grads(False)
        return y if s is None else (y, s)

    @staticmethod
    def backward(ctx, dy, ds=None):
        s, w, stats = ctx.saved_tensors
        rows, D, eps, dtype, rdtype, wdtype, bshape, need = ctx.meta
        dev = s.device
        dy = torch.zeros(s.shape, device=dev, dtype=dtype) if dy is None else dy.contiguous()
        ds = None if ds is None else ds.contiguous()
        # bf16 x on a bf16 residual: one gradient serves both
        dr = torch.empty(s.shape, device=dev, dtype=rdtype) if rdtype is not None and need[4] else None
        shared = dr is not None and rdtype == dtype
        dx = torch.empty(s.shape, device=dev, dtype=dtype) if not shared and (need[0] or dr is None) else None
        dw = torch.empty(D, device=dev, dtype=wdtype) if need[1] else None
        db = torch.empty(bshape, device=dev, dtype=wdtype) if need[2] else None
        ptr = _lib.ptr
        lib = _lib.load()
        args = _lib.LayerNormArgs(
            rows, D, eps, _DTYPES[dtype], _DTYPES[dtype if rdtype is None else rdtype],
            _DTYPES[torch.float32 if wdtype is None else wdtype], None, s.data_ptr() if rdtype is not None else None,
            ptr(w), None, None, None, stats.data_ptr(), stats.data_ptr() + 4 * rows)
        with _lib.on_device(dev):
            size = lib.gdn2_layer_norm_bwd_workspace_size(args) if need[1] or need[2] else 0
            ws = torch.empty(size, device=dev, dtype=torch.uint8)
            grads = _lib.LayerNormGrads(dy.data_ptr(), ptr(ds), s.data_ptr(), ptr(dx), ptr(dr), ptr(dw), ptr(db))
            _lib.check(lib.gdn2_layer_norm_bwd(args, grads, ws.data_ptr(), size, _lib.stream_ptr(dev)),
                       "gdn2_layer_norm_bwd")
        return (dr if shared else dx) if need[0] else None, dw, db, None, dr, None


@torch.compiler.disable
def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    eps: float = 1e-5,
    residual: torch.Tensor | None = None,
):
    r"""Layer norm over the last dimension D (at most 32768).

    ``y = (s - mean) / sqrt(var + eps) * weight + bias`` with ``s = x``, or
    ``s = x + residual``.  x: bf16 or fp32; weight, bias: ``[D]``, bf16 or
    fp32 (one type), either may be None; residual: the shape of x, x's type or
    fp32.  Returns ``y`` in x's type, or ``(y, s)`` with a residual, ``s`` in
    the residual's type (s is rounded to it before the statistics).
    Differentiable in every tensor.
    """
    if x.ndim < 1 or x.dtype not in _DTYPES:
        raise TypeError(f"layer_norm takes bf16 or fp32, got {x.dtype}.")
    D = x.shape[-1]
    if not 1 <= D <= 32768:
        raise ValueError(f"layer_norm takes rows of 1 to 32768 elements, got {D}.")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (D,):
            raise ValueError(f"{name} must have shape [{D}], got {tuple(t.shape)}.")
        if t is not None and t.dtype not in _DTYPES:
            raise TypeError(f"{name} must be bf16 or fp32, got {t.dtype}.")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}.")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}.")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"residual must be in x's type {x.dtype} or fp32, got {residual.dtype}.")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}.")
    _lib.require_device(x)
    return LayerNormFunction.apply(x, weight, bias, float(eps), residual, torch.is_grad_enabled())


class LayerNorm(nn.Module):
    """``layer_norm`` with its parameters (ones and zeros; names and shapes of ``torch.nn.LayerNorm``)."""

    def __init__(self, size: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True):
        super().__init__()
        self.size, self.eps = size, eps
        self.weight = nn.Parameter(torch.ones(size)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(size)) if elementwise_affine and bias else None

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        return layer_norm(x, self.weight, self.bias, self.eps, residual)
