"""Layer norm in front of the expert layer and its gradients (``csrc/kernels/layer_norm.cu``); CPU tensors take the PyTorch statements
below.  No counterpart in the reference, which has no norm.
"""
from typing import Optional, Tuple

import torch

from .. import _native
from .gemm import _by_type, _gradient_alone


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` as a matrix of rows with contiguous channels: a view where there is one."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(x - mean) * rstd * weight (+ bias)`` over the last axis of ``x [..., H]`` (bf16 or fp32, any strides) -> ``(y like x, mean, rstd)``,
    the statistics fp32, one of each per row, in ``x``'s leading shape (on a GPU they share an allocation).  ``weight`` and ``bias`` ``[H]``: both bf16 or both fp32.

    Carries gradients, by the kernel of :func:`layer_norm_backward`.  Tracers, function transforms, dispatch modes and forward mode see the PyTorch
    statement."""
    if not x.is_cuda:
        return layer_norm_ref(x, weight, bias, eps)
    res = _native.load().layer_norm(_rows(x), weight, bias, eps) if _by_type(x, weight, bias) else None
    if res is None:
        return _LayerNorm.apply(x, weight, bias, eps) if _gradient_alone(x, weight, bias) else layer_norm_ref(x, weight, bias, eps)
    if x.dim() == 2:
        return res
    y, mean, rstd = res
    return y.view(x.shape), mean.view(x.shape[:-1]), rstd.view(x.shape[:-1])


class _LayerNorm(torch.autograd.Function):
    """``apply(x, weight, bias or None, eps) -> (y, mean, rstd)``, all of them with gradients."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.with_bias = bias is not None
        ctx.set_materialize_grads(False)
        return y, mean, rstd

    @staticmethod
    def backward(ctx, dy, d_mean, d_rstd):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(torch.zeros_like(x) if dy is None else dy, x, weight, mean, rstd, with_bias=ctx.with_bias)
        if d_mean is not None or d_rstd is not None:
            # (hardly ever asked for: eager operations)
            d = 0.0 if d_mean is None else d_mean.unsqueeze(-1)
            if d_rstd is not None:
                d = d - (d_rstd * rstd**3).unsqueeze(-1) * (_wide(x) - mean.unsqueeze(-1))
            dx = (dx + d / x.shape[-1]).to(x.dtype)
        return dx, dw, db, None


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        with_bias: bool = False) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Gradients of :func:`layer_norm` from ``dy`` and what the forward pass was given and returned -> ``(dx like x, d_weight, d_bias or None)``.
    The parameters' gradients are summed over the rows in 32 bits, always in the same order.  Where these gradients are to carry gradients themselves, and
    for whoever watches, the PyTorch statement runs."""
    if not x.is_cuda:
        return layer_norm_backward_ref(dy, x, weight, mean, rstd, with_bias)
    if dy.shape != x.shape:
        raise ValueError('dy must have the shape of x, got %s and %s' % (tuple(dy.shape), tuple(x.shape)))
    res = None
    if _by_type(dy, x, weight, mean, rstd):
        flat = x.dim() == 2 and mean.dim() == rstd.dim() == 1
        res = _native.load().layer_norm_backward(_rows(dy), _rows(x), weight, mean if flat else mean.reshape(-1), rstd if flat else rstd.reshape(-1), with_bias)
    if res is None:
        return layer_norm_backward_ref(dy, x, weight, mean, rstd, with_bias)
    if x.dim() == 2:
        return res
    dx, dw, db = res
    return dx.view(x.shape), dw, db


def _wide(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float64 else t.float()


def layer_norm_ref(x, weight, bias=None, eps=1e-5):
    """:func:`layer_norm` stated with plain PyTorch operations (any device; what the kernel is tested against)."""
    v = _wide(x)
    mean = v.mean(-1)
    rstd = 1.0 / torch.sqrt((v - mean.unsqueeze(-1)).square().mean(-1) + eps)
    y = (v - mean.unsqueeze(-1)) * rstd.unsqueeze(-1) * _wide(weight)
    return (y if bias is None else y + _wide(bias)).to(x.dtype), mean, rstd


def layer_norm_backward_ref(dy, x, weight, mean, rstd, with_bias=False):
    """:func:`layer_norm_backward` stated with plain PyTorch operations."""
    d, xh = _wide(dy), (_wide(x) - mean.unsqueeze(-1)) * rstd.unsqueeze(-1)
    g = d * _wide(weight)
    dx = rstd.unsqueeze(-1) * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    H = x.shape[-1]
    dw, db = (d * xh).reshape(-1, H).sum(0), d.reshape(-1, H).sum(0)
    return dx.to(x.dtype), dw.to(weight.dtype), db.to(weight.dtype) if with_bias else None
