"""Orthogonalised updates of weight matrices (``csrc/kernels/newton_schulz.cu``): what the Muon optimiser makes of a matrix's momentum before
it is added to the weights, here for whole stacks such as the experts' ``w13`` and ``w2``.  CPU tensors take the PyTorch statement below.

No counterpart in the reference, which has no optimiser.
"""
import math
from typing import Optional, Tuple

import torch

from .. import _native
from .gemm import _by_type, _core_of

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(x: torch.Tensor, steps: int = 5, coefficients: Tuple[float, float, float] = COEFFICIENTS, eps: float = 1e-7,
                  out: Optional[torch.Tensor] = None, num_sms: int = 0, buffer=None) -> torch.Tensor:
    """Moves the singular values of every matrix of ``x [..., rows, cols]`` (bf16 or fp32) towards one: ``X = x / (|x|_F + eps)``, then ``steps``
    times ``X = a X + (b A + c A A) X`` with ``A = X X^T`` (of the smaller side) -> bf16, contiguous, in ``x``'s shape (``out``: its memory, which may be that of ``x``).

    Matrices may be stored by rows or by columns, with any distance between rows; other strides are copied first.  The products have fp16 operands and
    32-bit sums, and carry 22 bits of X and 32 bits of the diagonals from step to step, so that the result is
    mostly off by little more than its rounding to bf16 (1.7e-3 of its norm): 1.7e-3 to 2.3e-3.  Singular values on two levels far apart take the most: 2.7e-3 for 512 and
    more rows, 3.5e-3 for 256, 4.5e-3, 6e-3, 9e-3 and 2e-2 for 128, 64, 32 and 16.  The workspace comes from PyTorch's allocator: about 6 bytes per element and 2 to 6 per element of A, with rows of
    whole 128 bytes, and for few rows the parts of A that are summed along the columns, at most 64 KB per SM.
    Refused (on a GPU) are coefficients under which singular values between 0 and 1 may come to more than some 10 before the last step (A reaches the
    range of fp16); those that are made to move them towards one stay far below.
    Tensors that carry a gradient, tracers, function transforms, dispatch modes and forward mode get the PyTorch statement.
    ``num_sms``: SMs to run on (0: all).
    ``buffer``: see :func:`ops.gemm.gemm_nt`."""
    if x.dim() < 2:
        raise ValueError('matrices are needed, got shape %s' % (tuple(x.shape),))
    res = None
    if x.is_cuda and _by_type(x, out):
        m = x if x.dim() == 3 else x.reshape(math.prod(x.shape[:-2]), x.shape[-2], x.shape[-1])
        if 1 not in m.stride()[1:] and 1 not in m.shape[1:]:
            m = m.contiguous()
        res = _native.load().orthogonalize(m, steps, *coefficients, eps, None if out is None else out.view(m.shape), num_sms, _core_of(buffer))
    if res is not None:
        return res.view(x.shape) if out is None else out
    res = orthogonalize_ref(x, steps, coefficients, eps)
    return res if out is None else out.copy_(res)


def orthogonalize_ref(x: torch.Tensor, steps: int = 5, coefficients: Tuple[float, float, float] = COEFFICIENTS, eps: float = 1e-7) -> torch.Tensor:
    """The same result stated with plain PyTorch operations in 32 bits (any device; 64-bit matrices stay 64-bit)."""
    if steps < 1:
        raise ValueError('at least one step')
    a, b, c = coefficients
    X = x if x.dtype == torch.float64 else x.float()
    tall = x.shape[-2] > x.shape[-1]
    X = X.mT if tall else X
    X = X / (X.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        A = X @ X.mT
        X = a * X + (b * A + c * (A @ A)) @ X
    X = X.mT if tall else X
    return X.contiguous() if x.dtype == torch.float64 else X.to(torch.bfloat16).contiguous()
