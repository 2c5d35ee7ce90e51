"""RMS norm of query and key heads and their rotation by position, in one pass (``csrc/kernels/rotary.cu``): for training with gradients, for serving
straight into a paged cache.  CPU tensors take the PyTorch statements below.

No counterpart in the reference, which stops at the exchange of tokens.
"""
from typing import Tuple, Union

import torch

from .. import _native
from .gemm import _by_type, _gradient_alone


def rope_table(num_positions: int, dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """fp32 ``[num_positions, dim]``: the cosines, then the sines, of ``position * base ** (-2 i / dim)`` for ``i`` up to ``dim / 2``, from angles in 64 bits.  ``dim``: the
    channels that are rotated."""
    angles = torch.arange(num_positions, dtype=torch.float64, device=device)[:, None] * base**(-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    return torch.cat([angles.cos(), angles.sin()], -1).float()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, eps: float = 1e-6,
                 interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``q [T, heads, dim]`` and ``k [T, kv_heads, dim]`` (both bf16 or both fp32, any strides, ``dim`` a multiple of 8, at most 256) -> both normed and rotated, contiguous.

    Every head is divided by ``sqrt(mean(x^2) + eps)`` and multiplied by its weight (``[dim]``, both bf16 or both fp32); then pairs of its first ``R`` channels are turned by the
    angles of the token's position: ``table`` fp32 ``[num_positions, R]`` holds their cosines and sines (:func:`rope_table`; ``R`` a multiple of 16, at most ``dim``; the other channels are
    only normed).  Pairs are channels ``i`` and ``i + R / 2``, or with ``interleaved`` ``2 i`` and ``2 i + 1``.  ``positions`` int64 or int32 ``[T]``.

    A token with a negative position (padding) gets zeros and gives no gradient; one behind the table gets no numbers (NaN).  Heads whose channels are apart or that do
    not start on 16 bytes are copied first.  Carries gradients to heads and weights, by the kernel of :func:`qk_norm_rope_backward`.  Tracers, function transforms, dispatch
    modes and forward mode see the PyTorch statement, as does whoever wants a gradient of the table."""
    if q.is_cuda and _by_type(q, k, q_weight, k_weight, table, positions):
        res = _native.load().qk_norm_rope(q, k, q_weight, k_weight, table, positions, eps, interleaved)
        if res is not None:
            return res
        if _gradient_alone(q, k, q_weight, k_weight) and not table.requires_grad:
            return _QkNormRope.apply(q, k, q_weight, k_weight, table, positions, eps, interleaved)
    return qk_norm_rope_ref(q, k, q_weight, k_weight, table, positions, eps, interleaved)


class _QkNormRope(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, table, positions)
        ctx.options = eps, interleaved
        return qk_norm_rope(q, k, q_weight, k_weight, table, positions, eps, interleaved)

    @staticmethod
    def backward(ctx, dq, dk):
        return (*qk_norm_rope_backward(dq, dk, *ctx.saved_tensors, *ctx.options), None, None, None, None)


def qk_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, table: torch.Tensor,
                          positions: torch.Tensor, eps: float = 1e-6, interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of :func:`qk_norm_rope` from those of its results and what it was given -> ``(d_q, d_k, d_q_weight, d_k_weight)``.  The weights' gradients are summed over tokens
    and heads in 32 bits, always in the same order.  Where these gradients are to carry gradients themselves, and for whoever watches, the PyTorch statement runs."""
    if q.is_cuda and _by_type(dq, dk, q, k, q_weight, k_weight, table, positions):
        res = _native.load().qk_norm_rope_backward(dq, dk, q, k, q_weight, k_weight, table, positions, eps, interleaved)
        if res is not None:
            return res
    return qk_norm_rope_backward_ref(dq, dk, q, k, q_weight, k_weight, table, positions, eps, interleaved)


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, table: torch.Tensor, positions: torch.Tensor,
                        k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, eps: float = 1e-6, interleaved: bool = False,
                        keep_k: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """:func:`qk_norm_rope` whose keys, with the values ``v`` (like ``k``) as they are, go to their places in paged caches -> the queries, or with ``keep_k``
    ``(queries, keys)``, for a prompt whose attention is taken at once.

    ``k_cache`` and ``v_cache [pages, page_size, kv_heads, dim]``: of the heads' type, one layout, channels contiguous, heads on 16 bytes (views of one
    allocation, or with the heads in front of the places, are as good).  Token ``t`` goes to place ``slots[t] % page_size`` of page ``slots[t] // page_size`` (int64 or int32); tokens whose
    slot is not in the caches go nowhere.  What a place holds that several tokens name is not said.  What is in the caches carries no gradient; where
    the queries are to carry one (or the keys beside them), and for whoever watches, the PyTorch statement runs."""
    if q.is_cuda and _by_type(q, k, v, q_weight, k_weight, table, positions, k_cache, v_cache, slots):
        res = _native.load().qk_norm_rope_append(q, k, v, q_weight, k_weight, table, positions, k_cache, v_cache, slots, eps, interleaved, keep_k)
        if res is not None:
            return res if keep_k else res[0]
    return qk_norm_rope_append_ref(q, k, v, q_weight, k_weight, table, positions, k_cache, v_cache, slots, eps, interleaved, keep_k)


def _wide(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float64 else t.float()


def _angles(table, positions, like):
    """Cosines and sines of every token (``[T, 1, R / 2]``), and whether its position is in front of the table and in it (``[T, 1, 1]``)."""
    at = positions.long()
    inside = at < table.shape[0]
    if table.shape[0] == 0:                                          # (any row: nobody is in it)
        table = table.new_zeros(1, table.shape[1])
    rows = table[at.clamp(0, table.shape[0] - 1)].to(_wide(like).dtype).unsqueeze(1)
    half = table.shape[1] // 2
    return rows[..., :half], rows[..., half:], (at < 0)[:, None, None], inside[:, None, None]


def _turn(x, cos, sin, interleaved):
    R = 2 * cos.shape[-1]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1), x[..., R:]], -1)


def qk_norm_rope_ref(q, k, q_weight, k_weight, table, positions, eps=1e-6, interleaved=False):
    """:func:`qk_norm_rope` stated with plain PyTorch operations (any device; what the kernel is tested against)."""
    out = []
    for x, w in ((q, q_weight), (k, k_weight)):
        cos, sin, before, inside = _angles(table, positions, x)
        n = _wide(x)
        n = n / torch.sqrt(n.square().mean(-1, keepdim=True) + eps) * _wide(w)
        y = torch.where(inside, _turn(n, cos, sin, interleaved), float('nan'))
        out.append(torch.where(before, 0.0, y).to(x.dtype))
    return tuple(out)


def qk_norm_rope_backward_ref(dq, dk, q, k, q_weight, k_weight, table, positions, eps=1e-6, interleaved=False):
    """:func:`qk_norm_rope_backward` stated with plain PyTorch operations."""
    dx, dw = [], []
    for dy, x, w in ((dq, q, q_weight), (dk, k, k_weight)):
        cos, sin, before, inside = _angles(table, positions, x)
        v = _wide(x)
        rstd = 1.0 / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
        g = torch.where(before, 0.0, torch.where(inside, _turn(_wide(dy), cos, -sin, interleaved), float('nan')))
        u, n = g * _wide(w), v * rstd
        dx.append(torch.where(before, 0.0, rstd * (u - n * (u * n).mean(-1, keepdim=True))).to(x.dtype))
        dw.append(torch.where(before, 0.0, g * n).sum((0, 1)).to(w.dtype))
    return (*dx, *dw)


def qk_norm_rope_append_ref(q, k, v, q_weight, k_weight, table, positions, k_cache, v_cache, slots, eps=1e-6, interleaved=False, keep_k=False):
    """:func:`qk_norm_rope_append` stated with plain PyTorch operations."""
    q, k = qk_norm_rope_ref(q, k, q_weight, k_weight, table, positions, eps, interleaved)
    pages, size = k_cache.shape[:2]
    if pages * size > 0 and slots.shape[0] > 0:
        # (in shapes that do not depend on the slots: tokens without a place write what one that has one writes or, where nobody has, what stands in the first place)
        keep = (slots >= 0) & (slots < pages * size)
        some, one = keep.any(), keep.int().argmax(0, keepdim=True)
        at = torch.where(keep, slots.long(), torch.where(some, slots.long().index_select(0, one), 0))
        for cache, new in ((k_cache, k), (v_cache, v)):
            new = new.detach()
            cache[at // size, at % size] = torch.where(keep[:, None, None], new, torch.where(some, new.index_select(0, one), cache[:1, 0]))
    return (q, k) if keep_k else q
