"""Routing of tokens to experts: from the gate's logits to the ``topk_idx`` / ``topk_weights`` that ``ElasticBuffer.dispatch`` and
``FusedMoE`` take, and back from the gradient of the weights to the gradient of the logits.  One kernel each
(``csrc/kernels/router.cu``); CPU tensors take the PyTorch statements below.

No counterpart in the reference, whose callers bring their own gate.
"""
from typing import Optional, Tuple

import torch

from .. import _native
from ..buffers.elastic import topk_idx_t
from .gemm import _by_type, _gradient_alone

_SCORES = ('sigmoid', 'softmax')


def route(logits: torch.Tensor, num_topk: int, score: str = 'sigmoid', bias: Optional[torch.Tensor] = None, num_groups: int = 1,
          num_topk_groups: int = 1, group_top: int = 2, renormalize: bool = True, scale: float = 1.0,
          token_mask: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``logits [T, E]`` (fp32 or bf16, any row pitch, ``E <= 1024``) -> ``(topk_idx [T, K], topk_weights fp32 [T, K], count int32 [E])``.

    ``score``: ``'sigmoid'`` of each logit or ``'softmax'`` over the experts, in 32 bits.  The ``num_topk`` (at most 16) experts with the largest
    ``score + bias`` are chosen, equal ones by index, in that order; ``bias`` fp32 ``[E]`` (for balance) counts for the choice alone.
    ``num_groups`` (at most 32) > 1: the experts form that many equal groups of neighbours, and only those of the ``num_topk_groups`` groups with the
    largest sum of their ``group_top`` (1 or 2) best choices are eligible.  The weights are ``scale * score``, divided by the sum over the
    token's experts with ``renormalize``.  ``count[e]``: tokens that chose expert ``e``.

    Nobody chooses an expert whose logit is -inf, whose bias is -inf or whose choice is NaN; tokens with ``token_mask[t] == False`` choose none.
    Places without an expert hold index -1 and weight 0, which is what ``dispatch`` takes for "no selection".  (On a GPU the three results share an allocation: keep
    a clone of one that outlives the others.)

    The weights carry a gradient to the logits, by the kernel of :func:`route_backward`.  Tracers, function transforms, dispatch modes and forward mode
    see the PyTorch statement."""
    if score not in _SCORES:
        raise ValueError('score must be one of %s, got %r' % (_SCORES, score))
    if not logits.is_cuda:
        return route_ref(logits, num_topk, score, bias, num_groups, num_topk_groups, group_top, renormalize, scale, token_mask)
    if _by_type(logits, bias, token_mask):
        res = _native.load().route(logits, num_topk, score == 'softmax', bias, num_groups, num_topk_groups, group_top, renormalize, scale, token_mask,
                                   topk_idx_t == torch.int64)
        if res is not None:
            return res
        if _gradient_alone(logits):
            return RouteFunction.apply(logits, dict(num_topk=num_topk, score=score, bias=bias, num_groups=num_groups, num_topk_groups=num_topk_groups,
                                                    group_top=group_top, renormalize=renormalize, scale=scale, token_mask=token_mask))
    return route_ref(logits, num_topk, score, bias, num_groups, num_topk_groups, group_top, renormalize, scale, token_mask)


class RouteFunction(torch.autograd.Function):
    """:func:`route` with the gradient of its weights: ``apply(logits, options) -> (topk_idx, topk_weights, count)``, ``options`` a dict of
    ``route``'s other arguments."""

    @staticmethod
    def forward(ctx, logits, options):
        idx, weights, count = route(logits, **options)
        ctx.save_for_backward(logits, idx)
        ctx.options = {k: options[k] for k in ('score', 'renormalize', 'scale') if k in options}
        ctx.mark_non_differentiable(idx, count)
        return idx, weights, count

    @staticmethod
    def backward(ctx, _idx, d_weights, _count):
        logits, idx = ctx.saved_tensors
        return route_backward(d_weights.contiguous(), logits, idx, **ctx.options), None


def route_backward(d_weights: torch.Tensor, logits: torch.Tensor, topk_idx: torch.Tensor, score: str = 'sigmoid', renormalize: bool = True,
                   scale: float = 1.0) -> torch.Tensor:
    """Gradient of ``topk_weights`` with respect to the logits, the choice held fixed: ``d_weights`` fp32 ``[T, K]``, the ``logits`` and
    ``topk_idx`` of :func:`route` -> ``[T, E]`` in the logits' type.  Only a softmax without ``renormalize`` gives experts that were not chosen a
    gradient (and reads their logits); the others' is zero, as that of a token without experts.  Where this gradient is to carry gradients itself, and for
    whoever watches, the PyTorch statement runs."""
    if score not in _SCORES:
        raise ValueError('score must be one of %s, got %r' % (_SCORES, score))
    if not logits.is_cuda:
        return route_backward_ref(d_weights, logits, topk_idx, score, renormalize, scale)
    res = _native.load().route_backward(d_weights, logits, topk_idx, score == 'softmax', renormalize, scale) if _by_type(d_weights, logits, topk_idx) else None
    return route_backward_ref(d_weights, logits, topk_idx, score, renormalize, scale) if res is None else res


def _scores(logits: torch.Tensor, score: str) -> torch.Tensor:
    """Scores in 32 bits (64 for 64-bit logits).  The sum of a softmax is a tree: the experts, padded with zeros to a power of two, are halved
    and the upper half is added to the lower one until one value is left."""
    x = logits if logits.dtype == torch.float64 else logits.float()
    if score == 'sigmoid':
        return 1.0 / (1.0 + torch.exp(-x))
    e = torch.exp(x - x.max(dim=-1, keepdim=True).values)
    experts = int(e.shape[-1])                                      # (a number while tracing, too)
    width = 1 << (experts - 1).bit_length()
    total = torch.nn.functional.pad(e, (0, width - experts))
    while width > 1:
        width //= 2
        total = total[..., :width] + total[..., width:]
    return e / total


def _gathered(logits: torch.Tensor, topk_idx: torch.Tensor, score: str, renormalize: bool) -> torch.Tensor:
    """Scores of the chosen experts, 0 in empty places; renormalised ones of a softmax relative to the largest chosen logit."""
    live, at = topk_idx >= 0, topk_idx.clamp_min(0).to(torch.int64)
    if score == 'softmax' and renormalize:
        x = torch.where(live, (logits if logits.dtype == torch.float64 else logits.float()).gather(1, at), float('-inf'))
        top = x.max(dim=-1, keepdim=True).values
        return torch.where(live, torch.exp(x - top), 0.0)
    return torch.where(live, _scores(logits, score).gather(1, at), 0.0)


def route_ref(logits, num_topk, score='sigmoid', bias=None, num_groups=1, num_topk_groups=1, group_top=2, renormalize=True, scale=1.0,
              token_mask=None):
    """:func:`route` stated with plain PyTorch operations (any device; what the kernel is tested against)."""
    T, E = logits.shape
    if num_groups < 1 or E % num_groups or not 1 <= num_topk_groups <= num_groups or not 1 <= num_topk <= E // num_groups * num_topk_groups:
        raise ValueError('num_topk must be at most the experts of num_topk_groups of num_groups equal groups')
    if num_groups > 1 and not 1 <= group_top <= min(2, E // num_groups):
        raise ValueError('group_top must be 1 or 2, and at most the experts of a group')
    none, p = float('-inf'), _scores(logits, score)
    choice = p if bias is None else p + bias
    choice = torch.where(torch.isnan(choice) | (logits == none), none, choice)
    if num_groups > 1:
        groups = choice.view(T, num_groups, E // num_groups)
        best = groups.topk(group_top, dim=-1).values
        # (a place that nobody fills adds nothing; a group without an eligible expert comes last)
        total = torch.where(best[..., 0] == none, none, torch.where(best == none, 0.0, best).sum(-1))
        order = torch.sort(total, dim=-1, descending=True, stable=True).indices[:, :num_topk_groups]
        keep = torch.zeros_like(total).scatter(1, order, 1.0) > 0
        choice = torch.where(keep.unsqueeze(-1), groups, none).view(T, E)
    value, idx = torch.sort(choice, dim=-1, descending=True, stable=True)
    live = value[:, :num_topk] > none
    if token_mask is not None:
        live = live & token_mask.unsqueeze(1)
    idx = torch.where(live, idx[:, :num_topk], -1)
    w = _gathered(logits, idx, score, renormalize)
    if renormalize:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    count = torch.zeros(E + 1, dtype=torch.int32, device=idx.device).scatter_add(0, (idx + 1).flatten(), torch.ones_like(idx, dtype=torch.int32).flatten())[1:]
    return idx.to(topk_idx_t), w * scale, count


def route_backward_ref(d_weights, logits, topk_idx, score='sigmoid', renormalize=True, scale=1.0):
    """:func:`route_backward` stated with plain PyTorch operations."""
    live, at = topk_idx >= 0, topk_idx.clamp_min(0).to(torch.int64)
    w, d = _gathered(logits, topk_idx, score, renormalize), torch.where(live, d_weights, 0.0) * scale
    if renormalize:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
        d = d - (d * w).sum(-1, keepdim=True)
    d = torch.where(live, d * w, 0.0)                               # softmax: d loss / d logit through the chosen scores
    if score == 'sigmoid':
        d = d * (1.0 - _scores(logits, score).gather(1, at))
    out = torch.zeros(logits.shape[0], logits.shape[1] + 1, dtype=d.dtype, device=d.device).scatter(1, torch.where(live, at, logits.shape[1]), d)[:, :-1]
    if score == 'softmax' and not renormalize:
        out = torch.where(live.any(-1, keepdim=True), out - _scores(logits, score) * d.sum(-1, keepdim=True), 0.0)
    return out.to(logits.dtype)
