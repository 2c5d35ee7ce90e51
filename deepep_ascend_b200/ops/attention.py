"""Attention on the tensor cores: packed prompts, forward and backward (``csrc/kernels/attention.cu``), and single tokens over a paged cache
(``csrc/kernels/paged_attention.cu``).  CPU tensors take the PyTorch statements below.

No counterpart in the reference, which stops at the exchange of tokens.
"""
from typing import Optional, Tuple

import torch

from .. import _native
from .gemm import _by_type, _core_of, _gradient_alone


def _options(q: torch.Tensor, cu_seqlens, cu_seqlens_k, scale: Optional[float]):
    if cu_seqlens is None and cu_seqlens_k is not None:
        raise ValueError('cu_seqlens_k goes with cu_seqlens')
    return cu_seqlens, cu_seqlens if cu_seqlens_k is None else cu_seqlens_k, q.shape[-1]**-0.5 if scale is None else float(scale)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None, cu_seqlens_k: Optional[torch.Tensor] = None,
              causal: bool = True, scale: Optional[float] = None, buffer=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``q [tokens, heads, dim]``, ``k`` and ``v [keys, kv_heads, dim]`` (bf16, ``dim`` a multiple of 8, at most 128) -> ``(o`` like ``q``, contiguous,
    ``lse`` fp32 ``[heads, tokens])``: ``o = softmax(scale q k^T) v`` and ``lse = log sum exp(scale q k^T)`` within each sequence.  ``heads`` is a multiple of
    ``kv_heads``: as many neighbouring heads share keys and values.  ``scale``: ``dim ** -0.5`` if none is given, positive (a normal number of 32 bits).

    ``cu_seqlens`` int32 ``[sequences + 1]``: where the sequences start in ``q``, and where the last one ends; none: one sequence.  ``cu_seqlens_k``: the same of ``k``
    and ``v``, if their lengths are others (keys of earlier calls in front).  With ``causal`` both of a sequence end together: query ``i`` of ``n`` sees the keys up to
    ``i + keys - n``.  A query that sees no key, and one that belongs to no sequence, gets zeros and an ``lse`` of -inf.

    Scores, sums and ``lse`` are 32 bits; probabilities (and in the gradients what is made of them) are rounded to bf16 where they go into a product, so results are off by up to two
    roundings of bf16 of their terms.  Whatever lies behind a sequence is not looked at; within one, keys and values must be numbers (a value that is none reaches queries of its tile
    that do not see it).  Any strides;
    heads whose channels are apart or that do not start on 16 bytes are copied first.  ``buffer``: see :func:`ops.gemm.gemm_nt`.

    Both results carry gradients, by the kernels of :func:`attention_backward`.  Tracers, function transforms, dispatch modes (selective
    checkpoints are one) and forward mode see the PyTorch statement, which takes any floating type and holds the scores of all queries and all keys at once, ``4 heads tokens keys`` bytes
    several times over: for real batches it is too large."""
    cu_q, cu_k, scale = _options(q, cu_seqlens, cu_seqlens_k, scale)
    if q.is_cuda and _by_type(q, k, v, cu_q, cu_k):
        res = _native.load().attention(q, k, v, cu_q, cu_k, causal, scale, _core_of(buffer))
        if res is not None:
            return res
        if _gradient_alone(q, k, v):
            return _Attention.apply(q, k, v, cu_q, cu_k, causal, scale, buffer)
    return attention_ref(q, k, v, cu_q, cu_k, causal, scale)


class _Attention(torch.autograd.Function):
    """``apply(q, k, v, cu_seqlens, cu_seqlens_k, causal, scale, buffer) -> (o, lse)``, both with gradients."""

    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, causal, scale, buffer):
        o, lse = attention(q, k, v, cu_q, cu_k, causal, scale, buffer)
        ctx.save_for_backward(q, k, v, o, lse, cu_q, cu_k)
        ctx.options = dict(causal=causal, scale=scale, buffer=buffer)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    def backward(ctx, d_o, d_lse):
        q, k, v, o, lse, cu_q, cu_k = ctx.saved_tensors
        if d_o is None:
            d_o = torch.zeros_like(o)
        d_lse = None if d_lse is None else d_lse.contiguous()
        return (*attention_backward(d_o, q, k, v, o, lse, cu_q, cu_k, d_lse=d_lse, **ctx.options), None, None, None, None, None)


def attention_backward(d_o: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
                       cu_seqlens_k: Optional[torch.Tensor] = None, causal: bool = True, scale: Optional[float] = None, d_lse: Optional[torch.Tensor] = None,
                       buffer=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of :func:`attention` from ``d_o`` (like ``o``), optionally ``d_lse`` (like ``lse``), and what the forward pass was given and returned ->
    ``(d_q, d_k, d_v)``, contiguous.  Those of shared keys and values are added over their heads in 32 bits; every sum is taken in one order.  Queries and keys of no
    sequence, queries that see nothing and keys that nobody sees get zeros.  Where these gradients are to carry gradients themselves, and for whoever watches, the
    PyTorch statement runs (of any floating type, with all scores at once)."""
    cu_q, cu_k, scale = _options(q, cu_seqlens, cu_seqlens_k, scale)
    if q.is_cuda and _by_type(d_o, q, k, v, o, lse, d_lse, cu_q, cu_k):
        res = _native.load().attention_backward(d_o, q, k, v, o, lse, d_lse, cu_q, cu_k, causal, scale, _core_of(buffer))
        if res is not None:
            return res
    return attention_backward_ref(d_o, q, k, v, o, lse, cu_q, cu_k, causal, scale, d_lse)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One new token per sequence: ``q [sequences, heads, dim]`` (bf16, ``dim`` a multiple of 8, at most 128; at most 4096 sequences) over the keys and values of a paged cache,
    ``k_cache`` and ``v_cache [pages, page_size, kv_heads, dim]`` (as :func:`ops.rotary.qk_norm_rope_append` fills them) -> ``o`` like ``q``, contiguous, or ``out``.

    Sequence ``i`` has ``lengths[i]`` keys (int32), the new token's own among them; key ``p`` stands in place ``p % page_size`` of page ``page_table[i, p // page_size]``
    (int32 ``[sequences, at least as many pages]``).  Places behind the length are not looked at, nor are the table's.  A sequence without keys gets zeros; one that names a page which
    the caches do not have, or is longer than its row of the table, gets no numbers (NaN); what its other pages hold may be read, nothing outside the caches and the table is.
    Probabilities are rounded to bf16 where they go into the product with the values.  ``heads``, ``kv_heads`` and ``scale``: see
    :func:`attention`.  How the work is cut depends on the lengths of the whole batch: the last bits of a result can change with the batch that it is in.

    Carries no gradient of its own: where one is wanted, and for whoever watches, the PyTorch statement runs."""
    scale = q.shape[-1]**-0.5 if scale is None else float(scale)
    if q.is_cuda and _by_type(q, k_cache, v_cache, page_table, lengths, out):
        res = _native.load().paged_attention(q, k_cache, v_cache, page_table, lengths, scale, out)
        if res is not None:
            return res
    o = paged_attention_ref(q, k_cache, v_cache, page_table, lengths, scale)
    return o if out is None else out.copy_(o)


def _wide(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float64 else t.float()


def _places(t, cu):
    """Of every row: its sequence (-1: none), its place there, the sequence's length."""
    at = torch.arange(t.shape[0], device=t.device)
    if cu is None:
        return torch.zeros_like(at), at, torch.full_like(at, t.shape[0])
    if cu.numel() < 2:
        return torch.full_like(at, -1), at, at
    cu = cu.long()
    seq = (torch.searchsorted(cu, at, right=True) - 1).clamp(0, cu.numel() - 2)
    return torch.where((at >= cu[seq]) & (at < cu[seq + 1]), seq, -1), at - cu[seq], cu[seq + 1] - cu[seq]


def _of_sequences(t, cu):
    """``t`` in 32 bits (64 if it has them), zeros in rows of no sequence."""
    return torch.where((_places(t, cu)[0] >= 0)[:, None, None], _wide(t), 0.0)


def _scores(q, k, cu_q, cu_k, causal, scale):
    """``q`` and, for every query head, ``k`` in 32 bits; scores ``[heads, tokens, keys]`` and whether a query sees a key."""
    (sq, iq, nq), (sk, ik, nk) = _places(q, cu_q), _places(k, cu_k)
    sees = (sq[:, None] == sk) & (sq >= 0)[:, None]
    if causal:
        sees = sees & (ik - nk <= (iq - nq)[:, None])
    q, k = _of_sequences(q, cu_q), _of_sequences(k, cu_k).repeat_interleave(int(q.shape[1]) // int(k.shape[1]), 1)
    return q, k, torch.where(sees, torch.einsum('ihd,jhd->hij', q, k) * scale, float('-inf')), sees


def attention_ref(q, k, v, cu_seqlens=None, cu_seqlens_k=None, causal=True, scale=None):
    """:func:`attention` stated with plain PyTorch operations (any device; what the kernel is tested against).  All scores at once."""
    cu_q, cu_k, scale = _options(q, cu_seqlens, cu_seqlens_k, scale)
    if k.shape[0] == 0:
        return torch.zeros_like(q), _wide(q).new_full((q.shape[1], q.shape[0]), float('-inf'))
    _, _, s, sees = _scores(q, k, cu_q, cu_k, causal, scale)
    some = sees.any(-1)
    top = torch.where(some, s.max(-1).values, 0.0).detach()
    e = torch.exp(s - top.unsqueeze(-1))
    total = torch.where(some, e.sum(-1), 1.0)
    o = torch.einsum('hij,jhd->ihd', e / total.unsqueeze(-1), _of_sequences(v, cu_k).repeat_interleave(int(q.shape[1]) // int(k.shape[1]), 1))
    return o.to(q.dtype).contiguous(), torch.where(some, top + torch.log(total), float('-inf'))


def attention_backward_ref(d_o, q, k, v, o, lse, cu_seqlens=None, cu_seqlens_k=None, causal=True, scale=None, d_lse=None):
    """:func:`attention_backward` stated with plain PyTorch operations."""
    cu_q, cu_k, scale = _options(q, cu_seqlens, cu_seqlens_k, scale)
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    shape = (k.shape[0], k.shape[1], int(q.shape[1]) // int(k.shape[1]), k.shape[2])      # (numbers while tracing, too)
    types = q.dtype, k.dtype, v.dtype
    q, k, s, sees = _scores(q, k, cu_q, cu_k, causal, scale)
    some = sees.any(-1)
    p = torch.where(sees, torch.exp(s - torch.where(some, lse, 0.0).unsqueeze(-1)), 0.0)
    g = _of_sequences(d_o, cu_q)
    dp = torch.einsum('ihd,jhd->hij', g, _of_sequences(v, cu_k).repeat_interleave(shape[2], 1))
    delta = (g * _of_sequences(o, cu_q)).sum(-1).t()
    if d_lse is not None:
        delta = delta - torch.where(some, d_lse, 0.0)
    ds = torch.where(sees, p * (dp - delta.unsqueeze(-1)), 0.0) * scale
    dq = torch.einsum('hij,jhd->ihd', ds, k)
    dk, dv = (torch.einsum('hij,ihd->jhd', x, y).reshape(shape).sum(2) for x, y in ((ds, q), (p, g)))
    return tuple(t.to(dtype).contiguous() for t, dtype in zip((dq, dk, dv), types))


def paged_attention_ref(q, k_cache, v_cache, page_table, lengths, scale=None):
    """:func:`paged_attention` stated with plain PyTorch operations (any device; what the kernel is tested against).  All places of the table at once."""
    scale = q.shape[-1]**-0.5 if scale is None else float(scale)
    pages, size, kv_heads, dim = k_cache.shape
    n, group = lengths.long(), q.shape[1] // kv_heads
    at = torch.arange(page_table.shape[1] * size, device=q.device)
    there = at < n[:, None]
    page = page_table.long()[:, at // size]
    bad = (there & ((page < 0) | (page >= pages))).any(-1) | (n > at.numel())
    page, place = torch.where(there & (page >= 0) & (page < pages), page, 0), at % size
    if pages == 0 or at.numel() == 0:
        o = _wide(q).new_zeros(q.shape)
    else:
        k, v = (torch.where(there[:, :, None, None], _wide(c[page, place]), 0.0) for c in (k_cache, v_cache))
        s = torch.einsum('bhgd,bjhd->bhgj', _wide(q).reshape(q.shape[0], kv_heads, group, dim), k) * scale
        s = torch.where(there[:, None, None], s, float('-inf'))
        top = torch.where(n[:, None, None] > 0, s.amax(-1), 0.0)
        e = torch.exp(s - top.unsqueeze(-1))
        e = e / torch.where(n[:, None, None] > 0, e.sum(-1), 1.0).unsqueeze(-1)
        o = torch.einsum('bhgj,bjhd->bhgd', e, v).reshape(q.shape)
    return torch.where(bad[:, None, None], float('nan'), o).to(q.dtype)
