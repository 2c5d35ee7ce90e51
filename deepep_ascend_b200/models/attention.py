"""Pre-normed attention block: ``x + attention(norm(x))``, what stands in front of a ``MoEBlock`` in a layer, from this library's kernels

    layer norm (``ops.norm``) -> product to queries, keys and values (tcgen05 GEMM) -> norm and rotation of heads (``ops.rotary``)
      -> attention (``ops.attention``: packed prompts, or single tokens over a paged cache) -> product -> residual

forward and backward for packed sequences, and without gradients for prompts and single tokens over a paged cache.  The reference stops at the exchange of tokens.

    python -m deepep_ascend_b200.models.attention          trains a small layer (attention and experts) on one GPU and goes on with a prompt
"""
from typing import Optional, Tuple

import torch
import torch.nn as nn

from ..ops.attention import attention, paged_attention
from ..ops.rotary import qk_norm_rope, qk_norm_rope_append, rope_table
from .block import GateFunction, LayerNormFunction


def positions_of(cu_seqlens: Optional[torch.Tensor], num_tokens: int, device=None) -> torch.Tensor:
    """int64 ``[num_tokens]``: every token's place in its sequence (``cu_seqlens`` as of :func:`ops.attention.attention`), -1 behind the last one."""
    at = torch.arange(num_tokens, device=device if cu_seqlens is None else cu_seqlens.device)
    if cu_seqlens is None:
        return at
    seq = torch.searchsorted(cu_seqlens[1:].contiguous(), at.to(cu_seqlens.dtype), right=True)
    return torch.where(seq < cu_seqlens.numel() - 1, at - cu_seqlens[seq.clamp_max(max(cu_seqlens.numel() - 2, 0))], -1)


def slots_of(page_table: torch.Tensor, positions: torch.Tensor, page_size: int) -> torch.Tensor:
    """int64 slots (as of :func:`ops.rotary.qk_norm_rope_append`) of one position per row of ``page_table``; -1 for a negative one, or one that the row has no page for."""
    page = torch.div(positions, page_size, rounding_mode='floor').long()
    if page_table.shape[1] == 0:
        return torch.full_like(page, -1)
    there = (positions >= 0) & (page < page_table.shape[1])
    entry = page_table.gather(1, page.clamp(0, page_table.shape[1] - 1).unsqueeze(1)).squeeze(1).long()
    return torch.where(there & (entry >= 0), entry * page_size + positions % page_size, -1)


class AttentionBlock(nn.Module):
    """``forward(x bf16 [T, hidden], cu_seqlens=None, positions=None) -> x + out(attention(rotated(norm(x))))`` for packed sequences, causal, with gradients.

    ``hidden`` a multiple of 8, ``head_dim`` of 8 and at most 128, ``num_heads`` of ``num_kv_heads``; ``rotary_dim`` (a multiple of 16; ``head_dim`` if none is given) channels of
    every head are rotated, positions are below ``max_positions``.  ``buffer``: see :func:`ops.gemm.gemm_nt`.

    ``cu_seqlens``: see :func:`ops.attention.attention`; ``positions`` (int64 ``[T]``): places in the sequences, if none are given.  Tokens of no sequence come back as they are."""

    def __init__(self, hidden: int, num_heads: int, num_kv_heads: int, head_dim: int = 128, rotary_dim: Optional[int] = None, max_positions: int = 8192, base: float = 10000.0,
                 interleaved: bool = False, eps: float = 1e-5, init_std: float = 0.02, device='cuda', buffer=None):
        super().__init__()
        if hidden % 8 or head_dim % 8 or not 8 <= head_dim <= 128 or num_kv_heads < 1 or num_heads < 1 or num_heads % num_kv_heads:
            raise ValueError('hidden and head_dim (at most 128) must be multiples of 8, num_heads one of num_kv_heads')
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if rotary_dim % 16 or not 0 <= rotary_dim <= head_dim:
            raise ValueError('rotary_dim must be a multiple of 16 and at most head_dim')
        self.num_heads, self.num_kv_heads, self.head_dim, self.eps, self.interleaved, self.buffer = num_heads, num_kv_heads, head_dim, eps, interleaved, buffer
        normal = lambda *shape: nn.Parameter((torch.randn(*shape, device=device) * init_std).bfloat16())      # noqa: E731
        self.norm_weight = nn.Parameter(torch.ones(hidden, device=device))
        self.qkv = normal((num_heads + 2 * num_kv_heads) * head_dim, hidden)
        self.q_weight, self.k_weight = (nn.Parameter(torch.ones(head_dim, device=device)) for _ in range(2))
        self.out = normal(hidden, num_heads * head_dim)
        self.register_buffer('table', rope_table(max_positions, rotary_dim, base, device), persistent=False)

    def _heads(self, x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        qkv = GateFunction.apply(LayerNormFunction.apply(x, self.norm_weight, None, self.eps), self.qkv, self.buffer)
        return qkv.view(x.shape[0], self.num_heads + 2 * self.num_kv_heads, self.head_dim).split((self.num_heads, self.num_kv_heads, self.num_kv_heads), 1)

    def _result(self, x: torch.Tensor, o: torch.Tensor) -> torch.Tensor:
        return x + GateFunction.apply(o.view(x.shape[0], self.num_heads * self.head_dim), self.out, self.buffer)

    def forward(self, x: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        if x.shape[0] == 0:
            return x.clone()
        q, k, v = self._heads(x)
        positions = positions_of(cu_seqlens, x.shape[0], x.device) if positions is None else positions
        q, k = qk_norm_rope(q, k, self.q_weight, self.k_weight, self.table, positions, self.eps, self.interleaved)
        return self._result(x, attention(q, k, v, cu_seqlens, buffer=self.buffer)[0])

    def new_cache(self, num_pages: int, page_size: int = 64) -> Tuple[torch.Tensor, torch.Tensor]:
        """Caches of ``num_pages`` pages for keys and values, in one allocation (not filled)."""
        both = torch.empty(num_pages, 2, page_size, self.num_kv_heads, self.head_dim, dtype=torch.bfloat16, device=self.qkv.device)
        return both[:, 0], both[:, 1]

    @torch.no_grad()
    def prefill(self, x: torch.Tensor, cache: Tuple[torch.Tensor, torch.Tensor], slots: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
                positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        """:meth:`forward` of whole prompts, whose keys and values also go to ``slots`` (``[T]``, see :func:`ops.rotary.qk_norm_rope_append`) of ``cache``."""
        if x.shape[0] == 0:
            return x.clone()
        q, k, v = self._heads(x)
        positions = positions_of(cu_seqlens, x.shape[0], x.device) if positions is None else positions
        q, k = qk_norm_rope_append(q, k, v, self.q_weight, self.k_weight, self.table, positions, *cache, slots, self.eps, self.interleaved, keep_k=True)
        return self._result(x, attention(q, k, v, cu_seqlens, buffer=self.buffer)[0])

    @torch.no_grad()
    def decode(self, x: torch.Tensor, cache: Tuple[torch.Tensor, torch.Tensor], page_table: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
        """One new token per sequence, ``x [sequences, hidden]``, whose key and value go to their place; ``page_table`` and ``lengths`` (the new token counted) as of
        :func:`ops.attention.paged_attention`.  A sequence of length 0 takes no part.  Nothing waits for the host: it can be captured into a CUDA graph."""
        if x.shape[0] == 0:
            return x.clone()
        q, k, v = self._heads(x)
        positions = (lengths - 1).long()
        q = qk_norm_rope_append(q, k, v, self.q_weight, self.k_weight, self.table, positions, *cache, slots_of(page_table, positions, cache[0].shape[1]), self.eps, self.interleaved)
        return self._result(x, paged_attention(q, *cache, page_table, lengths))


def main(steps: int = 20, new_tokens: int = 8) -> None:
    from ..buffers.elastic import ElasticBuffer
    from ..optim import Muon
    from .block import MoEBlock
    torch.manual_seed(0)
    T, H, E, K = 512, 256, 16, 2
    buffer = ElasticBuffer(None, num_max_tokens_per_rank=T, hidden=H, num_topk=K)
    try:
        layer = nn.ModuleList([AttentionBlock(H, 8, 2, 64, max_positions=1024, buffer=buffer), MoEBlock(buffer, E, H, 256, K, num_groups=4, num_topk_groups=2, scale=2.0)])
        mixer, experts = layer
        matrices = Muon([mixer.qkv, mixer.out, experts.gate, experts.experts.w13, experts.experts.w2], lr=0.02, buffer=buffer)
        vectors = torch.optim.AdamW([p for p in layer.parameters() if p.dim() == 1], lr=1e-3)
        # every token's target is the input of the token before it in its sequence
        cu = torch.tensor([0, 200, 200, 512], dtype=torch.int32, device='cuda')
        x = torch.randn(T, H, device='cuda').bfloat16()
        target = x.roll(1, 0).float()
        for step in range(steps):
            loss = (experts(mixer(x, cu)).float() - target).square().mean()
            loss.backward()
            for opt in (matrices, vectors):
                opt.step()
                opt.zero_grad()
            if step % 5 == 0 or step == steps - 1:
                print('step %3d  loss %.4f' % (step, loss.item()))
        # a prompt, and tokens one by one behind it
        with torch.no_grad():
            cache, page_table = mixer.new_cache(8, 64), torch.arange(8, dtype=torch.int32, device='cuda')[None]
            n = 200
            y = experts(mixer.prefill(x[:n], cache, torch.arange(n, device='cuda')))
            for i in range(new_tokens):
                y = experts(mixer.decode(y[-1:], cache, page_table, torch.tensor([n + i + 1], dtype=torch.int32, device='cuda')))
            print('%d tokens behind a prompt of %d, last of size %.3f' % (new_tokens, n, y.float().abs().mean().item()))
        buffer.check_status()
    finally:
        buffer.destroy()


if __name__ == '__main__':
    main()
