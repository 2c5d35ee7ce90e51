"""Pre-normed mixture-of-experts block: ``x + experts(norm(x))`` with its own router, from this library's kernels

    layer norm (``ops.norm``) -> gate product (tcgen05 GEMM) -> routing (``ops.router``)
      -> ``FusedMoE`` (dispatch -> expert GEMMs -> combine) -> residual

forward and backward.  The reference stops at dispatch / combine; callers bring everything around them.

    python -m deepep_ascend_b200.models.block          trains a small block on one GPU with Muon and shows loss and balance
"""
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from ..buffers.elastic import ElasticBuffer
from ..ops import gemm as G
from ..ops.norm import layer_norm
from ..ops.router import RouteFunction
from .moe import FusedMoE


class LayerNormFunction:
    """``apply(x, weight, bias or None, eps) -> y``: the first result of :func:`ops.norm.layer_norm`, which carries gradients itself."""

    @staticmethod
    def apply(x, weight, bias, eps):
        return layer_norm(x, weight, bias, eps)[0]


class GateFunction(torch.autograd.Function):
    """``apply(h bf16 [T, H], gate bf16 [E, H], buffer=None) -> logits bf16 [T, E]`` on the tensor cores; ``H`` and ``E`` multiples of 8.  ``buffer``: see
    :func:`ops.gemm.gemm_nt`."""

    @staticmethod
    def forward(ctx, h, gate, buffer=None):
        ctx.save_for_backward(h, gate)
        ctx.buffer = buffer
        return G.gemm_nt(h, gate, buffer=buffer)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logits):
        h, gate = ctx.saved_tensors
        T, d_logits = h.shape[0], d_logits.contiguous()
        d_h = d_gate = None
        if ctx.needs_input_grad[0]:
            d_h = G.grouped_gemm_nn(d_logits, gate.unsqueeze(0), torch.zeros((T + G.BLOCK_M - 1) // G.BLOCK_M, dtype=torch.int32, device=h.device), buffer=ctx.buffer)
        if ctx.needs_input_grad[1]:
            rows = (T + 63) // 64 * 64                      # the sum over tokens runs in whole blocks of 64
            if rows != T:
                h, d_logits = (torch.nn.functional.pad(t, (0, 0, 0, rows - T)) for t in (h, d_logits))
            d_gate = G.gemm_kgrouped_tn(d_logits, h, torch.tensor([0, rows], dtype=torch.int32, device=h.device))[0]
        return d_h, d_gate, None


class MoEBlock(nn.Module):
    """``forward(x bf16 [T, hidden], token_mask bool [T] = None) -> x + FusedMoE(norm(x), route(gate(norm(x))))``.

    ``num_experts``: of all ranks, a multiple of 8; the experts of this rank are ``self.experts.w13`` and ``w2``, the gate is replicated.
    The logits are bf16 (the gate's product is rounded once), the scores that are made of them 32-bit: experts whose logits round alike tie, and go by index.
    ``score``, ``num_groups``, ``num_topk_groups``, ``group_top``, ``renormalize`` and ``scale`` are those of :func:`ops.router.route`.
    ``balance_bias`` (fp32 ``[num_experts]``, no parameter) is added to the scores for the choice of experts; :meth:`update_balance` moves it after
    a step so that crowded experts are chosen less.  ``self.last_count``: tokens of this rank that chose each expert in the last forward pass."""

    def __init__(self, buffer: ElasticBuffer, num_experts: int, hidden: int, intermediate: int, num_topk: int, score: str = 'sigmoid', num_groups: int = 1,
                 num_topk_groups: int = 1, scale: float = 1.0, eps: float = 1e-5, norm_bias: bool = False, init_std: float = 0.02, device='cuda',
                 renormalize: bool = True, group_top: int = 2, **moe):
        super().__init__()
        if num_experts % 8 or hidden % 8:
            raise ValueError('num_experts and hidden must be multiples of 8')
        self.options = dict(num_topk=num_topk, score=score, num_groups=num_groups, num_topk_groups=num_topk_groups, scale=scale, renormalize=renormalize,
                            group_top=group_top)
        self.eps = eps
        self.norm_weight = nn.Parameter(torch.ones(hidden, device=device))
        self.norm_bias = nn.Parameter(torch.zeros(hidden, device=device)) if norm_bias else None
        self.gate = nn.Parameter((torch.randn(num_experts, hidden, device=device) * hidden**-0.5).bfloat16())
        self.register_buffer('balance_bias', torch.zeros(num_experts, device=device))
        self.experts = FusedMoE(buffer, num_experts, hidden, intermediate, init_std=init_std, device=device, **moe)
        self.last_count: Optional[torch.Tensor] = None

    def forward(self, x: torch.Tensor, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        h = LayerNormFunction.apply(x, self.norm_weight, self.norm_bias, self.eps)
        logits = GateFunction.apply(h, self.gate, self.experts.buffer)
        idx, weights, count = RouteFunction.apply(logits, dict(self.options, bias=self.balance_bias, token_mask=token_mask))
        self.last_count = count.clone()                     # (the router's results share an allocation, which this would keep)
        return x + self.experts(h, idx, weights)

    @torch.no_grad()
    def update_balance(self, speed: float = 1e-3, group=None) -> None:
        """Moves every expert's bias by ``speed`` towards the mean load of the last forward pass, of all ranks of ``group`` (the buffer's, if none is given), which
        call this together and come to the same bias."""
        count = self.last_count.float()
        group = self.experts.buffer.group if group is None else group
        if group is not None and torch.distributed.get_world_size(group) > 1:
            torch.distributed.all_reduce(count, group=group)
        self.balance_bias += speed * torch.sign(count.mean() - count)


def main(steps: int = 30) -> None:
    from ..optim import Muon
    torch.manual_seed(0)
    T, H, I, E, K = 512, 256, 256, 16, 2
    buffer = ElasticBuffer(None, num_max_tokens_per_rank=T, hidden=H, num_topk=K)
    try:
        block = MoEBlock(buffer, E, H, I, K, num_groups=4, num_topk_groups=2, scale=2.0)
        matrices = Muon([block.gate, block.experts.w13, block.experts.w2], lr=0.05, buffer=buffer)
        vectors = torch.optim.AdamW([block.norm_weight], lr=1e-3)
        x, target = torch.randn(T, H, device='cuda').bfloat16(), torch.randn(T, H, device='cuda')
        for step in range(steps):
            loss = (block(x).float() - target).square().mean()
            loss.backward()
            matrices.param_groups[0]['lr'] = 0.05 * (1.0 - step / steps)
            for opt in (matrices, vectors):
                opt.step()
                opt.zero_grad()
            block.update_balance(0.01)
            if step % 5 == 0 or step == steps - 1:
                print('step %3d  loss %.4f  tokens per expert %d..%d' % (step, loss.item(), block.last_count.min().item(), block.last_count.max().item()))
        buffer.check_status()
    finally:
        buffer.destroy()


if __name__ == '__main__':
    main()
