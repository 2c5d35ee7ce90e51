"""What the block decides on the host, on CPU tensors: the experts and the gate's product, which run on a GPU alone, are stood in for."""
import os
import socket
from types import SimpleNamespace

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from deepep_ascend_b200.models import block as block_module
from deepep_ascend_b200.models.block import MoEBlock
from deepep_ascend_b200.ops.router import route_ref


def _block(group=None, num_ranks=1, **options):
    torch.manual_seed(0)
    buffer = SimpleNamespace(num_ranks=num_ranks, enable_expand=True, group=group, core=None)
    return MoEBlock(buffer, 16, 128, 128, 4, device='cpu', **options)


def _worker_balance(rank, port):
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port))
    dist.init_process_group('gloo', rank=rank, world_size=2)
    try:
        counts = torch.randint(0, 100, (2, 16), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
        total = counts.sum(0).float()
        want = 0.5 * torch.sign(total.mean() - total)
        for given in (None, dist.group.WORLD):
            block = _block(dist.group.WORLD, 2)
            block.last_count = counts[rank].clone()
            block.update_balance(0.5, *(() if given is None else (given,)))
            assert torch.equal(block.balance_bias, want)                     # the same on every rank
            assert torch.equal(block.last_count, counts[rank])
    finally:
        dist.destroy_process_group()


def test_the_bias_moves_alike_on_all_ranks_of_the_buffer():
    with socket.socket() as s:
        s.bind(('127.0.0.1', 0))
        port = s.getsockname()[1]
    mp.spawn(_worker_balance, args=(port,), nprocs=2, join=True)


def test_the_bias_of_a_single_rank():
    block = _block()
    block.last_count = torch.arange(16, dtype=torch.int32)
    block.update_balance(0.25)
    assert torch.equal(block.balance_bias, 0.25 * torch.sign(7.5 - torch.arange(16.0)))


class _Experts(torch.nn.Module):
    """Keeps what it is given, and is differentiable in the weights."""

    def forward(self, h, idx, weights):
        self.given = h, idx, weights
        return h * (weights * torch.arange(1.0, 5.0)).sum(1, keepdim=True)


def _stand_in(block, monkeypatch):
    monkeypatch.setattr(block_module.GateFunction, 'apply', staticmethod(lambda h, gate, *_: (h @ gate.float().t()).bfloat16()))
    buffer, block.experts = block.experts.buffer, _Experts()
    block.experts.buffer = buffer


@pytest.mark.parametrize('options', [dict(), dict(num_groups=4, num_topk_groups=2, scale=2.5),
                                     dict(score='softmax', num_groups=8, num_topk_groups=3, renormalize=False, group_top=1), dict(num_groups=16, num_topk_groups=5, group_top=1),
                                     dict(score='softmax', renormalize=True)])
def test_the_choice_is_the_routers(options, monkeypatch):
    """Every option, the balance bias and the mask come to the router: experts and weights are those of its statement for the gate's logits."""
    block = _block(**options)
    _stand_in(block, monkeypatch)
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        block.balance_bias.copy_(torch.randn(16, generator=g) * 0.3)             # large enough to change most choices
    x, mask = torch.randn(50, 128, generator=g), torch.arange(50) % 5 != 1
    out = block(x, mask)
    h, idx, weights = block.experts.given
    logits = (h @ block.gate.float().t()).bfloat16()
    want = route_ref(logits, 4, bias=block.balance_bias, token_mask=mask, **{'num_groups': 1, **options})
    assert torch.equal(idx, want[0]) and torch.equal(weights, want[1]) and torch.equal(block.last_count, want[2])
    assert torch.equal(out, x + h * (weights * torch.arange(1.0, 5.0)).sum(1, keepdim=True))
    # each of them counts
    given = dict(options, bias=block.balance_bias, token_mask=mask)
    for left_out in (['bias'], ['token_mask'], ['num_groups', 'num_topk_groups', 'group_top'], ['group_top'], ['score'], ['scale'], ['renormalize']):
        # (but the best four of 16 groups of one, which are the best four, and what is the router's own default)
        if left_out[0] in given and given[left_out[0]] is not True and not ('group_top' in left_out and given['num_groups'] == 16):
            other = route_ref(logits, 4, **{k: v for k, v in given.items() if k not in left_out})
            assert not (torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])), left_out


def test_the_gradient_of_a_softmax_that_is_not_renormalised(monkeypatch):
    """Every expert's row of the gate has one, which the other forms do not give."""
    for options, rows in ((dict(score='softmax', renormalize=False), 16), (dict(), 4)):
        block = _block(**options)
        _stand_in(block, monkeypatch)
        block(torch.randn(1, 128, generator=torch.Generator().manual_seed(2))).square().sum().backward()
        assert int((block.gate.grad.abs().sum(1) > 0).sum()) == rows


def _gate_on_cpu(monkeypatch):
    """The gate's products in PyTorch; returns which buffers they were given."""
    buffers = []
    G = block_module.G

    def nn(a, b, tile_group, out=None, num_sms=0, buffer=None):
        buffers.append(buffer)
        return a @ b[0]

    def nt(a, b, out=None, num_sms=0, buffer=None):
        buffers.append(buffer)
        return a @ b.t()
    monkeypatch.setattr(G, 'gemm_nt', nt)
    monkeypatch.setattr(G, 'grouped_gemm_nn', nn)
    monkeypatch.setattr(G, 'gemm_kgrouped_tn', lambda a, b, off: (a.t() @ b).unsqueeze(0))
    return buffers


def test_waits_of_the_gates_product_report_to_the_buffer(monkeypatch):
    buffers, block = _gate_on_cpu(monkeypatch), _block()
    block.experts = _Experts()
    block.experts.buffer = buffer = SimpleNamespace(group=None)
    block(torch.randn(10, 128).bfloat16().requires_grad_(True)).float().square().sum().backward()
    assert block.gate.grad is not None and buffers == [buffer, buffer]


def test_a_gradient_of_the_gates_gradient_is_refused(monkeypatch):
    """The products of its backward pass carry none: terms would be missing without a word."""
    _gate_on_cpu(monkeypatch)
    native = block_module.GateFunction
    h, gate = torch.randn(6, 8).bfloat16().requires_grad_(True), torch.randn(8, 8).bfloat16().requires_grad_(True)
    for name in ('grouped_gemm_nn', 'gemm_kgrouped_tn'):             # (native calls return results without a graph)
        f = getattr(block_module.G, name)
        monkeypatch.setattr(block_module.G, name, lambda *a, f=f, **k: f(*a, **k).detach())
    logits = native.apply(h, gate)
    d = torch.autograd.grad(logits.float().square().sum(), (h, gate), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(sum(t.float().square().sum() for t in d), h)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        ((d[0].float() * h.float()).sum() + (d[1].float() ** 2).sum()).backward()
