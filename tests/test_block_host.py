"""What the block decides on the host, on CPU tensors: the experts and the gate's product, which run on a GPU alone, are stood in for."""
import os
import socket
from types import SimpleNamespace

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from deepep_ascend_b200.models.block import MoEBlock


def _block(group=None, num_ranks=1, **options):
    torch.manual_seed(0)
    buffer = SimpleNamespace(num_ranks=num_ranks, enable_expand=True, group=group, core=None)
    return MoEBlock(buffer, 16, 128, 128, 2, device='cpu', **options)


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
