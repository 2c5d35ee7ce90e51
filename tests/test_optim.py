"""The optimiser of matrices: what it leaves alone, what it keeps between steps and across a checkpoint."""
import pytest
import torch

from deepep_ascend_b200.optim import Muon

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
BF16, F32 = torch.bfloat16, torch.float32


def _parameter(shape, dtype, device, seed=0, std=0.02):
    return torch.nn.Parameter((torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(device))


def _gradients(p, count, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(p.shape, generator=g).to(p.dtype).to(p.device) for _ in range(count)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('nesterov', [True, False])
def test_the_gradient_is_the_callers(dtype, nesterov, device):
    """Accumulating callers, norms that are logged and buckets of reduced gradients read it after the step."""
    p = _parameter((3, 24, 40), dtype, device)
    opt = Muon([p], nesterov=nesterov)
    for grad in _gradients(p, 3):
        p.grad = grad
        before = grad.clone()
        opt.step()
        assert p.grad is grad and torch.equal(grad, before)
