"""The optimiser of matrices: what it leaves alone, what it keeps between steps and across a checkpoint."""
import copy

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


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_a_checkpoint_keeps_every_bit(dtype, device):
    """A run that is saved and loaded goes on as the one that was not, although the base class casts loaded states to their parameter's type."""
    def fresh():
        p = _parameter((2, 48, 32), dtype, device)
        return p, Muon([p], lr=0.02, weight_decay=0.1)
    p, opt = fresh()
    grads = _gradients(p, 5)
    for grad in grads[:3]:
        p.grad = grad
        opt.step()
    saved, weights = copy.deepcopy(opt.state_dict()), p.detach().clone()
    resumed, other = fresh()
    with torch.no_grad():
        resumed.copy_(weights)
    other.load_state_dict(saved)
    assert opt.state[p].keys() == other.state[resumed].keys()
    for name, value in opt.state[p].items():
        loaded = other.state[resumed][name]
        assert loaded.dtype == value.dtype == F32 and loaded.device == value.device and torch.equal(loaded, value)
        assert loaded.data_ptr() != saved['state'][0][name].data_ptr()           # what was saved is not written to by later steps
    for grad in grads[3:]:
        for q, o in ((p, opt), (resumed, other)):
            q.grad = grad.clone()
            o.step()
        assert torch.equal(p, resumed) and torch.equal(opt.state[p]['momentum'], other.state[resumed]['momentum'])
