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


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('lr,decay', [(1e-3, 0.0), (1e-3, 0.1), (0.02, 0.1)])
def test_bf16_weights_move_as_fp32_ones_do(lr, decay, device):
    """Updates far below a weight's last place add up: the weights are those of an fp32 run, rounded."""
    p, q = _parameter((2, 96, 64), BF16, device), _parameter((2, 96, 64), BF16, device)
    q = torch.nn.Parameter(q.detach().float())
    a, b = Muon([p], lr=lr, weight_decay=decay), Muon([q], lr=lr, weight_decay=decay)
    start = p.detach().clone()
    for grad in _gradients(p, 30):
        p.grad, q.grad = grad, grad.float()
        a.step()
        b.step()
        assert torch.equal(p, q.bfloat16())
    assert (p != start).float().mean() > 0.9


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [F32, BF16, torch.float16])
def test_decay_alone_shrinks_the_weights(dtype, device):
    p = _parameter((64, 32), dtype, device)
    opt, start = Muon([p], lr=0.01, weight_decay=0.1), p.detach().float().clone()
    for _ in range(100):
        p.grad = torch.zeros_like(p)
        opt.step()
    # 100 fp32 products are off by a rounding each, the weight by that of its type
    half_ulp = {F32: 0.0, BF16: 2.0**-8, torch.float16: 2.0**-11}[dtype]
    torch.testing.assert_close(p.detach().float(), start * 0.999**100, rtol=half_ulp + 202 * 2.0**-24, atol=2.0**-25)


@pytest.mark.parametrize('device', DEVICES)
def test_weights_that_others_have_changed(device):
    """A weight that is set between two steps (loaded, clipped, tied) is the one that the next step starts from; the others go on with all their digits."""
    p = _parameter((32, 32), BF16, device)
    opt = Muon([p], lr=1e-3)
    grads = _gradients(p, 12)
    for grad in grads[:6]:
        p.grad = grad
        opt.step()
    q = torch.nn.Parameter(opt.state[p]['weight'].clone())
    with torch.no_grad():
        p[3], q[3] = 0.0, 0.0
        p[5, 7] = q[5, 7] = float('inf')
    other = Muon([q], lr=1e-3)
    other.load_state_dict({'state': {0: {'momentum': opt.state[p]['momentum']}}, 'param_groups': other.state_dict()['param_groups']})
    for grad in grads[6:]:
        p.grad, q.grad = grad, grad.float()
        opt.step()
        other.step()
        assert torch.equal(p, q.bfloat16())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('shape', [(0, 8, 4), (4, 0), (0, 4), (2, 3, 0), (2, 2, 0, 5)])
def test_parameters_without_elements(shape, device):
    """A rank that holds no expert, or a layer of no width, has nothing to update."""
    p, full = _parameter(shape, F32, device), _parameter((8, 8), F32, device)
    opt = Muon([p, full], weight_decay=0.1)
    before = full.detach().clone()
    p.grad, full.grad = torch.zeros_like(p), torch.ones_like(full)
    opt.step()
    assert p.shape == shape and not torch.equal(full, before)


def test_waits_of_the_products_report_to_the_buffer(monkeypatch):
    from deepep_ascend_b200 import optim
    seen = []
    monkeypatch.setattr(optim, 'orthogonalize', lambda x, *args, buffer=None: seen.append(buffer) or x.bfloat16())
    buffer = object()
    for given in (None, buffer):
        p = _parameter((8, 8), F32, 'cpu')
        opt = Muon([p], buffer=given)
        p.grad = torch.ones_like(p)
        opt.step()
        opt.load_state_dict(copy.deepcopy(opt.state_dict()))         # (a buffer is no state)
    assert seen == [None, buffer]


def test_what_others_have_put_into_a_checkpoint():
    """Entries that are not this optimiser's come through as the base class treats them: a count of steps is no tensor."""
    p = _parameter((8, 8), BF16, 'cpu')
    opt = Muon([p])
    p.grad = torch.ones_like(p)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    saved['state'][0].update(step=3, seen=torch.arange(2))
    opt.load_state_dict(saved)
    assert opt.state[p]['step'] == 3 and opt.state[p]['momentum'].dtype == F32
    assert torch.equal(opt.state[p]['seen'].float(), torch.arange(2).float())
