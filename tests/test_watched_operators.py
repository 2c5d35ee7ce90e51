"""Operators whose CPU form carries gradients and is seen by tracers, transforms and dispatch modes do the same on a GPU, where a kernel takes its place."""
import pytest
import torch

from deepep_ascend_b200 import _native
from deepep_ascend_b200.ops import gemm, muon, norm, router

from test_plain_tensor_guard import _watchers

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
EPS = 2.0**-24


@pytest.mark.parametrize('name', sorted(set(_watchers()) - {'gradient'}))
def test_native_calls_see_who_watches(name):
    """What the native calls ask for themselves, on CPU tensors."""
    watched = _native.load().watched
    seen = []

    def f(x):
        seen.append(watched([x]) or not gemm._by_type(x))
        return x * 2
    x = torch.randn(2, 4)
    assert not watched([x]) and not watched([x, torch.nn.Parameter(x)]) and gemm._by_type(x, None, torch.nn.Parameter(x))
    _watchers()[name](f, x)
    assert seen and all(seen)
    assert not watched([x])


def test_types_that_are_no_plain_tensors():
    class Named(torch.Tensor):
        pass
    x = torch.randn(2, 4)
    assert not gemm._by_type(x, x.as_subclass(Named)) and not gemm._by_type(x.as_subclass(Named))
    with torch.device('cpu'):                    # a mode that hands every call on
        assert gemm._by_type(x, None)
    x.requires_grad_(True)
    assert gemm._gradient_alone(None, x) and not gemm._gradient_alone(x.detach())
    with torch.no_grad():
        assert not gemm._gradient_alone(x)


def _norm_inputs(device, dtype, T=6, H=40):
    g = torch.Generator().manual_seed(0)
    return [t.to(dtype).to(device) for t in (torch.randn(T, H, generator=g) + 0.5, torch.randn(H, generator=g) + 1.0, torch.randn(H, generator=g))]


def test_the_norms_function_against_differences():
    """First and second derivatives of every result, statistics among them."""
    x, w, b = (t.requires_grad_(True) for t in _norm_inputs('cpu', torch.float64, 3, 7))
    f = lambda x, w, b: norm._LayerNorm.apply(x, w, b, 1e-3)      # noqa: E731
    assert torch.autograd.gradcheck(f, (x, w, b)) and torch.autograd.gradgradcheck(f, (x, w, b))
    g = lambda x, w: norm._LayerNorm.apply(x, w, None, 1e-3)[1:]      # noqa: E731
    assert torch.autograd.gradcheck(g, (x, w)) and torch.autograd.gradgradcheck(g, (x, w))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(6, 40), (2, 3, 40)])
def test_the_norm_carries_gradients(dtype, shape):
    x, w, b = _norm_inputs('cuda', dtype)
    leaves = [x.view(shape).clone().requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)]
    y, mean, rstd = norm.layer_norm(*leaves)
    assert y.shape == shape and mean.shape == rstd.shape == shape[:-1] and 'LayerNorm' in type(y.grad_fn).__name__
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    # the same kernel as by hand
    with torch.no_grad():
        want = norm.layer_norm_backward(dy, *leaves[:2], mean, rstd, with_bias=True)
        assert torch.equal(norm.layer_norm(*leaves)[0], y)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    # gradients of the statistics: (rows of 40 values: a few dozen roundings of terms no larger than the results' own scale)
    ref = [t.detach().double().requires_grad_(True) for t in leaves]
    _, m, r = norm.layer_norm_ref(*ref)
    size = 2.0**-8 if dtype == torch.bfloat16 else 64 * EPS
    for a, c in ((mean, m), (rstd, r), (mean * rstd, m * r)):
        d, = torch.autograd.grad(a.sum(), leaves[:1], retain_graph=True)
        e, = torch.autograd.grad(c.sum(), ref[:1], retain_graph=True)
        torch.testing.assert_close(d.double(), e, rtol=2 * size, atol=2 * size * e.abs().max().item())


@pytest.mark.gpu
def test_a_gradient_of_the_norms_gradient():
    x, w, b = (t.requires_grad_(True) for t in _norm_inputs('cuda', torch.float32))
    def second(x, w, b, f):
        y = f(x, w, b)[0]
        d = torch.autograd.grad((y**3).sum(), (x, w, b), create_graph=True)
        return torch.autograd.grad(sum((t**2).sum() for t in d), (x, w, b))
    got = second(x, w, b, norm.layer_norm)
    want = second(*(t.detach().double().requires_grad_(True) for t in (x, w, b)), norm.layer_norm_ref)
    for p, q in zip(got, want):
        torch.testing.assert_close(p.double(), q, rtol=1e-4, atol=1e-4 * q.abs().max().item())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('tracer', ['jit.trace', 'make_fx', 'functionalize', 'vmap', 'forward mode', 'dispatch mode'])
def test_the_norm_is_seen(tracer, device):
    """A recorded norm gives the result for rows that it has not seen, and a transformed one that of its statement."""
    x, w, b = _norm_inputs(device, torch.float32)
    stats = norm.layer_norm(x, w, b)[1:]
    dy = torch.randn_like(x)
    for f in (lambda x: norm.layer_norm(x, w, b)[0], lambda x: norm.layer_norm_backward(dy, x, w, *stats, with_bias=True)[0]):
        out = _watchers()[tracer](f, x)
        if callable(out):
            assert all(torch.allclose(out(v), f(v), rtol=1e-5, atol=1e-5) for v in (x, torch.randn_like(x) * 3))
        else:
            out = torch.autograd.forward_ad.unpack_dual(out)[0] if tracer == 'forward mode' else out
            assert torch.allclose(out.reshape(x.shape), f(x), rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_a_tangent_through_the_norm():
    x, w, b = _norm_inputs('cuda', torch.float32)
    t = torch.randn_like(x)
    got = torch.func.jvp(lambda x: norm.layer_norm(x, w, b)[0], (x,), (t,))[1]
    want = torch.func.jvp(lambda x: norm.layer_norm_ref(x, w.double(), b.double())[0], (x.double(),), (t.double(),))[1]
    torch.testing.assert_close(got.double(), want, rtol=1e-4, atol=1e-4)


ROUTES = [dict(), dict(score='softmax', renormalize=False), dict(score='softmax', scale=2.5), dict(renormalize=False, num_groups=4, num_topk_groups=2)]


@pytest.mark.parametrize('options', ROUTES)
def test_the_routing_function_against_differences(options):
    logits = torch.randn(4, 16, generator=torch.Generator().manual_seed(0), dtype=torch.float64).requires_grad_(True)
    f = lambda l: router.RouteFunction.apply(l, dict(options, num_topk=3))[1]      # noqa: E731
    assert torch.autograd.gradcheck(f, (logits,)) and torch.autograd.gradgradcheck(f, (logits,))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('options', ROUTES)
def test_routing_carries_gradients(options, dtype):
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(50, 32, generator=g).to(dtype).cuda().requires_grad_(True)
    bias = torch.randn(32, generator=g).mul(0.1).cuda().requires_grad_(True)
    mask = (torch.arange(50) % 7 != 2).cuda()
    idx, w, count = router.route(logits, 4, bias=bias, token_mask=mask, **options)
    assert 'RouteFunction' in type(w.grad_fn).__name__ and not idx.requires_grad and not count.requires_grad
    d = torch.randn_like(w)
    got, none = torch.autograd.grad(w, (logits, bias), d, allow_unused=True)
    assert none is None                                        # the bias counts for the choice alone
    keep = {k: options[k] for k in ('score', 'renormalize', 'scale') if k in options}
    with torch.no_grad():
        assert torch.equal(got, router.route_backward(d, logits, idx, **keep))
        again = router.route(logits, 4, bias=bias, token_mask=mask, **options)
    assert all(torch.equal(p, q) for p, q in zip((idx, w, count), again))
    # the gradient of a gradient, against the statement's: a few dozen roundings of 32 bits
    if dtype == torch.float32:
        def second(l, f):
            first, = torch.autograd.grad((f(l, 4, bias=bias.detach().to(l.dtype), **options)[1]**3).sum(), l, create_graph=True)
            return torch.autograd.grad((first**2).sum(), l)[0]
        want = second(logits.detach().double().requires_grad_(True), router.route_ref)
        torch.testing.assert_close(second(logits, router.route).double(), want, rtol=1e-4, atol=1e-4 * want.abs().max().item())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('tracer', ['jit.trace', 'make_fx', 'functionalize', 'vmap', 'forward mode', 'dispatch mode'])
def test_routing_is_seen(tracer, device):
    logits = torch.randn(20, 32, device=device)
    idx = router.route(logits, 4)[0]
    d = torch.randn(20, 4, device=device)
    for f in (lambda l: router.route(l, 4, num_groups=4, num_topk_groups=2)[1], lambda l: router.route(l, 4)[0] * 1, lambda l: router.route(l, 4)[2] * 1,
              lambda l: router.route_backward(d, l, idx), lambda l: router.route_backward(d, l, idx, 'softmax', False)):
        out = _watchers()[tracer](f, logits)
        want = f(logits)
        if callable(out):
            assert all(torch.allclose(out(v), f(v), rtol=1e-5, atol=1e-5) for v in (logits, torch.randn_like(logits) * 2))
        else:
            out = torch.autograd.forward_ad.unpack_dual(out)[0] if tracer == 'forward mode' else out
            assert torch.allclose(out.reshape(want.shape), want, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('tracer', ['jit.trace', 'make_fx', 'functionalize', 'vmap', 'forward mode', 'dispatch mode', 'fake tensors'])
def test_an_update_is_seen(tracer, device):
    """Against the statement: bf16 results whose last places differ (the kernel's errors are stated where it is tested)."""
    x = torch.randn(2, 24, 40, device=device)
    out = _watchers()[tracer](lambda x: muon.orthogonalize(x) * 1, x)
    if tracer == 'fake tensors':
        assert type(out).__name__ == 'FakeTensor' and out.shape == x.shape and out.dtype == torch.bfloat16
    elif callable(out):
        for v in (x, torch.randn_like(x) * 3):
            assert torch.allclose(out(v), muon.orthogonalize(v), rtol=2e-2, atol=5e-3)
    else:
        out = torch.autograd.forward_ad.unpack_dual(out)[0] if tracer == 'forward mode' else out
        assert torch.allclose(out.reshape(x.shape), muon.orthogonalize(x), rtol=2e-2, atol=5e-3)


@pytest.mark.parametrize('device', DEVICES)
def test_an_update_carries_gradients(device):
    x = torch.randn(3, 8, 5, generator=torch.Generator().manual_seed(0)).to(device).requires_grad_(True)
    d = torch.randn(3, 8, 5, generator=torch.Generator().manual_seed(1)).to(device)
    got, = torch.autograd.grad((muon.orthogonalize(x, steps=2).float() * d).sum(), x)
    y = x.detach().double().requires_grad_(True)
    want, = torch.autograd.grad((muon.orthogonalize_ref(y, steps=2) * d.double()).sum(), y)
    # (what comes back through the rounding to bf16 is rounded to it)
    assert (got.double() - want).norm() < 2.0**-7 * want.norm()
    with torch.no_grad():
        assert not muon.orthogonalize(x).requires_grad
