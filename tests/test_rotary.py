"""Norm and rotation of heads: the kernels and the PyTorch statements against the formulas in 64 bits."""
import pytest
import torch

from deepep_ascend_b200.ops import rotary as R
from deepep_ascend_b200.ops.rotary import qk_norm_rope, qk_norm_rope_append, qk_norm_rope_backward, rope_table

from test_plain_tensor_guard import _watchers

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
BF16, F32, EPS = torch.bfloat16, torch.float32, 2.0**-24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _make(T, Hq, Hk, D, rotary, dtype, param, seed=0, device='cpu', num_positions=500):
    g = torch.Generator().manual_seed(seed)
    r = lambda *shape: torch.randn(*shape, generator=g)      # noqa: E731
    size = torch.rand(T, 1, 1, generator=g) * 3
    q, k, dq, dk = r(T, Hq, D) * size, r(T, Hk, D) * size, r(T, Hq, D), r(T, Hk, D)
    positions = torch.randint(0, num_positions, (T,), generator=g)
    return dict(zip(('q', 'k', 'dq', 'dk'), (t.to(dtype).to(device) for t in (q, k, dq, dk)))), (r(D) * 0.3 + 1).to(param).to(device), (r(D) * 0.3 - 1).to(param).to(device), \
        rope_table(num_positions, rotary).to(device), positions.to(device)


def _rotation(table, positions, D, interleaved, back=False):
    """[T, D, D] matrices: rows are results."""
    rows = table.double().cpu()[positions.cpu()]
    T, half = rows.shape[0], rows.shape[1] // 2
    m = torch.eye(D, dtype=torch.float64).repeat(T, 1, 1)
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        cos, sin = rows[:, i], rows[:, half + i]
        m[:, a, a], m[:, b, b], m[:, a, b], m[:, b, a] = cos, cos, -sin, sin
    return m.transpose(1, 2) if back else m


def _check(given, qw, kw, table, positions, interleaved, eps=1e-6):
    """The square sum of D values, its root, their product with value and weight, and the rotation are off by at most D / 2 + 16 roundings in 32 bits of the magnitudes that go
    into a result, and half a step of the result's type; sums over n rows of the weight's gradient by n + 64 more."""
    D = given['q'].shape[2]
    out = qk_norm_rope(given['q'], given['k'], qw, kw, table, positions, eps, interleaved)
    grads = qk_norm_rope_backward(given['dq'], given['dk'], given['q'], given['k'], qw, kw, table, positions, eps, interleaved)
    few = (D / 2 + 16) * EPS
    for i, (name, w) in enumerate((('q', qw), ('k', kw))):
        x, dy = given[name], given['d' + name]
        assert out[i].dtype == x.dtype and out[i].shape == x.shape and out[i].is_contiguous() and grads[i].dtype == x.dtype and grads[2 + i].dtype == w.dtype
        half, x, dy, w64 = _half(x.dtype), x.double().cpu(), dy.double().cpu(), w.double().cpu()
        rstd = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
        m = _rotation(table, positions, D, interleaved)
        want = torch.einsum('tij,thj->thi', m, x * rstd * w64)
        err = few * torch.einsum('tij,thj->thi', m.abs(), (x * rstd * w64).abs())
        assert ((out[i].double().cpu() - want).abs() <= err + half * (want.abs() + err)).all()
        g = torch.einsum('tij,thj->thi', m.transpose(1, 2), dy)
        big = torch.einsum('tij,thj->thi', m.transpose(1, 2).abs(), dy.abs())
        n, u, u_big = x * rstd, g * w64, big * w64.abs()
        along, along_big = (u * n).mean(-1, keepdim=True), (u_big * n.abs()).mean(-1, keepdim=True)
        want = rstd * (u - n * along)
        err = 2 * few * rstd * (u_big + n.abs() * along_big)
        assert ((grads[i].double().cpu() - want).abs() <= err + half * (want.abs() + err)).all()
        want = (g * n).sum((0, 1))
        err = (few + (x.shape[0] * x.shape[1] + 64) * EPS) * (big * n.abs()).sum((0, 1))
        assert ((grads[2 + i].double().cpu() - want).abs() <= err + _half(w.dtype) * (want.abs() + err) + 1e-38).all()
    return out, grads


SHAPES = [(1, 1, 1, 8, 0), (1, 4, 2, 64, 64), (3, 5, 1, 40, 32), (7, 3, 3, 80, 80), (5, 9, 3, 96, 48), (33, 14, 2, 128, 128), (2, 17, 1, 192, 96), (9, 2, 2, 256, 256), (4, 1, 1, 16, 16)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('dtype,param', [(BF16, F32), (F32, F32), (BF16, BF16), (F32, BF16)])
@pytest.mark.parametrize('T,Hq,Hk,D,rotary', SHAPES)
def test_against_the_formulas(T, Hq, Hk, D, rotary, dtype, param, interleaved, device):
    _check(*_make(T, Hq, Hk, D, rotary, dtype, param, T + D, device), interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize('T,Hq,Hk,D,rotary,dtype', [(1500, 16, 4, 128, 128, BF16), (3001, 7, 1, 64, 32, F32), (700, 8, 8, 192, 192, BF16), (2000, 33, 11, 40, 32, BF16)])
def test_many_rows(T, Hq, Hk, D, rotary, dtype):
    for interleaved in (False, True):
        _check(*_make(T, Hq, Hk, D, rotary, dtype, F32, T, 'cuda'), interleaved)


def test_angles_of_far_positions():
    """Of every position to the last bit of 32: the angles are made in 64."""
    table = rope_table(200000, 16, base=500000.0)
    for p in (0, 1, 65535, 199999):
        angles = [p * 500000.0**(-2 * i / 16) for i in range(8)]
        import math
        want = torch.tensor([math.cos(a) for a in angles] + [math.sin(a) for a in angles], dtype=torch.float64)
        assert ((table[p].double() - want).abs() <= EPS * want.abs() + 1e-10).all()
    assert rope_table(0, 16).shape == (0, 16)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [torch.int64, torch.int32])
def test_positions_outside_the_table(dtype, device):
    given, qw, kw, table, positions = _make(6, 3, 2, 64, 32, BF16, F32, 1, device)
    want = qk_norm_rope(given['q'], given['k'], qw, kw, table, positions)
    p = positions.to(dtype)
    p[1], p[4] = -1, table.shape[0]
    given['q'][1] = float('inf')                              # padding may hold anything
    out = qk_norm_rope(given['q'], given['k'], qw, kw, table, p)
    for got, ref in zip(out, want):
        assert not got[1].any() and got[4].isnan().all() and torch.equal(got[[0, 2, 3, 5]], ref[[0, 2, 3, 5]])
    p[4] = 0
    dq, dk, dqw, dkw = qk_norm_rope_backward(given['dq'], given['dk'], given['q'], given['k'], qw, kw, table, p)
    assert not dq[1].any() and not dk[1].any()
    keep = [0, 2, 3, 4, 5]
    rest = qk_norm_rope_backward(*(given[n][keep] for n in ('dq', 'dk', 'q', 'k')), qw, kw, table, p[keep])
    # (fewer rows: sums in another order, of 15 and 10 terms of ordinary size)
    assert torch.allclose(dqw, rest[2], rtol=0, atol=64 * EPS * 16) and torch.allclose(dkw, rest[3], rtol=0, atol=64 * EPS * 16)
    p[4] = 10**6
    assert all(t.isnan().all() for t in qk_norm_rope_backward(given['dq'], given['dk'], given['q'], given['k'], qw, kw, table, p)[2:])


def _caches(pages, size, Hk, D, dtype, device, layout):
    """Contiguous ones; both in one allocation; heads in front of places."""
    if layout == 'fused':
        both = torch.full((pages, 2, size, Hk, D), 7.0, dtype=dtype, device=device)
        return both[:, 0], both[:, 1]
    if layout == 'heads first':
        return tuple(torch.full((pages, Hk, size, D), 7.0, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))
    return tuple(torch.full((pages, size, Hk, D), 7.0, dtype=dtype, device=device) for _ in range(2))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('layout', ['plain', 'fused', 'heads first'])
@pytest.mark.parametrize('T,Hq,Hk,D,size,dtype,index', [(1, 4, 1, 64, 16, BF16, torch.int64), (19, 8, 2, 128, 24, BF16, torch.int32), (50, 3, 3, 80, 1, F32, torch.int64)])
def test_into_paged_caches(T, Hq, Hk, D, size, dtype, index, layout, device):
    given, qw, kw, table, positions = _make(T, Hq, Hk, D, 16, dtype, F32, T, device)
    q, k = qk_norm_rope(given['q'], given['k'], qw, kw, table, positions)
    v = given['dk']
    pages = (T + size - 1) // size + 2
    k_cache, v_cache = _caches(pages, size, Hk, D, dtype, device, layout)
    slots = torch.randperm(pages * size, generator=torch.Generator().manual_seed(T))[:T].to(index).to(device)
    if T > 4:
        slots[1], slots[3], slots[4] = -1, pages * size, 2**31 - 1      # nowhere
    out = qk_norm_rope_append(given['q'], given['k'], v, qw, kw, table, positions, k_cache, v_cache, slots)
    assert torch.equal(out, q)
    for cache, new in ((k_cache, k), (v_cache, v)):
        want = torch.full((pages * size, Hk, D), 7.0, dtype=dtype, device=device)
        keep = (slots >= 0) & (slots < pages * size)
        want[slots[keep].long()] = new[keep]
        assert torch.equal(cache.reshape(-1, Hk, D), want)
    # the keys as a result too, those that go nowhere among them
    again = qk_norm_rope_append(given['q'], given['k'], v, qw, kw, table, positions, k_cache, v_cache, slots, keep_k=True)
    assert torch.equal(again[0], q) and torch.equal(again[1], k)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('keep_k', [False, True])
def test_caches_without_pages(keep_k, device):
    """Have a place for nobody: nothing is written, and the results are those of any caches."""
    given, qw, kw, table, positions = _make(5, 4, 2, 64, 32, BF16, F32, 9, device)
    want = qk_norm_rope(given['q'], given['k'], qw, kw, table, positions)
    k_cache, v_cache = _caches(0, 16, 2, 64, BF16, device, 'plain')
    for slots in (torch.arange(5, device=device), torch.tensor([-1, 0, 2**31 - 1, 7, -16], dtype=torch.int32, device=device)):
        out = qk_norm_rope_append(given['q'], given['k'], given['dk'], qw, kw, table, positions, k_cache, v_cache, slots, keep_k=keep_k)
        assert torch.equal(out[0] if keep_k else out, want[0]) and (not keep_k or torch.equal(out[1], want[1]))


@pytest.mark.parametrize('slots', [[3, -1, 40, 0, 31, -5], [-1, 32, 99, -2, 40, 50], [7, 6, 5, 4, 3, 2], [-1, -1, -1, -1, -1, 9]])
@pytest.mark.parametrize('device', DEVICES)
def test_the_statement_appends_without_looking(slots, device):
    """Its shapes do not depend on the slots, and nobody waits for them: on a GPU it can be captured into a graph, with gradients to carry as well."""
    from torch.utils._python_dispatch import TorchDispatchMode
    given, qw, kw, table, positions = _make(6, 3, 2, 32, 16, F32, F32, 18, device)
    leaf = given['q'].clone().requires_grad_(True)
    at, caches = torch.full((6,), -1, device=device), _caches(2, 16, 2, 32, F32, device, 'fused')

    def f(at, k_cache, v_cache):
        return R.qk_norm_rope_append(leaf, given['k'], given['dk'], qw, kw, table, positions, k_cache, v_cache, at)

    class Seen(TorchDispatchMode):
        names = set()

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.add(func.overloadpacket.__name__)
            return func(*args, **(kwargs or {}))
    with Seen() as seen:
        f(at, *caches)
    assert not seen.names & {'nonzero', '_local_scalar_dense', 'item'} and 'index_put_' in seen.names
    want = [c.clone().view(32, 2, 32) for c in caches]
    for i, s in enumerate(slots):
        if 0 <= s < 32:
            want[0][s], want[1][s] = qk_norm_rope(given['q'], given['k'], qw, kw, table, positions)[1][i], given['dk'][i]
    if device == 'cuda':
        f(at, *caches)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f(at, *caches)
        at.copy_(torch.tensor(slots))
        graph.replay()
    else:
        at.copy_(torch.tensor(slots))
        out = f(at, *caches)
    assert out.requires_grad
    # (two ways to the same norm in 32 bits)
    assert torch.allclose(caches[0].reshape(32, 2, 32), want[0], rtol=1e-5, atol=1e-5) and torch.equal(caches[1].reshape(32, 2, 32), want[1])
    assert all(torch.equal(c[~hit], torch.full_like(c[~hit], 7.0)) for c in (x.reshape(32, 2, 32) for x in caches)
               for hit in [torch.tensor([p in slots for p in range(32)], device=device)])


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('layout', ['plain', 'fused'])
def test_caches_that_a_gradient_needs(layout, device):
    """Whoever kept them hears that they have been written; inference tensors have nobody to tell."""
    given, qw, kw, table, positions = _make(4, 2, 1, 32, 16, F32, F32, 19, device)
    args = given['q'], given['k'], given['dk'], qw, kw, table, positions
    for which in range(2):
        caches = _caches(2, 16, 1, 32, F32, device, layout)
        w = torch.ones((), device=device, requires_grad=True)
        y = (caches[which] * w).sum()
        qk_norm_rope_append(*args, *caches, torch.arange(4, device=device))
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            y.backward()
    with torch.inference_mode():
        caches = _caches(2, 16, 1, 32, F32, device, layout)
        qk_norm_rope_append(*args, *caches, torch.arange(4, device=device))
        assert (caches[0][0, :4] != 7).all() and torch.equal(caches[1][0, :4], given['dk'])


@pytest.mark.gpu
@pytest.mark.parametrize('layout', ['plain', 'heads first'])
@pytest.mark.parametrize('T,Hq,Hk,D,rotary,dtype', [(900, 33, 11, 128, 128, BF16), (1600, 33, 11, 64, 32, BF16), (600, 33, 11, 256, 256, BF16), (600, 14, 10, 192, 96, F32), (3, 5, 2, 192, 192, BF16),
                                                    (2, 4, 1, 256, 64, F32)])
def test_prompts_into_paged_caches(T, Hq, Hk, D, rotary, dtype, layout):
    """Enough rows that a warp takes several at once, heads that do not divide by them, and the widest heads."""
    given, qw, kw, table, positions = _make(T, Hq, Hk, D, rotary, dtype, F32, T, 'cuda')
    q, k = qk_norm_rope(given['q'], given['k'], qw, kw, table, positions)
    _check(given, qw, kw, table, positions, False)
    pages, size = T // 48 + 3, 48
    k_cache, v_cache = _caches(pages, size, Hk, D, dtype, 'cuda', layout)
    slots = torch.randperm(pages * size, generator=torch.Generator().manual_seed(T))[:T].cuda()
    slots[1] = -1
    out = qk_norm_rope_append(given['q'], given['k'], given['dk'], qw, kw, table, positions, k_cache, v_cache, slots, keep_k=True)
    assert torch.equal(out[0], q) and torch.equal(out[1], k)
    for cache, new in ((k_cache, k), (v_cache, given['dk'])):
        want = torch.full((pages * size, Hk, D), 7.0, dtype=dtype, device='cuda')
        want[slots[slots >= 0]] = new[slots >= 0]
        assert torch.equal(cache.reshape(-1, Hk, D), want)


@pytest.mark.gpu
def test_strides_and_alignment():
    given, qw, kw, table, positions = _make(37, 6, 2, 96, 64, BF16, F32, 3, 'cuda')
    want = qk_norm_rope(given['q'], given['k'], qw, kw, table, positions)
    grads = qk_norm_rope_backward(given['dq'], given['dk'], given['q'], given['k'], qw, kw, table, positions)
    fused = torch.cat([given['q'], given['k'], given['k']], 1)
    odd = lambda t: torch.zeros(t.numel() + 1, dtype=t.dtype, device='cuda')[1:].view(t.shape).copy_(t)      # noqa: E731
    front = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)                                         # noqa: E731
    every_other = torch.stack([positions, positions], -1)[:, 0]
    for q, k, w, tab, pos in ((fused[:, :6], fused[:, 6:8], qw, table, positions), (odd(given['q']), odd(given['k']), odd(qw), odd(table), positions),
                              (front(given['q']), front(given['k']), qw, table, every_other)):
        got = qk_norm_rope(q, k, w, kw, tab, pos)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        again = qk_norm_rope_backward(front(given['dq']), odd(given['dk']), q, k, w, kw, tab, pos)
        assert all(torch.equal(a, b) for a, b in zip(again, grads))


def test_the_function_against_differences():
    g = torch.Generator().manual_seed(0)
    q, k, qw, kw = (torch.randn(*s, dtype=torch.float64, generator=g).requires_grad_(True) for s in ((3, 2, 24), (3, 1, 24), (24,), (24,)))
    table, positions = rope_table(10, 16), torch.tensor([3, -1, 9])
    for interleaved in (False, True):
        assert torch.autograd.gradcheck(lambda *a: R._QkNormRope.apply(*a, table, positions, 1e-3, interleaved), (q, k, qw, kw))


@pytest.mark.gpu
def test_gradients_through_the_call():
    given, qw, kw, table, positions = _make(21, 4, 2, 64, 64, BF16, F32, 4, 'cuda')
    leaves = [t.clone().requires_grad_(True) for t in (given['q'], given['k'], qw, kw)]
    out = qk_norm_rope(*leaves, table, positions)
    assert all(torch.equal(a, b) for a, b in zip(out, qk_norm_rope(given['q'], given['k'], qw, kw, table, positions)))
    got = torch.autograd.grad(out, leaves, [given['dq'], given['dk']])
    want = qk_norm_rope_backward(given['dq'], given['dk'], given['q'], given['k'], qw, kw, table, positions)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a gradient that one of the two alone has, broadcast on its way
    out = qk_norm_rope(*leaves, table, positions)
    got = torch.autograd.grad(out[0].float().sum(), leaves, allow_unused=True)
    want = qk_norm_rope_backward(torch.ones_like(given['q']), torch.zeros_like(given['k']), given['q'], given['k'], qw, kw, table, positions)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # what goes into the caches carries none; the queries do
    k_cache, v_cache = _caches(2, 16, 2, 64, BF16, 'cuda', 'plain')
    y = qk_norm_rope_append(leaves[0], leaves[1], given['dk'], *leaves[2:], table, positions, k_cache, v_cache, torch.arange(21, device='cuda'))
    assert y.requires_grad and not k_cache.requires_grad


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('tracer', ['jit.trace', 'make_fx', 'functionalize', 'vmap', 'forward mode', 'dispatch mode'])
def test_it_is_seen(tracer, device):
    given, qw, kw, table, positions = _make(6, 2, 1, 32, 16, F32, F32, 5, device)
    k = given['k']
    for f in (lambda x: qk_norm_rope(x, k, qw, kw, table, positions)[0],
              lambda x: qk_norm_rope_backward(given['dq'], given['dk'], x, k, qw, kw, table, positions)[0]):
        out = _watchers()[tracer](f, given['q'])
        if callable(out):
            assert all(torch.allclose(out(x), f(x), rtol=1e-5, atol=1e-5) for x in (given['q'], given['q'].flip(0)))
        else:
            out = torch.autograd.forward_ad.unpack_dual(out)[0] if tracer == 'forward mode' else out
            assert torch.allclose(out.reshape(6, 2, 32), f(given['q']), rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_in_two_graphs():
    made = [_make(300, 4, 2, 64, 64, BF16, F32, seed, 'cuda') for seed in (6, 7)]
    want, graphs = [], []
    for given, qw, kw, table, positions in made:
        args = given['q'], given['k'], qw, kw, table, positions
        want.append((*qk_norm_rope(*args), *qk_norm_rope_backward(given['dq'], given['dk'], *args)))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = (*qk_norm_rope(*args), *qk_norm_rope_backward(given['dq'], given['dk'], *args))
        graphs.append((graph, out))
    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for (_, out), ref in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(out, ref))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('Hq,Hk', [(0, 3), (3, 0), (0, 0)])
@pytest.mark.parametrize('T', [4, 700])
def test_without_heads(T, Hq, Hk, device):
    """Of one kind, or of both: the other one's results and gradients are what they are beside heads."""
    given, qw, kw, table, positions = _make(T, 3, 3, 64, 32, BF16, F32, 17, device)
    want = qk_norm_rope(given['q'], given['k'], qw, kw, table, positions)
    grads = qk_norm_rope_backward(given['dq'], given['dk'], given['q'], given['k'], qw, kw, table, positions)
    q, dq, k, dk = given['q'][:, :Hq], given['dq'][:, :Hq], given['k'][:, :Hk], given['dk'][:, :Hk]
    out = qk_norm_rope(q, k, qw, kw, table, positions)
    assert torch.equal(out[0], want[0][:, :Hq]) and torch.equal(out[1], want[1][:, :Hk])
    got = qk_norm_rope_backward(dq, dk, q, k, qw, kw, table, positions)
    assert torch.equal(got[0], grads[0][:, :Hq]) and torch.equal(got[1], grads[1][:, :Hk])
    # (the weights' sums may be in another order: of 64 rows in 32 bits, or 3 T)
    for x, y, H in ((got[2], grads[2], Hq), (got[3], grads[3], Hk)):
        assert not x.any() if H == 0 else torch.allclose(x, y, rtol=0, atol=(3 * T + 64) * EPS * 3 * T * 16)
    behind = torch.full_like(positions, 10**6)
    got = qk_norm_rope_backward(dq, dk, q, k, qw, kw, table, behind)
    assert all(not x.any() if H == 0 else x.isnan().all() for x, H in ((got[2], Hq), (got[3], Hk)))
    k_cache, v_cache = _caches(T, 1, Hk, 64, BF16, device, 'plain')
    append = qk_norm_rope_append(q, k, k, qw, kw, table, positions, k_cache, v_cache, torch.arange(T, device=device), keep_k=True)
    assert all(torch.equal(a, b) for a, b in zip(append, out)) and torch.equal(k_cache[:, 0], out[1])


@pytest.mark.parametrize('device', DEVICES)
def test_a_table_without_positions(device):
    """Nobody has one: no numbers, and zeros for padding."""
    given, qw, kw, table, positions = _make(4, 2, 1, 64, 64, BF16, F32, 8, device)
    positions[2] = -1
    rest = [0, 1, 3]
    for t in (*qk_norm_rope(given['q'], given['k'], qw, kw, table[:0], positions),
              *qk_norm_rope_backward(given['dq'], given['dk'], given['q'], given['k'], qw, kw, table[:0], positions)[:2]):
        assert t[rest].isnan().all() and not t[2].any()


@pytest.mark.gpu
def test_nothing_to_do():
    given, qw, kw, table, positions = _make(4, 2, 1, 64, 64, BF16, F32, 8, 'cuda')
    q, k = qk_norm_rope(given['q'][:0], given['k'][:0], qw, kw, table, positions[:0])
    assert q.shape == (0, 2, 64) and k.shape == (0, 1, 64)
    dq, dk, dqw, dkw = qk_norm_rope_backward(q, k, q, k, qw, kw, table, positions[:0])
    assert not dqw.any() and not dkw.any()
    # a table without positions: nobody has one
    q, _ = qk_norm_rope(given['q'], given['k'], qw, kw, table[:0], positions)
    assert q.isnan().all()


@pytest.mark.gpu
def test_refusals():
    given, qw, kw, table, positions = _make(4, 2, 1, 64, 64, BF16, F32, 8, 'cuda')
    ok = dict(q=given['q'], k=given['k'], q_weight=qw, k_weight=kw, table=table, positions=positions)
    wide = torch.zeros(4, 2, 264, dtype=BF16, device='cuda')
    for bad in (dict(q=given['q'].half()), dict(k=given['k'].float()), dict(k=given['k'][:3]), dict(q_weight=qw[:32]), dict(k_weight=kw.bfloat16()), dict(table=table.double()),
                dict(table=table[:, :24]), dict(table=torch.zeros(5, 80, device='cuda')), dict(positions=positions.float()), dict(positions=positions[:2]), dict(positions=positions.cpu()),
                dict(q=wide, k=wide, q_weight=torch.zeros(264, device='cuda'), k_weight=torch.zeros(264, device='cuda')), dict(q=given['q'][..., :60], k=given['k'][..., :60])):
        with pytest.raises(RuntimeError):
            qk_norm_rope(**{**ok, **bad})
    with pytest.raises(RuntimeError):
        qk_norm_rope_backward(given['dq'][:2], given['dk'], *ok.values())
    k_cache, v_cache = _caches(2, 16, 1, 64, BF16, 'cuda', 'plain')
    slots = torch.arange(4, device='cuda')
    ok = dict(ok, v=given['k'], k_cache=k_cache, v_cache=v_cache, slots=slots)
    odd = torch.zeros(2 * 16 * 64 + 1, dtype=BF16, device='cuda')[1:].view(2, 16, 1, 64)
    for bad in (dict(v=given['q']), dict(k_cache=k_cache.float(), v_cache=v_cache.float()), dict(v_cache=v_cache[:1]), dict(k_cache=odd), dict(slots=slots[:2]), dict(slots=slots.float()),
                dict(k_cache=k_cache.expand(2, 16, 2, 64), v_cache=v_cache.expand(2, 16, 2, 64)), dict(k_cache=k_cache[..., ::2], v_cache=v_cache[..., ::2])):
        with pytest.raises(RuntimeError):
            qk_norm_rope_append(**{**ok, **bad})
    assert (k_cache == 7).all()
