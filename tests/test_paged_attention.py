"""Attention of single tokens over a paged cache: the kernel and the PyTorch statement against the formulas in 64 bits."""
import pytest
import torch

from deepep_ascend_b200.ops.attention import paged_attention

from test_plain_tensor_guard import _watchers

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
BF16, HALF, EPS = torch.bfloat16, 2.0**-8, 2.0**-23


def _make(lengths, H, Hk, D, size, seed=0, device='cpu', layout='plain', extra=2):
    """Pages anywhere; places that nobody may look at hold no numbers, places of the table that nobody needs hold anything."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + size - 1) // size for n in lengths]
    pages, width = sum(need) + 3, max(need + [0]) + extra
    order = torch.randperm(pages, generator=g).int()
    table = torch.randint(-5, 10**6, (len(lengths), width), generator=g).int()
    k, v = (torch.full((pages, size, Hk, D), float('nan')) for _ in range(2))
    at = 0
    for b, (n, m) in enumerate(zip(lengths, need)):
        mine = order[at:at + m]
        table[b, :m] = mine
        at += m
        for c in (k, v):
            flat = torch.full((m * size, Hk, D), float('nan'))
            flat[:n] = torch.randn(n, Hk, D, generator=g)
            c[mine.long()] = flat.view(m, size, Hk, D)
    k, v = k.bfloat16().to(device), v.bfloat16().to(device)
    if layout == 'fused':
        both = torch.stack([k, v], 1)
        k, v = both[:, 0], both[:, 1]
    elif layout == 'heads first':
        k, v = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (k, v))
    q = (1.5 * torch.randn(len(lengths), H, D, generator=g)).bfloat16().to(device)
    return q, k, v, table.to(device), torch.tensor(lengths, dtype=torch.int32, device=device)


def _check(q, k, v, table, lengths, scale=None, skip=()):
    """As of packed prompts: a score is off by E = scale (D + 8) EPS sum |q k|, a probability by E, roundings of its exponent and half a step, a sum of n terms by n EPS."""
    o = paged_attention(q, k, v, table, lengths, scale)
    assert o.shape == q.shape and o.dtype == BF16 and o.is_contiguous()
    B, H, D = q.shape
    size, Hk = k.shape[1], k.shape[2]
    c = D**-0.5 if scale is None else scale
    O, Q, K, V, T = (t.double().cpu() if t.dtype == BF16 else t.long().cpu() for t in (o, q, k, v, table))
    for b, n in enumerate(lengths.tolist()):
        if b in skip:
            continue
        if n == 0:
            assert not O[b].any()
            continue
        at = torch.arange(n)
        page, place = T[b, at // size], at % size
        for h in range(H):
            x, y, z = Q[b, h], K[page, place, h // (H // Hk)], V[page, place, h // (H // Hk)]
            s = c * y @ x
            E = c * (D + 8) * EPS * (y.abs() @ x.abs())
            p = torch.softmax(s, 0)
            want, err = p @ z, (p * (HALF + E + E.max() + 4 * EPS * (1 + s.abs()) + (2 * n + 64) * EPS)) @ z.abs()
            assert ((O[b, h] - want).abs() <= err + HALF * (want.abs() + err)).all(), (b, h)
    return o


CASES = [([1], 1, 1, 128, 16), ([17, 0, 64, 65, 1], 8, 2, 64, 16), ([200], 32, 8, 128, 64), ([300, 1000, 5], 14, 2, 128, 24), ([130, 7], 3, 3, 96, 1), ([63, 129, 500], 24, 1, 80, 256),
         ([40, 41], 34, 2, 32, 8), ([0, 0], 4, 1, 64, 16), ([1500], 1, 1, 8, 48), ([513, 512, 511], 16, 1, 128, 128)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('lengths,H,Hk,D,size', CASES)
def test_against_the_formulas(lengths, H, Hk, D, size, device):
    args = _make(lengths, H, Hk, D, size, sum(lengths) + D, device)
    o = _check(*args)
    _check(*args, scale=0.4)
    assert torch.equal(o, paged_attention(*args, out=torch.full_like(o, 3.0)))


@pytest.mark.gpu
@pytest.mark.parametrize('lengths,H,Hk,D,size', [([9000], 4, 1, 128, 64), ([40000, 3, 0, 700], 8, 2, 64, 16), ([2000 + 37 * i for i in range(40)], 4, 2, 128, 32),
                                                 ([i % 70 for i in range(600)], 8, 4, 128, 16), ([33] * 4096, 2, 1, 32, 16), ([70000, 1, 70000], 7, 1, 128, 128)])
def test_longer_and_more(lengths, H, Hk, D, size):
    """Stretches that begin and end inside sequences, sequences that many share, many short ones in a stretch."""
    _check(*_make(lengths, H, Hk, D, size, 5, 'cuda'))


@pytest.mark.gpu
@pytest.mark.parametrize('layout', ['plain', 'fused', 'heads first'])
def test_layouts(layout):
    args = _make([700, 30, 1], 8, 2, 64, 16, 6, 'cuda', layout)
    want = _check(*_make([700, 30, 1], 8, 2, 64, 16, 6, 'cuda'))
    assert torch.equal(paged_attention(*args), want)
    q, k, v, table, lengths = args
    wide = torch.full((3, table.shape[1] + 9), -7, dtype=torch.int32, device='cuda')
    wide[:, 2:2 + table.shape[1]] = table
    odd = torch.zeros(q.numel() + 1, dtype=BF16, device='cuda')[1:].view(q.shape).copy_(q)
    assert torch.equal(paged_attention(odd, k, v, wide[:, 2:2 + table.shape[1]], lengths), want)
    assert torch.equal(paged_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, table, lengths), want)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('lengths', [[40, 90, 20, 50], [4000, 900, 20, 5000]])
def test_pages_that_are_none(lengths, device):
    """Sequences that name them, or are longer than their row of the table, get no numbers; the others theirs."""
    q, k, v, table, n = _make(lengths, 4, 2, 64, 16, 7, device, extra=0)
    table[0, 1], table[1, 2] = -1, k.shape[0]
    if len(lengths) > 3:
        n[3] = table.shape[1] * 16 + 1
    o = paged_attention(q, k, v, table, n)
    assert all(o[b].isnan().all() for b in (0, 1, 3))
    _check(q, k, v, table, n, skip=(0, 1, 3))
    n[3] = 2**31 - 1
    assert paged_attention(q, k, v, table, n)[3].isnan().all()
    n[2] = -3                                              # as of a sequence without keys
    assert not paged_attention(q, k, v, table, n)[2].any()
    o = paged_attention(q, k, v, table[:, :0], torch.tensor([0, 0, 0, 1], dtype=torch.int32, device=device))
    assert not o[:3].any() and o[3].isnan().all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('page', [-1, -2, -3, -2**31, 2**31 - 1])
@pytest.mark.parametrize('n', [30, 5000])
def test_any_number_that_is_no_page(n, page, device):
    """First, in the middle and last of a sequence's pages; in tables that cut the work and in those that do not."""
    lengths = [n, 20, n, n - 5]
    q, k, v, table, lens = _make(lengths, 4, 2, 64, 16, 14, device)
    for b, at in ((0, 0), (2, n // 32), (3, (n - 6) // 16)):
        table[b, at] = page
    o = paged_attention(q, k, v, table, lens)
    assert all(o[b].isnan().all() for b in (0, 2, 3))
    _check(q, k, v, table, lens, skip=(0, 2, 3))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('width', [1, 100])
def test_caches_without_pages(width, device):
    """Every page is one that they do not have."""
    q, k, v, _, _ = _make([1, 1, 1], 4, 2, 64, 16, 13, device)
    table = torch.zeros(3, width, dtype=torch.int32, device=device)
    o = paged_attention(q, k[:0].clone(), v[:0].clone(), table, torch.tensor([1, 0, 16 * width], dtype=torch.int32, device=device))
    assert o[0].isnan().all() and not o[1].any() and o[2].isnan().all()


@pytest.mark.gpu
def test_the_same_bits_and_graphs():
    """Graphs of one shape, each with data of its own, replayed in turn; lengths that change between replays."""
    made = [_make([3000, 17, 1200], 8, 2, 128, 16, seed, 'cuda') for seed in (8, 9)]
    want = [paged_attention(*args) for args in made]
    graphs = []
    for args in made:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged_attention(*args)
        graphs.append((graph, out))
    for _ in range(4):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, ref) for (_, out), ref in zip(graphs, want))
    made[0][4].copy_(torch.tensor([10, 16, 700], dtype=torch.int32))
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], _check(*made[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [paged_attention(*made[1]) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(t, want[1]) for t in got)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A cache of 9 GB whose last pages are used: element offsets pass 2^32."""
    size, Hk, D = 64, 8, 128
    pages = 2**32 // (size * Hk * D) + 40
    k = torch.empty(pages, size, Hk, D, dtype=BF16, device='cuda')
    v = torch.empty_like(k)
    table = torch.tensor([[pages - 1, 3, pages - 7]], dtype=torch.int32, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(0)
    for p in table[0].tolist():
        for c in (k, v):
            c[p] = torch.randn(size, Hk, D, device='cuda', generator=g).bfloat16()
    q = torch.randn(1, 16, D, device='cuda', generator=g).bfloat16()
    n = torch.tensor([150], dtype=torch.int32, device='cuda')
    got = paged_attention(q, k, v, table, n)
    small = table[0].long()
    want = _check(q, k[small], v[small], torch.arange(3, dtype=torch.int32, device='cuda')[None], n)
    assert torch.equal(got, want)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('tracer', ['jit.trace', 'make_fx', 'functionalize', 'vmap', 'forward mode', 'dispatch mode'])
def test_it_is_seen(tracer, device):
    q, k, v, table, lengths = _make([20, 3], 2, 1, 16, 8, 10, device)
    f = lambda x: paged_attention(x, k, v, table, lengths)      # noqa: E731
    out = _watchers()[tracer](f, q)
    if callable(out):
        assert all(torch.allclose(out(x).float(), f(x).float(), rtol=8 * HALF, atol=8 * HALF) for x in (q, q.flip(0)))
    else:
        out = torch.autograd.forward_ad.unpack_dual(out)[0] if tracer == 'forward mode' else out
        assert torch.allclose(out.reshape(q.shape).float(), f(q).float(), rtol=8 * HALF, atol=8 * HALF)


@pytest.mark.parametrize('device', DEVICES)
def test_a_result_that_a_gradient_needs(device):
    """Whoever kept what is given for the result hears that it has been written."""
    args = _make([20, 3], 2, 1, 16, 8, 10, device)
    out, w = torch.zeros_like(args[0]), torch.ones((), device=device, requires_grad=True)
    y = (out * w).sum()
    assert paged_attention(*args, out=out) is out or out.any()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()
    with torch.inference_mode():
        assert torch.equal(paged_attention(*args, out=torch.zeros_like(out)), out)


@pytest.mark.gpu
def test_a_gradient_goes_through_the_statement():
    q, k, v, table, lengths = _make([20, 3], 2, 1, 16, 8, 11, 'cuda')
    x = q.clone().requires_grad_(True)
    o = paged_attention(x, k, v, table, lengths)
    assert o.requires_grad and torch.allclose(o.float(), paged_attention(q, k, v, table, lengths).float(), rtol=8 * HALF, atol=8 * HALF)
    assert torch.autograd.grad(o.float().sum(), x)[0].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize('scale', [1e-50, 1e-39, 3e38, 1e300, -1.0, float('nan')])
def test_scales_that_32_bits_do_not_hold(scale):
    with pytest.raises(RuntimeError, match='scale'):
        paged_attention(*_make([20], 4, 2, 64, 16, 12, 'cuda'), scale)


@pytest.mark.gpu
def test_refusals():
    q, k, v, table, lengths = _make([20, 30], 4, 2, 64, 16, 12, 'cuda')
    ok = dict(q=q, k_cache=k, v_cache=v, page_table=table, lengths=lengths)
    odd = torch.zeros(k.numel() + 1, dtype=BF16, device='cuda')[1:].view(k.shape)
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(k_cache=k.float()), dict(v_cache=v[:1]), dict(v_cache=v.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(k_cache=odd, v_cache=odd), dict(k_cache=k[0], v_cache=v[0]), dict(page_table=table.long()), dict(page_table=table[:1]), dict(page_table=table.cpu()),
                dict(page_table=torch.stack([table, table], -1)[..., 0]), dict(lengths=lengths.long()), dict(lengths=lengths[:1]), dict(scale=0.0), dict(scale=float('inf')),
                dict(out=torch.zeros(2, 4, 64, device='cuda')), dict(out=torch.zeros(2, 4, 128, dtype=BF16, device='cuda')[..., :64])):
        with pytest.raises(RuntimeError):
            paged_attention(**{**ok, **bad})
    many = torch.zeros(4097, 4, 64, dtype=BF16, device='cuda')
    with pytest.raises(RuntimeError):
        paged_attention(many, k, v, torch.zeros(4097, 1, dtype=torch.int32, device='cuda'), torch.ones(4097, dtype=torch.int32, device='cuda'))
    none = paged_attention(q[:0], k, v, table[:0], lengths[:0])
    assert none.shape == (0, 4, 64)
