"""Attention of packed sequences and its gradients: the kernels and the PyTorch statements against the formulas in 64 bits."""
import pytest
import torch

from deepep_ascend_b200.ops import attention as A
from deepep_ascend_b200.ops.attention import attention, attention_backward

from test_plain_tensor_guard import _watchers

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
BF16, HALF, EPS = torch.bfloat16, 2.0**-8, 2.0**-23      # EPS: sums of the tensor cores may cut off where others round


def _cu(lengths, device='cpu'):
    return torch.tensor([0] + list(lengths)).cumsum(0).int().to(device)


def _make(tq, tk, H, Hk, D, seed=0, device='cpu'):
    g = torch.Generator().manual_seed(seed)
    r = lambda *shape: torch.randn(*shape, generator=g)      # noqa: E731
    k = r(tk, Hk, D)
    k[torch.rand(tk, generator=g) < 0.05] *= 3.0              # keys that many look at
    return [t.bfloat16().to(device) for t in (r(tq, H, D), k, r(tk, Hk, D), r(tq, H, D))] + [r(H, tq).to(device)]


def _check(q, k, v, d_o, d_lse, lq, lk, causal, scale=None, cu=True):
    """Forward and backward pass against 64 bits, sequence by sequence and head by head.

    A score is a sum of D products in 32 bits: off by E = scale (D + 8) EPS sum |q k|, and by roundings of its size in the exponent.  A probability is then off by the relative
    r = E + 4 EPS (|s| + |lse|) + 4 EPS, and by half a step of bf16 as an operand; sums of n terms by n EPS of their terms' magnitudes, and results by half a step."""
    D, H = q.shape[2], q.shape[1]
    c = D**-0.5 if scale is None else scale
    cq, ck = (_cu(lq, q.device), _cu(lk, q.device)) if cu else (None, None)
    o, lse = attention(q, k, v, cq, ck, causal, scale)
    assert o.dtype == BF16 and o.shape == q.shape and o.is_contiguous() and lse.shape == (H, q.shape[0]) and lse.dtype == torch.float32
    grads = attention_backward(d_o, q, k, v, o, lse, cq, ck, causal, scale, d_lse=d_lse)
    assert [t.shape for t in grads] == [q.shape, k.shape, v.shape] and all(t.dtype == BF16 and t.is_contiguous() for t in grads)
    Q, K, V, G, L = (t.double().cpu() for t in (q, k, v, d_o, d_lse))
    O, S = o.double().cpu(), lse.double().cpu()
    dq, dk, dv = (t.double().cpu() for t in grads)
    group = H // k.shape[1]
    near = lambda got, want, err: bool(((got - want).abs() <= err + HALF * (want.abs() + err) + 1e-30).all())      # noqa: E731
    a = b = 0
    for nq, nk in zip(lq, lk):
        i, j = slice(a, a + nq), slice(b, b + nk)
        a, b = a + nq, b + nk
        sum_k, err_k, sum_v, err_v = ([torch.zeros(nk, D, dtype=torch.float64) for _ in range(k.shape[1])] for _ in range(4))
        for h in range(H):
            kh = h // group
            x, y, z, g = Q[i, h], K[j, kh], V[j, kh], G[i, h]
            s = c * x @ y.t()
            sees = torch.ones(nq, nk, dtype=torch.bool)
            if causal:
                sees = torch.arange(nk) <= torch.arange(nq)[:, None] + nk - nq
            some = sees.any(-1)
            s = torch.where(sees, s, -torch.inf)
            want = torch.where(some, torch.logsumexp(s, -1) if nk else torch.zeros(nq, dtype=torch.float64), -torch.inf)
            E = c * (D + 8) * EPS * (x.abs() @ y.abs().t())
            most = torch.where(sees, E, 0.0).amax(-1) if nk else torch.zeros(nq, dtype=torch.float64)
            assert (torch.isinf(S[h, i]) == ~some).all()
            assert ((S[h, i] - want)[some].abs() <= (most + (nk + 16) * EPS + 4 * EPS * (1.0 + want.abs()))[some]).all()
            sized = torch.where(sees, s, 0.0).abs()
            p = torch.where(some[:, None], torch.exp(s - want[:, None]), 0.0) if nk else s
            rel = E + 4 * EPS * (1 + sized) + most[:, None] + (2 * nk + 32) * EPS
            assert near(O[i, h], p @ z, (p * (HALF + rel)) @ z.abs())
            # the gradient of what the forward pass returned: o and lse are inputs
            p = torch.where(some[:, None], torch.exp(s - S[h, i][:, None]), 0.0) if nk else s
            p = torch.where(sees, p, 0.0)
            rel = E + 4 * EPS * (2 + sized + torch.where(some, S[h, i], 0.0).abs()[:, None])
            dp, delta = g @ z.t(), (g * O[i, h]).sum(-1) - L[h, i]
            ds = p * (dp - delta[:, None])
            e_dp = (D + 8) * EPS * (g.abs() @ z.abs().t() + ((g * O[i, h]).abs().sum(-1) + L[h, i].abs())[:, None])
            e_ds = p * e_dp + ds.abs() * (rel + HALF) + (p * e_dp) * (rel + HALF)
            assert near(dq[i, h], c * ds @ y, c * (e_ds + (nk + 8) * EPS * ds.abs()) @ y.abs())
            n = group * nq + 8
            sum_k[kh] += c * ds.t() @ x
            err_k[kh] += c * (e_ds + n * EPS * ds.abs()).t() @ x.abs()
            sum_v[kh] += p.t() @ g
            err_v[kh] += (p * (rel + HALF + n * EPS)).t() @ g.abs()
        for kh in range(k.shape[1]):
            assert near(dk[j, kh], sum_k[kh], err_k[kh]) and near(dv[j, kh], sum_v[kh], err_v[kh])
    # rows of no sequence
    assert not O[a:].any() and (S[:, a:] == -torch.inf).all() and not dq[a:].any() and not dk[b:].any() and not dv[b:].any()
    return o, lse, grads


CASES = [
    ([1], [1], 1, 1, 128), ([1], [300], 4, 2, 64), ([64], [64], 2, 1, 8), ([127], [127], 3, 3, 80), ([128], [128], 2, 1, 128), ([129], [129], 2, 2, 72),
    ([256, 257], [256, 257], 2, 1, 64), ([5, 0, 130, 1, 63], [5, 0, 130, 1, 63], 6, 2, 96), ([0, 0], [0, 0], 2, 1, 64), ([3, 0, 40], [10, 7, 300], 4, 1, 128),
    ([385], [385], 14, 2, 128), ([70, 200], [20, 0], 2, 2, 64), ([300], [40], 2, 1, 128), ([65], [65], 16, 1, 24),
]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('lq,lk,H,Hk,D', CASES)
def test_against_the_formulas(lq, lk, H, Hk, D, causal, device):
    _check(*_make(sum(lq), sum(lk), H, Hk, D, sum(lk) + D, device), lq, lk, causal)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('group', [5, 11, 12, 17, 26, 48])
def test_groups_of_heads(group, causal, device):
    """Numbers of heads that do not divide 128, or have no divisor that a tile could take; sequences that end inside a tile."""
    lq, lk = [1, 30, 23, 131], [1, 30, 140, 131]
    _check(*_make(sum(lq), sum(lk), 2 * group, 2, 32, group, device), lq, lk, causal)


@pytest.mark.gpu
@pytest.mark.parametrize('lq,lk,H,Hk,D,causal', [([1100], [1100], 2, 1, 128, True), ([513, 700], [1900, 700], 4, 2, 64, True), ([640], [1333], 2, 2, 128, False)])
def test_longer_sequences(lq, lk, H, Hk, D, causal):
    _check(*_make(sum(lq), sum(lk), H, Hk, D, 3, 'cuda'), lq, lk, causal)


@pytest.mark.gpu
def test_long_sequences_of_many_heads():
    """Enough tiles of long sequences that a CTA takes two, of heads apart."""
    lq = [2000, 2110]
    _check(*_make(sum(lq), sum(lq), 28, 4, 72, 6, 'cuda'), lq, lq, True)


@pytest.mark.gpu
@pytest.mark.parametrize('H,Hk,D,causal', [(70, 10, 128, True), (70, 10, 64, False), (64, 64, 40, True), (72, 24, 104, True)])
def test_many_heads_are_what_few_are(H, Hk, D, causal):
    """Rows do not depend on one another: a launch with many tiles, and those of its heads by themselves, have the same bits."""
    lq, lk = [2049, 2311], [2049, 2400]
    q, k, v, d_o, d_lse = _make(sum(lq), sum(lk), H, Hk, D, 7, 'cuda')
    cq, ck = _cu(lq, 'cuda'), _cu(lk, 'cuda')
    o, lse = attention(q, k, v, cq, ck, causal)
    dq, dk, dv = attention_backward(d_o, q, k, v, o, lse, cq, ck, causal, d_lse=d_lse)
    group = H // Hk
    for h in range(0, Hk, max(1, Hk // 3)):
        a, b = slice(h * group, h * group + group), slice(h, h + 1)
        some = attention(q[:, a], k[:, b], v[:, b], cq, ck, causal)
        assert torch.equal(o[:, a], some[0]) and torch.equal(lse[a], some[1])
        grads = attention_backward(d_o[:, a], q[:, a], k[:, b], v[:, b], *some, cq, ck, causal, d_lse=d_lse[a].contiguous())
        assert torch.equal(dq[:, a], grads[0])
        # (sums over the heads may be in another order: within a rounding of the size that they have on the whole)
        for x, y in ((dk[:, b], grads[1]), (dv[:, b], grads[2])):
            assert float((x.float() - y.float()).norm()) <= 2 * HALF * float(y.float().norm())


@pytest.mark.parametrize('device', DEVICES)
def test_one_sequence_and_a_scale(device):
    q, k, v, d_o, d_lse = _make(150, 190, 4, 2, 64, 1, device)
    o, lse, grads = _check(q, k, v, d_o, d_lse, [150], [190], True, scale=0.31, cu=False)
    with_cu = attention(q, k, v, _cu([150], device), _cu([190], device), scale=0.31)
    assert torch.equal(o, with_cu[0]) and torch.equal(lse, with_cu[1])
    # scores far apart: references that move, probabilities that vanish
    _check(*(t * 8 if t is k else t for t in (q, k, v, d_o, d_lse)), [150], [190], True, scale=1.0, cu=False)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('D', [64, 128])
def test_what_lies_behind_the_sequences_is_not_looked_at(D, device):
    """Padding that holds no numbers; its rows get zeros, and no gradient."""
    lq, lk = [70, 3, 131], [75, 3, 200]
    q, k, v, d_o, d_lse = _make(300, 400, 4, 2, D, 2, device)
    want = attention(q, k, v, _cu(lq, device), _cu(lk, device))
    for t, n in ((q, 204), (k, 278), (v, 278), (d_o, 204)):
        t[n:] = float('nan')
    d_lse[:, 204:] = float('inf')
    o, lse, _ = _check(q, k, v, d_o, d_lse, lq, lk, True)
    assert torch.equal(o[:204], want[0][:204]) and torch.equal(lse[:, :204], want[1][:, :204])


@pytest.mark.gpu
@pytest.mark.parametrize('H,Hk,D', [(14, 2, 128), (6, 6, 64), (22, 2, 32)])
def test_sequences_do_not_reach_one_another(H, Hk, D, device='cuda'):
    """One that holds no numbers anywhere, between others that share its tiles: theirs, results and gradients, keep their bits."""
    lq, lk = [100, 50, 1, 290], [100, 61, 1, 290]
    q, k, v, d_o, d_lse = _make(441, 452, H, Hk, D, 15, device)
    cq, ck = _cu(lq, device), _cu(lk, device)
    kept = attention(q, k, v, cq, ck)
    want = attention_backward(d_o, q, k, v, *kept, cq, ck, d_lse=d_lse)
    bad = [t.clone() for t in (q, k, v, d_o)]
    for t, a, n in zip(bad, (100, 100, 100, 100), (50, 61, 61, 50)):
        t[a:a + n] = float('nan')
    o, lse = attention(*bad[:3], cq, ck)
    grads = attention_backward(bad[3], *bad[:3], o, lse, cq, ck, d_lse=d_lse)
    rows, keys = (torch.cat([torch.arange(100), torch.arange(100 + n, 391 + n)]).to(device) for n in (50, 61))
    assert torch.equal(o[rows], kept[0][rows]) and torch.equal(lse[:, rows], kept[1][:, rows])
    assert all(torch.equal(a[i], b[i]) for a, b, i in zip(grads, want, (rows, keys, keys)))
    assert o[100:150].isnan().all()


@pytest.mark.parametrize('H,n,device', [(2, 300, 'cpu'), pytest.param(2, 300, 'cuda', marks=pytest.mark.gpu), pytest.param(56, 2200, 'cuda', marks=pytest.mark.gpu)])
def test_a_key_that_is_no_number(H, n, device):
    """Wherever it stands, who sees it gets no numbers, in both results; who does not keeps what there was."""
    q, k, v, _, _ = _make(n, n, H, 1, 64, 16, device)
    o, lse = attention(q, k, v)
    for at in [*range(16, 24), 130, 135, 255, n - 1]:
        for bad in (float('nan'), float('inf')):
            x = k.clone()
            x[at] = bad if bad != bad else (x[at].sign() * bad)      # (products of both signs: their sum is no number)
            got = attention(q, x, v)
            assert got[0][at:].isnan().all() and got[1][:, at:].isnan().all(), (at, bad)
            assert torch.equal(got[0][:at], o[:at]) and torch.equal(got[1][:, :at], lse[:, :at])


@pytest.mark.gpu
@pytest.mark.parametrize('H', [1, 512])
def test_powers(H):
    """2^x of the keys whose powers go by a polynomial, seen in lse: 128 keys of score 0, which the reference stays at, and of the 128 behind them those 32 with score x, the others far below.

    x is exact in bf16 halves, its product with scale log2 e off by 2^-23 of it, the polynomial by 2.9e-6; the sum of 160 terms, its logarithm and their product by 2^-24 of their size each."""
    x = torch.cat([torch.arange(-160, -20) + 0.3125, torch.arange(-20 * 128, 8 * 128 - 1) / 128]).double()
    tokens = x.numel()
    high = x.bfloat16().double()
    low = (x - high).bfloat16().double()
    assert (high + low == x).all()
    q, k = torch.zeros(tokens, H, 8), torch.zeros(256, 1, 8)
    q[:, :, 0], q[:, :, 1], q[:, :, 2] = high[:, None], low[:, None], 1.0
    by_polynomial = torch.arange(128) % 8 >= 6
    k[128:][by_polynomial, :, :2] = 1.0
    k[128:][~by_polynomial, :, 2] = -1000.0
    scale = float(torch.tensor(2.0).log())
    lse = attention(q.bfloat16().cuda(), k.bfloat16().cuda(), torch.ones(256, 1, 8, dtype=BF16, device='cuda'), causal=False, scale=scale)[1].double().cpu()
    part = 32 * 2.0**x
    want = torch.log(128 + part)
    err = part / (128 + part) * (2.9e-6 + x.abs() * 2.0**-23) + 8 * 2.0**-24 * (1 + want) + 160 * 2.0**-24
    assert ((lse - want).abs() <= err).all(), float(((lse - want).abs() - err).max())


@pytest.mark.gpu
@pytest.mark.parametrize('cu_q,cu_k', [([9, 40, 100], [30, 80, 120]), ([0, 400, 100], [0, 50, 900]), ([0, 50, 30], [0, 90, 20]), ([-5, 30, 100], [0, 50, 120])])
def test_bounds_that_are_out_of_order_stay_inside(cu_q, cu_k):
    """Gaps in front give zeros; whatever the bounds are, nothing outside the tensors is read or written."""
    q, k, v, d_o, d_lse = _make(100, 120, 2, 1, 64, 4, 'cuda')
    cq, ck = (torch.tensor(c, dtype=torch.int32, device='cuda') for c in (cu_q, cu_k))
    o, lse = attention(q, k, v, cq, ck)
    grads = attention_backward(d_o, q, k, v, o, lse, cq, ck)
    torch.cuda.synchronize()
    if cu_q[0] == 9:
        assert not o[:9].any() and (lse[:, :9] == -torch.inf).all() and not grads[0][:9].any() and not grads[1][:30].any() and not grads[2][:30].any()
        want = attention(q[9:].contiguous(), k[30:].contiguous(), v[30:].contiguous(), cq - 9, ck - 30)
        assert torch.equal(o[9:], want[0]) and torch.equal(lse[:, 9:], want[1])


@pytest.mark.gpu
def test_strides_and_alignment():
    """Views of one projection, heads in front of tokens, rows that start anywhere, a head that all share, channels apart: the same bits as contiguous tensors."""
    lq, H, Hk, D = [120, 77], 4, 2, 64
    q, k, v, d_o, d_lse = _make(197, 197, H, Hk, D, 5, 'cuda')
    cu = _cu(lq, 'cuda')
    want = attention(q, k, v, cu)
    grads = attention_backward(d_o, q, k, v, *want, cu, d_lse=d_lse)
    fused = torch.cat([q, k, v], 1)
    in_front = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    odd = [torch.zeros(t.numel() + 3, dtype=BF16, device='cuda')[3:].view(t.shape).copy_(t) for t in (q, k, v)]
    apart = [torch.stack([t, t], -1)[..., 0] for t in (q, k, v)]
    for a, b, c in ((fused[:, :H], fused[:, H:H + Hk], fused[:, H + Hk:]), in_front, odd, apart):
        got = attention(a, b, c, cu)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        d = d_o.transpose(0, 1).contiguous().transpose(0, 1)
        again = attention_backward(d, a, b, c, *want, cu, d_lse=d_lse)
        assert all(torch.equal(x, y) for x, y in zip(again, grads))
    shared = k[:, :1].expand(-1, Hk, -1)
    assert torch.equal(attention(q, shared, shared, cu)[0], attention(q, shared.contiguous(), shared.contiguous(), cu)[0])


@pytest.mark.gpu
def test_the_same_bits_every_time():
    q, k, v, d_o, d_lse = _make(900, 900, 8, 1, 128, 6, 'cuda')
    cu = _cu([300, 600], 'cuda')
    first = attention(q, k, v, cu)
    grads = attention_backward(d_o, q, k, v, *first, cu)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(attention(q, k, v, cu), first))
        assert all(torch.equal(a, b) for a, b in zip(attention_backward(d_o, q, k, v, *first, cu), grads))


def test_the_function_against_differences():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h, 4, dtype=torch.float64, generator=g).requires_grad_(True) for n, h in ((7, 4), (9, 2), (9, 2)))
    cq, ck = _cu([2, 0, 4]), _cu([3, 1, 4])
    seen = torch.isfinite(attention(q, k, v, cq, ck)[1])

    def f(q, k, v):
        o, lse = A._Attention.apply(q, k, v, cq, ck, True, 0.7, None)
        return o, torch.where(seen, lse, 0.0)
    assert torch.autograd.gradcheck(f, (q, k, v)) and torch.autograd.gradcheck(lambda *a: f(*a)[0], (q, k, v)) and torch.autograd.gradcheck(lambda *a: f(*a)[1], (q, k, v))


@pytest.mark.gpu
def test_gradients_through_the_call():
    lq = [90, 41]
    q, k, v, d_o, d_lse = _make(131, 131, 4, 2, 64, 7, 'cuda')
    cu = _cu(lq, 'cuda')
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o, lse = attention(*leaves, cu)
    want = attention(q, k, v, cu)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    grads = attention_backward(d_o, q, k, v, *want, cu, d_lse=d_lse)
    got = torch.autograd.grad([o, lse], leaves, [d_o, d_lse], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, grads))
    only = torch.autograd.grad(lse, leaves, d_lse, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(only, attention_backward(torch.zeros_like(d_o), q, k, v, *want, cu, d_lse=d_lse)))
    # one head that all queries share, given as a view: its gradient is the sum
    shared = k[:, :1].clone().requires_grad_(True)
    o = attention(q, shared.expand(-1, 2, -1), v, cu)[0]
    got, = torch.autograd.grad(o, shared, d_o)
    parts = attention_backward(d_o, q, shared.detach().expand(-1, 2, -1), v, o.detach(), attention(q, shared.detach().expand(-1, 2, -1), v, cu)[1], cu)[1]
    torch.testing.assert_close(got.float(), parts.float().sum(1, keepdim=True), rtol=2 * HALF, atol=2 * HALF)


@pytest.mark.gpu
def test_a_gradient_of_the_gradient():
    """Given away to the statement, which carries it: (its 32 bits against its 64 bits, sums of 20 terms)"""
    q, k, v, d_o, _ = (t.float() for t in _make(20, 20, 2, 1, 8, 8, 'cuda'))
    def second(q, k, v, o, lse, d_o):
        d = attention_backward(d_o, q, k, v, o, lse)
        return torch.autograd.grad(sum((t**2).sum() for t in d), (q, k, v))
    o, lse = (t.detach() for t in A.attention_ref(q, k, v))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = second(*leaves, o, lse, d_o)
    want = second(*(t.detach().double().requires_grad_(True) for t in leaves), o.double(), lse.double(), d_o.double())
    for a, b in zip(got, want):
        torch.testing.assert_close(a.double(), b, rtol=1e-4, atol=1e-4 * b.abs().max().item())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('tracer', ['jit.trace', 'make_fx', 'functionalize', 'vmap', 'forward mode', 'dispatch mode'])
def test_it_is_seen(tracer, device):
    q, k, v, d_o, _ = _make(12, 12, 2, 1, 16, 9, device)
    cu = _cu([5, 7], device)
    kept = attention(q, k, v, cu)
    for f in (lambda x: attention(x, k, v, cu)[0], lambda x: attention_backward(d_o, x, k, v, *kept, cu)[0]):
        out = _watchers()[tracer](f, q)
        if callable(out):
            # (bf16 results of two ways to the same formula)
            assert all(torch.allclose(out(x).float(), f(x).float(), rtol=8 * HALF, atol=8 * HALF) for x in (q, q.flip(0)))
        else:
            out = torch.autograd.forward_ad.unpack_dual(out)[0] if tracer == 'forward mode' else out
            assert torch.allclose(out.reshape(q.shape).float(), f(q).float(), rtol=8 * HALF, atol=8 * HALF)


@pytest.mark.gpu
def test_in_a_graph_and_on_another_stream():
    """Two graphs of one size that are replayed in turn, with inputs and bounds of their own, and a call on a side stream."""
    made = [_make(200, 200, 4, 2, 64, seed, 'cuda') for seed in (10, 11)]
    bounds = [_cu([200], 'cuda'), _cu([40, 160], 'cuda')]
    bounds[0] = torch.tensor([0, 200, 200], dtype=torch.int32, device='cuda')
    want = []
    for (q, k, v, d_o, d_lse), cu in zip(made, bounds):
        o, lse = attention(q, k, v, cu)
        want.append((o, lse, *attention_backward(d_o, q, k, v, o, lse, cu)))
    graphs = []
    for (q, k, v, d_o, _), cu in zip(made, bounds):
        x = [t.clone() for t in (q, k, v, d_o)]
        c = cu.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, lse = attention(*x[:3], c)
            out = (o, lse, *attention_backward(x[3], *x[:3], o, lse, c))
        graphs.append((graph, x, c, out))
    for order in ((0, 1), (1, 0)):                   # (each with its own data, then with the other's)
        for g, data in zip(graphs, order):
            for t, new in zip(g[1], made[data]):
                t.copy_(new)
            g[2].copy_(bounds[data])
        for _ in range(3):
            for g in graphs:
                g[0].replay()
        torch.cuda.synchronize()
        for g, data in zip(graphs, order):
            assert all(torch.equal(a, b) for a, b in zip(g[3], want[data]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o, lse = attention(*made[1][:3], bounds[1])
    side.synchronize()
    assert torch.equal(o, want[1][0]) and torch.equal(lse, want[1][1])


@pytest.mark.gpu
def test_in_threads_that_have_done_nothing_yet():
    import threading
    q, k, v, d_o, _ = _make(200, 200, 4, 2, 64, 12, 'cuda')
    want = attention(q, k, v)
    grads = attention_backward(d_o, q, k, v, *want)
    got = {}
    for name, f in (('forward', lambda: attention(q, k, v)), ('backward', lambda: attention_backward(d_o, q, k, v, *want))):
        thread = threading.Thread(target=lambda: got.update({name: f()}))
        thread.start()
        thread.join()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*got['forward'], *got['backward']), (*want, *grads)))


@pytest.mark.gpu
@pytest.mark.parametrize('D,H,Hk', [(128, 12, 4), (64, 16, 16)])
def test_more_blocks_than_processors(D, H, Hk):
    """Every CTA takes many blocks of unlike length, empty sequences among them: against the same sequences one by one."""
    lengths = [700, 0, 33, 128, 1500, 129, 1, 256, 640] * 3
    q, k, v, d_o, _ = _make(sum(lengths), sum(lengths), H, Hk, D, 13, 'cuda')
    cu = _cu(lengths, 'cuda')
    o, lse = attention(q, k, v, cu)
    grads = attention_backward(d_o, q, k, v, o, lse, cu)
    a = 0
    for n in lengths[:9]:
        i = slice(a, a + n)
        a += n
        if n == 0:
            continue
        one = attention(q[i], k[i], v[i])
        assert torch.equal(one[0], o[i]) and torch.equal(one[1], lse[:, i])
        # (keys' gradients may be added in other parts: half a step of bf16, and of what the products round)
        for x, y in zip(attention_backward(d_o[i], q[i], k[i], v[i], *one), grads):
            assert (x.float() - y[i].float()).abs().max() <= 4 * HALF * y[i].float().abs().max()


@pytest.mark.gpu
def test_nothing_to_do():
    q, k, v, d_o, d_lse = _make(10, 12, 2, 1, 64, 0, 'cuda')
    o, lse = attention(q[:0], k, v)
    assert o.shape == (0, 2, 64) and lse.shape == (2, 0)
    assert all(not t.any() for t in attention_backward(d_o[:0], q[:0], k, v, o, lse))
    o, lse = attention(q, k[:0], v[:0])
    assert not o.any() and (lse == -torch.inf).all()
    assert all(not t.any() for t in attention_backward(d_o, q, k[:0], v[:0], o, lse))
    none = torch.zeros(1, dtype=torch.int32, device='cuda')
    o, lse = attention(q, k, v, none)
    assert not o.any() and (lse == -torch.inf).all()
    assert all(not t.any() for t in attention_backward(d_o, q, k, v, o, lse, none))


@pytest.mark.gpu
@pytest.mark.parametrize('scale', [1e-50, 1e-39, 3e38, 1e300, -1.0, float('nan')])
def test_scales_that_32_bits_do_not_hold(scale):
    with pytest.raises(RuntimeError, match='scale'):
        attention(*_make(10, 10, 2, 1, 64, 0, 'cuda')[:3], scale=scale)


@pytest.mark.gpu
def test_refusals():
    q, k, v, d_o, d_lse = _make(10, 10, 4, 2, 64, 0, 'cuda')
    cu = _cu([10], 'cuda')
    o, lse = attention(q, k, v, cu)
    for bad in (dict(q=q.float()), dict(k=k[:, :, :32]), dict(v=v[:5]), dict(q=q[:, :3]), dict(k=k.cpu()), dict(q=q[..., :4], k=k[..., :4], v=v[..., :4]), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float('nan')), dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu.cpu()), dict(cu_seqlens=cu[None]), dict(cu_seqlens_k=cu[:1]), dict(q=q[0])):
        with pytest.raises((RuntimeError, ValueError)):
            attention(**{**dict(q=q, k=k, v=v, cu_seqlens=cu), **bad})
    with pytest.raises(ValueError):
        attention(q, k, v, cu_seqlens_k=cu)
    wide = torch.zeros(4, 1, 136, dtype=BF16, device='cuda')
    with pytest.raises(RuntimeError):
        attention(wide, wide, wide)
    for bad in (dict(d_o=d_o[:5]), dict(d_o=d_o.float()), dict(o=o[:, :2]), dict(lse=lse.t()), dict(lse=lse.double()), dict(d_lse=d_lse[:1])):
        with pytest.raises(RuntimeError):
            attention_backward(**{**dict(d_o=d_o, q=q, k=k, v=v, o=o, lse=lse, cu_seqlens=cu), **bad})


_SHORT_LIMIT = """
import torch
from deepep_ascend_b200 import ElasticBuffer, _native
from deepep_ascend_b200.ops.attention import attention, attention_backward
torch.manual_seed(0)
make = lambda n: [torch.randn(n, 1, 64, device='cuda').bfloat16() for _ in range(4)]
q, k, v, g = make(1000)
want = attention(q, k, v)
grads = attention_backward(g, q, k, v, *want)
buf = ElasticBuffer(None, num_max_tokens_per_rank=16, hidden=256, num_topk=2)
assert torch.equal(attention(q, k, v, buffer=buf)[0], want[0])
assert all(torch.equal(a, b) for a, b in zip(attention_backward(g, q, k, v, *want, buffer=buf), grads))
torch.cuda.synchronize()
buf.check_status()
x, y, z, d = make(100000)
if BACKWARD:
    o, lse = attention(x, y, z, causal=False)
    torch.cuda.synchronize()
buf.core.set_gpu_timeout(3e-4)
if BACKWARD:
    attention_backward(d, x, y, z, o, lse, causal=False, buffer=buf)
else:
    attention(x, y, z, causal=False, buffer=buf)
torch.cuda.synchronize()
code, phase, peer, expected, observed, rank = buf.core.read_status()
assert (code, phase, rank) == (1, 14, 0) and expected in (1, 7), (code, phase, expected, rank)
assert _native.load().gemm_error(0) == expected
try:
    buf.check_status()
except RuntimeError as e:
    assert 'timed out' in str(e)
else:
    raise AssertionError('the wait was not reported')
# shared and tensor memory have been given back, and what follows is right
for _ in range(3):
    o, lse = attention(q, k, v)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    assert all(torch.equal(a, b) for a, b in zip(attention_backward(g, q, k, v, *want), grads))
print('reported')
"""


@pytest.mark.gpu
@pytest.mark.parametrize('backward', [False, True])
def test_a_wait_that_runs_out_is_reported(backward):
    """A block of 128 rows against 100000 takes a millisecond, while who waits for its end has 0.3.  (In a process of its own: the device's error flag stays up.)"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, '-c', _SHORT_LIMIT.replace('BACKWARD', str(backward))], cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True,
                         timeout=120)
    assert run.returncode == 0 and run.stdout.strip().endswith('reported'), run.stderr[-2000:]
