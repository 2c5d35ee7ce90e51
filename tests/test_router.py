"""Routing: the kernels and the PyTorch statements against the definition in 64 bits, token by token."""
import math

import numpy as np
import pytest
import torch

from deepep_ascend_b200.ops import router

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def _definition(logits, K, score, bias, G, TG, top, renormalize, scale, mask):
    """-> (idx, weights, clear): numpy in 64 bits.  ``clear``: tokens whose choice 32 bits cannot change: what decides is
    equal, or differs by more than its rounding."""
    T, E = logits.shape
    idx, weights, clear = -np.ones((T, K), np.int64), np.zeros((T, K)), np.ones(T, bool)
    for t in range(T):
        l = logits[t]
        with np.errstate(all='ignore'):
            p = 1 / (1 + np.exp(-l)) if score == 'sigmoid' else np.exp(l - np.max(l)) / np.sum(np.exp(l - np.max(l)))
        choice = p + (0 if bias is None else bias)
        choice[np.isnan(choice) | (l == -np.inf)] = -np.inf
        # 32 bits are off by at most 40 x 2^-24 of a score, and by 2^-24 of what is added to it
        width = 0 if bias is None else np.max(np.abs(bias[np.isfinite(bias)]), initial=0)
        def decided(values, n):
            """Whether the first n of falling values and their order are the same in 32 bits (equal ones by index, wherever they stand)."""
            for i, (a, b) in enumerate(zip(values, values[1:])):
                if b == -np.inf or (i >= n and a != values[n - 1]):
                    break
                if a != b and a - b <= 1e-5 * (abs(a) + width) + 1e-37:
                    return False
            return True
        if G > 1:
            total = np.full(G, -np.inf)
            for g in range(G):
                best = sorted((c for c in choice[g * (E // G):(g + 1) * (E // G)] if c > -np.inf), reverse=True)[:top]
                total[g] = sum(best) if best else -np.inf
            order = sorted(range(G), key=lambda g: (-total[g], g))
            clear[t] &= TG == G or decided(total[order], TG)
            for g in order[TG:]:
                choice[g * (E // G):(g + 1) * (E // G)] = -np.inf
        order = sorted((e for e in range(E) if choice[e] > -np.inf), key=lambda e: (-choice[e], e))
        clear[t] &= decided(choice[order], K)
        order = order[:K]
        clear[t] &= not order or p[order].sum() > 1e-36              # scores that vanish in 32 bits are equal there, and their weights zero
        if mask is not None and not mask[t]:
            order = []
        if order:
            with np.errstate(all='ignore'):
                w = p[order]
                if renormalize:
                    if score == 'softmax':
                        w = np.exp(l[order] - np.max(l[order]))
                    w = w / w.sum() if w.sum() > 0 else 0 * w
            idx[t, :len(order)], weights[t, :len(order)] = order, scale * w
    return idx, weights, clear


def _logits(T, E, dtype, seed, device):
    """Logits on a grid of 1/8, so that many experts tie and the others are well apart; rows with every kind of special value."""
    g = torch.Generator().manual_seed(seed)
    l = torch.round(torch.randn(T, E, generator=g) * 16) / 8
    lowest = torch.finfo(dtype).min
    if T >= 12:
        l[1] = -math.inf                                        # nobody can be chosen
        l[2] = -math.inf
        l[2, E // 2] = 0.5                                      # one expert is left
        l[3] = 0.25                                             # all are as good
        l[4, ::2] = -math.inf
        l[5, : E // 2] = lowest                                 # masked by the type's lowest value
        l[6] = lowest
        l[7, E // 3] = math.nan
        l[8, 0] = math.inf
        l[9] *= 100                                             # saturated scores
        l[10] = -200.0
    return l.to(dtype).to(device)


SHAPES = [
    # E, K, groups, topk_groups, group_top
    (1, 1, 1, 1, 1), (2, 2, 1, 1, 1), (5, 3, 1, 1, 2), (8, 6, 4, 3, 2), (31, 4, 1, 1, 1), (32, 8, 8, 4, 2), (33, 16, 3, 2, 1), (64, 6, 1, 1, 1),
    (100, 7, 10, 3, 2), (160, 6, 8, 3, 1), (256, 8, 8, 4, 2), (256, 8, 1, 1, 1), (320, 9, 32, 5, 2), (509, 16, 1, 1, 1), (512, 16, 2, 1, 2),
    (768, 12, 24, 7, 2), (1024, 16, 32, 32, 2), (1000, 1, 8, 1, 1),
]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('score', ['sigmoid', 'softmax'])
@pytest.mark.parametrize('E,K,G,TG,top', SHAPES)
def test_choice_and_weights(E, K, G, TG, top, score, device):
    for case, (dtype, renormalize, with_bias, masked) in enumerate([(torch.float32, True, True, False), (torch.bfloat16, False, False, True),
                                                                    (torch.float32, False, True, True), (torch.bfloat16, True, False, False)]):
        T = (1, 13, 40, 64)[case]
        logits = _logits(T, E, dtype, 7 * E + case, device)
        bias = torch.round(torch.randn(E, generator=torch.Generator().manual_seed(E)) * 64).div(512) if with_bias else None
        if with_bias and E > 2:
            bias[E - 1] = -math.inf                             # switched off for everybody
        mask = torch.arange(T) % 5 != 0 if masked else None
        scale = 2.5
        idx, w, count = router.route(logits, K, score, None if bias is None else bias.to(device), G, TG, top, renormalize, scale,
                                     None if mask is None else mask.to(device))
        assert idx.dtype == router.topk_idx_t and w.dtype == torch.float32 and count.dtype == torch.int32
        idx, w = idx.cpu().numpy(), w.cpu().numpy()
        assert np.array_equal(count.cpu().numpy(), np.bincount(idx[idx >= 0], minlength=E))
        want_idx, want_w, clear = _definition(logits.double().cpu().numpy(), K, score, None if bias is None else bias.double().numpy(), G, TG, top,
                                              renormalize, scale, None if mask is None else mask.numpy())
        assert clear.mean() > 0.5 or T == 1
        assert np.array_equal(idx[clear], want_idx[clear])
        assert np.all(w[idx < 0] == 0)
        # exp of an argument of up to 40 is off by the argument's rounding (40 x 2^-24), the few operations after it by 2^-24 each
        ok = clear & np.isfinite(want_w).all(1)
        np.testing.assert_allclose(w[ok], want_w[ok], rtol=80 * 2.0**-24, atol=1e-37)


@pytest.mark.parametrize('device', DEVICES)
def test_special_rows(device):
    """What is chosen where the scores are no ordinary numbers, in words."""
    l = _logits(16, 32, torch.float32, 3, device)
    for score in ('sigmoid', 'softmax'):
        idx, w, _ = router.route(l, 4, score, renormalize=False)
        idx, w = idx.cpu(), w.cpu()
        assert (idx[1] == -1).all() and (w[1] == 0).all()
        assert idx[2].tolist() == [16, -1, -1, -1]
        assert idx[3].tolist() == [0, 1, 2, 3]
        assert all(e % 2 for e in idx[4].tolist())
        assert all(e >= 16 for e in idx[5].tolist())
        assert idx[6].tolist() == [0, 1, 2, 3]
        assert 10 not in idx[7].tolist()
    sig, soft = router.route(l, 4, 'sigmoid', renormalize=False)[0].cpu(), router.route(l, 4, 'softmax', renormalize=False)[0].cpu()
    assert sig[8, 0] == 0 and (sig[7] >= 0).all()
    assert (soft[7] == -1).all() and (soft[8] == -1).all()          # a sum with a NaN in it leaves no score
    # a group of which one expert is left stays ahead of groups that nobody can be chosen from
    l = torch.full((1, 16), -math.inf, device=device)
    l[0, 13] = 1.0
    assert router.route(l, 2, num_groups=4, num_topk_groups=1, group_top=2)[0].tolist() == [[13, -1]]
    # weights of chosen experts whose softmax vanishes in 32 bits still add up to one
    l = torch.tensor([[200.0, 0.0, math.log(3.0)]], device=device)
    _, w, _ = router.route(l, 2, 'softmax', bias=torch.tensor([-math.inf, 0.0, 0.0], device=device))
    np.testing.assert_allclose(sorted(w.cpu().numpy()[0]), [0.25, 0.75], rtol=8 * 2.0**-24)


@pytest.mark.gpu
@pytest.mark.parametrize('score', ['sigmoid', 'softmax'])
@pytest.mark.parametrize('E,K,G,TG,top', [s for s in SHAPES if s[0] in (5, 64, 160, 256, 512, 768)])
def test_kernel_chooses_what_32_bit_scores_say(E, K, G, TG, top, score):
    """Random logits, where neighbours in 32 bits are common: bit for bit the choice of the PyTorch statement."""
    T = 4000
    for dtype in (torch.float32, torch.bfloat16):
        logits = (torch.randn(T, E, generator=torch.Generator().manual_seed(E)) * 2).to(dtype).cuda()
        bias = torch.randn(E, generator=torch.Generator().manual_seed(1)).mul(0.05).cuda()
        for b in (None, bias):
            got = router.route(logits, K, score, b, G, TG, top)
            want = router.route_ref(logits, K, score, b, G, TG, top)
            assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


@pytest.mark.gpu
@pytest.mark.parametrize('score', ['sigmoid', 'softmax'])
@pytest.mark.parametrize('E,K', [(8, 8), (40, 16), (256, 8), (1000, 16)])
def test_scores_of_every_size(E, K, score):
    """Bit by bit what 32-bit scores say over the whole range: logits around and beyond what the kernel's short reciprocal and quotient take, groups of eight
    neighbours of ordinary ones, of small ones and mixed, with and without a bias of ordinary numbers."""
    g = torch.Generator().manual_seed(E)
    l = torch.randn(4096, E, generator=g) * torch.logspace(-3, 2.2, 4096)[:, None]
    l[::3] -= torch.randint(0, 140, (len(l[::3]), 1), generator=g)
    l[1::3, : E // 2] -= 75 + 10 * torch.rand(len(l[1::3]), 1, generator=g)
    l = l.cuda()
    for bias in (None, (torch.randn(E, generator=g) * 0.1).cuda(), torch.full((E, ), -0.5, device='cuda')):
        want = router.route_ref(l, K, score, bias, renormalize=False)
        got = router.route(l, K, score, bias, renormalize=False)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('score,renormalize', [('sigmoid', True), ('sigmoid', False), ('softmax', True), ('softmax', False)])
@pytest.mark.parametrize('E,K', [(1, 1), (7, 3), (32, 8), (65, 6), (160, 6), (256, 8), (500, 16), (1024, 9)])
def test_gradient(E, K, score, renormalize, device):
    T, scale = 37, 2.5
    g = torch.Generator().manual_seed(E + K)
    for dtype in (torch.float32, torch.bfloat16):
        logits = (torch.randn(T, E, generator=g) * 2).to(dtype)
        if E >= 32:
            logits[2, : E // 2] = -math.inf
            logits[3] *= 40
        mask = torch.arange(T) % 7 != 1
        idx, w, _ = router.route_ref(logits, K, score, renormalize=renormalize, scale=scale, token_mask=mask)
        idx[5, K // 2:] = -1                                    # selections that were dropped later
        d = torch.randn(T, K, generator=g)
        got = router.route_backward(d.to(device), logits.to(device), idx.to(device), score, renormalize, scale)
        assert got.dtype == dtype
        # the definition: the chain rule through the scores of the whole row, in 64 bits
        l = logits.double().requires_grad_(True)
        p = torch.sigmoid(l) if score == 'sigmoid' else torch.softmax(l, -1)
        ps = p.gather(1, idx.clamp_min(0)) * (idx >= 0)
        if renormalize:
            ps = ps / ps.sum(-1, keepdim=True).clamp_min(1e-300)
        want, = torch.autograd.grad((scale * ps * d.double()).sum(), l)
        want = torch.where((idx >= 0).any(-1, keepdim=True), torch.nan_to_num(want, nan=0.0), 0.0)
        # terms no larger than scale x |d|, each off by the rounding of exp's argument (up to 300 x 2^-24 in the row times 40) or of a few operations,
        # with at most K of them added up; bf16 results are rounded once more
        size = scale * d.abs().max(-1, keepdim=True).values.double()
        rounding = torch.full((T, 1), 64.0, dtype=torch.float64)
        rounding[3] += 400
        bound = (rounding + 2 * K) * 2.0**-24 * size + (2.0**-8 * want.abs() if dtype == torch.bfloat16 else 0)
        assert ((got.cpu().double() - want).abs() <= bound).all()
        assert (got.cpu()[1::7][: (T - 1) // 7] == 0).all()


def test_gradient_against_differences():
    """64-bit central differences of the statement's weights, the choice held."""
    T, E, K, h = 3, 12, 4, 1e-6
    g = torch.Generator().manual_seed(0)
    logits, d = torch.randn(T, E, generator=g, dtype=torch.float64), torch.randn(T, K, generator=g, dtype=torch.float64)
    for score in ('sigmoid', 'softmax'):
        for renormalize in (True, False):
            idx = router.route_ref(logits, K, score, renormalize=renormalize, scale=1.5)[0].long()

            def loss(l):
                w = router._gathered(l, idx, score, renormalize)
                return (1.5 * (w / w.sum(-1, keepdim=True) if renormalize else w) * d).sum()
            got = router.route_backward_ref(d, logits, idx, score, renormalize, 1.5)
            for t in range(T):
                for e in range(E):
                    step = torch.zeros_like(logits)
                    step[t, e] = h
                    assert abs((loss(logits + step) - loss(logits - step)).item() / (2 * h) - got[t, e].item()) < 1e-8


@pytest.mark.gpu
def test_pitched_logits_streams_and_empty_batches():
    wide = torch.randn(300, 300, device='cuda')
    view = wide[:, 17:17 + 256]
    assert not view.is_contiguous()
    want = router.route(view.contiguous(), 8, num_groups=8, num_topk_groups=4)
    got = router.route(view, 8, num_groups=8, num_topk_groups=4)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    d = torch.randn(300, 8, device='cuda')
    for score in ('sigmoid', 'softmax'):
        assert torch.equal(router.route_backward(d, view, got[0], score, False), router.route_backward(d, view.contiguous(), got[0], score, False))
    # another stream than the current one's tensors were made on; the same bits on every run
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = router.route(view, 8, num_groups=8, num_topk_groups=4)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    # int32 ids serve the gradient as well
    assert torch.equal(router.route_backward(d, view, got[0].int()), router.route_backward(d, view, got[0]))
    idx, w, count = router.route(wide[:0], 4)
    assert idx.shape == w.shape == (0, 4) and count.tolist() == [0] * 300
    assert router.route_backward(d[:0], wide[:0, :8], idx.new_zeros(0, 8)).shape == (0, 8)


@pytest.mark.gpu
def test_replay_from_a_graph():
    logits = torch.randn(64, 256, device='cuda')
    router.route(logits, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = router.route(logits, 8)
    for seed in range(3):
        logits.copy_(torch.randn(64, 256, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, router.route_ref(logits, 8)) if a.dtype != torch.float32)


@pytest.mark.gpu
def test_refusals():
    l = torch.randn(4, 64, device='cuda')
    bad = [dict(num_topk=0), dict(num_topk=17), dict(num_topk=9, num_groups=8, num_topk_groups=1), dict(num_topk=2, num_groups=7), dict(num_topk=2, num_groups=64),
           dict(num_topk=2, num_groups=8, num_topk_groups=9), dict(num_topk=2, num_groups=8, num_topk_groups=0), dict(num_topk=2, num_groups=8, group_top=3),
           dict(num_topk=2, bias=torch.zeros(63, device='cuda')), dict(num_topk=2, bias=torch.zeros(64)), dict(num_topk=2, bias=torch.zeros(64, device='cuda').bfloat16()),
           dict(num_topk=2, token_mask=torch.ones(4, device='cuda')), dict(num_topk=2, token_mask=torch.ones(5, device='cuda', dtype=torch.bool))]
    for kw in bad:
        with pytest.raises(RuntimeError):
            router.route(l, **kw)
    for x in (l.half(), l[0], l.t(), torch.randn(4, 1025, device='cuda'), l[:, :0], l[:1].expand(4, 64)):
        with pytest.raises(RuntimeError):
            router.route(x, 1)
    with pytest.raises(ValueError):
        router.route(l, 2, 'relu')
    idx = torch.zeros(4, 2, dtype=torch.int64, device='cuda')
    d = torch.zeros(4, 2, device='cuda')
    for args in ((d[:3], l, idx), (d.double(), l, idx), (d, l, idx[:, :1]), (d, l, idx.short()), (d.cpu(), l, idx), (d, l, idx[:2]),
                 (torch.zeros(4, 17, device='cuda'), l, torch.zeros(4, 17, dtype=torch.int64, device='cuda'))):
        with pytest.raises(RuntimeError):
            router.route_backward(*args)


def test_refusals_of_the_statements():
    l = torch.randn(4, 64)
    for kw in (dict(num_topk=0), dict(num_topk=9, num_groups=8), dict(num_topk=2, num_groups=7), dict(num_topk=2, num_groups=8, num_topk_groups=9),
               dict(num_topk=2, num_groups=8, group_top=3)):
        with pytest.raises(ValueError):
            router.route(l, **kw)
    with pytest.raises(ValueError):
        router.route_backward(torch.zeros(4, 2), l, torch.zeros(4, 2, dtype=torch.int64), 'relu')


@pytest.mark.gpu
def test_short_divisions_have_the_bits_of_the_general_ones(tmp_path):
    """Every reciprocal of the range that the kernel takes it in, and six thousand million quotients."""
    import shutil
    import subprocess
    from pathlib import Path
    nvcc = shutil.which('nvcc') or '/usr/local/cuda/bin/nvcc'
    if not Path(nvcc).exists():
        pytest.skip('no compiler')
    root = Path(__file__).resolve().parents[1]
    program = tmp_path / 'division'
    subprocess.run([nvcc, '-gencode', 'arch=compute_100a,code=sm_100a', '-O3', '-std=c++17', '-I', root / 'deepep_ascend_b200' / 'csrc' / 'kernels',
                    root / 'tests' / 'probes' / 'division.cu', '-o', program], check=True)
    state, reciprocals, quotients, count = subprocess.run([program], check=True, capture_output=True, text=True).stdout.split()
    assert (state, int(reciprocals), int(quotients)) == ('cudaSuccess', 0, 0) and int(count) > 6e9


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('score,renormalize', [('sigmoid', True), ('sigmoid', False), ('softmax', True), ('softmax', False)])
def test_gradients_of_empty_places_count_for_nothing(score, renormalize, device):
    """Whatever stands there: no number, or none at all."""
    g = torch.Generator().manual_seed(0)
    logits, d = torch.randn(9, 24, generator=g).to(device), torch.randn(9, 4, generator=g).to(device)
    idx = router.route_ref(logits, 4, score)[0]
    idx[2, 1], idx[4, 3], idx[5, 0], idx[7] = -1, -1, -1, -1
    want = router.route_backward(torch.where(idx >= 0, d, 0.0), logits, idx, score, renormalize)
    for nothing in (math.nan, math.inf, -math.inf, 1e30):
        assert torch.equal(router.route_backward(torch.where(idx >= 0, d, nothing), logits, idx, score, renormalize), want)
    assert torch.isfinite(want).all()
