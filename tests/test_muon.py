"""Orthogonalised updates: the kernels and the PyTorch statement against the Newton-Schulz steps in 64 bits, and what they are for."""
import pytest
import torch

from deepep_ascend_b200.ops.muon import COEFFICIENTS, orthogonalize, orthogonalize_ref

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
BF16, F32 = torch.bfloat16, torch.float32


def _exact(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    X = x.double()
    X = X / (torch.linalg.matrix_norm(X, keepdim=True) + eps)
    for _ in range(steps):
        if X.shape[-2] <= X.shape[-1]:
            A = X @ X.mT
            X = a * X + (b * A + c * A @ A) @ X
        else:
            A = X.mT @ X
            X = a * X + X @ (b * A + c * A @ A)
    return X


def _matrix(kind, count, rows, cols, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(count, rows, cols, generator=g)
    if kind == 'strong directions':           # momentum: a few directions far above the noise
        x = 0.1 * x + torch.randn(count, rows, 8, generator=g) @ (torch.randn(count, 8, cols, generator=g) * torch.logspace(0, -1, 8)[:, None])
    elif kind == 'one direction':
        x = 0.01 * x + torch.randn(count, rows, 1, generator=g) @ torch.randn(count, 1, cols, generator=g)
    elif kind == 'rows of all sizes':
        x = x * torch.logspace(0, -3, rows)[torch.randperm(rows, generator=g)][:, None]
    return 1e-3 * x


def _error(got, want):
    """Per matrix: 2-norm of the difference over that of the result."""
    return (torch.linalg.matrix_norm(got.double().cpu() - want.cpu()) / torch.linalg.matrix_norm(want.cpu())).max().item()


# Rounding the result to bf16 is off by 1.7e-3 of its norm.  Simulated in 64 bits, the steps' own roundings add at most 1e-3 to that for matrices of 64 and
# more rows (2.2e-3 where one direction holds nearly all of the norm); matrices of fewer rows are held to the same.
BOUND = {'normal': 2.5e-3, 'strong directions': 2.7e-3, 'one direction': 3.5e-3, 'rows of all sizes': 2.5e-3}

SHAPES = [(1, 64, 64), (2, 128, 256), (1, 129, 130), (3, 77, 301), (2, 300, 77), (1, 256, 1024), (1, 1000, 257), (1, 511, 513), (2, 640, 384), (5, 65, 1001), (1, 31, 2000),
          (1, 2056, 100)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('kind', sorted(BOUND))
@pytest.mark.parametrize('count,rows,cols', SHAPES)
def test_against_64_bits(count, rows, cols, kind, device):
    for dtype in (BF16, F32):
        x = _matrix(kind, count, rows, cols, rows + cols).to(dtype)
        got = orthogonalize(x.to(device))
        assert got.dtype == BF16 and got.shape == x.shape and got.is_contiguous()
        assert _error(got, _exact(x)) < BOUND[kind]


@pytest.mark.gpu
@pytest.mark.parametrize('count,rows,cols', [(1, 1024, 4096), (2, 2000, 1100), (9, 520, 776), (1, 264, 7168), (40, 128, 160)])
def test_more_tiles_than_one_wave_and_few_sms(count, rows, cols):
    x = _matrix('strong directions', count, rows, cols).bfloat16().cuda()
    want = _exact(x)
    got = orthogonalize(x)
    assert _error(got, want) < BOUND['strong directions']
    assert torch.equal(orthogonalize(x), got)                  # the same bits on every run
    for sms in (1, 7):
        assert _error(orthogonalize(x, num_sms=sms), want) < BOUND['strong directions']
    # each matrix by itself: the others change nothing but the order of a sum
    for i in range(0, count, 3):
        assert _error(orthogonalize(x[i]), want[i]) < BOUND['strong directions']


@pytest.mark.gpu
@pytest.mark.parametrize('kind', sorted(BOUND))
@pytest.mark.parametrize('count,rows,cols', [(1, 256, 9000), (2, 130, 4800), (4, 128, 4096), (2, 6001, 255), (1, 129, 200), (70, 96, 250), (3, 64, 5000)])
def test_short_matrices_in_either_form(count, rows, cols, kind):
    """Polynomial and update in one kernel, or (more tiles than SMs) in two."""
    x = _matrix(kind, count, rows, cols).bfloat16().cuda()
    want = _exact(x)
    for sms in (0, 100, 20):
        got = orthogonalize(x, num_sms=sms)
        assert _error(got, want) < BOUND[kind]
        assert torch.equal(orthogonalize(x, num_sms=sms), got)


def _falling(count, rows, cols, orders):
    """Singular values that fall off evenly by 10^orders."""
    g = torch.Generator().manual_seed(orders)
    u = torch.linalg.qr(torch.randn(count, rows, rows, generator=g, dtype=torch.float64))[0]
    v = torch.linalg.qr(torch.randn(count, cols, rows, generator=g, dtype=torch.float64))[0]
    return ((u * torch.logspace(0, -orders, rows, dtype=torch.float64)) @ v.mT).float()


# Wide enough for steps in pairs, and enough of them.  Simulated in 64 bits, pairs add up to 8e-4 to the rounding of the result for the kinds above, less than
# the bounds above leave; 2.2e-3 in another direction for singular values that fall off evenly (together 2.8e-3).
@pytest.mark.gpu
@pytest.mark.parametrize('kind', sorted(BOUND) + ['falling by 3', 'falling by 6'])
@pytest.mark.parametrize('count,rows,cols', [(5, 1000, 2017), (2, 1530, 2930), (32, 512, 1032), (3, 2600, 1208)])
def test_steps_in_pairs(count, rows, cols, kind):
    if kind in BOUND:
        x, bound = _matrix(kind, count, rows, cols), BOUND[kind]
    else:
        x, bound = _falling(count, min(rows, cols), max(rows, cols), int(kind[-1])), 3.3e-3
        x = x.mT if rows > cols else x
    x = x.bfloat16().cuda()
    got, one = orthogonalize(x), orthogonalize(x[0])       # (a single one is too few)
    assert torch.equal(orthogonalize(x), got)
    want = _exact(x)
    assert _error(got, want) < bound
    assert _error(one, want[0]) < bound


@pytest.mark.gpu
def test_pairs_of_other_steps_and_coefficients():
    x = _matrix('strong directions', 5, 1000, 2016).cuda()
    for steps, coefficients in ((1, COEFFICIENTS), (2, COEFFICIENTS), (3, COEFFICIENTS), (4, COEFFICIENTS), (6, (1.875, -1.25, 0.375)), (4, (1.5, -0.5, 0.0)),
                                (2, (6.0, -9.0, 4.0))):
        assert _error(orthogonalize(x, steps, coefficients), _exact(x, steps, coefficients)) < 2.7e-3
    # bad matrices are their own
    x = x.bfloat16()
    want = orthogonalize(x)
    x[1, 999, 2015], x[3] = float('inf'), 0.0
    got = orthogonalize(x)
    assert torch.isnan(got[1]).all() and not got[3].any()
    assert all(torch.equal(got[i], want[i]) for i in (0, 2, 4))


@pytest.mark.parametrize('device', DEVICES)
def test_tiny_matrices(device):
    for shape in ((1, 1, 1), (3, 1, 9), (2, 9, 1), (1, 2, 2), (4, 3, 17), (2, 8, 5)):
        x = _matrix('normal', *shape).to(device)
        assert _error(orthogonalize(x), _exact(x)) < 3e-3
    assert orthogonalize(torch.zeros(0, 4, 5, device=device)).shape == (0, 4, 5)
    assert orthogonalize(torch.zeros(2, 0, 5, device=device)).shape == (2, 0, 5)


@pytest.mark.parametrize('device', DEVICES)
def test_scales_zeros_and_bad_matrices(device):
    x = _matrix('normal', 1, 96, 200)
    want = _exact(x, eps=0.0)
    for scale in (1e-25, 1e-10, 1.0, 1e12, 1e16):            # the norm divides out (and is no square that leaves the range of its type)
        if device == 'cuda' or 1e-12 < scale < 1e14:
            assert _error(orthogonalize((x * scale).to(device), eps=0.0), want) < BOUND['normal']
    # eps decides where the norm is smaller
    assert _error(orthogonalize((x * 1e-9).to(device), eps=1e-3), _exact(x * 1e-9, eps=1e-3)) < BOUND['normal']
    stack = torch.stack([x[0], torch.zeros(96, 200), x[0], x[0]]).to(device)
    stack[2, 3, 5] = float('nan')
    got = orthogonalize(stack)
    assert _error(got[:1], _exact(x)) < BOUND['normal'] and not got[1].any()
    assert torch.isnan(got[2]).all() and torch.equal(got[3], got[0])


@pytest.mark.parametrize('device', DEVICES)
def test_strides_shapes_and_out(device):
    wide = _matrix('strong directions', 3, 150, 310).to(device)
    for x in (wide, wide[:, 3:140, 5:300], wide.mT, wide[::2], wide[:, ::2], wide[:1].expand(2, 150, 310), wide[0], wide[:, :, ::2], wide.transpose(0, 1)[:100],
              wide.view(3, 1, 150, 310).expand(3, 2, 150, 310), wide[:, 3:140, 5:300].mT):
        got = orthogonalize(x)
        assert got.shape == x.shape and got.is_contiguous()
        assert _error(got, _exact(x)) < 5e-3
        out = torch.empty(x.shape, dtype=BF16, device=device)
        assert orthogonalize(x, out=out) is out and torch.equal(out, got)
    own = wide.bfloat16()                                     # in place
    want = orthogonalize(own)
    assert orthogonalize(own, out=own) is own and torch.equal(own, want)


@pytest.mark.parametrize('device', DEVICES)
def test_other_steps_and_coefficients(device):
    x = _matrix('normal', 2, 100, 260)
    for steps, coefficients in ((1, COEFFICIENTS), (2, COEFFICIENTS), (8, COEFFICIENTS), (12, (1.875, -1.25, 0.375)), (3, (1.5, -0.5, 0.0))):
        assert _error(orthogonalize(x.to(device), steps, coefficients), _exact(x, steps, coefficients)) < 2.7e-3
    # what it is for: with enough steps of the fifth-order polynomial whose fixed point is one, rows are orthonormal
    got = orthogonalize(x.to(device), 25, (1.875, -1.25, 0.375)).float().cpu()
    assert (got @ got.mT - torch.eye(100)).abs().max() < 0.02


@pytest.mark.gpu
def test_streams_and_graphs():
    x = _matrix('strong directions', 2, 200, 520).cuda()
    want = orthogonalize(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = orthogonalize(x)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = orthogonalize(x)
    x.copy_(_matrix('strong directions', 2, 200, 520, seed=5))
    graph.replay()
    assert torch.equal(out, orthogonalize(x))


@pytest.mark.gpu
def test_waits_report_to_the_buffer():
    """A buffer's limit and status block serve the products, which end within it."""
    from deepep_ascend_b200 import ElasticBuffer, _native
    buf = ElasticBuffer(None, num_max_tokens_per_rank=16, hidden=256, num_topk=2)
    try:
        x = _matrix('normal', 1, 128, 256).cuda()
        assert torch.equal(orthogonalize(x, buffer=buf), orthogonalize(x))
        torch.cuda.synchronize()
        buf.check_status()
        assert _native.load().gemm_error(0) == 0
    finally:
        buf.destroy()


@pytest.mark.gpu
def test_refusals():
    x = torch.randn(2, 64, 64, device='cuda')
    for bad in (x.half(), x.double()):
        with pytest.raises(RuntimeError):
            orthogonalize(bad)
    for kw in (dict(steps=0), dict(out=torch.empty_like(x)), dict(out=torch.empty(2, 64, 64, dtype=BF16)), dict(out=torch.empty(2, 64, 65, dtype=BF16, device='cuda')[:, :, :64])):
        with pytest.raises(RuntimeError):
            orthogonalize(x, **kw)
    with pytest.raises(ValueError):
        orthogonalize(x[0, 0])


def test_refusals_of_the_statement():
    with pytest.raises(ValueError):
        orthogonalize(torch.randn(4))
    with pytest.raises(ValueError):
        orthogonalize_ref(torch.randn(4, 4), steps=0)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('shape', [(0, 5), (5, 0), (0, 0), (0, 4, 5), (2, 0, 5), (2, 3, 0, 5), (2, 3, 5, 0), (2, 0, 4, 5)])
def test_no_elements_in_any_number_of_axes(shape, device):
    x = torch.empty(shape, device=device)
    got = orthogonalize(x)
    assert got.shape == shape and got.dtype == BF16
    out = torch.empty(shape, dtype=BF16, device=device)
    assert orthogonalize(x, out=out) is out


@pytest.mark.gpu
def test_coefficients_that_leave_the_range_of_the_operands():
    """A matrix whose norm is all in one element, or in one pair of equal rows, takes the largest singular values that steps can make.  They are right
    up to where a step's A or B would leave fp16, and refused beyond.  (Right: the result's rounding is 2e-3, that of the operands 5e-4 per step, which a
    step that grows with the cube of what it is given triples.)"""
    one, pair = torch.zeros(1, 80, 96), torch.zeros(1, 80, 96)
    one[0, 3, 5], pair[0, 2:4, 7] = 2.0, 1.0
    for steps, coefficients in ((3, (3.0, 0.0, 0.0)), (5, (1.7, 0.0, 0.0)), (2, (2.0, 3.0, 0.0))):
        for x in (one, pair):
            assert _error(orthogonalize(x.cuda(), steps, coefficients), _exact(x, steps, coefficients)) < 6e-3
    for steps, coefficients in ((2, (6.0, -9.0, 4.0)), (1, (8.2872, -23.5959, 17.3004)), (3, (4.0848, -6.8946, 2.9270)), (8, COEFFICIENTS)):
        assert _error(orthogonalize(one.cuda(), steps, coefficients), _exact(one, steps, coefficients)) < 6e-3
    for steps, coefficients in ((4, (3.0, 0.0, 0.0)), (5, (4.0, 0.0, 0.0)), (3, (2.0, 3.0, 0.0)), (2, (1.0, 40.0, 40.0)), (3, (8.2872, -23.5959, 17.3004)),
                                (2, (float('nan'), 0.0, 0.0)), (2, (1.0, 0.0, float('inf'))), (1, (1.0, 0.0, float('nan')))):
        with pytest.raises(RuntimeError, match='singular values'):
            orthogonalize(one.cuda(), steps, coefficients)


@pytest.mark.gpu
def test_pairs_only_where_singular_values_stay_small():
    """Coefficients under which they grow step by step, for matrices that would be taken in pairs.  Bound as above."""
    x = torch.zeros(5, 1000, 2016)
    x[:, 3:5, 5] = 2.0
    x[1] += _matrix('normal', 1, 1000, 2016)[0]
    for steps, coefficients in ((5, (1.7, 0.0, 0.0)), (3, (2.0, 0.05, 0.0))):
        want = _exact(x.cuda(), steps, coefficients)
        assert _error(orthogonalize(x.cuda(), steps, coefficients), want) < 6e-3


def _two_levels(count, rows, cols, share, low):
    """A share of the singular values at one, the others at `low`: strong directions over a floor."""
    g = torch.Generator().manual_seed(rows)
    u = torch.linalg.qr(torch.randn(count, rows, rows, generator=g, dtype=torch.float64))[0]
    v = torch.linalg.qr(torch.randn(count, cols, rows, generator=g, dtype=torch.float64))[0]
    s = torch.full((rows,), low, dtype=torch.float64)
    s[: int(rows * share)] = 1.0
    return ((u * s) @ v.mT).float()


@pytest.mark.gpu
@pytest.mark.parametrize('share,low', [(0.1, 0.1), (0.05, 0.07), (0.2, 0.14), (0.2, 1e-3), (0.5, 1e-3), (0.03, 0.0)])
@pytest.mark.parametrize('count,rows,cols', [(32, 512, 1032), (4, 1024, 1800), (2, 512, 1032), (2, 1024, 640)])
def test_singular_values_on_two_levels(count, rows, cols, share, low):
    """Simulated in 64 bits, the steps' roundings add at most 1.9e-3 for these (single steps or with a pair in front) to the result's 1.7e-3 in another
    direction, together 2.6e-3.  A pair in any other place than in front adds up to 6.8e-3."""
    x = _two_levels(1, min(rows, cols), max(rows, cols), share, low).repeat(count, 1, 1)
    x = (x.mT if rows > cols else x).cuda()
    for y in (x, x.bfloat16()):
        got, want = orthogonalize(y), _exact(y[:1])
        assert all(torch.equal(m, got[0]) for m in got[1:])
        assert _error(got[:1], want) < 3e-3


@pytest.mark.gpu
@pytest.mark.parametrize('rows,cols,simulated', [(256, 1024, 2.9e-3), (256, 256, 2.5e-3), (300, 128, 3.9e-3), (64, 256, 5.1e-3), (128, 32, 7.9e-3), (16, 64, 2e-2)])
def test_two_levels_in_few_rows(rows, cols, simulated):
    """What five steps add at most in a simulation in 64 bits over shares from 0.02 to 0.8 and floors from 0.5 to 1e-4, half as much again for other singular vectors, and the
    result's rounding (2e-3 of a matrix of few elements)."""
    m, n = min(rows, cols), max(rows, cols)
    for share in (1.01 / m, 0.3, 0.5, 0.8):
        for low in (0.1, 3e-3, 1e-4):
            x = _two_levels(1, m, n, share, low)
            x = (x.mT if rows > cols else x).cuda()
            assert _error(orthogonalize(x), _exact(x)) < 1.5 * simulated + 2e-3


_SHORT_LIMIT = """
import torch
from deepep_ascend_b200 import ElasticBuffer, _native
from deepep_ascend_b200.ops.muon import orthogonalize
torch.manual_seed(0)
small = torch.randn(3, 300, 500, device='cuda')
want = orthogonalize(small)
buf = ElasticBuffer(None, num_max_tokens_per_rank=16, hidden=256, num_topk=2)
x = torch.randn(128, 1000000, device='cuda', dtype=torch.bfloat16)
buf.core.set_gpu_timeout(3e-4)
orthogonalize(x, steps=1, num_sms=1, buffer=buf)
torch.cuda.synchronize()
code, phase, peer, expected, observed, rank = buf.core.read_status()
assert (code, phase, expected, rank) == (1, 14, 5, 0), (code, phase, expected, rank)
assert _native.load().gemm_error(0) == 5
try:
    buf.check_status()
except RuntimeError as e:
    assert 'timed out' in str(e)
else:
    raise AssertionError('the wait was not reported')
try:
    orthogonalize(small, buffer=buf)
except RuntimeError:
    pass
else:
    raise AssertionError('a buffer whose wait has failed was taken')
# the memory of the products has been given back, and what follows is right
for _ in range(3):
    assert torch.equal(orthogonalize(small), want)
print('reported')
"""


@pytest.mark.gpu
def test_a_wait_that_runs_out_is_reported():
    """One SM sums 15625 blocks of K, for milliseconds, while the warps that wait for the sum have 0.3 ms.  (In a process of its own: the device's error flag stays up.)"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, '-c', _SHORT_LIMIT], cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip().endswith('reported'), run.stderr[-2000:]
