"""Layer norm and its gradients: the kernels and the PyTorch statements against the formulas in 64 bits."""
import pytest
import torch

from deepep_ascend_b200.ops.norm import layer_norm, layer_norm_backward, layer_norm_backward_ref

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
EPS = 2.0**-24
BF16, F32 = torch.bfloat16, torch.float32


def _make(T, H, dtype, param, seed, device, std=1.0, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, H, generator=g) * std + offset).to(dtype)
    w, b = (torch.randn(H, generator=g) * 0.3 + 1).to(param), torch.randn(H, generator=g).to(param)
    return x.to(device), w.to(device), b.to(device), torch.randn(T, H, generator=g).to(dtype).to(device)


def _half_ulp(dtype):
    return 2.0**-8 if dtype == BF16 else EPS


def _check(x, w, b, dy, eps=1e-5):
    """Forward and backward pass against 64 bits.  A sum of n terms is off by at most (n / 256 + 32) roundings of its terms' magnitudes however
    it is split over the threads of a row (256 or more of them where the row has that many channels; n roundings otherwise)."""
    (T, H), out = x.shape, {}
    x64, w64, b64, d64 = (t.double().cpu() for t in (x, w, b, dy))
    n = H if H < 512 else H / 256 + 32
    y, mean, rstd = layer_norm(x, w, b, eps)
    assert y.dtype == x.dtype and mean.dtype == rstd.dtype == F32 and mean.shape == rstd.shape == (T,)
    m64 = x64.mean(-1, keepdim=True)
    v64 = (x64 - m64).square().mean(-1, keepdim=True)
    r64 = (v64 + eps).rsqrt()
    big = x64.abs().amax(-1, keepdim=True)
    m_err = (n + 4) * EPS * big
    assert ((mean.double().cpu()[:, None] - m64).abs() <= m_err).all()
    # a mean that is off by e adds e^2 to the variance; the squares' sum and the root are off by their roundings
    r_err = r64 * ((n + 16) * EPS + 0.5 * r64**2 * (m_err**2 + 4 * EPS * big * v64.sqrt() + (EPS * big)**2 * 4))
    assert ((rstd.double().cpu()[:, None] - r64).abs() <= r_err).all()
    xh = (x64 - m64) * r64
    xh_err = (m_err + 4 * EPS * big) * r64 + xh.abs() * (r_err / r64 + 4 * EPS)
    want = xh * w64 + b64
    y_err = xh_err * w64.abs() + 4 * EPS * (want.abs() + b64.abs())
    assert ((y.double().cpu() - want).abs() <= y_err + _half_ulp(y.dtype) * (want.abs() + y_err)).all()
    out['y'] = y

    # the gradient of what the forward pass returned: mean and rstd are inputs
    dx, dw, db = layer_norm_backward(dy, x, w, mean, rstd, with_bias=True)
    assert dx.dtype == x.dtype and dw.dtype == db.dtype == w.dtype
    m, r = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    xh, g = (x64 - m) * r, d64 * w64
    xh_err = (2 * EPS * (x64.abs() + m.abs())) * r + 2 * EPS * xh.abs()
    mg, mgx = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    mg_err = (n + 4) * EPS * g.abs().mean(-1, keepdim=True)
    mgx_err = (n + 8) * EPS * (g * xh).abs().mean(-1, keepdim=True) + (g.abs() * xh_err).mean(-1, keepdim=True)
    want = r * (g - mg - xh * mgx)
    dx_err = r * (8 * EPS * (g.abs() + mg.abs() + (xh * mgx).abs()) + mg_err + xh.abs() * mgx_err + xh_err * mgx.abs())
    assert ((dx.double().cpu() - want).abs() <= dx_err + _half_ulp(dx.dtype) * (want.abs() + dx_err)).all()
    # columns: at most one rounding per row
    for got, terms, err in ((dw, d64 * xh, (d64.abs() * xh_err).sum(0)), (db, d64, 0.0)):
        err = (T + 64) * EPS * terms.abs().sum(0) + err
        want = terms.sum(0)
        assert ((got.double().cpu() - want).abs() <= err + _half_ulp(got.dtype) * (want.abs() + err) + 1e-38).all()
    no_bias = layer_norm_backward(dy, x, w, mean, rstd)
    assert no_bias[2] is None and torch.equal(no_bias[0], dx) and torch.equal(no_bias[1], dw)
    assert torch.equal(layer_norm(x, w, torch.zeros_like(b), eps)[0], layer_norm(x, w, None, eps)[0])
    return out


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype,param', [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize('T,H', [(1, 1), (3, 2), (5, 7), (2, 31), (9, 64), (4, 100), (17, 255), (33, 256), (150, 520), (300, 1000), (40, 2049), (7, 4096), (3, 7168),
                                 (2, 8192), (1, 12344), (2, 20001), (1, 40000)])
def test_against_the_formulas(T, H, dtype, param, device):
    _check(*_make(T, H, dtype, param, T + H, device))


@pytest.mark.gpu
@pytest.mark.parametrize('T,H', [(8192, 1024), (3000, 7168), (20011, 129), (70001, 8)])
def test_many_rows(T, H):
    _check(*_make(T, H, BF16, F32, 1, 'cuda'))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('T,H', [(9001, 200), (9001, 512), (5001, 1040), (2001, 4104), (1001, 8200), (1001, 12280), (701, 16392), (701, 24576), (301, 32776)])
def test_every_width_over_many_rows(T, H, dtype):
    """One, two and four pieces of 16 bytes per thread, rows of a warp, of up to 256, 384 and 1024 threads and wider ones, each with several rows per CTA."""
    _check(*_make(T, H, dtype, F32, 3, 'cuda'))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('std,offset', [(1e-3, 100.0), (1e-18, 0.0), (1e15, 0.0), (1.0, -1e4)])
def test_scales_and_offsets(std, offset, device):
    """Rows far from zero (no difference of squares), tiny ones that eps decides, huge ones."""
    _check(*_make(6, 600, F32, F32, 5, device, std, offset))


@pytest.mark.parametrize('device', DEVICES)
def test_equal_channels_and_no_rows(device):
    x, w, b, dy = _make(4, 300, F32, F32, 2, device)
    x[1] = 2.5
    y, mean, rstd = layer_norm(x, w, b)
    assert torch.equal(y[1], b) and mean[1] == 2.5
    y, mean, rstd = layer_norm(x[:0], w, b)
    assert y.shape == (0, 300) and mean.shape == rstd.shape == (0,)
    dx, dw, db = layer_norm_backward(dy[:0], x[:0], w, mean, rstd, with_bias=True)
    assert dx.shape == (0, 300) and not dw.any() and not db.any()


@pytest.mark.parametrize('device', DEVICES)
def test_a_bad_row_stays_alone(device):
    x, w, b, dy = _make(6, 520, BF16, BF16, 3, device)
    good, stats = layer_norm(x, w, b)[0].clone(), layer_norm(x, w, b)[1:]
    good_dx = layer_norm_backward(dy, x, w, *stats)[0]
    x[2, 5], x[4, 7] = float('nan'), float('inf')
    y, mean, rstd = layer_norm(x, w, b)
    rest = torch.tensor([0, 1, 3, 5], device=device)
    assert torch.equal(y[rest], good[rest]) and torch.isnan(y[2]).all() and torch.isnan(y[4]).all()
    dx, dw, _ = layer_norm_backward(dy, x, w, mean, rstd)
    assert torch.equal(dx[rest], good_dx[rest]) and torch.isnan(dx[2]).all() and torch.isnan(dw).all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('H', [64, 333, 1024, 7168])
def test_strides_and_starts(H, dtype, device):
    """Rows of a wider matrix that start anywhere, broadcast inputs and gradients, channels apart, parameters that start anywhere, leading axes."""
    wide, w, b, d_wide = _make(10, H + 37, dtype, dtype, 4, device)
    for start in (0, 1, 4, 8):
        x, dy, ww, bb = wide[:, start:start + H], d_wide[:, start + 3:start + 3 + H], w[start:start + H], b[7:7 + H]
        _check(x, ww, bb, dy)
        _check(x[::3], ww, bb, d_wide[:4, :H])
        _check(x[:1].expand(5, H), ww, bb, dy[:1].expand(5, H))
        _check(x.t().contiguous().t(), ww, bb, dy.t().contiguous().t())
    ww, bb = w[:H].clone(), b[:H].clone()
    want = layer_norm(wide[:, :H].contiguous(), ww, bb)
    deep = wide[:, :H].contiguous().view(2, 5, H)
    y, mean, rstd = layer_norm(deep, ww, bb)
    assert y.shape == deep.shape and mean.shape == (2, 5) and torch.equal(y.view(10, H), want[0])
    dx, dw, db = layer_norm_backward(torch.ones_like(deep), deep, ww, mean, rstd, with_bias=True)
    assert dx.shape == deep.shape and torch.equal(db, torch.full_like(db, 10.0))


@pytest.mark.gpu
def test_the_same_bits_on_every_run_and_stream():
    x, w, b, dy = _make(5000, 2048, BF16, F32, 6, 'cuda')
    y, mean, rstd = layer_norm(x, w, b)
    want = layer_norm_backward(dy, x, w, mean, rstd, with_bias=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(layer_norm_backward(dy, x, w, mean, rstd, with_bias=True), want))
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y2, m2, r2 = layer_norm(x, w, b)
        out = layer_norm_backward(dy, x, w, m2, r2, with_bias=True)
    for t in (y2, *out):
        t.zero_()
    graph.replay()
    assert torch.equal(y2, y) and all(torch.equal(p, q) for p, q in zip(out, want))


def test_gradient_against_differences():
    g = torch.Generator().manual_seed(0)
    T, H, h = 3, 11, 1e-6
    x, w, b, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((T, H), (H,), (H,), (T, H)))

    def loss(x, w, b):
        return (layer_norm(x, w, b)[0] * dy).sum()
    _, mean, rstd = layer_norm(x, w, b)
    for k, got in enumerate(layer_norm_backward_ref(dy, x, w, mean, rstd, with_bias=True)):
        for i in range(got.numel()):
            args = [[x.clone(), w.clone(), b.clone()] for _ in range(2)]
            args[0][k].view(-1)[i] += h
            args[1][k].view(-1)[i] -= h
            assert abs((loss(*args[0]) - loss(*args[1])).item() / (2 * h) - got.reshape(-1)[i].item()) < 1e-7


@pytest.mark.gpu
def test_refusals():
    x, w, b, dy = _make(4, 64, BF16, BF16, 0, 'cuda')
    _, mean, rstd = layer_norm(x, w, b)
    for args in ((x.half(), w, b), (x, w[:63], b), (x, w.half(), b), (x, w, b.float()), (x, w.cpu(), b), (x, w, b[:63]), (x, w.view(1, 64), b), (x[:, :0], w[:0], None)):
        with pytest.raises(RuntimeError):
            layer_norm(*args)
    for args in ((dy.float(), x, w, mean, rstd), (dy, x, w, mean[:3], rstd), (dy, x, w, mean, rstd.double()), (dy, x, w, mean.cpu(), rstd), (dy.cpu(), x, w, mean, rstd)):
        with pytest.raises(RuntimeError):
            layer_norm_backward(*args)
    with pytest.raises(ValueError):
        layer_norm_backward(dy[:3], x, w, mean, rstd)


@pytest.mark.gpu
def test_gradients_of_the_parameters_have_a_storage_each():
    """Whatever frees, saves or resizes the one leaves the other alone."""
    x, w, b, dy = _make(5, 72, BF16, F32, 0, 'cuda')
    _, mean, rstd = layer_norm(x, w, b)
    _, dw, db = layer_norm_backward(dy, x, w, mean, rstd, with_bias=True)
    for t in (dw, db):
        assert t.untyped_storage().nbytes() == 72 * 4 and t.storage_offset() == 0
