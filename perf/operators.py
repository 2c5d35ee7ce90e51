"""The operators around the expert layer on one GPU, for timing and for comparing outputs: routing (``ops.router``), layer norm
(``ops.norm``) and the orthogonalised update of expert matrices (``ops.muon``).

``own`` chooses what ``run`` computes with: elementary PyTorch operations in 32 bits, or this library's kernels.  Sizes are those of the
repository's own benchmarks and tests: up to 65536 tokens (8192 of each of eight ranks), hidden 7168 and 2048, top-8 of 256 / top-6 of
160 experts, intermediate 2048.  Data is synthetic.

    listed()        the cases
    draw(rng)       one more case of the same ranges
    prepare / run   inputs of a case / one pass
    work            bytes and operations that one pass cannot do without
    exact           the computed outputs in 64 bits
"""
import math

import torch

own = False


def listed():
    return [
        # Routing of a decode step: a handful of tokens between two layers, so launch and host time are all there is.
        dict(name='route_decode_8', op='route', dir='fwd', tokens=8, experts=256, topk=8, score='sigmoid', bias=True, groups=8, topk_groups=4,
             group_top=2, renormalize=True, scale=2.5, dtype='float32', masked=0.0),
        # Routing of a whole training batch (8192 tokens of each of eight ranks), the grouped sigmoid gate with a balance bias.
        dict(name='route_65536', op='route', dir='fwd', tokens=65536, experts=256, topk=8, score='sigmoid', bias=True, groups=8, topk_groups=4,
             group_top=2, renormalize=True, scale=2.5, dtype='float32', masked=0.0),
        # Gradient of a plain softmax gate (every expert's logit has one): bf16 logits, a ragged batch with padding tokens, 160 experts.
        dict(name='route_grad_softmax_4097', op='route', dir='bwd', tokens=4097, experts=160, topk=6, score='softmax', bias=False, groups=8,
             topk_groups=3, group_top=1, renormalize=False, scale=1.0, dtype='bfloat16', masked=0.1),
        # Gradient of the grouped sigmoid gate over a whole training batch.
        dict(name='route_grad_65536', op='route', dir='bwd', tokens=65536, experts=256, topk=8, score='sigmoid', bias=True, groups=8,
             topk_groups=4, group_top=2, renormalize=True, scale=2.5, dtype='float32', masked=0.0),
        # The norm in front of the expert layer in a decode step.
        dict(name='norm_decode_3', op='norm', dir='fwd', tokens=3, hidden=7168, dtype='bfloat16', param='bfloat16', bias=False),
        # ... of a prefill or training batch.
        dict(name='norm_8192', op='norm', dir='fwd', tokens=8192, hidden=7168, dtype='bfloat16', param='bfloat16', bias=False),
        # Gradients in 32 bits with a bias, odd width (no row but the first starts on 16 bytes).
        dict(name='norm_grad_odd_1001', op='norm', dir='bwd', tokens=1001, hidden=2049, dtype='float32', param='float32', bias=True),
        # Gradients of a training batch, 32-bit parameters.
        dict(name='norm_grad_8192', op='norm', dir='bwd', tokens=8192, hidden=7168, dtype='bfloat16', param='float32', bias=False),
        # Update of three small matrices of odd size (an adapter or a shared projection), 32-bit momentum.
        dict(name='muon_3x777x1001', op='muon', count=3, rows=777, cols=1001, dtype='float32'),
        # Update of the gate's weights: one wide matrix, little parallel work.
        dict(name='muon_gate_256x7168', op='muon', count=1, rows=256, cols=7168, dtype='bfloat16'),
        # Update of the down projections of four experts (tall matrices).
        dict(name='muon_4x7168x2048', op='muon', count=4, rows=7168, cols=2048, dtype='bfloat16'),
        # Update of the gate | up projections of eight experts.
        dict(name='muon_8x4096x7168', op='muon', count=8, rows=4096, cols=7168, dtype='bfloat16'),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n + 1 if n == 3072 else n


def _muon_flops(count, rows, cols):
    m, n = min(rows, cols), max(rows, cols)
    return MUON_STEPS * count * (m * m * n + m * m * m + 2 * m * m * n)


def draw(rng):
    op = rng.choice(['route', 'norm', 'muon'])
    if op == 'route':
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = max(groups, _log_int(rng, 8, 512) // groups * groups)
        topk_groups = rng.randint(1, groups)
        topk = rng.randint(1, min(16, experts // groups * topk_groups))
        return dict(op=op, dir=rng.choice(['fwd', 'bwd']), tokens=_log_int(rng, 1, 65536 * 256 // max(experts, 256)), experts=experts, topk=topk,
                    score=rng.choice(['sigmoid', 'softmax']), bias=rng.random() < 0.5, groups=groups, topk_groups=topk_groups,
                    group_top=1 if experts // groups < 2 else rng.choice([1, 2]), renormalize=topk > 1 and rng.random() < 0.6, scale=rng.choice([1.0, 2.5]),
                    dtype=rng.choice(['float32', 'bfloat16']), masked=rng.choice([0.0, 0.1]))
    if op == 'norm':
        hidden = _log_int(rng, 64, 8192)
        if rng.random() < 0.6:
            hidden = max(64, hidden // 64 * 64)
        hidden += hidden == 3072
        return dict(op=op, dir=rng.choice(['fwd', 'bwd']), tokens=_log_int(rng, 1, 8192 * 7168 // max(hidden, 7168)), hidden=hidden,
                    dtype=rng.choice(['bfloat16', 'float32']), param=rng.choice(['bfloat16', 'float32']), bias=rng.random() < 0.5)
    while True:
        case = dict(op=op, count=_log_int(rng, 1, 8), rows=_log_int(rng, 64, 7168), cols=_log_int(rng, 64, 7168), dtype=rng.choice(['bfloat16', 'float32']))
        if _muon_flops(case['count'], case['rows'], case['cols']) <= _muon_flops(8, 4096, 7168):
            return case


# ---------------------------------------------------------------------------------------------------------------- inputs
MUON_STEPS, MUON_COEFFICIENTS, MUON_EPS, NORM_EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7, 1e-5


def _normal(gen, *shape, dtype=torch.float32, std=1.0):
    return torch.empty(shape, dtype=dtype, device='cuda').normal_(0.0, std, generator=gen)


def _prepare_route(c, gen):
    T, E, K = c['tokens'], c['experts'], c['topk']
    # gate logits: some experts are liked better than others, which is what the balance bias answers
    logits = _normal(gen, T, E, std=1.5) + _normal(gen, E, std=0.7)
    s = dict(logits=logits.to(getattr(torch, c['dtype'])), bias=_normal(gen, E, std=0.05) if c['bias'] else None, mask=None)
    if c['masked']:
        s['mask'] = torch.rand(T, generator=gen, device='cuda') >= c['masked']       # False: a padding token
    if c['dir'] == 'bwd':
        s['idx'] = _choose(c, s)[1]
        s['d_weights'] = _normal(gen, T, K)
    return s


def _prepare_norm(c, gen):
    T, H, dtype, param = c['tokens'], c['hidden'], getattr(torch, c['dtype']), getattr(torch, c['param'])
    # activations of a residual stream: rows of different size, a few channels far larger than the others
    x = _normal(gen, T, H) * (0.5 + torch.rand(T, 1, generator=gen, device='cuda'))
    x[:, torch.randint(0, H, (max(1, H // 512),), generator=gen, device='cuda')] *= 12.0
    x = x.to(dtype)
    s = dict(x=x, weight=(1.0 + _normal(gen, H, std=0.1)).to(param), bias=_normal(gen, H, std=0.1).to(param) if c['bias'] else None)
    if c['dir'] == 'bwd':
        s['dy'] = _normal(gen, T, H, dtype=dtype)
        s['mean'], s['rstd'] = _moments(x.float())
    return s


def _prepare_muon(c, gen):
    # momentum of a weight matrix: a few strong directions over a floor of noise
    G, M, N = c['count'], c['rows'], c['cols']
    strong = _normal(gen, G, M, 16) * torch.logspace(0, -1, 16, device='cuda')
    g = torch.baddbmm(_normal(gen, G, M, N, std=0.3), strong, _normal(gen, G, 16, N))
    return dict(g=(1e-3 * g).to(getattr(torch, c['dtype'])))


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    return case, {'route': _prepare_route, 'norm': _prepare_norm, 'muon': _prepare_muon}[case['op']](case, gen)


# ------------------------------------------------------------------------------------------------------- the plain forms
def _sum_by_halves(e):
    """Sum along the last axis as a tree: padded with zeros to a power of two, the upper half is added to the lower one."""
    width = 1 << (e.shape[-1] - 1).bit_length()
    e = torch.nn.functional.pad(e, (0, width - e.shape[-1]))
    # (the tree's levels, not its elements)
    while e.shape[-1] > 1:
        h = e.shape[-1] // 2
        e = e[..., :h] + e[..., h:]
    return e


def _scores(c, logits):
    l = logits.float()
    if c['score'] == 'sigmoid':
        return 1.0 / (1.0 + torch.exp(-l))
    e = torch.exp(l - l.max(dim=-1, keepdim=True).values)
    return e / _sum_by_halves(e)


def _choose(c, s):
    """(scores, chosen experts): what the weights are made of."""
    T, E, K, G = c['tokens'], c['experts'], c['topk'], c['groups']
    p = _scores(c, s['logits'])
    choice = p if s['bias'] is None else p + s['bias']
    none = float('-inf')
    choice = torch.where(torch.isnan(choice) | (s['logits'] == none), none, choice)
    if G > 1:
        best = torch.sort(choice.view(T, G, E // G), dim=-1, descending=True).values[..., :c['group_top']].sum(-1)
        order = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :c['topk_groups']]
        keep = torch.zeros(T, G, dtype=torch.bool, device=choice.device).scatter(1, order, True)
        choice = torch.where(keep.unsqueeze(-1), choice.view(T, G, E // G), none).view(T, E)
    value, idx = torch.sort(choice, dim=-1, descending=True, stable=True)
    value, idx = value[:, :K], idx[:, :K]
    live = value > none
    if s['mask'] is not None:
        live = live & s['mask'].unsqueeze(1)
    return p, torch.where(live, idx, -1)


def _weights(c, p, idx):
    """Scores of the chosen experts (0 in empty places), and their sum."""
    w = torch.where(idx >= 0, p.gather(1, idx.clamp_min(0)), 0.0)
    return w, w.sum(-1, keepdim=True)


def _run_route(c, s):
    p, idx = _choose(c, s)
    w, total = _weights(c, p, idx)
    if c['renormalize']:
        w = torch.where(total > 0, w / total, 0.0)
    ones = torch.ones(idx.numel(), dtype=torch.int32, device=idx.device)
    count = torch.zeros(c['experts'] + 1, dtype=torch.int32, device=idx.device).scatter_add_(0, idx.reshape(-1) + 1, ones)[1:]
    return dict(idx=idx, weights=w * c['scale'], count=count)


def _run_route_grad(c, s):
    idx, dw = s['idx'], s['d_weights'] * c['scale']
    p = _scores(c, s['logits'])
    live = idx >= 0
    w, total = _weights(c, p, idx)
    if c['renormalize']:
        dw = torch.where(live & (total > 0), (dw - (dw * w).sum(-1, keepdim=True) / total) / total, 0.0)
    # one column more than experts takes what empty places would add
    place = torch.where(live, idx, c['experts'])
    dp = torch.zeros(c['tokens'], c['experts'] + 1, device=dw.device).scatter(1, place, torch.where(live, dw, 0.0))[:, :-1]
    dl = dp * p * (1.0 - p) if c['score'] == 'sigmoid' else p * (dp - (p * dp).sum(-1, keepdim=True))
    return torch.where(live.any(-1, keepdim=True), dl, 0.0).to(s['logits'].dtype)


def _moments(x):
    mean = x.mean(-1)
    return mean, 1.0 / torch.sqrt((x - mean.unsqueeze(-1)).square().mean(-1) + NORM_EPS)


def _run_norm(c, s):
    x = s['x'].float()
    mean, rstd = _moments(x)
    y = (x - mean.unsqueeze(-1)) * rstd.unsqueeze(-1) * s['weight'].float()
    if s['bias'] is not None:
        y = y + s['bias'].float()
    return dict(y=y.to(s['x'].dtype), mean=mean, rstd=rstd)


def _run_norm_grad(c, s):
    x, dy, rstd = s['x'].float(), s['dy'].float(), s['rstd'].unsqueeze(-1)
    xh = (x - s['mean'].unsqueeze(-1)) * rstd
    g = dy * s['weight'].float()
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    out = dict(dx=dx.to(s['x'].dtype), dw=(dy * xh).sum(0).to(s['weight'].dtype))
    if s['bias'] is not None:
        out['db'] = dy.sum(0).to(s['bias'].dtype)
    return out


def _run_muon(c, s):
    a, b, k = MUON_COEFFICIENTS
    x = s['g'].float()
    tall = c['rows'] > c['cols']
    if tall:
        x = x.transpose(1, 2)
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + MUON_EPS)
    # (one step behind the other)
    for _ in range(MUON_STEPS):
        gram = x @ x.transpose(1, 2)
        x = a * x + (b * gram + k * (gram @ gram)) @ x
    return (x.transpose(1, 2) if tall else x).to(torch.bfloat16).contiguous()


def run(state):
    c, s = state
    if own:
        return _run_own(c, s)
    if c['op'] == 'muon':
        return _run_muon(c, s)
    if c['op'] == 'norm':
        return _run_norm(c, s) if c['dir'] == 'fwd' else _run_norm_grad(c, s)
    return _run_route(c, s) if c['dir'] == 'fwd' else _run_route_grad(c, s)


# ------------------------------------------------------------------------------------------------------ this library's calls
def _run_own(c, s):
    if c['op'] == 'muon':
        from deepep_ascend_b200.ops.muon import orthogonalize
        return orthogonalize(s['g'], steps=MUON_STEPS, coefficients=MUON_COEFFICIENTS, eps=MUON_EPS)
    if c['op'] == 'norm':
        from deepep_ascend_b200.ops.norm import layer_norm, layer_norm_backward
        if c['dir'] == 'fwd':
            y, mean, rstd = layer_norm(s['x'], s['weight'], s['bias'], eps=NORM_EPS)
            return dict(y=y, mean=mean, rstd=rstd)
        dx, dw, db = layer_norm_backward(s['dy'], s['x'], s['weight'], s['mean'], s['rstd'], with_bias=c['bias'])
        return dict(dx=dx, dw=dw, db=db) if c['bias'] else dict(dx=dx, dw=dw)
    from deepep_ascend_b200.ops.router import route, route_backward
    if c['dir'] == 'bwd':
        return route_backward(s['d_weights'], s['logits'], s['idx'], score=c['score'], renormalize=c['renormalize'], scale=c['scale'])
    idx, weights, count = route(s['logits'], c['topk'], score=c['score'], bias=s['bias'], num_groups=c['groups'], num_topk_groups=c['topk_groups'],
                                group_top=c['group_top'], renormalize=c['renormalize'], scale=c['scale'], token_mask=s['mask'])
    return dict(idx=idx, weights=weights, count=count)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    size = {'float32': 4, 'bfloat16': 2}
    if c['op'] == 'muon':
        elements = c['count'] * c['rows'] * c['cols']
        # the two symmetric products need one half each
        return dict(bytes=elements * (size[c['dtype']] + 2), flops=_muon_flops(c['count'], c['rows'], c['cols']))
    T = c['tokens']
    if c['op'] == 'norm':
        H, rows, params = c['hidden'], 2 if c['dir'] == 'fwd' else 3, size[c['param']] * (2 if c['bias'] else 1)
        return dict(bytes=rows * T * H * size[c['dtype']] + 8 * T + H * params + (H * params if c['dir'] == 'bwd' else 0),
                    flops=(8 if c['dir'] == 'fwd' else 14) * T * H)
    E, K, logits = c['experts'], c['topk'], T * c['experts'] * size[c['dtype']]
    if c['dir'] == 'fwd':
        return dict(bytes=logits + T * K * 12 + 4 * E * (2 if c['bias'] else 1) + (T if c['masked'] else 0), flops=10 * T * E)
    # a gradient that only the chosen experts have needs their logits only
    read = logits if c['score'] == 'softmax' and not c['renormalize'] else T * K * size[c['dtype']]
    return dict(bytes=read + T * K * 12 + logits, flops=10 * T * (E if read == logits else K))


# ----------------------------------------------------------------------------------------------------------------- exact
def _exact_choice(c, s):
    """Probabilities in 64 bits, chosen experts and which of them count, from the definition: one selection after the other."""
    T, E, K, G = c['tokens'], c['experts'], c['topk'], c['groups']
    l = s['logits'].double()
    p = torch.sigmoid(l) if c['score'] == 'sigmoid' else torch.softmax(l, dim=-1)
    left = (p + s['bias'].double() if s['bias'] is not None else p.clone()).view(T, G, E // G)
    if G > 1:
        best = left.topk(c['group_top'], dim=-1).values.sum(-1)
        chosen = torch.zeros_like(best, dtype=torch.bool)
        for _ in range(c['topk_groups']):
            chosen[torch.arange(T), best.masked_fill(chosen, -math.inf).argmax(-1)] = True
        left = left.masked_fill(~chosen.unsqueeze(-1), -math.inf)
    left, idx = left.reshape(T, E).clone(), []
    for _ in range(K):
        k = left.argmax(-1, keepdim=True)
        idx.append(k)
        left.scatter_(1, k, -math.inf)
    live = torch.ones(T, 1, dtype=torch.bool, device=l.device) if s['mask'] is None else s['mask'].unsqueeze(1)
    return l, p, torch.cat(idx, dim=1), live.expand(T, K)


def _exact_route(c, s):
    _, p, idx, live = _exact_choice(c, s)
    w = p.gather(1, idx)
    if c['renormalize']:
        w = w / w.sum(1, keepdim=True)
    # whole numbers are compared with the plain form's: experts that tie in 32 bits need not tie here
    return dict(idx=None, weights=torch.where(live, c['scale'] * w, 0.0), count=None)


def _exact_route_grad(c, s):
    """Derivative of sum(d_weights * weights) by the chain rule through the whole row, the chosen experts given."""
    idx, live = s['idx'].clamp_min(0), (s['idx'] >= 0).double()
    with torch.enable_grad():
        l = s['logits'].double().requires_grad_(True)
        w = (torch.sigmoid(l) if c['score'] == 'sigmoid' else torch.softmax(l, dim=-1)).gather(1, idx) * live
        if c['renormalize']:
            w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
        grad, = torch.autograd.grad((w * s['d_weights'].double()).sum() * c['scale'], l)
    return grad


def _exact_norm(c, s):
    x = s['x'].double()
    var, mean = torch.var_mean(x, dim=-1, correction=0)
    y = torch.nn.functional.layer_norm(x, (c['hidden'],), s['weight'].double(), None if s['bias'] is None else s['bias'].double(), NORM_EPS)
    return dict(y=y, mean=mean, rstd=(var + NORM_EPS).rsqrt())


def _exact_norm_grad(c, s):
    x, dy, rstd = s['x'].double(), s['dy'].double(), s['rstd'].double()[:, None]
    xh = (x - s['mean'].double()[:, None]) * rstd
    dw, g = (dy * xh).sum(0), dy * s['weight'].double()
    along = (g * xh).sum(1, keepdim=True) / c['hidden']
    out = dict(dx=(g - xh * along - g.sum(1, keepdim=True) / c['hidden']) * rstd, dw=dw)
    if c['bias']:
        out['db'] = dy.sum(0)
    return out


def _exact_muon(c, s):
    # one matrix after the other, by the smaller side
    a, b, k = MUON_COEFFICIENTS
    out = []
    for g in s['g']:
        x = g.double()
        x = x / (torch.linalg.matrix_norm(x) + MUON_EPS)
        for _ in range(MUON_STEPS):
            if x.shape[0] > x.shape[1]:
                gram = x.t() @ x
                x = torch.addmm(x, x, b * gram + k * gram @ gram, beta=a)
            else:
                gram = x @ x.t()
                x = torch.addmm(x, b * gram + k * gram @ gram, x, beta=a)
        out.append(x)
    return torch.stack(out)


def exact(case, seed):
    c, s = prepare(case, seed)
    if c['op'] == 'muon':
        return _exact_muon(c, s)
    if c['op'] == 'norm':
        return _exact_norm(c, s) if c['dir'] == 'fwd' else _exact_norm_grad(c, s)
    return _exact_route(c, s) if c['dir'] == 'fwd' else _exact_route_grad(c, s)
