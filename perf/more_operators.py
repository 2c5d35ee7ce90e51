"""The attention half of a layer on one GPU, for timing and for comparing outputs: norm and rotation of queries and keys (``ops.rotary``),
attention over packed prompts, forward and backward, and attention of single tokens over a paged cache (``ops.attention``).

``own`` chooses what ``run`` computes with: elementary PyTorch operations in 32 bits, or this library's kernels.  Sizes are generic, or those of the
repository's own benchmarks: hidden 7168 (56 heads of 128 channels) and 2048 (16 of 128, 32 of 64), 8192 tokens per rank, decode batches of up to 128 tokens.
Data is synthetic.

    listed()        the cases
    draw(rng)       one more case of the same ranges
    prepare / run   inputs of a case / one pass
    work            bytes and operations that one pass cannot do without
    exact           the computed outputs in 64 bits
"""
import math
import random

import torch

own = False


def listed():
    return [
        # A decode step: queries and keys of sixteen sequences, keys and values go to their places in the paged cache.  Launch and host time.
        dict(name='rope_append_16', op='rope', dir='append', tokens=16, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, dtype='bfloat16',
             param='float32', page=64, positions=8192),
        # A prefill or training batch.
        dict(name='rope_8192', op='rope', dir='fwd', tokens=8192, heads=56, kv_heads=8, dim=128, rotary=128, interleaved=False, dtype='bfloat16',
             param='float32', page=0, positions=8192),
        # Gradients of a ragged batch in 32 bits, neighbouring channels as pairs, half of the channels rotated.
        dict(name='rope_grad_odd_1003', op='rope', dir='bwd', tokens=1003, heads=16, kv_heads=4, dim=96, rotary=48, interleaved=True, dtype='float32',
             param='float32', page=0, positions=131072),
        # Gradients of a training batch.
        dict(name='rope_grad_8192', op='rope', dir='bwd', tokens=8192, heads=56, kv_heads=8, dim=128, rotary=128, interleaved=False, dtype='bfloat16',
             param='float32', page=0, positions=8192),
        # One short prompt.
        dict(name='prompt_97', op='prompt', dir='fwd', tokens=97, seqs=1, context=0, heads=32, kv_heads=8, dim=128, causal=True),
        # A prefill batch of 31 prompts of different lengths.
        dict(name='prompt_packed_8191', op='prompt', dir='fwd', tokens=8191, seqs=31, context=0, heads=56, kv_heads=8, dim=128, causal=True),
        # One long prompt.
        dict(name='prompt_16384', op='prompt', dir='fwd', tokens=16384, seqs=1, context=0, heads=56, kv_heads=8, dim=128, causal=True),
        # Gradients of a ragged micro-batch of narrower heads.
        dict(name='prompt_grad_odd_2011', op='prompt', dir='bwd', tokens=2011, seqs=7, context=0, heads=32, kv_heads=4, dim=64, causal=True),
        # Gradients of a training batch: two documents of about 4096 tokens.
        dict(name='prompt_grad_8192', op='prompt', dir='bwd', tokens=8192, seqs=2, context=0, heads=56, kv_heads=8, dim=128, causal=True),
        # A single user's short answer: one token over a few pages.
        dict(name='decode_1x200', op='decode', seqs=1, longest=200, heads=32, kv_heads=8, dim=128, page=64),
        # A server's batch: sequences of very different lengths, pages of 16.
        dict(name='decode_128x8192', op='decode', seqs=128, longest=8192, heads=56, kv_heads=8, dim=128, page=16),
        # Few very long sequences: all of the work along the cache.
        dict(name='decode_3x131072', op='decode', seqs=3, longest=131072, heads=32, kv_heads=4, dim=128, page=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, most, groups):
    group = rng.choice([g for g in groups if g <= most])
    kv = _log_int(rng, 1, most // group)
    return dict(heads=kv * group, kv_heads=kv)


def _largest(op, dir=None):
    sizes = [work(c) for c in listed() if c['op'] == op and c.get('dir') in (dir, 'fwd' if dir == 'append' else dir)]
    return max(w['bytes'] for w in sizes), max(w['flops'] for w in sizes)


def draw(rng):
    op = rng.choice(['rope', 'prompt', 'decode'])
    while True:
        if op == 'rope':
            case = dict(op=op, dir=rng.choice(['fwd', 'bwd', 'append']), tokens=_log_int(rng, 1, 16384), dim=rng.choice([64, 80, 96, 128, 128, 192, 256]),
                        interleaved=rng.random() < 0.4, dtype=rng.choice(['bfloat16', 'bfloat16', 'float32']), param=rng.choice(['bfloat16', 'float32']),
                        positions=_log_int(rng, 4096, 262144), **_heads(rng, 64, [1, 1, 2, 4, 7, 8]))
            case['rotary'] = case['dim'] if rng.random() < 0.6 else max(16, case['dim'] // 32 * 16)
            case['page'] = rng.choice([1, 16, 24, 64, 256]) if case['dir'] == 'append' else 0
            if case['page']:
                case['dtype'] = 'bfloat16'
        elif op == 'prompt':
            tokens = _log_int(rng, 1, 16384)
            case = dict(op=op, dir=rng.choice(['fwd', 'bwd']), tokens=tokens, seqs=_log_int(rng, 1, min(64, tokens)),
                        context=0 if rng.random() < 0.7 else _log_int(rng, 1, 4096), dim=rng.choice([32, 64, 64, 80, 96, 128, 128, 128]), causal=rng.random() < 0.8,
                        **_heads(rng, 64, [1, 1, 2, 4, 7, 8, 16]))
        else:
            case = dict(op=op, seqs=_log_int(rng, 1, 256), longest=_log_int(rng, 1, 131072), dim=rng.choice([64, 64, 96, 128, 128, 128]),
                        page=rng.choice([1, 16, 24, 64, 128, 256]), **_heads(rng, 64, [1, 2, 4, 7, 8, 8, 16, 24]))
        most, now = _largest(op, case.get('dir')), work(case)
        if now['bytes'] <= most[0] and now['flops'] <= most[1]:
            return case


# --------------------------------------------------------------------------------------------------------------- lengths
def _split(total, parts, seed):
    """`total` tokens in `parts` sequences of very different lengths."""
    if parts == 1:
        return [total]
    rng = random.Random(seed)
    if parts == 2:
        first = total // 2 - rng.randint(0, total // 16)
        return [first, total - first]
    weights = [math.exp(rng.gauss(0.0, 1.0)) for _ in range(parts)]
    lengths = [int(total * w / sum(weights)) for w in weights]
    lengths[rng.randrange(parts)] += total - sum(lengths)
    return lengths


def _prompt_lengths(c):
    """Lengths of the sequences' queries and keys: with `context`, a sequence has up to so many keys from earlier calls in front."""
    lq = _split(c['tokens'], c['seqs'], c['tokens'] * 64 + c['seqs'])
    rng = random.Random(c['context'])
    return lq, [n + (rng.randint(0, c['context']) if c['context'] else 0) for n in lq]


def _decode_lengths(c):
    """One sequence of the longest length, the others spread below it over the logarithm."""
    rng = random.Random(c['seqs'] * 1000003 + c['longest'])
    return [c['longest']] + [_log_int(rng, max(1, c['longest'] // 32), c['longest']) for _ in range(c['seqs'] - 1)]


# ---------------------------------------------------------------------------------------------------------------- inputs
EPS = 1e-6


def _normal(gen, *shape, dtype=torch.float32, std=1.0):
    return torch.empty(shape, dtype=dtype, device='cuda').normal_(0.0, std, generator=gen)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device='cuda')


def _pages(gen, lengths, page):
    """(page table, pages in all): every sequence's pages lie anywhere in the cache; places that nobody needs hold -1."""
    need = [(n + page - 1) // page for n in lengths]
    total, width = sum(need) + 5, max(1, max(need))
    order = torch.randperm(total, generator=gen, device='cuda').to(torch.int32)
    first, need = _ints([sum(need[:i]) for i in range(len(need))], torch.int64), _ints(need, torch.int64)
    at = torch.arange(width, device='cuda')
    return torch.where(at < need[:, None], order[(first[:, None] + at).clamp_max(total - 1)], -1), total


def _prepare_rope(c, gen):
    T, Hq, Hk, D, R = c['tokens'], c['heads'], c['kv_heads'], c['dim'], c['rotary']
    dtype, param = getattr(torch, c['dtype']), getattr(torch, c['param'])
    # queries, keys and values lie side by side, as the projection writes them
    qkv = _normal(gen, T, Hq + 2 * Hk, D)
    qkv *= 0.5 + torch.rand(T, Hq + 2 * Hk, 1, generator=gen, device='cuda')
    qkv = qkv.to(dtype)
    angles = torch.arange(c['positions'], dtype=torch.float64, device='cuda')[:, None] * 10000.0**(-torch.arange(0, R, 2, dtype=torch.float64, device='cuda') / R)
    s = dict(q=qkv[:, :Hq], k=qkv[:, Hq:Hq + Hk], v=qkv[:, Hq + Hk:], qw=(1.0 + _normal(gen, D, std=0.1)).to(param), kw=(1.0 + _normal(gen, D, std=0.1)).to(param),
             table=torch.cat([angles.cos(), angles.sin()], -1).float())
    if c['dir'] == 'append':
        total = (T + c['page'] - 1) // c['page'] + 3
        s['slots'] = torch.randperm(total * c['page'], generator=gen, device='cuda')[:T]
        s['positions'] = torch.randint(0, c['positions'], (T,), generator=gen, device='cuda')
        s['k_cache'] = _normal(gen, total, c['page'], Hk, D, dtype=dtype)
        s['v_cache'] = _normal(gen, total, c['page'], Hk, D, dtype=dtype)
    else:
        # a few sequences behind one another, the positions of each count from an offset
        s['positions'] = (torch.arange(T, device='cuda') + torch.randint(0, c['positions'], (1,), generator=gen, device='cuda')) % c['positions']
    if c['dir'] == 'bwd':
        s['dq'], s['dk'] = _normal(gen, T, Hq, D, dtype=dtype), _normal(gen, T, Hk, D, dtype=dtype)
    return s


def _prepare_prompt(c, gen):
    lq, lk = _prompt_lengths(c)
    Hq, Hk, D, bf16 = c['heads'], c['kv_heads'], c['dim'], torch.bfloat16
    # normed heads: scores of size one, a few keys that many queries look at
    q, k = _normal(gen, sum(lq), Hq, D), _normal(gen, sum(lk), Hk, D)
    k = torch.where(torch.rand(sum(lk), 1, 1, generator=gen, device='cuda') < 0.02, 2.5 * k, k)
    s = dict(q=q.to(bf16), k=k.to(bf16), v=_normal(gen, sum(lk), Hk, D, dtype=bf16), lq=lq, lk=lk, scale=D**-0.5,
             cu_q=_ints([0] + lq).cumsum(0).to(torch.int32), cu_k=_ints([0] + lk).cumsum(0).to(torch.int32))
    if c['dir'] == 'bwd':
        s['do'] = _normal(gen, sum(lq), Hq, D, dtype=bf16)
        s['o'], s['lse'] = _run_prompt(c, s).values()                # what a training step has kept
    return s


def _prepare_decode(c, gen):
    lengths, Hq, Hk, D = _decode_lengths(c), c['heads'], c['kv_heads'], c['dim']
    table, total = _pages(gen, lengths, c['page'])
    return dict(q=_normal(gen, c['seqs'], Hq, D, std=1.5).to(torch.bfloat16), k_cache=_normal(gen, total, c['page'], Hk, D, dtype=torch.bfloat16),
                v_cache=_normal(gen, total, c['page'], Hk, D, dtype=torch.bfloat16), table=table, lengths=_ints(lengths), host_lengths=lengths, scale=D**-0.5)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    return case, {'rope': _prepare_rope, 'prompt': _prepare_prompt, 'decode': _prepare_decode}[case['op']](case, gen)


# ------------------------------------------------------------------------------------------------------- the plain forms
def _pairs(c, x):
    """First and second channels of the rotated pairs."""
    R = c['rotary']
    return (x[..., 0:R:2], x[..., 1:R:2]) if c['interleaved'] else (x[..., :R // 2], x[..., R // 2:R])


def _rotate(c, s, x, back=False):
    cs = s['table'][s['positions']].unsqueeze(1)
    cos, sin = cs[..., :c['rotary'] // 2], cs[..., c['rotary'] // 2:]
    sin = -sin if back else sin
    a, b = _pairs(c, x)
    y = x.clone()
    for to, value in zip(_pairs(c, y), (a * cos - b * sin, b * cos + a * sin)):
        to.copy_(value)
    return y


def _rstd(x):
    return 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)


def _run_rope(c, s):
    q, k = (_rotate(c, s, x.float() * _rstd(x.float()) * w.float()).to(x.dtype) for x, w in ((s['q'], s['qw']), (s['k'], s['kw'])))
    if c['dir'] == 'fwd':
        return dict(q=q, k=k)
    page, place = s['slots'] // c['page'], s['slots'] % c['page']
    s['k_cache'][page, place] = k
    s['v_cache'][page, place] = s['v']
    return dict(q=q, k_cache=s['k_cache'], v_cache=s['v_cache'])


def _run_rope_grad(c, s):
    out = {}
    for name, x, w, dy in (('q', s['q'], s['qw'], s['dq']), ('k', s['k'], s['kw'], s['dk'])):
        v = x.float()
        rstd = _rstd(v)
        g, xh = _rotate(c, s, dy.float(), back=True), v * rstd
        u = g * w.float()
        out['d' + name] = (rstd * (u - xh * (u * xh).mean(-1, keepdim=True))).to(x.dtype)
        out['d' + name + 'w'] = (g * xh).sum((0, 1)).to(w.dtype)
    return out


def _blocks(lq, lk, causal, most=1 << 27):
    """Pieces that fit: sequence, its queries [q0, q1), its keys [k0, k1), and how many keys the piece's first query does not see at the end."""
    q0 = k0 = 0
    for nq, nk in zip(lq, lk):
        step = max(1, most // max(1, nk))
        for a in range(0, nq, step):
            b = min(a + step, nq)
            last = nk - nq + b if causal else nk
            yield q0 + a, q0 + b, k0, k0 + last, nk - nq + a
        q0, k0 = q0 + nq, k0 + nk


def _seen(nq, nk, first, causal):
    """[nq, nk]: query i of the piece sees the keys up to first + i."""
    if not causal:
        return torch.ones(nq, nk, dtype=torch.bool, device='cuda')
    return torch.arange(nk, device='cuda') <= first + torch.arange(nq, device='cuda')[:, None]


def _run_prompt(c, s):
    Hq, group = c['heads'], c['heads'] // c['kv_heads']
    o = torch.zeros(s['q'].shape, dtype=torch.bfloat16, device='cuda')
    lse = torch.empty(Hq, s['q'].shape[0], device='cuda')
    for h in range(Hq):
        q, k, v = s['q'][:, h].float(), s['k'][:, h // group].float(), s['v'][:, h // group].float()
        for q0, q1, k0, k1, first in _blocks(s['lq'], s['lk'], c['causal']):
            x = (q[q0:q1] @ k[k0:k1].t()) * s['scale']
            x = torch.where(_seen(q1 - q0, k1 - k0, first, c['causal']), x, -math.inf)
            top = x.max(-1, keepdim=True).values
            x = torch.exp(x - top)
            total = x.sum(-1, keepdim=True)
            o[q0:q1, h] = ((x @ v[k0:k1]) / total).to(torch.bfloat16)
            lse[h, q0:q1] = (top + torch.log(total)).squeeze(-1)
    return dict(o=o, lse=lse)


def _run_prompt_grad(c, s):
    Hq, Hk = c['heads'], c['kv_heads']
    group = Hq // Hk
    dq = torch.zeros(s['q'].shape, dtype=torch.bfloat16, device='cuda')
    dk, dv = (torch.zeros(s['k'].shape, dtype=torch.bfloat16, device='cuda') for _ in range(2))
    for kh in range(Hk):
        k, v = s['k'][:, kh].float(), s['v'][:, kh].float()
        sum_k, sum_v = torch.zeros_like(k), torch.zeros_like(v)
        for h in range(kh * group, (kh + 1) * group):
            q, do, lse = s['q'][:, h].float(), s['do'][:, h].float(), s['lse'][h]
            delta = (do * s['o'][:, h].float()).sum(-1, keepdim=True)
            for q0, q1, k0, k1, first in _blocks(s['lq'], s['lk'], c['causal']):
                x = (q[q0:q1] @ k[k0:k1].t()) * s['scale']
                p = torch.where(_seen(q1 - q0, k1 - k0, first, c['causal']), torch.exp(x - lse[q0:q1, None]), 0.0)
                sum_v[k0:k1] += p.t() @ do[q0:q1]
                ds = p * (do[q0:q1] @ v[k0:k1].t() - delta[q0:q1]) * s['scale']
                dq[q0:q1, h] = (ds @ k[k0:k1]).to(torch.bfloat16)
                sum_k[k0:k1] += ds.t() @ q[q0:q1]
        dk[:, kh], dv[:, kh] = sum_k.to(torch.bfloat16), sum_v.to(torch.bfloat16)
    return dict(dq=dq, dk=dk, dv=dv)


def _run_decode(c, s):
    Hk, D, group = c['kv_heads'], c['dim'], c['heads'] // c['kv_heads']
    out = torch.empty_like(s['q'])
    for b, n in enumerate(s['host_lengths']):
        page = s['table'][b, :(n + c['page'] - 1) // c['page']].long()
        k, v = (cache[page].reshape(-1, Hk, D)[:n].float().transpose(0, 1) for cache in (s['k_cache'], s['v_cache']))
        x = (s['q'][b].float().view(Hk, group, D) @ k.transpose(1, 2)) * s['scale']
        x = torch.exp(x - x.max(-1, keepdim=True).values)
        out[b] = ((x @ v) / x.sum(-1, keepdim=True)).reshape(c['heads'], D).to(out.dtype)
    return out


def run(state):
    c, s = state
    if own:
        return _run_own(c, s)
    if c['op'] == 'decode':
        return _run_decode(c, s)
    if c['op'] == 'prompt':
        return _run_prompt(c, s) if c['dir'] == 'fwd' else _run_prompt_grad(c, s)
    return _run_rope_grad(c, s) if c['dir'] == 'bwd' else _run_rope(c, s)


# ------------------------------------------------------------------------------------------------------ this library's calls
def _run_own(c, s):
    if c['op'] == 'rope':
        from deepep_ascend_b200.ops.rotary import qk_norm_rope, qk_norm_rope_append, qk_norm_rope_backward
        given, options = (s['qw'], s['kw'], s['table'], s['positions']), dict(eps=EPS, interleaved=c['interleaved'])
        if c['dir'] == 'fwd':
            q, k = qk_norm_rope(s['q'], s['k'], *given, **options)
            return dict(q=q, k=k)
        if c['dir'] == 'append':
            q = qk_norm_rope_append(s['q'], s['k'], s['v'], *given, s['k_cache'], s['v_cache'], s['slots'], **options)
            return dict(q=q, k_cache=s['k_cache'], v_cache=s['v_cache'])
        dq, dk, dqw, dkw = qk_norm_rope_backward(s['dq'], s['dk'], s['q'], s['k'], *given, **options)
        return dict(dq=dq, dqw=dqw, dk=dk, dkw=dkw)
    from deepep_ascend_b200.ops.attention import attention, attention_backward, paged_attention
    if c['op'] == 'decode':
        return paged_attention(s['q'], s['k_cache'], s['v_cache'], s['table'], s['lengths'], scale=s['scale'])
    options = dict(cu_seqlens=s['cu_q'], cu_seqlens_k=s['cu_k'], causal=c['causal'], scale=s['scale'])
    if c['dir'] == 'fwd':
        o, lse = attention(s['q'], s['k'], s['v'], **options)
        return dict(o=o, lse=lse)
    dq, dk, dv = attention_backward(s['do'], s['q'], s['k'], s['v'], s['o'], s['lse'], **options)
    return dict(dq=dq, dk=dk, dv=dv)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    Hq, Hk, D = c['heads'], c['kv_heads'], c['dim']
    if c['op'] == 'rope':
        T, size = c['tokens'], {'float32': 4, 'bfloat16': 2}[c['dtype']]
        rows = dict(fwd=2 * (Hq + Hk), append=2 * (Hq + 2 * Hk), bwd=3 * (Hq + Hk))[c['dir']]
        # (every token has a row of the table of its own)
        small = T * (4 * c['rotary'] + (16 if c['dir'] == 'append' else 8)) + 2 * D * {'float32': 4, 'bfloat16': 2}[c['param']] * (2 if c['dir'] == 'bwd' else 1)
        return dict(bytes=rows * T * D * size + small, flops=(16 if c['dir'] == 'bwd' else 8) * T * (Hq + Hk) * D)
    if c['op'] == 'decode':
        lengths = _decode_lengths(c)
        keys, places = sum(lengths), sum((n + c['page'] - 1) // c['page'] for n in lengths)
        return dict(bytes=4 * keys * Hk * D + 4 * c['seqs'] * Hq * D + 4 * places + 4 * c['seqs'], flops=4 * keys * Hq * D)
    lq, lk = _prompt_lengths(c)
    seen = sum(a * (b - a) + a * (a + 1) // 2 if c['causal'] else a * b for a, b in zip(lq, lk))
    queries, keys, statistics = sum(lq) * Hq * D * 2, sum(lk) * Hk * D * 2, 4 * sum(lq) * Hq
    if c['dir'] == 'fwd':
        return dict(bytes=2 * queries + 2 * keys + statistics, flops=4 * seen * Hq * D)
    return dict(bytes=4 * queries + 4 * keys + statistics, flops=10 * seen * Hq * D)


# ----------------------------------------------------------------------------------------------------------------- exact
def _exact_heads(c, s, x, w):
    """Norm and rotation of heads by complex numbers."""
    R = c['rotary']
    y = torch.nn.functional.rms_norm(x, (c['dim'],), w, EPS)
    angle = torch.complex(*(s['table'][s['positions']].double()[:, None, a:a + R // 2] for a in (0, R // 2)))
    turned = y[..., :R]
    pairs = turned.unflatten(-1, (R // 2, 2)) if c['interleaved'] else turned.unflatten(-1, (2, R // 2)).transpose(-1, -2)
    pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * angle)
    return torch.cat([(pairs if c['interleaved'] else pairs.transpose(-1, -2)).flatten(-2), y[..., R:]], -1)


def _exact_rope(c, s):
    leaves = [t.double().requires_grad_(c['dir'] == 'bwd') for t in (s['q'], s['qw'], s['k'], s['kw'])]
    with torch.enable_grad():
        q, k = _exact_heads(c, s, *leaves[:2]), _exact_heads(c, s, *leaves[2:])
        if c['dir'] == 'bwd':
            return dict(zip(('dq', 'dqw', 'dk', 'dkw'), torch.autograd.grad((q, k), leaves, (s['dq'].double(), s['dk'].double()))))
    if c['dir'] == 'fwd':
        return dict(q=q, k=k)
    caches = s['k_cache'].double(), s['v_cache'].double()
    for cache, new in zip(caches, (k, s['v'].double())):
        cache.view(-1, c['kv_heads'], c['dim'])[s['slots']] = new
    return dict(q=q, k_cache=caches[0], v_cache=caches[1])


def _exact_prompt(c, s):
    """Head by head, in pieces of queries; gradients by the rules of a softmax's derivative, from queries, keys and values alone."""
    group, back = c['heads'] // c['kv_heads'], c['dir'] == 'bwd'
    o, lse = torch.empty(s['q'].shape, dtype=torch.float64, device='cuda'), torch.empty(c['heads'], s['q'].shape[0], dtype=torch.float64, device='cuda')
    dq, dk, dv = (torch.zeros(s[n].shape, dtype=torch.float64, device='cuda') for n in ('q', 'k', 'v'))
    for h in range(c['heads']):
        q, k, v = s['q'][:, h].double(), s['k'][:, h // group].double(), s['v'][:, h // group].double()
        for q0, q1, k0, k1, first in _blocks(s['lq'], s['lk'], c['causal'], 1 << 26):
            x = torch.einsum('id,jd->ij', q[q0:q1] * s['scale'], k[k0:k1])
            x.masked_fill_(~_seen(q1 - q0, k1 - k0, first, c['causal']), -math.inf)
            lse[h, q0:q1] = torch.logsumexp(x, -1)
            p = torch.softmax(x, -1)
            o[q0:q1, h] = p @ v[k0:k1]
            if back:
                do = s['do'][q0:q1, h].double()
                dv[k0:k1, h // group] += torch.einsum('ij,id->jd', p, do)
                dp = torch.einsum('id,jd->ij', do, v[k0:k1])
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * s['scale']
                dq[q0:q1, h] = torch.einsum('ij,jd->id', ds, k[k0:k1])
                dk[k0:k1, h // group] += torch.einsum('ij,id->jd', ds, q[q0:q1])
    return dict(dq=dq, dk=dk, dv=dv) if back else dict(o=o, lse=lse)


def _exact_decode(c, s):
    out, group = torch.empty(s['q'].shape, dtype=torch.float64, device='cuda'), c['heads'] // c['kv_heads']
    for b, n in enumerate(s['host_lengths']):
        at = torch.arange(n, device='cuda')
        page, place = s['table'][b].long()[at // c['page']], at % c['page']
        for h in range(c['kv_heads']):
            k, v = s['k_cache'][page, place, h].double(), s['v_cache'][page, place, h].double()
            p = torch.softmax(s['q'][b, h * group:(h + 1) * group].double() @ k.t() * s['scale'], -1)
            out[b, h * group:(h + 1) * group] = p @ v
    return out


def exact(case, seed):
    c, s = prepare(case, seed)
    return {'rope': _exact_rope, 'prompt': _exact_prompt, 'decode': _exact_decode}[c['op']](c, s)
