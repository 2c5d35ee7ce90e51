"""The attention block: norm, products, rotation and attention together, packed, over a cache, and in front of the experts."""
import pytest
import torch

from deepep_ascend_b200.models.attention import AttentionBlock, positions_of, slots_of

BF16, HALF = torch.bfloat16, 2.0**-8


def _cu(lengths, device='cpu'):
    return torch.tensor([0] + list(lengths)).cumsum(0).int().to(device)


def test_positions():
    assert positions_of(None, 4).tolist() == [0, 1, 2, 3]
    assert positions_of(_cu([2, 0, 3]), 7).tolist() == [0, 1, 0, 1, 2, -1, -1]
    assert positions_of(_cu([]), 2).tolist() == [-1, -1]


def test_slots():
    table = torch.tensor([[5, 2], [-1, 3], [0, -1]], dtype=torch.int32)
    assert slots_of(table, torch.tensor([0, 17, 15]), 16).tolist() == [80, 49, 15]
    assert slots_of(table, torch.tensor([-1, 3, 32]), 16).tolist() == [-1, -1, -1]


def test_a_table_without_pages():
    """Has a slot for nobody; nothing is looked up in it."""
    assert slots_of(torch.empty(2, 0, dtype=torch.int32), torch.tensor([0, -1]), 16).tolist() == [-1, -1]


def test_sizes_that_do_not_fit():
    for bad in (dict(hidden=100), dict(head_dim=136), dict(head_dim=60), dict(num_heads=5), dict(rotary_dim=24), dict(rotary_dim=80)):
        with pytest.raises(ValueError):
            AttentionBlock(**{**dict(hidden=64, num_heads=4, num_kv_heads=2, head_dim=64, device='cpu'), **bad})


def _block(seed=0, **options):
    torch.manual_seed(seed)
    block = AttentionBlock(**{**dict(hidden=256, num_heads=4, num_kv_heads=2, head_dim=64, rotary_dim=32, max_positions=2048, init_std=0.06), **options})
    with torch.no_grad():
        for p in (block.norm_weight, block.q_weight, block.k_weight):
            p.add_(0.2 * torch.randn_like(p))
    return block


def _reference(p, block, x, lengths):
    """With plain operations in 32 bits, sequence by sequence."""
    H, Hk, D = block.num_heads, block.num_kv_heads, block.head_dim
    h = torch.nn.functional.layer_norm(x, x.shape[1:], p['norm_weight'], None, block.eps)
    q, k, v = (h @ p['qkv'].t()).view(-1, H + 2 * Hk, D).split((H, Hk, Hk), 1)
    out, a = [], 0
    half = block.table.shape[1] // 2
    for n in lengths:
        def turned(t, w):
            t = t[a:a + n]
            t = t * (t.square().mean(-1, keepdim=True) + block.eps).rsqrt() * w
            cos, sin = (block.table[:n, None, i * half:(i + 1) * half] for i in range(2))
            u, z = t[..., :half], t[..., half:2 * half]
            return torch.cat([u * cos - z * sin, z * cos + u * sin, t[..., 2 * half:]], -1)
        y, z = turned(q, p['q_weight']), turned(k, p['k_weight']).repeat_interleave(H // Hk, 1)
        s = torch.einsum('ihd,jhd->hij', y, z) * D**-0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -torch.inf)
        out.append(torch.einsum('hij,jhd->ihd', torch.softmax(s, -1), v[a:a + n].repeat_interleave(H // Hk, 1)).reshape(n, H * D))
        a += n
    o = torch.cat(out + [x.new_zeros(x.shape[0] - a, H * D)])
    return x + o @ p['out'].t()


@pytest.mark.gpu
@pytest.mark.parametrize('lengths,pad', [([200], 0), ([70, 0, 1, 130], 11)])
def test_forward_and_gradients(lengths, pad):
    from deepep_ascend_b200.utils.math import calc_diff
    block = _block()
    T = sum(lengths) + pad
    x = torch.randn(T, 256, device='cuda').bfloat16().requires_grad_(True)
    g = torch.randn(T, 256, device='cuda').bfloat16()
    out = block(x, _cu(lengths, 'cuda'))
    out.backward(g)
    if pad:
        assert torch.equal(out[-pad:], x[-pad:]) and torch.equal(x.grad[-pad:], g[-pad:])
    ref = {n: p.detach().float().requires_grad_(True) for n, p in block.named_parameters()}
    y = x.detach().float().requires_grad_(True)
    want = _reference(ref, block, y, lengths)
    want.backward(g.float())
    # five roundings to bf16 on the way there, seven on the way back, each 2^-9 of its values' size as a root of squares; calc_diff is half the square of a relative error:
    # below (7 x 2^-9)^2, 1.9e-4, were they all to add up
    pairs = dict(result=(out, want), x=(x.grad, y.grad), **{n: (p.grad, ref[n].grad) for n, p in block.named_parameters()})
    diffs = {n: calc_diff(a.detach().float(), b.detach()) for n, (a, b) in pairs.items()}
    assert all(v < 2e-4 for v in diffs.values()), diffs


@pytest.mark.gpu
@pytest.mark.parametrize('page_size', [16, 24])
def test_prompts_and_tokens_behind_them(page_size):
    """A prompt through the cache and tokens one by one give what the whole sequences give at once."""
    block = _block(1)
    prompts, new = [37, 5, 64], 6
    xs = [torch.randn(n + new, 256, device='cuda').bfloat16() for n in prompts]
    want = [block(x) for x in xs]
    pages = [(n + new + page_size - 1) // page_size for n in prompts]
    cache = block.new_cache(sum(pages) + 2, page_size)
    cache[0].fill_(float('nan')), cache[1].fill_(float('nan'))          # (what nobody has written is not looked at)
    order, table, a = torch.randperm(sum(pages) + 2), torch.full((4, max(pages)), -1, dtype=torch.int32), 0
    for i, n in enumerate(pages):
        table[i, :n] = order[a:a + n]
        a += n
    table = table.cuda()
    cu = _cu(prompts, 'cuda')
    positions = positions_of(cu, sum(prompts))
    slots = torch.cat([slots_of(table[i:i + 1].expand(n, -1), torch.arange(n, device='cuda'), page_size) for i, n in enumerate(prompts)])
    x = torch.cat([t[:n] for t, n in zip(xs, prompts)])
    y = block.prefill(x, cache, slots, cu, positions)
    assert torch.equal(y, block(x, cu).detach())
    # the fourth sequence takes no part
    lengths = torch.tensor([n + 1 for n in prompts] + [-1], dtype=torch.int32, device='cuda')
    token = torch.zeros(4, 256, device='cuda', dtype=BF16)
    step = lambda: block.decode(token, cache, table, lengths)      # noqa: E731
    step()                                                         # (places that are written again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for j in range(new):
        lengths.copy_(torch.tensor([n + j + 1 for n in prompts] + [0], dtype=torch.int32))
        token.copy_(torch.stack([t[n + j] for t, n in zip(xs, prompts)] + [xs[0][0]]))
        graph.replay()
        assert torch.equal(out[3], token[3])
        for i, n in enumerate(prompts):
            # (probabilities, heads and products rounded apart: a few halves of bf16 of the values' size)
            assert float((out[i].float() - want[i][n + j].detach().float()).abs().max()) <= 8 * HALF * float(want[i][n + j].abs().max())


@pytest.mark.gpu
def test_no_tokens():
    block = _block(3)
    x = torch.zeros(0, 256, dtype=BF16, device='cuda', requires_grad=True)
    y = block(x, _cu([0, 0], 'cuda'))
    y.sum().backward()
    assert y.shape == x.shape == x.grad.shape
    cache, none = block.new_cache(2, 16), torch.zeros(0, dtype=torch.int32, device='cuda')
    assert block.prefill(x.detach(), cache, none).shape == x.shape and block.decode(x.detach(), cache, none.view(0, 1), none).shape == x.shape


@pytest.mark.gpu
def test_a_cache_without_pages():
    """A prompt is what it is without a cache; a single token, which has no place for its key, gets no numbers, and one of no sequence comes back."""
    block = _block(4)
    x = torch.randn(20, 256, device='cuda').bfloat16()
    cache = block.new_cache(0, 16)
    assert torch.equal(block.prefill(x, cache, torch.arange(20, device='cuda')), block(x).detach())
    y = block.decode(x[:2], cache, torch.zeros(2, 1, dtype=torch.int32, device='cuda'), torch.tensor([1, 0], dtype=torch.int32, device='cuda'))
    assert y[0].isnan().all() and torch.equal(y[1], x[1])


@pytest.mark.gpu
def test_a_layer_runs(capsys):
    from deepep_ascend_b200.models import attention
    attention.main(steps=3, new_tokens=3)
    lines = capsys.readouterr().out.splitlines()
    assert all(float(line.split()[3]) > 0 for line in lines[:-1]) and lines[-1].startswith('3 tokens behind a prompt')


@pytest.mark.gpu
def test_gradients_reach_every_parameter_of_a_layer():
    from deepep_ascend_b200 import ElasticBuffer
    from deepep_ascend_b200.models.block import MoEBlock
    T, H = 200, 256
    buf = ElasticBuffer(None, num_max_tokens_per_rank=T, hidden=H, num_topk=2)
    try:
        mixer, experts = _block(2, buffer=buf), MoEBlock(buf, 8, H, 128, 2)
        x = torch.randn(T, H, device='cuda').bfloat16().requires_grad_(True)
        experts(mixer(x, _cu([90, 110], 'cuda'))).float().square().mean().backward()
        torch.cuda.synchronize()
        buf.check_status()
        for name, p in [('x', x), *mixer.named_parameters(), *experts.named_parameters()]:
            assert p.grad is not None and p.grad.isfinite().all() and p.grad.any(), name
    finally:
        buf.destroy()
