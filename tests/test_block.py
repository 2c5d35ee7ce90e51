"""The block that runs the norm, the router, the experts and the orthogonalised update together, and the optimiser by itself."""
import pytest
import torch

from deepep_ascend_b200.ops.muon import orthogonalize
from deepep_ascend_b200.optim import Muon


def _reference(block, x, idx, w13, w2):
    """The block with plain fp32 operations, the experts chosen as the block chose them."""
    from deepep_ascend_b200.models.moe import moe_reference
    h = torch.nn.functional.layer_norm(x, x.shape[1:], block['norm_weight'], block['norm_bias'], 1e-5)
    p = torch.sigmoid(h @ block['gate'].t())
    w = p.gather(1, idx.clamp_min(0)) * (idx >= 0)
    w = 2.0 * w / w.sum(-1, keepdim=True).clamp_min(1e-20)
    return x + moe_reference(h, idx, w, w13, w2)


@pytest.mark.gpu
@pytest.mark.parametrize('T,fp8_backward', [(200, False), (512, True), (64, False)])
def test_forward_and_gradients(T, fp8_backward):
    from deepep_ascend_b200 import ElasticBuffer
    from deepep_ascend_b200.models.block import MoEBlock
    from deepep_ascend_b200.utils.math import calc_diff
    torch.manual_seed(0)
    H, I, E, K = 256, 128, 16, 3
    buf = ElasticBuffer(None, num_max_tokens_per_rank=T, hidden=H, num_topk=K)
    try:
        block = MoEBlock(buf, E, H, I, K, num_groups=4, num_topk_groups=2, scale=2.0, norm_bias=True, init_std=0.05, fp8_backward=fp8_backward)
        with torch.no_grad():
            block.norm_weight.add_(0.1 * torch.randn(H, device='cuda'))
            block.norm_bias.add_(0.1 * torch.randn(H, device='cuda'))
            block.balance_bias.add_(0.02 * torch.randn(E, device='cuda'))
        x = torch.randn(T, H, device='cuda').bfloat16().requires_grad_(True)
        mask = torch.arange(T, device='cuda') % 11 != 3
        chosen = {}
        hook = block.experts.register_forward_pre_hook(lambda m, args: chosen.update(idx=args[1]))
        out = block(x, mask)
        hook.remove()
        g = torch.randn_like(out)
        out.backward(g)
        torch.cuda.synchronize()
        buf.check_status()
        idx = chosen['idx']
        assert (idx[~mask] == -1).all() and torch.equal(out[~mask], x[~mask])
        assert torch.equal(block.last_count, torch.bincount(idx.flatten() + 1, minlength=E + 1)[1:].int())

        names = ('norm_weight', 'norm_bias', 'gate')
        ref = {n: getattr(block, n).detach().float().requires_grad_(True) for n in names}
        xr = x.detach().float().requires_grad_(True)
        w13, w2 = block.experts.w13.detach().float().requires_grad_(True), block.experts.w2.detach().float().requires_grad_(True)
        want = _reference(ref, xr, idx, w13, w2)
        want.backward(g.float())
        # the bounds of the layer's own tests: its e4m3 products are what differs
        pairs = dict(out=(out, want), x=(x.grad, xr.grad), w13=(block.experts.w13.grad, w13.grad), w2=(block.experts.w2.grad, w2.grad),
                     **{n: (getattr(block, n).grad, ref[n].grad) for n in names})
        diffs = {n: calc_diff(a.float(), b) for n, (a, b) in pairs.items()}
        assert all(v < 5e-3 for v in diffs.values()), diffs
        # the load moves the bias the other way
        before = block.balance_bias.clone()
        block.update_balance(0.5)
        count = block.last_count.float()
        assert torch.equal(torch.sign(block.balance_bias - before), torch.sign(count.mean() - count))
    finally:
        buf.destroy()


@pytest.mark.gpu
def test_training_lowers_the_loss(capsys):
    from deepep_ascend_b200.models import block
    block.main(steps=31)
    losses = [float(line.split()[3]) for line in capsys.readouterr().out.splitlines()]
    assert losses[-1] < 0.7 * losses[0], losses


def _by_hand(p, grads, lr, beta, nesterov, decay):
    m = torch.zeros_like(p)
    for g in grads:
        m = beta * m + g
        update = orthogonalize(g + beta * m if nesterov else m).float()
        p = p * (1 - lr * decay) - lr * max(1.0, p.shape[-2] / p.shape[-1])**0.5 * update
    return p


@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('shape', [(24, 40), (3, 48, 16)])
@pytest.mark.parametrize('nesterov,decay', [(True, 0.0), (False, 0.1)])
def test_optimizer(shape, nesterov, decay, device):
    g = torch.Generator().manual_seed(0)
    start, grads = torch.randn(shape, generator=g).to(device), [torch.randn(shape, generator=g).to(device) for _ in range(3)]
    p = torch.nn.Parameter(start.clone())
    unused = torch.nn.Parameter(torch.ones(4, 4, device=device))
    opt = Muon([p, unused], lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=decay)
    for grad in grads:
        p.grad = grad.clone()
        opt.step()
    # the same products in another order of a few fp32 operations: bf16 updates may differ by their rounding
    torch.testing.assert_close(p.detach(), _by_hand(start, grads, 0.1, 0.9, nesterov, decay), rtol=0, atol=3 * 0.1 * 2**-7)
    assert torch.equal(unused, torch.ones_like(unused)) and opt.state[p]['momentum'].dtype == torch.float32
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.ones(4))])


@pytest.mark.gpu
def test_refusals():
    from deepep_ascend_b200 import ElasticBuffer
    from deepep_ascend_b200.models.block import MoEBlock
    buf = ElasticBuffer(None, num_max_tokens_per_rank=16, hidden=256, num_topk=2)
    try:
        with pytest.raises(ValueError):
            MoEBlock(buf, 12, 256, 128, 2)
    finally:
        buf.destroy()


@pytest.mark.gpu
def test_what_is_kept_of_a_batch_is_its_counts():
    """`last_count` outlives the batch; its ids and weights do not, and a forward pass gives the block's own choice."""
    from deepep_ascend_b200 import ElasticBuffer
    from deepep_ascend_b200.models.block import MoEBlock
    from deepep_ascend_b200.ops import gemm
    from deepep_ascend_b200.ops.norm import layer_norm
    from deepep_ascend_b200.ops.router import route_ref
    torch.manual_seed(0)
    T, H, E, K = 300, 256, 16, 3
    buf = ElasticBuffer(None, num_max_tokens_per_rank=T, hidden=H, num_topk=K)
    try:
        for options in (dict(num_groups=4, num_topk_groups=2, scale=2.0), dict(score='softmax', num_groups=8, num_topk_groups=3, group_top=1, renormalize=False)):
            block = MoEBlock(buf, E, H, 128, K, norm_bias=True, **options)
            block.balance_bias.copy_(0.3 * torch.randn(E, device='cuda'))
            x, mask = torch.randn(T, H, device='cuda').bfloat16(), torch.arange(T, device='cuda') % 11 != 3
            chosen = {}
            hook = block.experts.register_forward_pre_hook(lambda m, args: chosen.update(idx=args[1], weights=args[2]))
            block(x, mask).float().sum().backward()
            hook.remove()
            with torch.no_grad():
                logits = gemm.gemm_nt(layer_norm(x, block.norm_weight, block.norm_bias, block.eps)[0], block.gate, buffer=buf)
            idx, weights, count = route_ref(logits, K, bias=block.balance_bias, token_mask=mask, **options)
            plain = route_ref(logits, K, **options)[0]
            assert torch.equal(chosen['idx'], idx) and torch.equal(block.last_count, count) and not torch.equal(plain, idx)
            # (a sum of three weights and a few operations in another order)
            torch.testing.assert_close(chosen['weights'].detach(), weights, rtol=1e-5, atol=1e-6)
            assert block.last_count.untyped_storage().nbytes() == 4 * E
            assert block.norm_weight.grad.untyped_storage().data_ptr() != block.norm_bias.grad.untyped_storage().data_ptr()
        buf.check_status()
    finally:
        buf.destroy()
