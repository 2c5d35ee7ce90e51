"""Optimiser for the matrices of the library's layers: Muon, whose update is the orthogonalised momentum (``ops.muon``).

An expert's matrices live whole on one rank, so the update of a stack of experts needs no communication; replicated matrices (a gate) get the
same update on every rank from gradients that the caller has averaged.  No counterpart in the reference.
"""
import torch

from .ops.muon import COEFFICIENTS, orthogonalize


class Muon(torch.optim.Optimizer):
    """``momentum = beta * momentum + grad``; ``update = orthogonalize(grad + beta * momentum)`` (``nesterov``; otherwise of the momentum);
    ``p = p * (1 - lr * weight_decay) - lr * sqrt(max(1, rows / cols)) * update``.

    Parameters are matrices or stacks of them (``[experts, rows, cols]``: every expert's matrix by itself).  The momentum is fp32, and so is a copy of
    16-bit parameters (``state[p]['weight']``, 4 bytes per element) that steps are added to, since most of an update is below the last place of a bf16 weight: ``p``
    is that copy, rounded.  Where a weight has been set by others since, its value counts.  ``buffer``: see :func:`ops.gemm.gemm_nt`."""

    buffer = None

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5,
                 coefficients=COEFFICIENTS, eps: float = 1e-7, buffer=None):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps, coefficients=coefficients, eps=eps))
        self.buffer = buffer
        for group in self.param_groups:
            for p in group['params']:
                if p.dim() < 2:
                    raise ValueError('Muon updates matrices, got a parameter of shape %s' % (tuple(p.shape),))

    def load_state_dict(self, state_dict) -> None:
        """As the base class's, which casts a state to its parameter's type; what is kept in fp32 is taken as it was saved."""
        given = {}

        def restore(_):
            ids = (i for group in given['param_groups'] for i in group['params'])
            for p, i in zip((p for group in self.param_groups for p in group['params']), ids):
                saved = given['state'].get(i, {})
                for name in saved.keys() & {'momentum', 'weight'}:
                    self.state[p][name] = saved[name].to(p.device, torch.float32, copy=True)
        # (behind the caller's hooks, which may give another dict, and ahead of those that look at what was loaded)
        hooks = (self.register_load_state_dict_pre_hook(lambda _, loaded: given.update(loaded)),
                 self.register_load_state_dict_post_hook(restore, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group['params']:
                if p.grad is None or p.numel() == 0:
                    continue
                state = self.state[p]
                if 'momentum' not in state:
                    state['momentum'] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                m, grad = state['momentum'], p.grad.float()
                m.mul_(group['momentum']).add_(grad)
                update = orthogonalize(torch.add(grad, m, alpha=group['momentum']) if group['nesterov'] else m, group['steps'], group['coefficients'], group['eps'],
                                       buffer=self.buffer)
                w = self._weight(p, state)
                if group['weight_decay']:
                    w.mul_(1.0 - group['lr'] * group['weight_decay'])
                w.add_(update, alpha=-group['lr'] * max(1.0, p.shape[-2] / p.shape[-1])**0.5)
                if w is not p:
                    p.copy_(w)
        return loss

    @staticmethod
    def _weight(p, state):
        """What a step is added to: ``p``, or the fp32 copy of a 16-bit one."""
        if p.dtype.itemsize > 2:
            return p
        w = state.get('weight')
        if w is None:
            w = state['weight'] = p.to(torch.float32, copy=True)
        else:
            w.copy_(torch.where(w.to(p.dtype) == p, w, p))
        return w
