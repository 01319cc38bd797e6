"""Calls of the packed-batch operators that need no GPU to be wrong: derivatives that they do not have, on fake tensors."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode

import pytorch_scatter_b200 as ts


def cuda(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device='cuda')


def calls():
    """name -> (function of one differentiable input, that input)"""
    slot, p = cuda(6, 2, dtype=torch.long), cuda(4, dtype=torch.long)
    x, many, weight, state = cuda(6, 8), cuda(12, 8), cuda(6, 2), cuda(3, 8)
    return {
        'topk': (lambda a: ts.expert_topk(a, 2)[0], x),
        'topk, all experts': (lambda a: ts.expert_topk(a, 2, False)[0], x),
        'dispatch': (lambda a: ts.expert_dispatch(a, slot, p), x),
        'dispatch weights': (lambda a: ts.expert_dispatch(x, slot, p, a), weight),
        'combine': (lambda a: ts.expert_combine(a, slot, p), many),
        'combine weights': (lambda a: ts.expert_combine(many, slot, p, a), weight),
        'scan': (lambda a: ts.scan_csr(a, x, p), x),
        'scan gate': (lambda a: ts.scan_csr(x, a, p), x),
        'scan shared gate': (lambda a: ts.scan_csr(x, a, p), cuda(6, 1)),
        'scan constant gate': (lambda a: ts.scan_csr(x, a, p), cuda(1, 8)),
        'scan state': (lambda a: ts.scan_csr_state(x, x, p, a)[1], state),
        'step': (lambda a: ts.scan_step(a, x, cuda(6, 8)), x),
        'step gate': (lambda a: ts.scan_step(x, a, cuda(6, 8)), cuda(6, 1)),
        'step state': (lambda a: ts.scan_step(x, x, a), cuda(6, 8)),
    }


with FakeTensorMode():
    NAMES = sorted(calls())


@pytest.mark.parametrize('grad', [True, False])
@pytest.mark.parametrize('name', NAMES)
def test_forward_mode_raises(name, grad):
    """An input with a tangent and no requires_grad: an error, not an output without a tangent."""
    with FakeTensorMode(), fwd.dual_level(), torch.set_grad_enabled(grad):
        f, a = calls()[name]
        with pytest.raises(RuntimeError, match='jvp|forward-mode'):
            f(fwd.make_dual(a, torch.ones_like(a)))


@pytest.mark.parametrize('transform', ['jvp', 'jacfwd', 'jvp of vmap'])
@pytest.mark.parametrize('name', NAMES)
def test_forward_transforms_raise(name, transform):
    with FakeTensorMode():
        f, a = calls()[name]
        with pytest.raises(RuntimeError):
            if transform == 'jvp':
                torch.func.jvp(f, (a,), (torch.ones_like(a),))
            elif transform == 'jacfwd':
                torch.func.jacfwd(f)(a)
            else:
                two = torch.stack([a, a])
                torch.func.jvp(torch.vmap(f), (two,), (torch.ones_like(two),))


def test_calls_without_a_tangent_still_run():
    with FakeTensorMode():
        for f, a in calls().values():
            f(a)
            with fwd.dual_level():
                f(a)
