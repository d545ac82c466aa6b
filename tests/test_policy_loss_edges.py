"""Clipped policy loss where it is easiest to get wrong.  Helpers and tolerances
are those of test_policy_loss.py."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from handyrl_amd import ops
from handyrl_amd.losses import clipped_policy_loss
from test_policy_loss import COEFS, make

gpu = pytest.mark.gpu


@pytest.mark.skipif(not ops.available(), reason='extension not built')
def test_extension_refuses_forward_mode():
    """The refusal comes before the extension looks at the device."""
    args = make((5,), 4)
    with fwd.dual_level():
        args['logits'] = fwd.make_dual(args['logits'], torch.ones_like(args['logits']))
        with pytest.raises(ValueError, match='forward-mode'):
            ops.require().clipped_policy_loss(*args.values(), 0.2, 0.2, 0.0, 0.0)


def test_eager_forward_mode():
    """Along a gradient the derivative is its square."""
    args = {k: v.double() if v.is_floating_point() else v for k, v in make((5,), 4).items()}
    z = args.pop('logits').requires_grad_()
    grad, = torch.autograd.grad(clipped_policy_loss(z, **args, **COEFS)[0], z)
    with fwd.dual_level():
        loss, _ = clipped_policy_loss(fwd.make_dual(z.detach(), grad), **args, **COEFS)
        got = fwd.unpack_dual(loss).tangent
    torch.testing.assert_close(got, grad.square().sum(), rtol=1e-10, atol=1e-10)


@gpu
@pytest.mark.parametrize('name', ['logits', 'old_log_probs', 'advantages', 'mask', 'entropy_scale'])
def test_kernel_refuses_forward_mode(name):
    args = make((5,), 4, device='cuda')
    with fwd.dual_level():
        args[name] = fwd.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(ValueError, match='forward-mode'):
            clipped_policy_loss(**args, **COEFS)


@gpu
def test_captured_backward_beside_an_eager_graph():
    """Refused while the eager graph of the same leaf lives, and right once it is gone."""
    args = make((64,), 9, device='cuda')
    leaf = args['logits'].requires_grad_()
    kept = clipped_policy_loss(**args, **COEFS)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = clipped_policy_loss(**args, **COEFS)
        with pytest.raises(RuntimeError, match='living eager graph'):
            torch.autograd.grad(out[0], leaf)
    want, = torch.autograd.grad(kept[0], leaf)
    del kept, out, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(clipped_policy_loss(**args, **COEFS)[0], leaf)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
