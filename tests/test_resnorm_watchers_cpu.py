"""What follows a computation by watching it is refused before anything is launched: the kernels' outputs would look like constants to it."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from semseg_amd import _lib
from semseg_amd.resnorm import gated_residual_norm


@pytest.fixture(params=['native', 'python'])
def node(request):
    """the C++ node, and the Python one that traced calls take"""
    old = _lib.TRACE
    _lib.TRACE = [] if request.param == 'python' else None
    yield request.param
    _lib.TRACE = old


def inputs():
    t = {k: torch.rand(8) for k in ('post_weight', 'post_bias', 'pre_weight', 'pre_bias', 'scale')}
    return dict(t, x=torch.rand(2, 3, 8), branch=torch.rand(2, 3, 8), gate=torch.rand(2, 8), keep=torch.ones(2))


@pytest.mark.parametrize('requires_grad', [False, True])
@pytest.mark.parametrize('which', list(inputs()))
def test_forward_mode_is_refused_for_every_input(node, which, requires_grad):
    t = inputs()
    t['branch'].requires_grad_(requires_grad)
    call = lambda: gated_residual_norm(post='layer', pre='layer', **t)  # noqa: E731
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match='HIP device'):  # no tangent anywhere: only the host's tensors are refused
            call()
        t[which] = fwd.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(NotImplementedError, match='forward-mode'):
            call()
        with torch.no_grad(), pytest.raises(NotImplementedError, match='forward-mode'):
            call()


def test_jvp_is_refused(node):
    t = inputs()
    with pytest.raises(NotImplementedError, match='forward-mode'):
        torch.func.jvp(lambda v: gated_residual_norm(v, t['branch'])[0], (t['x'],), (t['x'],))
