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


def joined(v):
    return gated_residual_norm(v, v + 1)[0]


def test_jit_trace_is_refused(node):
    with pytest.raises(NotImplementedError, match='tracing'):
        torch.jit.trace(joined, (torch.rand(2, 3, 8),), check_trace=False)


@pytest.mark.parametrize('kw', [{}, {'tracing_mode': 'fake'}, {'tracing_mode': 'symbolic'}, {'pre_dispatch': True}, {'tracing_mode': 'symbolic', 'pre_dispatch': True}])
def test_make_fx_is_refused(node, kw):
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(NotImplementedError, match='tracing'):
        make_fx(joined, **kw)(torch.rand(2, 3, 8))
    with pytest.raises(NotImplementedError, match='tracing'):
        make_fx(torch.no_grad()(joined), **kw)(torch.rand(2, 3, 8))


def test_nothing_is_refused_once_tracing_ended(node):
    from torch.fx.experimental.proxy_tensor import make_fx
    for _ in range(2):
        with pytest.raises(NotImplementedError, match='tracing'):
            make_fx(joined)(torch.rand(2, 3, 8))
        with pytest.raises(RuntimeError, match='HIP device'):
            joined(torch.rand(2, 3, 8))


def test_export_is_refused(node):
    class Join(torch.nn.Module):
        def forward(self, v):
            return joined(v)
    with pytest.raises(Exception):                            # whatever the exporter wraps it in
        torch.export.export(Join(), (torch.rand(2, 3, 8),), strict=False)
