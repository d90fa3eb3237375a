"""Residual update between two norms: what is refused before anything reaches the device, and the 64-bit restatement against torch's own layers."""
import pytest
import torch

from oracle.resnorm import resnorm as oracle_resnorm


def test_restatement_matches_torch_autograd():
    """The oracle's written-out gradients against autograd over torch's LayerNorm, in 64 bits, and against differences."""
    torch.manual_seed(0)
    B, N, C = 3, 5, 12
    t = lambda *s: torch.randn(*s, dtype=torch.float64)  # noqa: E731
    x, b, gate, scale, keep = t(B * N, C), t(B * N, C), t(B, C), t(C), torch.tensor([1.25, 0.0, 1.25], dtype=torch.float64)
    pw, pb, w, bias, dh, dy = t(C), t(C), t(C), t(C), t(B * N, C), t(B * N, C)
    leaves = {'x': x, 'b': b, 'gate': gate, 'scale': scale, 'post_w': pw, 'post_b': pb, 'pre_w': w, 'pre_b': bias}
    for v in leaves.values():
        v.requires_grad_()
    ln = torch.nn.functional.layer_norm
    rows = torch.arange(B * N) // N

    def f(L):
        h = 0.5 * L['x'] + keep[rows, None] * L['scale'] * torch.sigmoid(L['gate'])[rows] * ln(L['b'], (C,), L['post_w'], L['post_b'], 1e-5)
        return h, ln(h, (C,), L['pre_w'], L['pre_b'], 1e-5)
    h, y = f(leaves)
    want = dict(zip(leaves, torch.autograd.grad((h, y), list(leaves.values()), (dh, dy))))
    got = oracle_resnorm(x, b, None, dh, dy, N, gate, 'sigmoid', scale, keep, 0.5, 'layer', pw, pb, 'layer', w, bias, 1e-5)
    assert torch.allclose(got['h'][0], h) and torch.allclose(got['y'][0], y)
    for k, v in want.items():
        assert torch.allclose(got[k][0], v, rtol=1e-9, atol=1e-9), k
    for k, v in leaves.items():                               # a directional difference of the whole function, central, step 1e-5
        d = torch.randn_like(v)
        with torch.no_grad():
            def at(s):
                hh, yy = f({**leaves, k: v + s * d})
                return (hh * dh).sum() + (yy * dy).sum()
            num = (at(1e-5) - at(-1e-5)) / 2e-5
        assert abs(num - (want[k] * d).sum()) < 1e-6 * (1 + abs(num)), k


def _code(name, *args):
    from semseg_amd._lib import lib
    return getattr(lib(), name)(*args), lib().ss_last_error().decode()


def _fwd(**kw):
    a = dict(xd=0, bd=0, x=16, ldx=8, b=16, ldb=8, gate=None, ldg=0, mode=0, act=0, scale=None, keep=None, alpha=1.0, post=0, pw=None, pb=None, pre=0,
             w=None, bias=None, eps=1e-6, h=16, y=None, stats=None, rows=4, n=4, C=8, stream=None)
    a.update(kw)
    return _code('ss_resnorm_fwd', *a.values())


@pytest.mark.parametrize('bad,text', [
    (dict(xd=1, bd=0), 'types'), (dict(xd=2), 'types'), (dict(rows=0), 'row counts'), (dict(rows=1 << 31, n=1), 'row counts'), (dict(n=3), 'row counts'),
    (dict(C=0), 'C=0'), (dict(C=4097), 'C=4097'), (dict(post=3), 'codes'), (dict(act=2), 'codes'), (dict(mode=1), 'gate'), (dict(gate=16), 'gate'),
    (dict(post=1), 'weight'), (dict(pre=2, y=16), 'weight'), (dict(post=2, pw=16, pb=16), 'bias'), (dict(pb=16), 'bias'), (dict(x=None), 'bad arguments'),
    (dict(pre=1, w=16), 'bad arguments'), (dict(ldx=-8), 'bad arguments'), (dict(eps=-1.0), 'bad arguments')])
def test_forward_refusals_at_the_c_entry(bad, text):
    rc, msg = _fwd(**bad)
    assert rc != 0 and 'ss_resnorm_fwd' in msg and text in msg


def _bwd(**kw):
    a = dict(xd=0, bd=0, dh=16, lddh=8, dy=None, lddy=8, h=16, ldh=8, b=16, ldb=8, gate=None, ldg=0, mode=0, act=0, scale=None, keep=None, alpha=1.0,
             post=0, pw=None, pb=None, pre=0, w=None, stats=16, dx=16, db=16, dgate=None, dvec=None, rows=4, n=4, C=8, ws=None, wsb=0, stream=None)
    a.update(kw)
    return _code('ss_resnorm_bwd', *a.values())


@pytest.mark.parametrize('bad,text', [
    (dict(dh=None), 'bad arguments'), (dict(dy=16), 'bad arguments'), (dict(pre=2, w=16, dy=16, h=None, dvec=16), 'bad arguments'),
    (dict(gate=16, mode=2), 'bad arguments'), (dict(stats=None), 'bad arguments'), (dict(scale=16, dvec=16), 'workspace'),
    (dict(scale=16, dvec=16, ws=16, wsb=31), 'workspace'), (dict(scale=16, ws=16, wsb=1 << 20), 'workspace'), (dict(C=5000), 'C=5000')])
def test_backward_refusals_at_the_c_entry(bad, text):
    rc, msg = _bwd(**bad)
    assert rc != 0 and 'ss_resnorm_bwd' in msg and text in msg


def test_workspace_of_bad_sizes_is_zero():
    from semseg_amd._lib import lib
    assert lib().ss_resnorm_bwd_workspace(0, 1, 8, 1, 1, 0, 1) == 0 and lib().ss_resnorm_bwd_workspace(8, 8, 5000, 1, 1, 0, 1) == 0
    assert lib().ss_resnorm_bwd_workspace(8, 8, 64, 1, 1, 0, 1) >= 5 * 64 * 4


def test_python_refusals():
    from semseg_amd import ops
    from semseg_amd.resnorm import GatedResidualNorm, gated_residual_norm
    x = torch.zeros(2, 3, 8)
    with pytest.raises(RuntimeError, match='HIP device'):
        gated_residual_norm(x, x)
    with pytest.raises(ValueError, match='must be alike'):
        gated_residual_norm(x, x[:, :2])
    with pytest.raises(ValueError, match='gate must be'):
        gated_residual_norm(x, x, gate=torch.zeros(3, 8))
    with pytest.raises(ValueError, match='divide'):
        gated_residual_norm(x, x, samples=4)
    w = torch.ones(8)
    r = x.view(6, 8)
    check = lambda **kw: ops._resnorm_args(**{**dict(x=r, b=r, rows_per_sample=3, gate=None, gate_act='none', scale=None, keep=None, post='none',  # noqa: E731
                                                     post_w=None, post_b=None, pre='none', pre_w=None, pre_b=None, who='t'), **kw})
    assert check()[:4] == (6, 8, 3, 0) and check(gate=torch.zeros(2, 8))[3] == 1 and check(gate=r)[3] == 2
    for kw in (dict(post='batch'), dict(gate=r, gate_act='tanh'), dict(post='layer'), dict(pre_w=w), dict(pre='rms', pre_w=w, pre_b=w),
               dict(pre='rms', pre_w=w[:7]), dict(keep=torch.ones(3)), dict(scale=w.double()), dict(rows_per_sample=4), dict(b=r[:3]),
               dict(x=torch.zeros(0, 8), b=torch.zeros(0, 8)), dict(gate=torch.zeros(2, 8, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            check(**kw)
    with pytest.raises(TypeError):
        check(x=r.bfloat16())
    with pytest.raises(ValueError):
        GatedResidualNorm(8, post='group')
    with pytest.raises(ValueError):
        GatedResidualNorm(8, gate_act='tanh')
