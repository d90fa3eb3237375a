"""Residual update between two norms (ss_resnorm_fwd / _bwd, semseg_amd/resnorm.py) against its 64-bit restatement.

Tolerance of a value: half a step of its type relative to it, plus K 2^-24 times the sum of the absolute values of its terms (the oracle's
``mag``), a rounding in 32 bits each.  Element-wise values go through at most 20 roundings in a row, two of them of row sums in 32 bits with
64 terms a lane and join: K = 64.  Column sums add up to 256 rows in a register before they are joined over at most 1024 workgroups in
chains of 32 and 32: 256 + 64 + 20 roundings, K = 384.  The sigmoid adds v_exp_f32 of an argument scaled in 32 bits: |v| roundings,
|v| < 16 here, inside both."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


def close(got, want, column=False):
    value, mag = want
    g = got.detach().double().cpu().reshape(value.shape)
    tol = HALF[got.dtype] * value.abs() + (384 if column else 64) * U * mag + 1e-38
    bad = ~((g - value).abs() <= tol)
    assert not bad.any(), f'{int(bad.sum())} of {bad.numel()} off, worst {float(((g - value).abs() / tol).max()):.3g} x the tolerance'


def make(rows, C, stream, branch, seed, *, samples=1, post='none', pre='none', gate='none', act='none', scale=True, keep=False, alpha=1.0, bias=True,
         offset=0.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, dt=torch.float32, m=0.0, k=1.0: (torch.randn(*s, generator=g) * k + m).to(dt)  # noqa: E731
    t = {'x': r(rows, C, dt=stream, k=2.0, m=offset), 'b': r(rows, C, dt=branch, m=offset - 0.2),
         'gate': None if gate == 'none' else r(samples if gate == 'sample' else rows, C, dt=branch), 'scale': r(C, k=0.3, m=0.2) if scale else None,
         'keep': (torch.rand(samples, generator=g) < 0.7).float() / 0.7 if keep else None}
    for k, kind in (('post', post), ('pre', pre)):
        t[k + '_w'] = r(C, k=0.3, m=1.0) if kind != 'none' else None
        t[k + '_b'] = r(C, k=0.3) if kind == 'layer' and bias else None
    meta = dict(rows_per_sample=rows // samples, gate_act=act, alpha=alpha, post=post, pre=pre)
    return t, meta, r(rows, C, dt=stream), r(rows, C, dt=branch)


def run_and_check(t, meta, dh, dy, eps=1e-6):
    from semseg_amd import ops
    from oracle.resnorm import resnorm as oracle
    d = {k: None if v is None else v.cuda() for k, v in t.items()}
    fwd = {k: v for k, v in d.items()}
    h, y, stats = ops.resnorm_fwd(**fwd, **meta, eps=eps)
    h2, y2, none = ops.resnorm_fwd(**fwd, **meta, eps=eps, want_stats=False)
    assert torch.equal(h, h2) and none is None and (y is None or torch.equal(y, y2))
    if meta['pre'] == 'none':
        dy = None
    want = oracle(t['x'], t['b'], h.cpu(), dh, dy, eps=eps, **{k: v for k, v in t.items() if k not in 'xb'}, **meta)
    close(h, want['h'])
    if y is not None:
        close(y, want['y'])
    back = {k: v for k, v in d.items() if k not in ('x', 'b', 'pre_b')}
    dx, db, dg, G = ops.resnorm_bwd(None if dh is None else dh.cuda(), None if dy is None else dy.cuda(), h, d['b'], stats, **back, **meta)
    close(dx, want['x']), close(db, want['b'])
    if dg is not None:
        close(dg, want['gate'], column=dg.shape[0] != dx.shape[0])
    assert set(G) == {k for k in ('pre_w', 'pre_b', 'post_w', 'post_b', 'scale') if k in want}
    for k, v in G.items():
        close(v, want[k], column=True)
    return h, y, (dx, db, dg, G)


F, H = torch.float32, torch.bfloat16
TYPES = [(F, F), (H, H), (F, H)]


@pytest.mark.parametrize('types', TYPES)
@pytest.mark.parametrize('rows,C', [(1, 1), (1, 8), (3, 7), (5, 64), (130, 97), (37, 511), (66, 512), (9, 513), (11, 1000), (4, 1024), (6, 1025), (3, 2048),
                                    (5, 2049), (2, 4095), (7, 4096)])
def test_widths_both_norms(rows, C, types):
    run_and_check(*make(rows, C, *types, seed=rows * 7 + C, post='layer', pre='layer', gate='row'))


@pytest.mark.parametrize('types', TYPES)
@pytest.mark.parametrize('pre', ['none', 'layer', 'rms'])
@pytest.mark.parametrize('post', ['none', 'layer', 'rms'])
@pytest.mark.parametrize('gate,act', [('none', 'none'), ('sample', 'none'), ('sample', 'sigmoid'), ('row', 'none'), ('row', 'sigmoid')])
def test_every_form(types, post, pre, gate, act):
    for i, (rows, C, samples, scale, keep, alpha) in enumerate([(60, 40, 4, True, True, 1.0), (21, 33, 3, False, False, 0.75), (14, 640, 7, True, False, -1.5)]):
        run_and_check(*make(rows, C, *types, seed=i, samples=samples, post=post, pre=pre, gate=gate, act=act, scale=scale, keep=keep, alpha=alpha, bias=i != 1))


@pytest.mark.parametrize('rows,C,samples', [(20000, 64, 4), (30001, 8, 1), (4097, 320, 17), (600, 1500, 3), (5000, 24, 5000), (3000, 768, 1500)])
def test_many_rows(rows, C, samples):
    """more rows than one step of all workgroups; samples of many rows, of two, of one; several units to a workgroup"""
    run_and_check(*make(rows, C, H, H, seed=C, samples=samples, post='rms', pre='layer', gate='sample', keep=True))


def test_sums_do_not_cancel_far_from_zero():
    """rows around 1000 with deviation 1: a variance from 32-bit sums of squares would have no digit left"""
    run_and_check(*make(50, 768, F, F, seed=3, post='layer', pre='layer', offset=1000.0))


@pytest.mark.parametrize('which', ['dh', 'dy'])
def test_one_gradient_alone(which):
    t, meta, dh, dy = make(33, 72, H, H, seed=5, post='layer', pre='rms')
    run_and_check(t, meta, dh if which == 'dh' else None, dy if which == 'dy' else None)


def test_constant_rows_and_zero_rows():
    """no deviation at all: 1 / sqrt(eps), finite everywhere"""
    t, meta, dh, dy = make(6, 40, F, F, seed=1, post='layer', pre='layer', scale=False)
    t['b'][:3], t['x'][:3] = 0.0, 0.0
    t['b'][3:] = 2.5
    run_and_check(t, meta, dh, dy)


def test_rows_with_nan_or_infinity_stay_alone():
    from semseg_amd import ops
    t, meta, _, _ = make(40, 48, H, H, seed=2, post='rms', pre='layer')
    d = {k: None if v is None else v.cuda() for k, v in t.items()}
    h, y, _ = ops.resnorm_fwd(**d, **meta)
    d['b'][7, 3], d['b'][21, 5] = float('nan'), float('inf')
    h2, y2, _ = ops.resnorm_fwd(**d, **meta)
    ok = torch.ones(40, dtype=torch.bool)
    ok[[7, 21]] = False
    assert torch.equal(h[ok.cuda()], h2[ok.cuda()]) and torch.equal(y[ok.cuda()], y2[ok.cuda()])
    assert y2[7].isnan().all() and y2[21].isnan().all()


@pytest.mark.parametrize('types', TYPES)
@pytest.mark.parametrize('C', [64, 97, 640])
def test_strided_and_unaligned_rows(types, C):
    """slices of wider buffers that start anywhere, rows repeated with stride 0: same bits as from dense rows"""
    from semseg_amd import ops
    rows = 50
    t, meta, dh, dy = make(rows, C, *types, seed=C, samples=5, post='layer', pre='rms', gate='sample', act='none', keep=True)
    d = {k: None if v is None else v.cuda() for k, v in t.items()}

    def inside(v, lead):
        wide = torch.full((v.shape[0], v.shape[1] + lead + 3), float('nan'), dtype=v.dtype, device='cuda')
        wide[:, lead:lead + v.shape[1]] = v
        return wide[:, lead:lead + v.shape[1]]
    s = dict(d, x=inside(d['x'], 1), b=inside(d['b'], 3), gate=inside(d['gate'], 5))
    h, y, st = ops.resnorm_fwd(**d, **meta)
    h2, y2, st2 = ops.resnorm_fwd(**s, **meta)
    assert torch.equal(h, h2) and torch.equal(y, y2) and torch.equal(st, st2)
    back = lambda q: {k: v for k, v in q.items() if k not in ('x', 'b', 'pre_b')}  # noqa: E731
    a = ops.resnorm_bwd(dh.cuda(), dy.cuda(), h, d['b'], st, **back(d), **meta)
    b = ops.resnorm_bwd(inside(dh.cuda(), 7), inside(dy.cuda(), 1), inside(h, 2), s['b'], st, **back(s), **meta)
    assert all(torch.equal(p, q) for p, q in zip(a[:3], b[:3])) and all(torch.equal(a[3][k], b[3][k]) for k in a[3])
    one = d['x'][:1]
    h3, _, _ = ops.resnorm_fwd(**dict(d, x=one.expand(rows, C)), **meta)
    h4, _, _ = ops.resnorm_fwd(**dict(d, x=one.expand(rows, C).contiguous()), **meta)
    assert torch.equal(h3, h4)


@pytest.mark.parametrize('C,dtype', [(64, H), (97, F), (4096, H)])
def test_same_bits_every_time_and_for_every_split(C, dtype):
    """no atomics: a call repeats itself; and a row's outputs do not depend on how many rows stand beside it"""
    from semseg_amd import ops
    t, meta, dh, dy = make(257, C, dtype, dtype, seed=9, post='layer', pre='layer', gate='row')
    d = {k: None if v is None else v.cuda() for k, v in t.items()}
    h, y, st = ops.resnorm_fwd(**d, **meta)
    back = {k: v for k, v in d.items() if k not in ('x', 'b', 'pre_b')}
    a = ops.resnorm_bwd(dh.cuda(), dy.cuda(), h, d['b'], st, **back, **meta)
    b = ops.resnorm_bwd(dh.cuda(), dy.cuda(), h, d['b'], st, **back, **meta)
    assert all(torch.equal(p, q) for p, q in zip(a[:3], b[:3])) and all(torch.equal(a[3][k], b[3][k]) for k in a[3])
    one = {k: v if v is None or v.dim() == 1 else v[100:101] for k, v in d.items()}
    h1, y1, _ = ops.resnorm_fwd(**one, **dict(meta, rows_per_sample=1))
    assert torch.equal(h1, h[100:101]) and torch.equal(y1, y[100:101])


# ---------------------------------------------------------------------------------- through autograd and the module
def _leaves(t):
    return {k: v.cuda().requires_grad_() if k != 'keep' else v.cuda() for k, v in t.items() if v is not None}


@pytest.mark.parametrize('shape', [(4, 15, 40), (2, 3, 5, 24), (30, 40)])
def test_function_gradients_and_shapes(shape):
    from semseg_amd import ops
    from semseg_amd.resnorm import gated_residual_norm
    C, samples = shape[-1], shape[0] if len(shape) > 2 else 1
    rows = torch.Size(shape[:-1]).numel()
    t, meta, dh, dy = make(rows, C, F, H, seed=rows, samples=samples, post='rms', pre='layer', gate='sample', act='sigmoid', keep=True)
    L = _leaves(t)
    h, y = gated_residual_norm(L['x'].view(shape), L['b'].view(shape), post='rms', post_weight=L['post_w'], gate=L['gate'], gate_act='sigmoid',
                               scale=L['scale'], keep=L['keep'], pre='layer', pre_weight=L['pre_w'], pre_bias=L['pre_b'])
    assert h.shape == y.shape == torch.Size(shape) and h.dtype == F and y.dtype == H
    names = [k for k in L if k != 'keep']
    got = dict(zip(names, torch.autograd.grad((h, y), [L[k] for k in names], (dh.cuda().view(shape), dy.cuda().view(shape)))))
    D = {k: v.detach() for k, v in L.items()}
    h2, y2, st = ops.resnorm_fwd(**D, **meta)
    assert torch.equal(h.detach().view(rows, C), h2) and torch.equal(y.detach().view(rows, C), y2)
    dx, db, dg, G = ops.resnorm_bwd(dh.cuda(), dy.cuda(), h2, D['b'], st, **{k: v for k, v in D.items() if k not in ('x', 'b', 'pre_b')}, **meta)
    for k, v in dict(G, x=dx, b=db, gate=dg).items():
        assert torch.equal(got[k], v), k


def test_gradients_against_differences():
    """a directional difference of the fp32 operator itself: step 1e-2 along random directions; the third-order term and the rounding of
    a sum of 400 terms around 1 are below 2e-3 of it"""
    from semseg_amd.resnorm import gated_residual_norm
    t, meta, dh, dy = make(10, 40, F, F, seed=4, samples=2, post='layer', pre='rms', gate='sample', act='sigmoid')
    L = _leaves(t)
    dh, dy = dh.cuda().view(2, 5, 40), dy.cuda().view(2, 5, 40)

    def f(P):
        h, y = gated_residual_norm(P['x'].view(2, 5, 40), P['b'].view(2, 5, 40), post='layer', post_weight=P['post_w'], post_bias=P['post_b'],
                                   gate=P['gate'], gate_act='sigmoid', scale=P['scale'], pre='rms', pre_weight=P['pre_w'])
        return (h.double() * dh).sum() + (y.double() * dy).sum()
    grads = dict(zip(L, torch.autograd.grad(f(L), list(L.values()))))
    g = torch.Generator(device='cuda').manual_seed(1)
    for k, v in L.items():
        d = torch.randn(v.shape, generator=g, device='cuda')
        with torch.no_grad():
            num = (f({**L, k: v + 1e-2 * d}) - f({**L, k: v - 1e-2 * d})) / 2e-2
        exact = (grads[k].double() * d).sum()
        assert abs(num - exact) <= 2e-3 * (grads[k].double().abs() * d.abs()).sum(), k


def test_broadcast_gradients_unused_outputs_and_no_grad():
    from semseg_amd.resnorm import GatedResidualNorm
    torch.manual_seed(0)
    m = GatedResidualNorm(48, post='rms', pre='layer', layer_scale=0.1).cuda()
    x, b = torch.randn(2, 7, 48, device='cuda', requires_grad=True), torch.randn(2, 7, 48, device='cuda', requires_grad=True)
    h, y = m(x, b)
    y.sum().backward()                                        # a gradient with stride 0 everywhere, none for h
    gx = x.grad.clone()
    x.grad = None
    h, y = m(x, b)
    torch.autograd.backward([y], [torch.ones(2, 7, 48, device='cuda')])
    assert torch.equal(gx, x.grad)
    h, y = m(x, b)
    h.mean().backward()                                       # h alone: the norm behind it gets zero gradients, not garbage
    assert m.pre_weight.grad is not None and torch.isfinite(m.pre_weight.grad).all()
    only = GatedResidualNorm(48, pre='none').cuda()
    h, y = only(x, b)
    assert y is None and torch.equal(h.detach(), (x + b).detach())
    h.sum().backward()
    with torch.no_grad():
        h2, _ = m(x, b)
    assert not h2.requires_grad and h2.grad_fn is None
    wide = torch.randn(2, 7, 96, device='cuda', requires_grad=True)      # a branch and its gate from one projection, row stride 96
    bb, gg = wide.chunk(2, -1)
    g = GatedResidualNorm(48, pre='rms', gate_act='sigmoid').cuda()
    h, y = g(x, bb, gate=gg)
    (h.sum() + y.sum()).backward()
    dense = [t.detach().contiguous().requires_grad_() for t in (bb, gg)]
    h3, y3 = g(x, dense[0], gate=dense[1])
    (h3.sum() + y3.sum()).backward()
    assert torch.equal(h, h3) and torch.equal(wide.grad, torch.cat([dense[0].grad, dense[1].grad], -1))


def test_retained_graph_backward_twice():
    from semseg_amd.resnorm import GatedResidualNorm
    m = GatedResidualNorm(32, pre='layer', layer_scale=1.0).cuda()
    x = torch.randn(3, 4, 32, device='cuda', requires_grad=True)
    h, y = m(x, torch.randn(3, 4, 32, device='cuda'))
    loss = (h * y).sum()
    a = torch.autograd.grad(loss, [x, m.scale], retain_graph=True)
    b = torch.autograd.grad(loss, [x, m.scale])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_drop_path_draws_like_the_framework():
    from semseg_amd.resnorm import GatedResidualNorm
    from semseg_amd.runtime import drop_path_keep
    m = GatedResidualNorm(16, pre='none', drop_path=0.5).cuda().train()
    x, b = torch.randn(64, 3, 16, device='cuda'), torch.randn(64, 3, 16, device='cuda')
    torch.manual_seed(5)
    h, _ = m(x, b)
    torch.manual_seed(5)
    keep = drop_path_keep(64, 0.5, torch.float32, x.device)
    assert 0 < int((keep > 0).sum()) < 64 and torch.equal(h, x + b * keep[:, None, None])
    assert torch.equal(m.eval()(x, b)[0], x + b)


def test_side_stream_and_graph_replays():
    """the call runs on the caller's stream; captured, it repeats the eager bits at every replay, with eager work in between"""
    from semseg_amd import ops
    t, meta, dh, dy = make(700, 96, H, H, seed=8, samples=7, post='layer', pre='layer', gate='sample', keep=True)
    d = {k: None if v is None else v.cuda() for k, v in t.items()}
    dh, dy = dh.cuda(), dy.cuda()
    back = {k: v for k, v in d.items() if k not in ('x', 'b', 'pre_b')}

    def step():
        h, y, st = ops.resnorm_fwd(**d, **meta)
        return (h, y) + ops.resnorm_bwd(dh, dy, h, d['b'], st, **back, **meta)
    flat = lambda r: list(r[:-1]) + list(r[-1].values())  # noqa: E731
    want = [v.clone() for v in flat(step())]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = flat(step())
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(side, want))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = flat(step())
        graphs.append((g, out))
    x0 = d['x'].clone()
    for k in range(3):
        d['x'].copy_(x0 * (k + 1))
        eager = [v.clone() for v in flat(step())]
        for g, out in graphs:
            for v in out:
                v.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, eager)), k


def test_python_refusals_on_the_device():
    from semseg_amd import ops
    x = torch.randn(6, 8, device='cuda')
    with pytest.raises(ValueError):
        ops.resnorm_fwd(x, x, pre='layer', pre_w=torch.ones(8))                  # a weight on the host
    with pytest.raises(ValueError):
        ops.resnorm_fwd(x.t(), x.t())                                            # inner stride
    h, y, st = ops.resnorm_fwd(x, x, pre='rms', pre_w=torch.ones(8, device='cuda'))
    with pytest.raises(ValueError):
        ops.resnorm_bwd(None, None, h, x, st, pre='rms', pre_w=torch.ones(8, device='cuda'))
    with pytest.raises(ValueError):
        ops.resnorm_bwd(x, x, h, x, st)                                          # dy without a norm behind h
    with pytest.raises(ValueError):
        ops.resnorm_bwd(x.bfloat16(), None, h, x, st)
    with pytest.raises(ValueError):
        ops.resnorm_bwd(x, None, h, x, st[:3])
    wide = torch.zeros(2, 5000, device='cuda')
    with pytest.raises(RuntimeError, match='C=5000'):
        ops.resnorm_fwd(wide, wide)


def test_gradients_of_gradients_are_refused():
    from semseg_amd.resnorm import GatedResidualNorm
    m = GatedResidualNorm(16).cuda()
    x = torch.randn(2, 3, 16, device='cuda', requires_grad=True)
    h, y = m(x, x * 2)
    with pytest.raises(RuntimeError, match='gradients of gradients'):
        torch.autograd.grad(y.square().sum(), x, create_graph=True)


@pytest.mark.parametrize('C,types', [(40, (H, H)), (512, (F, F)), (700, (F, H)), (4000, (H, H))])
@pytest.mark.parametrize('samples,n', [(3000, 2), (900, 7), (770, 1), (2, 1500)])
def test_gates_of_many_and_of_few_samples(C, types, samples, n):
    """a workgroup that walks whole samples writes their gates' gradients itself; several that share one leave partial sums"""
    if C >= 700 and samples > 1000:
        samples //= 4
    run_and_check(*make(samples * n, C, *types, seed=n, samples=samples, post='layer', pre='rms', gate='sample', act='sigmoid', keep=True))


@pytest.mark.parametrize('dtype', [H, F])
@pytest.mark.parametrize('C', [40, 100, 384, 512, 768, 1000])
def test_a_row_has_the_same_bits_in_any_company(C, dtype):
    """few rows are spread over more lanes each than many: same h, y and statistics"""
    from semseg_amd import ops
    t, meta, _, _ = make(20000, C, dtype, dtype, seed=C, post='layer', pre='rms', gate='row')
    d = {k: None if v is None else v.cuda() for k, v in t.items()}
    h, y, st = ops.resnorm_fwd(**d, **meta)
    for lo, hi in ((0, 1), (19990, 20000), (7000, 7300)):
        part = {k: v if v is None or v.dim() == 1 else v[lo:hi] for k, v in d.items()}
        h1, y1, st1 = ops.resnorm_fwd(**part, **dict(meta, rows_per_sample=hi - lo))
        assert torch.equal(h1, h[lo:hi]) and torch.equal(y1, y[lo:hi]) and torch.equal(st1, st[lo:hi])


@pytest.mark.parametrize('post,pre,gate,act,keep', [('layer', 'layer', 'sample', 'sigmoid', True), ('rms', 'none', 'row', 'none', False),
                                                    ('none', 'layer', 'none', 'none', True), ('none', 'none', 'none', 'none', False)])
def test_both_nodes_agree_bit_for_bit(post, pre, gate, act, keep):
    """the C++ node, and the Python one that parameters of engine.FlatParams and traced calls take"""
    from semseg_amd import _lib
    from semseg_amd.resnorm import gated_residual_norm
    t, meta, dh, dy = make(60, 72, F, H, seed=3, samples=4, post=post, pre=pre, gate=gate, act=act, keep=keep, alpha=0.5)

    def run():
        L = _leaves(t)
        view = {k: v.view(4, 15, 72) if k in 'xb' or (k == 'gate' and gate == 'row') else v for k, v in L.items()}
        h, y = gated_residual_norm(view['x'], view['b'], post=post, post_weight=L.get('post_w'), post_bias=L.get('post_b'), gate=view.get('gate'),
                                   gate_act=act, scale=L['scale'], keep=L.get('keep'), alpha=0.5, pre=pre, pre_weight=L.get('pre_w'), pre_bias=L.get('pre_b'))
        outs, grads = ([h, y], [dh.cuda().view(4, 15, 72), dy.cuda().view(4, 15, 72)]) if y is not None else ([h], [dh.cuda().view(4, 15, 72)])
        names = [k for k in L if k != 'keep']
        return outs + list(torch.autograd.grad(outs, [L[k] for k in names], grads))
    native = run()
    _lib.TRACE = []
    try:
        python = run()
        assert {e[0] for e in _lib.TRACE} == {'ss_resnorm_fwd', 'ss_resnorm_bwd'}
    finally:
        _lib.TRACE = None
    assert len(native) == len(python) and all(torch.equal(a, b) for a, b in zip(native, python))


def test_parameters_of_other_shapes_and_flat_parameters():
    """a vector shaped [1, C] gets its gradient in that shape; parameters in FlatParams' buffer find theirs there, added to what is there"""
    from semseg_amd.engine import FlatParams
    from semseg_amd.resnorm import GatedResidualNorm, gated_residual_norm
    torch.manual_seed(0)
    x, b = torch.randn(5, 40, device='cuda'), torch.randn(5, 40, device='cuda')
    w = torch.rand(1, 40, device='cuda', requires_grad=True)
    h, y = gated_residual_norm(x, b, pre='rms', pre_weight=w)
    y.sum().backward()
    flat_w = w.detach().view(40).clone().requires_grad_()
    gated_residual_norm(x, b, pre='rms', pre_weight=flat_w)[1].sum().backward()
    assert w.grad.shape == (1, 40) and torch.equal(w.grad.view(40), flat_w.grad)
    a, c = (GatedResidualNorm(40, post='rms', layer_scale=0.3).cuda() for _ in range(2))
    flat = FlatParams(c)
    for m in (a, c):
        for _ in range(2):                                     # gradients accumulate
            h, y = m(x.view(1, 5, 40), b.view(1, 5, 40))
            (h.sum() + (y * y).sum()).backward()
    for p, q in zip(a.parameters(), c.parameters()):
        assert torch.equal(p.grad, q.grad) and q.grad.data_ptr() >= flat.grad.data_ptr()


def test_leaves_changed_in_place_before_backward_are_noticed():
    from semseg_amd.resnorm import GatedResidualNorm
    m = GatedResidualNorm(16).cuda()
    x, b = torch.randn(2, 3, 16, device='cuda', requires_grad=True), torch.randn(2, 3, 16, device='cuda')
    h, y = m(x, b)
    b.mul_(2.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_flat_parameters_with_a_reducer_take_the_python_node():
    """a GradReducer's callbacks are counted as for every other node (one process: the reducer is made active by hand)"""
    from semseg_amd.engine import FlatParams
    from semseg_amd.resnorm import GatedResidualNorm
    torch.manual_seed(1)
    a, c = (GatedResidualNorm(24, post='layer', layer_scale=0.3).cuda() for _ in range(2))
    FlatParams(a), FlatParams(c)
    seen = []
    for p in c.parameters():
        p._ss_grad_ready = lambda q: seen.append(q)
    x, b = torch.randn(2, 5, 24, device='cuda'), torch.randn(2, 5, 24, device='cuda')
    for m in (a, c):
        h, y = m(x, b)
        (h.sum() + (y * y).sum()).backward()
    assert len(seen) == 5 and {id(p) for p in seen} == {id(p) for p in c.parameters()}
    assert all(torch.equal(p.grad, q.grad) for p, q in zip(a.parameters(), c.parameters()))


def test_frozen_flat_parameters_and_replaced_gradients():
    from semseg_amd.engine import FlatParams
    from semseg_amd.resnorm import GatedResidualNorm
    torch.manual_seed(2)
    m = GatedResidualNorm(24, post='rms', layer_scale=0.3).cuda()
    flat = FlatParams(m)
    m.pre_weight.requires_grad_(False)                         # frozen after the buffer was laid out: its slot stays zero
    slot = m.scale.grad
    m.scale.grad = torch.zeros(24, device='cuda')              # no longer the slot: the gradient goes to what .grad is
    x, b = torch.randn(2, 5, 24, device='cuda'), torch.randn(2, 5, 24, device='cuda')
    h, y = m(x, b)
    (h.sum() + (y * y).sum()).backward()
    assert (m.pre_weight.grad == 0).all() and (slot == 0).all() and (m.scale.grad != 0).any() and (m.post_weight.grad != 0).any()
    assert m.post_weight.grad.data_ptr() >= flat.grad.data_ptr()


@pytest.mark.parametrize('C', [8, 64, 200])
@pytest.mark.parametrize('rows', [1, 3, 70])
def test_an_infinity_in_the_last_row_reaches_the_sums_as_it_is(rows, C):
    """lanes behind the last row read that row again: they add zero, not zero times infinity"""
    from semseg_amd import ops
    t, meta, dh, _ = make(rows, C, F, F, seed=5)
    d = {k: None if v is None else v.cuda() for k, v in t.items()}
    dh = dh.cuda()
    d['b'][-1, 3] = float('inf')
    back = {k: v for k, v in d.items() if k not in ('x', 'b', 'pre_b')}
    h, _, st = ops.resnorm_fwd(**d, **meta)
    *_, G = ops.resnorm_bwd(dh, None, h, d['b'], st, **back, **meta)
    assert G['scale'][3] == float('inf') * torch.sign(dh[-1, 3]) and torch.isfinite(torch.cat([G['scale'][:3], G['scale'][4:]])).all()
    d['b'][-1, 3] = 1.0
    d['gate'] = back['gate'] = torch.ones(rows, C, device='cuda')
    d['gate'][-1, 3] = float('inf')
    h, _, st = ops.resnorm_fwd(**d, **meta)
    *_, G = ops.resnorm_bwd(dh, None, h, d['b'], st, **back, **meta)
    assert G['scale'][3] == float('inf') * torch.sign(dh[-1, 3])


def test_rows_far_apart():
    """strides past the lanes' offsets are copied"""
    from semseg_amd.resnorm import gated_residual_norm
    torch.manual_seed(0)
    x = torch.randn(3, (1 << 23) + 8, device='cuda', dtype=H)[:, :64]
    b = torch.randn(3, 64, device='cuda', dtype=H)
    w = torch.rand(64, device='cuda') + 0.5
    far, near = (gated_residual_norm(v, b, pre='rms', pre_weight=w) for v in (x, x.contiguous()))
    assert x.stride(0) > 1 << 23 and all(torch.equal(p, q) for p, q in zip(far, near))
    grads = []
    for dy in (x, x.contiguous()):
        leaf = b.clone().requires_grad_()
        _, y = gated_residual_norm(x.contiguous(), leaf, pre='rms', pre_weight=w)
        grads += torch.autograd.grad(y, leaf, dy)
    assert torch.equal(*grads)


def test_offsets_past_32_bits():
    """the last rows of 2^32 + elements have the bits that they have alone"""
    from semseg_amd import ops
    C, rows = 4096, (1 << 20) + 5
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip('needs 100 GB')
    t, meta, _, _ = make(5, C, H, H, seed=3, post='rms', pre='layer')
    v = {k: u.cuda() for k, u in t.items() if u is not None and k not in 'xb'}
    meta.pop('rows_per_sample')
    big = lambda seed: torch.empty(rows, C, device='cuda', dtype=H).normal_(generator=torch.Generator('cuda').manual_seed(seed))  # noqa: E731
    x, b, dh, dy = (big(k) for k in range(4))
    last = slice(rows - 5, rows)
    back = {k: u for k, u in v.items() if k != 'pre_b'}
    h, y, st = ops.resnorm_fwd(x, b, **v, **meta, rows_per_sample=rows)
    dx, db, _, _ = ops.resnorm_bwd(dh, dy, h, b, st, **back, **meta, rows_per_sample=rows)
    h1, y1, st1 = ops.resnorm_fwd(x[last], b[last], **v, **meta, rows_per_sample=5)
    dx1, db1, _, _ = ops.resnorm_bwd(dh[last], dy[last], h1, b[last], st1, **back, **meta, rows_per_sample=5)
    for p, q in ((h, h1), (y, y1), (st, st1), (dx, dx1), (db, db1)):
        assert torch.equal(p[last], q)
    del x, b, dh, dy, h, y, dx, db, st
    torch.cuda.empty_cache()


def captured_training(C=48):
    torch.manual_seed(3)
    leaves = [torch.randn(2, 9, C, device='cuda').requires_grad_(), torch.randn(2, 9, C, device='cuda').requires_grad_(),
              (torch.rand(C, device='cuda') + 0.5).requires_grad_(), (torch.rand(C, device='cuda') + 0.5).requires_grad_()]
    dh, dy = torch.randn(2, 9, C, device='cuda'), torch.randn(2, 9, C, device='cuda')

    def forward():
        from semseg_amd.resnorm import gated_residual_norm
        return gated_residual_norm(leaves[0], leaves[1], post='rms', post_weight=leaves[2], pre='rms', pre_weight=leaves[3])
    return leaves, (dh, dy), forward


@pytest.mark.parametrize('accumulate', [False, True])
def test_captured_autograd_backward(accumulate):
    """two captured training passes of the same leaves replay the eager bits, with eager passes in between"""
    leaves, dout, forward = captured_training()

    def step():
        if not accumulate:
            return list(torch.autograd.grad(forward(), leaves, dout))
        torch.autograd.backward(forward(), dout)
        return [p.grad for p in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        for p in leaves:
            p.grad = None
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for k in range(4):
        with torch.no_grad():
            leaves[0].mul_(1.5), leaves[1].add_(0.25)
        for p in leaves:
            p.grad = None
        eager = torch.autograd.grad(forward(), leaves, dout)
        for g, out in graphs:
            for v in out:
                v.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, eager)), k


def test_a_captured_backward_is_refused_while_an_eager_graph_of_its_leaves_lives():
    leaves, dout, forward = captured_training()
    alive = forward()                                          # made on the default stream, never run backward
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match='eager graph of the same leaves'):
            torch.autograd.grad(forward(), leaves, dout)
        with pytest.raises(RuntimeError, match='eager graph of the same leaves'):
            torch.autograd.backward(forward(), dout)
        out = forward()                                        # the forward alone is taken
    assert all(p.grad is None for p in leaves)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, alive))


def test_checkpointing_and_saved_tensor_hooks():
    """recomputed and offloaded activations give the gradients of the plain graph; a second backward of a freed graph is refused"""
    from torch.utils.checkpoint import checkpoint
    leaves, dout, forward = captured_training()
    want = torch.autograd.grad(forward(), leaves, dout)
    for reentrant in (False, True):
        got = torch.autograd.grad(checkpoint(lambda *a: forward(), *leaves, use_reentrant=False), leaves, dout) if not reentrant else None
        if reentrant:
            torch.autograd.backward(checkpoint(lambda *a: forward(), *leaves, use_reentrant=True), dout)
            got = [p.grad for p in leaves]
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    with torch.autograd.graph.save_on_cpu():
        out = forward()
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(out, leaves, dout), want))
    with pytest.raises(RuntimeError, match='second time|already been freed'):
        torch.autograd.grad(out, leaves, dout)
    out = forward()
    assert out[0].requires_grad and not out[0].is_leaf and out[1].grad_fn is out[0].grad_fn or out[1].grad_fn.name() == out[0].grad_fn.name()
    with torch.no_grad():
        assert not forward()[0].requires_grad
    seen = []
    out[0].register_hook(lambda g: seen.append(tuple(g.shape)))
    torch.autograd.grad(out, leaves[:1], dout)                 # one input alone
    assert seen == [(2, 9, 48)]


@pytest.mark.parametrize('types', TYPES)
@pytest.mark.parametrize('C', [2, 3, 6, 7, 9, 11, 12, 18, 23, 90, 96, 200, 330, 384, 385, 600, 767, 768, 1023, 1100, 1535, 1536, 2047, 2100, 2500])
def test_chunks_of_one_six_and_eight_channels(C, types):
    """both norms, gates and DropPath where the chunk's width or the waves of a row change, one workgroup and many"""
    for rows, samples, gate in ((7, 1, 'row'), (390, 3, 'sample')):
        t, meta, dh, dy = make(rows, C, *types, seed=C, samples=samples, post='layer', pre='rms', gate=gate, act='sigmoid', keep=True, alpha=0.75)
        run_and_check(t, meta, dh, dy)


@pytest.mark.parametrize('C', [5, 96, 700, 1300])
def test_views_of_every_chunk_width(C):
    """rows at odd offsets and strides: the bits of the dense call, and nothing written next to the rows"""
    from semseg_amd import ops
    for types in TYPES:
        t, meta, dh, dy = make(33, C, *types, seed=1, samples=3, post='rms', pre='layer', gate='sample')
        d = {k: None if v is None else v.cuda() for k, v in t.items()}

        def odd(v):
            wide = torch.zeros(v.shape[0], C + 5, device='cuda', dtype=v.dtype)
            wide[:, 3:3 + C] = v.cuda()
            return wide[:, 3:3 + C]
        o = {**d, 'x': odd(t['x']), 'b': odd(t['b'])}
        dense, view = ops.resnorm_fwd(**d, **meta), ops.resnorm_fwd(**o, **meta)
        assert all(torch.equal(p, q) for p, q in zip(dense, view))
        back = {k: v for k, v in d.items() if k not in ('x', 'b', 'pre_b')}
        one = ops.resnorm_bwd(dh.cuda(), dy.cuda(), dense[0], d['b'], dense[2], **back, **meta)
        two = ops.resnorm_bwd(odd(dh), odd(dy), dense[0], o['b'], dense[2], **back, **meta)
        assert all(torch.equal(p, q) for p, q in zip(one[:3], two[:3])) and all(torch.equal(one[3][k], two[3][k]) for k in one[3])
