"""AdamW over many tensors (ss_multi_sqnorm / ss_adamw_prepare / ss_adamw_step, engine.AdamW) against its restatements.

32-bit moments: m and v are two products and a sum of floats, 4 roundings: 8 2^-24 of the terms.  The update divides by sqrt(v)
(v_sqrt_f32, v_rcp_f32: 1 unit each) and multiplies three times more: 16 2^-24 of the update and 3 2^-24 of p, then half a step of p's type.
8-bit moments: every product and sum that a code depends on is rounded once, so codes and scales are compared for EQUALITY with the
operation-by-operation restatement."""
import numpy as np
import pytest
import torch

from oracle import adamw as oracle

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
SIZES = [(1,), (3,), (64,), (255,), (256,), (257,), (33, 31), (1024,), (1025,), (7, 5, 3), (90, 100), (0,), (4099,)]


def build(sizes, p_dtype=torch.float32, g_dtype=torch.float32, seed=0, lead=0, **kw):
    """parameters of their own storage that start `lead` elements into it"""
    from semseg_amd.engine import AdamW
    g = torch.Generator().manual_seed(seed)
    params = []
    for s in sizes:
        n = int(np.prod(s))
        store = torch.zeros(n + lead + 1).to(p_dtype)
        store[lead:lead + n] = torch.randn(n, generator=g)
        store = store.cuda()
        params.append(torch.nn.Parameter(store[lead:lead + n].view(s)))
    return params, AdamW(params, **kw), g


def give(params, g, dtype, scale=1.0):
    out = []
    for i, p in enumerate(params):
        grad = (torch.randn(p.shape, generator=g) * scale * 10.0 ** (i % 5 - 2)).to(dtype)
        if p.dtype != dtype:
            p.grad_dtype = dtype
        p.grad = grad.cuda()
        out.append(grad.double().numpy())
    return out


def state(opt, name, i):
    o, n = opt.plan.first_run[i] * 256, opt.numels[i]
    return getattr(opt, name)[o:o + n].cpu()


def close(got, want, mag, half):
    got = got.detach().double().cpu().numpy().reshape(want.shape)
    tol = half * np.abs(want) + mag + 1e-38
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize('p_dtype,g_dtype', [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16),
                                             (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize('clip,grad_scale', [(None, 1.0), (0.5, 1.0), (1e9, 0.125)])
def test_steps_with_32_bit_moments(p_dtype, g_dtype, clip, grad_scale):
    hy = dict(lr=1e-2, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.1, max_grad_norm=clip)
    params, opt, g = build(SIZES, p_dtype, seed=1, lead=3, per_param=lambda p: {'weight_decay': 0.0, 'lr_scale': 0.5} if p.dim() == 1 else {}, **hy)
    for t in range(1, 5):
        grads = give(params, g, g_dtype)
        before = [(p.detach().double().cpu().numpy(), *(state(opt, k, i).double().numpy().reshape(p.shape) for k in ('exp_avg', 'exp_avg_sq')))
                  for i, p in enumerate(params)]
        norm = opt.step(grad_scale)
        want_norm, coef = oracle.clip_coef(grads, clip, grad_scale)
        assert (norm is None) == (clip is None)
        if clip:
            assert abs(float(norm) - want_norm) <= U * want_norm
        for i, (p, gr, (p0, m0, v0)) in enumerate(zip(params, grads, before)):
            lr, wd = (hy['lr'] * 0.5, 0.0) if p.dim() == 1 else (hy['lr'], 0.1)
            pw, mw, vw = oracle.step64(p0, gr, m0, v0, t, lr, hy['betas'], hy['eps'], wd, coef)
            close(state(opt, 'exp_avg', i), mw, 8 * U * (np.abs(m0) + np.abs(gr * coef)), 0)
            close(state(opt, 'exp_avg_sq', i), vw, 8 * U * (v0 + (gr * coef) ** 2), 0)
            # sqrt(v) and m carry those errors into the update: m's is relative to its terms
            update = lr / (1 - 0.9 ** t) / (np.sqrt(vw) / np.sqrt(1 - 0.98 ** t) + 1e-8)
            close(p, pw, 3 * U * np.abs(p0) + 32 * U * update * (np.abs(mw) + np.abs(m0) + np.abs(gr * coef)), HALF[p_dtype])


def _padded(x, runs):
    out = np.zeros(runs * 256, np.float32)
    out[:x.size] = x.reshape(-1)
    return out.reshape(runs, 256)


@pytest.mark.parametrize('p_dtype,g_dtype', [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16),
                                             (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize('clip', [None, 0.3])
def test_steps_with_8_bit_moments_bit_for_bit(p_dtype, g_dtype, clip):
    betas = (0.9, 0.999)
    params, opt, g = build(SIZES, p_dtype, seed=2, lead=1, lr=1e-2, betas=betas, weight_decay=0.05, max_grad_norm=clip, state_bits=8)
    opt.seed = 77
    for t in range(1, 7):
        grads = give(params, g, g_dtype, scale=1.0 if t < 4 else 1e-3)
        if t == 3:
            params[6].grad.zero_()
            grads[6] = grads[6] * 0
        before = [p.detach().double().cpu().numpy() for p in params]
        old = [x.cpu().numpy().copy() for x in (opt.exp_avg, opt.exp_avg_scale, opt.exp_avg_sq, opt.exp_avg_sq_scale)]
        opt.step()
        _, coef = oracle.clip_coef(grads, clip)
        coef = np.float32(coef)
        for i, p in enumerate(params):
            n, r0 = opt.numels[i], opt.plan.first_run[i]
            runs = -(-n // 256)
            if runs == 0:
                continue
            sl, rs = slice(r0 * 256, (r0 + runs) * 256), slice(r0, r0 + runs)
            cm, qm, cv, qv, m, v = oracle.moments8(_padded(grads[i].astype(np.float32), runs), old[0][sl].reshape(runs, 256), old[1][rs],
                                                   old[2][sl].reshape(runs, 256), old[3][rs], t, 77, np.arange(r0, r0 + runs), betas, coef)
            for got, want, name in ((opt.exp_avg[sl], cm, 'm'), (opt.exp_avg_sq[sl], cv, 'v'), (opt.exp_avg_scale[rs], qm, 'm scale'),
                                    (opt.exp_avg_sq_scale[rs], qv, 'v scale')):
                assert np.array_equal(got.cpu().numpy(), want.reshape(-1)), (t, i, name)
            m, v = (z.reshape(-1)[:n].reshape(p.shape).astype(np.float64) for z in (m, v))
            u = 1e-2 / (1 - 0.9 ** t) * m / (np.sqrt(v) / np.sqrt(1 - 0.999 ** t) + 1e-8)
            close(p, before[i] * (1 - 1e-2 * 0.05) - u, 3 * U * np.abs(before[i]) + 16 * U * np.abs(u), HALF[p_dtype])
    m, v = opt.state_values()
    assert np.array_equal(m.cpu().numpy().reshape(-1, 256), oracle.decode(opt.exp_avg.cpu().numpy().reshape(-1, 256), opt.exp_avg_scale.cpu().numpy(), 2))
    assert np.array_equal(v.cpu().numpy().reshape(-1, 256), oracle.decode(opt.exp_avg_sq.cpu().numpy().reshape(-1, 256), opt.exp_avg_sq_scale.cpu().numpy(), 4))


@pytest.mark.parametrize('bits', [8, 32])
@pytest.mark.parametrize('align', [64, 256])
def test_flat_parameters_take_the_same_steps_as_a_list(bits, align):
    """FlatParams: one address, tensors in reverse order; each tensor's step is that of a list in the same order, padding stays zero"""
    from semseg_amd.engine import AdamW, FlatParams
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(37, 19), torch.nn.Linear(19, 301), torch.nn.Linear(301, 5)).cuda()
    flat = FlatParams(net, align=align)
    copies = [torch.nn.Parameter(p.detach().clone()) for p in flat.params]
    rule = lambda p: {'weight_decay': 0.0} if p.dim() == 1 else {}  # noqa: E731
    a = AdamW(flat, lr=1e-2, max_grad_norm=1.0, state_bits=bits, per_param=rule)
    b = AdamW(copies, lr=1e-2, max_grad_norm=1.0, state_bits=bits, per_param=rule)
    for _ in range(3):
        for p, c in zip(flat.params, copies):
            p.grad.copy_(torch.randn_like(p))
            c.grad = p.grad.clone()
        na, nb = a.step(), b.step()
        assert torch.equal(na, nb)
    for p, c in zip(flat.params, copies):
        assert torch.equal(p, c)
    assert torch.equal(a.exp_avg, b.exp_avg) and torch.equal(a.exp_avg_sq, b.exp_avg_sq)
    used = torch.zeros(flat.numel, dtype=torch.bool, device='cuda')
    for p, o in zip(flat.params, flat.offsets):
        used[o:o + p.numel()] = True
    assert (flat.data[~used] == 0).all()


def test_many_small_tensors_take_several_launches():
    """more tensors than one launch carries addresses for"""
    sizes = [(1 + i % 7, 1 + i % 11) for i in range(451)]
    params, opt, g = build(sizes, seed=3, max_grad_norm=1.0, lr=1e-2, weight_decay=0.0)
    ref = [torch.nn.Parameter(p.detach().double().cpu()) for p in params]
    ropt = torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.0)
    for _ in range(3):
        grads = give(params, g, torch.float32)
        norm = opt.step()
        want, coef = oracle.clip_coef(grads, 1.0)
        assert abs(float(norm) - want) <= U * want
        for r, gr in zip(ref, grads):
            r.grad = torch.from_numpy(gr * coef)
        ropt.step()
    for p, r in zip(params, ref):                              # three steps of at most 1e-2 each, errors of one step as in the test above
        assert (p.detach().double().cpu() - r).abs().max() <= 3 * (4 * U * float(r.detach().abs().max()) + 64 * U * 1e-2 * 30)


def test_parameters_without_gradients_stay():
    params, opt, g = build([(300,), (20, 20), (513,)], seed=4, max_grad_norm=10.0, state_bits=8)
    give(params, g, torch.float32)
    opt.step()
    kept = [p.detach().clone() for p in params]
    before = [x.clone() for x in (opt.exp_avg, opt.exp_avg_sq, opt.exp_avg_scale)]
    give(params, g, torch.float32)
    params[1].grad = None
    only = [params[0].grad.clone(), params[2].grad.clone()]
    norm = opt.step()
    assert torch.equal(params[1], kept[1]) and not torch.equal(params[0], kept[0]) and not torch.equal(params[2], kept[2])
    lo, hi = opt.plan.first_run[1] * 256, opt.plan.first_run[2] * 256
    assert torch.equal(opt.exp_avg[lo:hi], before[0][lo:hi]) and torch.equal(opt.exp_avg_scale[lo // 256:hi // 256], before[2][lo // 256:hi // 256])
    assert not torch.equal(opt.exp_avg[:lo], before[0][:lo])
    want = sum(float(x.double().square().sum()) for x in only) ** 0.5
    assert abs(float(norm) - want) <= U * want


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
@pytest.mark.parametrize('bits', [8, 32])
def test_nonfinite_gradients(bad, bits):
    """skip_nonfinite: nothing changes, the step is not counted, the next one is as if it had not been; without it NaN shows in the parameters"""
    params, opt, g = build([(700,), (30, 30)], seed=5, max_grad_norm=1.0, state_bits=bits, skip_nonfinite=True)
    twin, opt2, g2 = build([(700,), (30, 30)], seed=5, max_grad_norm=1.0, state_bits=bits)
    for k in range(4):
        give(params, g, torch.float32), give(twin, g2, torch.float32)
        assert torch.equal(opt.step(), opt2.step())
        if k == 1:
            keep = [p.grad.clone() for p in params]
            params[0].grad[5] = bad
            norm = opt.step()
            assert not torch.isfinite(norm)
            for p, q in zip(params, keep):
                p.grad.copy_(q)
    assert opt.t == opt2.t == 4
    assert all(torch.equal(a, b) for a, b in zip(params, twin)) and torch.equal(opt.exp_avg, opt2.exp_avg)
    twin[0].grad[5] = bad
    opt2.step()
    assert twin[0].isnan().any()


def test_a_nan_marks_its_run_without_clipping():
    params, opt, g = build([(1000,)], seed=6, state_bits=8)
    give(params, g, torch.float32)
    params[0].grad[300] = float('nan')
    opt.step()
    m, v = opt.state_values()
    assert m[256:512].isnan().all() and v[256:512].isnan().all() and torch.isfinite(m[:256]).all() and torch.isfinite(m[512:]).all()
    assert params[0].isnan().sum() == 1


def test_state_dict_resumes_bit_for_bit():
    for bits in (8, 32):
        params, opt, g = build(SIZES, seed=7, max_grad_norm=1.0, state_bits=bits, lr=1e-2)
        for _ in range(2):
            give(params, g, torch.float32), opt.step()
        sd = opt.state_dict()
        copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
        from semseg_amd.engine import AdamW
        other = AdamW(copies, max_grad_norm=1.0, state_bits=bits)
        other.load_state_dict(sd)
        assert other.lr == 1e-2 and other.t == 2
        for _ in range(2):
            give(params, g, torch.float32)
            for p, c in zip(params, copies):
                c.grad = p.grad.clone()
            opt.step(), other.step()
        assert all(torch.equal(p, c) for p, c in zip(params, copies)) and torch.equal(opt.exp_avg, other.exp_avg)


def test_scheduler_and_weight_copies_follow():
    """OneCycleLR moves lr and betas; the bf16 copies of the weights are refreshed after a step"""
    from semseg_amd import weightprep
    from semseg_amd.engine import AdamW, FlatParams, OneCycleLR
    net = torch.nn.Linear(64, 32).cuda()
    opt = AdamW(FlatParams(net), max_grad_norm=1.0)
    sched = OneCycleLR(opt, max_lr=0.1, total_steps=5)
    before = weightprep.cast(net.weight, torch.bfloat16).clone()
    net.weight.grad.normal_(), net.bias.grad.normal_()
    for _ in range(2):
        opt.step(), sched.step()
    after = weightprep.cast(net.weight, torch.bfloat16)
    assert not torch.equal(before, after) and torch.equal(after, net.weight.detach().bfloat16())


def test_captured_steps_count_and_read_the_rate():
    """two graphs of one optimizer, replayed with eager work between: each replay is the next step, at the rate last pushed"""
    params, opt, g = build([(5000,), (40, 40)], seed=8, max_grad_norm=1.0, state_bits=8, capturable=True, lr=1e-2)
    twin, opt2, g2 = build([(5000,), (40, 40)], seed=8, max_grad_norm=1.0, state_bits=8, lr=1e-2)
    give(params, g, torch.float32), give(twin, g2, torch.float32)
    opt.step(), opt2.step()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            norm = opt.step()
        graphs.append((gr, norm))
    assert opt.t == 1                                          # capturing takes no step
    for k in range(4):
        fresh = [torch.randn(p.shape, generator=g).cuda() for p in params]
        for p, q, f in zip(params, twin, fresh):
            p.grad.copy_(f), q.grad.copy_(f)
        if k == 2:
            opt.lr = opt2.lr = 3e-3
            opt.push_lr()
        gr, norm = graphs[k % 2]
        gr.replay()
        assert torch.equal(norm, opt2.step())
        assert all(torch.equal(a, b) for a, b in zip(params, twin)), k
        assert torch.equal(opt.exp_avg, opt2.exp_avg) and torch.equal(opt.exp_avg_sq_scale, opt2.exp_avg_sq_scale)
    assert opt.t == opt2.t == 5


def test_runs_on_the_current_stream():
    params, opt, g = build([(200000,)], seed=9, max_grad_norm=1.0)
    twin, opt2, g2 = build([(200000,)], seed=9, max_grad_norm=1.0)
    give(params, g, torch.float32), give(twin, g2, torch.float32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        opt.step()
    torch.cuda.current_stream().wait_stream(s)
    opt2.step()
    assert torch.equal(params[0], twin[0])


def test_changed_parameters_and_gradients_are_refused():
    params, opt, g = build([(64,), (8, 8)], seed=1)
    give(params, g, torch.float32)
    params[1].grad = None
    params[0].grad = None
    opt.step()                                                 # nothing to do is a step of nothing
    give(params, g, torch.float32)
    params[1].data = torch.zeros(9, 8, device='cuda')
    with pytest.raises(RuntimeError):
        opt.step()


def test_training_run_of_block_norm_and_optimizer_together():
    """blocks joined by the gated residual norm, trained by AdamW over FlatParams with clipping, in 32 and in 8 bits: the gradients of the
    whole are those of the plain formulas in 64 bits at every step"""
    from semseg_amd.engine import AdamW, FlatParams
    from semseg_amd.resnorm import GatedResidualNorm

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.first = torch.nn.LayerNorm(24)
            self.blocks = torch.nn.ModuleList([torch.nn.Linear(24, 24) for _ in range(3)])
            self.joins = torch.nn.ModuleList([GatedResidualNorm(24, post='rms', pre='layer', layer_scale=0.5) for _ in range(3)])

        def forward(self, x):
            y = self.first(x)
            for f, j in zip(self.blocks, self.joins):
                x, y = j(x, f(y))
            return y

    def plain(P, x):
        ln = torch.nn.functional.layer_norm
        y = ln(x, (24,), P['first.weight'], P['first.bias'])
        for i in range(3):
            b = y @ P[f'blocks.{i}.weight'].t() + P[f'blocks.{i}.bias']
            n = b / (b.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * P[f'joins.{i}.post_weight']
            x = x + P[f'joins.{i}.scale'] * n
            y = ln(x, (24,), P[f'joins.{i}.pre_weight'], P[f'joins.{i}.pre_bias'], 1e-6)
        return y
    for bits in (32, 8):
        torch.manual_seed(0)
        net = Net().cuda()
        flat = FlatParams(net)
        opt = AdamW(flat, lr=1e-2, max_grad_norm=1.0, state_bits=bits, per_param=lambda p: {'weight_decay': 0.0} if p.dim() == 1 else {})
        x, want = torch.randn(2, 50, 24, device='cuda'), torch.randn(2, 50, 24, device='cuda')
        for _ in range(3):
            P = {k: p.detach().double().cpu().requires_grad_() for k, p in net.named_parameters()}
            flat.zero_grad()
            (net(x) - want).square().mean().backward()
            (plain(P, x.double().cpu()) - want.double().cpu()).square().mean().backward()
            for k, p in net.named_parameters():
                # three blocks of two norms and a product each, some 300 roundings in 32 bits deep
                assert (p.grad.double().cpu() - P[k].grad).abs().max() <= 300 * U * max(float(P[k].grad.abs().max()), float(P[k].grad.norm())) + 1e-9, k
            opt.step()


def test_capture_is_refused_without_a_device_count():
    params, opt, g = build([(64,)], seed=1, max_grad_norm=1.0)
    give(params, g, torch.float32)
    opt.step()
    torch.cuda.synchronize()
    before = params[0].detach().clone()
    with pytest.raises(RuntimeError, match='capturable'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.zeros(1, device='cuda')                      # a graph of something, so that capturing itself is in order
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(params[0], before) and opt.t == 1


def test_an_eager_capturable_step_follows_lr():
    """the rate moved by a scheduler reaches eager steps without push_lr"""
    a, opt, g = build([(1000,)], seed=2, lr=1e-2, capturable=True)
    b, opt2, g2 = build([(1000,)], seed=2, lr=1e-2)
    for k in range(3):
        opt.lr = opt2.lr = 1e-2 / (k + 1)
        give(a, g, torch.float32), give(b, g2, torch.float32)
        opt.step(), opt2.step()
    assert torch.equal(a[0], b[0])


def test_zero_sized_and_single_element_models():
    params, opt, g = build([(0,), (1,)], seed=3, max_grad_norm=1.0, state_bits=8)
    give(params, g, torch.float32)
    assert float(opt.step()) == pytest.approx(abs(float(params[1].grad)), rel=1e-6)
    params, opt, g = build([(0,)], seed=3, max_grad_norm=1.0)
    give(params, g, torch.float32)
    assert float(opt.step()) == 0.0 and opt.t == 1


def test_the_norm_is_written_when_the_first_tensors_are_empty():
    params, opt, g = build([(0,)] * 230 + [(7,)], seed=3, max_grad_norm=1.0)
    give(params, g, torch.float32)
    assert float(opt.step()) == pytest.approx(float(params[-1].grad.norm()), rel=1e-6)


def test_a_refused_step_is_not_counted():
    params, opt, g = build([(7,)], seed=3)
    give(params, g, torch.float32)
    before = params[0].detach().clone()
    opt.betas = (0.9, 1.0)
    with pytest.raises(RuntimeError, match='betas'):
        opt.step()
    assert opt.t == 0 and torch.equal(params[0], before)
    opt.betas = (0.9, 0.999)
    opt.step()
    assert opt.t == 1 and not torch.equal(params[0], before)


def test_elements_past_32_bits():
    """the last elements of 2^32 + take the step that they take alone"""
    from semseg_amd.engine import AdamW
    n, tail = (1 << 32) + 300, 556                             # whole runs from n - 556 on
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip('needs 80 GB')
    p = torch.full((n,), 0.5, device='cuda', dtype=torch.bfloat16)
    p.grad = torch.full((n,), 0.25, device='cuda', dtype=torch.bfloat16)
    q = torch.randn(tail, device='cuda').bfloat16()
    p[-tail:].copy_(q)
    q.grad = torch.randn(tail, device='cuda').bfloat16()
    p.grad[-tail:].copy_(q.grad)
    kw = dict(lr=0.05, max_grad_norm=1e9, state_bits=8)        # no clipping: every element is on its own
    big, small = AdamW([p], **kw), AdamW([q], **kw)
    norm = float(big.step())
    small.step()
    assert norm == pytest.approx(((n - tail) * 0.0625 + float((q.grad.double() ** 2).sum())) ** 0.5, rel=1e-6)
    assert torch.equal(p[-tail:], q)
    assert torch.equal(big.exp_avg_scale[-3:], small.exp_avg_scale) and torch.equal(big.exp_avg_sq_scale[-3:], small.exp_avg_sq_scale)
    assert int((big.exp_avg[-768:].int() - small.exp_avg.int()).abs().max()) <= 1        # other draws, by the element's place
    assert float(p[:1 << 20].float().std()) == 0.0 and float(p[0]) != 0.5
    del p, big
    torch.cuda.empty_cache()
