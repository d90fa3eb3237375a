"""Gradients added into engine.FlatParams' slots (ss_multi_add_f32) where destinations repeat, overlap, or the caller wants them elsewhere.

Sums of two or three floats in a fixed order: equal to the last bit wherever the order is the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('n', [1, 7, 64, 4096, 5000, 300000])
def test_repeated_destinations_are_added_in_order(n):
    from semseg_amd import ops
    torch.manual_seed(n)
    a, b = torch.randn(n, device='cuda'), torch.randn(n, device='cuda')
    srcs = [torch.randn(n, device='cuda') for _ in range(100)]
    dsts = [(a, b)[i % 3 == 2] for i in range(100)]
    want = {id(a): a.clone(), id(b): b.clone()}
    for s, d in zip(srcs, dsts):
        want[id(d)] = want[id(d)] + s
    ops.multi_add(srcs, dsts)
    assert torch.equal(a, want[id(a)]) and torch.equal(b, want[id(b)])


def test_overlapping_destinations_are_added_in_order():
    from semseg_amd import ops
    torch.manual_seed(0)
    pool = torch.randn(20000, device='cuda')
    spans = [(0, 9000), (8999, 9000), (17999, 1), (18000, 2000), (3, 15000), (0, 20000)]      # touching, by one element, inside, around
    srcs = [torch.randn(n, device='cuda') for _, n in spans]
    want = pool.clone()
    for (o, n), s in zip(spans, srcs):
        want[o:o + n] += s
    ops.multi_add(srcs, [pool[o:o + n] for o, n in spans])
    assert torch.equal(pool, want)


@pytest.mark.parametrize('roles', [('post_weight', 'pre_weight'), ('post_weight', 'scale'), ('pre_bias', 'post_bias'), ('post_weight', 'pre_weight', 'scale')])
@pytest.mark.parametrize('python', [False, True])
@pytest.mark.parametrize('C', [24, 300, 4096])
def test_one_parameter_in_several_roles_of_a_call(C, python, roles):
    """each role's gradient reaches the parameter's slot, through the C++ node and through the Python one (whose callback a reducer counts)"""
    from semseg_amd.engine import FlatParams
    from semseg_amd.resnorm import gated_residual_norm
    torch.manual_seed(C)
    x, b, dh, dy = (torch.randn(40, C, device='cuda') for _ in range(4))
    names = ('post_weight', 'post_bias', 'pre_weight', 'pre_bias', 'scale')
    values = {k: torch.rand(C, device='cuda') + 0.5 for k in names}

    def run(flat):
        model = torch.nn.Module()
        shared = torch.nn.Parameter(values[roles[0]].clone())
        P = {k: shared if k in roles else torch.nn.Parameter(values[k].clone()) for k in names}
        for k, p in P.items():
            if k not in roles[1:]:
                model.register_parameter(k, p)
        seen = []
        if flat:
            FlatParams(model)
            if python:
                for p in model.parameters():
                    p._ss_grad_ready = lambda q: seen.append(q)
        for _ in range(2):                                    # gradients accumulate
            h, y = gated_residual_norm(x, b, post='layer', pre='layer', **P)
            torch.autograd.backward((h, y), (dh, dy))
        assert not flat or not python or sum(q is shared for q in seen) == 2 * len(roles)
        return {k: p.grad.clone() for k, p in P.items()}
    want, got = run(False), run(True)
    for k in want:
        if k in roles:                                         # autograd adds the roles up before the passes, the slots one by one: at most 3 + 5 roundings of the sum of all parts
            assert ((got[k] - want[k]).abs() <= 8 * 2.0 ** -24 * (want[k].abs() + 2 * sum_of_parts(run_parts(x, b, dh, dy, values, roles, names)))).all(), k
        else:
            assert torch.equal(got[k], want[k]), k


def run_parts(x, b, dh, dy, values, roles, names):
    """the gradient of each role by itself, as parameters of their own"""
    from semseg_amd.resnorm import gated_residual_norm
    P = {k: values[roles[0] if k in roles else k].clone().requires_grad_() for k in names}
    h, y = gated_residual_norm(x, b, post='layer', pre='layer', **P)
    return torch.autograd.grad((h, y), [P[k] for k in roles], (dh, dy))


def sum_of_parts(parts):
    return sum(p.abs() for p in parts)


@pytest.mark.parametrize('python', [False, True])
def test_flat_parameters_under_autograd_grad_and_some_inputs(python):
    """the gradients of a plain module, handed to the caller or put into the slots that are asked for, and nothing anywhere else"""
    from semseg_amd.engine import FlatParams
    from semseg_amd.resnorm import GatedResidualNorm
    torch.manual_seed(5)
    plain, flat = (GatedResidualNorm(40, post='layer', pre='rms', layer_scale=0.5).cuda() for _ in range(2))
    buffer = FlatParams(flat)
    if python:
        for p in flat.parameters():
            p._ss_grad_ready = lambda q: None
    x, b = (torch.randn(3, 5, 40, device='cuda', requires_grad=True) for _ in range(2))

    def loss(m):
        h, y = m(x, b)
        return h.square().sum() + (y * x.detach()).sum()
    for pick in (lambda m: [x, *m.parameters()], lambda m: [b], lambda m: [m.scale, m.pre_weight]):
        want, got = torch.autograd.grad(loss(plain), pick(plain)), torch.autograd.grad(loss(flat), pick(flat))
        assert all(torch.equal(p, q) for p, q in zip(want, got)) and not buffer.grad.any()
    loss(plain).backward(inputs=[plain.scale, plain.post_bias])
    loss(flat).backward(inputs=[flat.scale, flat.post_bias])
    assert torch.equal(flat.scale.grad, plain.scale.grad) and torch.equal(flat.post_bias.grad, plain.post_bias.grad)
    assert not flat.pre_weight.grad.any() and not flat.post_weight.grad.any() and x.grad is None
    assert flat.scale.grad.data_ptr() == flat.scale._ss_grad_sink.data_ptr()


@pytest.mark.parametrize('python', [False, True])
def test_a_forward_on_another_stream_than_the_leaves(python):
    """leaves whose accumulators belong to the caller's stream, a graph made on a side stream: the caller sees its gradients without waiting itself"""
    from semseg_amd.engine import FlatParams
    from semseg_amd.resnorm import GatedResidualNorm
    torch.manual_seed(6)
    m = GatedResidualNorm(40, post='layer', pre='rms', layer_scale=0.5).cuda()
    flat = FlatParams(m)
    if python:
        for p in m.parameters():
            p._ss_grad_ready = lambda q: None
    x, b = torch.randn(3, 5, 40, device='cuda'), torch.randn(3, 5, 40, device='cuda')

    def loss():
        h, y = m(x, b)
        return h.square().sum() + (y * x).sum()
    loss().backward()
    torch.cuda.synchronize()
    want = flat.grad.clone()
    flat.zero_grad()
    alive = [p * 1.0 for p in m.parameters()]                  # accumulators on the caller's stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for k in range(3):
        with torch.cuda.stream(side):
            value = loss()
            torch.cuda._sleep(20_000_000)                      # some 10 ms: the backward's kernels wait behind it
        value.backward()
        got = flat.grad.clone()                                # on the caller's stream, without a word to the side stream
        torch.cuda.synchronize()
        assert torch.allclose(got, (k + 1) * want, rtol=2.0 ** -23, atol=0), k      # the third sum and product are rounded once each
    assert all(p.grad.data_ptr() == p._ss_grad_sink.data_ptr() for p in m.parameters()) and alive
