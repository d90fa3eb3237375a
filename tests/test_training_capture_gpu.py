"""A whole training step captured: gradients cleared, blocks joined by the gated residual norm forward and backward, gradients delivered into FlatParams'
buffer, one weight in two roles, and the clipped AdamW step.  Every replay is the next step of an eager twin, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def build(bits):
    from semseg_amd.engine import AdamW, FlatParams
    from semseg_amd.resnorm import GatedResidualNorm
    torch.manual_seed(1)
    net = torch.nn.ModuleList([GatedResidualNorm(40, post='rms', pre='layer', layer_scale=0.5, gate_act='sigmoid') for _ in range(3)]).cuda()
    net[1].scale = net[1].post_weight                          # one parameter in two roles
    flat = FlatParams(net)
    opt = AdamW(flat, lr=1e-2, max_grad_norm=0.5, state_bits=bits, capturable=True, skip_nonfinite=True)
    x, want, gate = (torch.empty(2, 9, 40, device='cuda') for _ in range(3))

    def step():
        flat.zero_grad()
        h, y = x, x
        for join in net:
            h, y = join(h, y * 0.5, gate=gate)
        torch.autograd.backward([h, y], [h.detach() - want, y.detach() * 0.1])
        return opt.step(grad_scale=0.5)
    return net, flat, opt, (x, want, gate), step


@pytest.mark.parametrize('bits', [8, 32])
def test_captured_training_steps_are_the_eager_ones(bits):
    from semseg_amd import weightprep
    a, flat_a, opt_a, in_a, step_a = build(bits)
    b, flat_b, opt_b, in_b, step_b = build(bits)
    g = torch.Generator().manual_seed(2)

    def feed():
        for p, q in zip(in_a, in_b):
            v = torch.randn(p.shape, generator=g).cuda()
            p.copy_(v), q.copy_(v)
    side = torch.cuda.Stream()
    feed()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step_a()
    torch.cuda.current_stream().wait_stream(side)
    step_b()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = step_a()
        graphs.append((graph, norm))
    assert opt_a.t == 1
    for k in range(5):
        feed()
        graph, norm = graphs[k % 2]
        graph.replay()
        weightprep.bump()
        eager = step_b()
        torch.cuda.synchronize()
        assert torch.equal(norm, eager) and torch.equal(flat_a.grad, flat_b.grad) and torch.equal(flat_a.data, flat_b.data), k
        assert torch.equal(opt_a.exp_avg, opt_b.exp_avg) and torch.equal(opt_a.exp_avg_sq, opt_b.exp_avg_sq), k
    assert opt_a.t == opt_b.t == 6
