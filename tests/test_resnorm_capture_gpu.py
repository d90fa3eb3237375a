"""Captured backward passes of the gated residual norm whose leaves lie behind other nodes: replayed like the eager ones, or refused where a part
of the graph belongs to the default stream (the capture could not take it in, and the process would end)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def network(python):
    """leaves behind a view, a product and a slice; ``python``: a parameter whose callback makes the call take the Python node"""
    torch.manual_seed(3)
    x = torch.randn(18, 48, device='cuda').requires_grad_()
    wide = torch.randn(2, 9, 96, device='cuda').requires_grad_()
    w, v = ((torch.rand(48, device='cuda') + 0.5).requires_grad_() for _ in range(2))
    dh, dy = torch.randn(2, 9, 48, device='cuda'), torch.randn(2, 9, 48, device='cuda')
    if python:
        v._ss_grad_ready = lambda p: None

    def forward():
        from semseg_amd.resnorm import gated_residual_norm
        return gated_residual_norm(x.view(2, 9, 48), wide[..., 48:], post='rms', post_weight=w * 2.0, pre='rms', pre_weight=v)
    return [x, wide, w, v], (dh, dy), forward


@pytest.mark.parametrize('python', [False, True])
def test_a_captured_backward_through_other_nodes_replays(python):
    leaves, dout, forward = network(python)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(forward(), leaves, dout)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = torch.autograd.grad(forward(), leaves, dout)
        graphs.append((g, out))
    for k in range(4):
        with torch.no_grad():
            leaves[0].mul_(1.5), leaves[1].add_(0.25)
        eager = torch.autograd.grad(forward(), leaves, dout)
        for g, out in graphs:
            for t in out:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, eager)), k


@pytest.mark.parametrize('python', [False, True])
@pytest.mark.parametrize('leaf', [0, 1, 2, 3])
def test_refused_while_an_eager_graph_of_one_leaf_lives(leaf, python):
    """the accumulator of that leaf alone belongs to the default stream, behind whatever stands between"""
    leaves, dout, forward = network(python)
    alive = leaves[leaf] * 1.0                                 # on the default stream, never run backward
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match='eager graph of the same leaves'):
            torch.autograd.backward(forward(), dout)
        with pytest.raises(RuntimeError, match='eager graph of the same leaves'):
            torch.autograd.grad(forward(), leaves, dout)
        out = forward()
    assert all(p.grad is None for p in leaves)
    g.replay()
    torch.cuda.synchronize()
    assert alive.requires_grad and all(torch.equal(p, q) for p, q in zip(out, forward()))


@pytest.mark.parametrize('python', [False, True])
def test_what_is_not_asked_for_does_not_count(python):
    """autograd.grad of other leaves: the living graph's leaf takes no part"""
    leaves, dout, forward = network(python)
    alive = leaves[0] * 1.0
    eager = torch.autograd.grad(forward(), leaves[1:], dout)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = torch.autograd.grad(forward(), leaves[1:], dout)
    for _ in range(3):
        for t in out:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager))
    assert alive.requires_grad
