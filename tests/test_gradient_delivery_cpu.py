"""Where a backward node's gradients of parameters with a slot in a flat buffer go (runtime.deliver_grads), on the host."""
import pytest
import torch

from semseg_amd import ops, runtime
from semseg_amd.engine import FlatParams


class Scale(runtime.GradAwareFunction):
    """y = x * p * q, delivering the gradients of p and q as the package's nodes do"""
    @staticmethod
    def forward(ctx, x, p, q):
        ctx.params = [p, q]
        ctx.save_for_backward(x)
        return x * p * q

    @staticmethod
    def backward(ctx, dy):
        x, (p, q) = ctx.saved_tensors[0], ctx.params
        grads = runtime.deliver_grads(ctx.params, [(dy * x * q).sum(0).detach(), (dy * x * p).sum(0).detach()])
        return (dy * p * q, *grads)


@pytest.fixture
def model(monkeypatch):
    def add(srcs, dsts):
        for s, d in zip(srcs, dsts):
            d.add_(s.reshape(d.shape))
    monkeypatch.setattr(ops, 'multi_add', add)
    m = torch.nn.Module()
    m.p, m.q = torch.nn.Parameter(torch.tensor([1.0, 2.0])), torch.nn.Parameter(torch.tensor([3.0, 4.0]))
    FlatParams(m)
    m.x = torch.tensor([[1.0, 1.0], [2.0, 3.0]], requires_grad=True)
    m.y = lambda: Scale.apply(m.x, m.p, m.q).sum()
    return m


P, Q, X = torch.tensor([9.0, 16.0]), torch.tensor([3.0, 8.0]), torch.tensor([[3.0, 8.0], [3.0, 8.0]])


def test_backward_fills_the_slots(model):
    model.y().backward()
    model.y().backward()
    assert torch.equal(model.p.grad, 2 * P) and torch.equal(model.q.grad, 2 * Q) and model.p.grad.data_ptr() == model.p._ss_grad_sink.data_ptr()


def test_autograd_grad_hands_the_gradients_over_and_leaves_the_slots(model):
    gx, gp = torch.autograd.grad(model.y(), [model.x, model.p])
    assert torch.equal(gx, X) and torch.equal(gp, P) and not model.p.grad.any() and not model.q.grad.any()
    assert torch.equal(torch.autograd.grad(model.y(), model.x)[0], X) and not model.p.grad.any()


def test_backward_of_some_inputs_fills_theirs_only(model):
    model.y().backward(inputs=[model.q])
    assert torch.equal(model.q.grad, Q) and not model.p.grad.any() and model.x.grad is None
    model.y().backward(inputs=[model.p, model.x])
    assert torch.equal(model.q.grad, Q) and torch.equal(model.p.grad, P) and torch.equal(model.x.grad, X)
    assert model.p.grad.data_ptr() == model.p._ss_grad_sink.data_ptr()
