"""AdamW over FlatParams steps what the parameters and their .grad hold, or refuses."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def net_and_optimizer(**kw):
    from semseg_amd.engine import AdamW, FlatParams
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(8, 5), torch.nn.Linear(5, 3)).cuda()
    flat = FlatParams(net)
    return net, flat, AdamW(flat, lr=1e-2, **kw)


def test_gradients_that_left_the_buffer_are_refused():
    """torch's zero_grad() drops the slots: the next gradients are new tensors, and the buffer still holds the last step's"""
    net, flat, opt = net_and_optimizer(max_grad_norm=1.0)
    x = torch.randn(4, 8, device='cuda')
    net(x).square().sum().backward()
    opt.step()
    before = [p.detach().clone() for p in net.parameters()]
    net.zero_grad()
    for backward in (False, True):
        if backward:
            net(x).square().sum().backward()
        with pytest.raises(RuntimeError, match='lies elsewhere'):
            opt.step()
        assert opt.t == 1 and all(torch.equal(p, q) for p, q in zip(net.parameters(), before))
    flat.zero_grad()
    net(x).square().sum().backward()
    opt.step()
    net.zero_grad(set_to_none=False)
    net(x).square().sum().backward()
    opt.step()
    assert opt.t == 3


def test_parameters_that_left_the_buffer_are_refused():
    net, flat, opt = net_and_optimizer()
    net[1].weight.data = net[1].weight.data.clone()
    with pytest.raises(RuntimeError, match='lies elsewhere'):
        opt.step()
    assert opt.t == 0


def test_frozen_and_untouched_parameters_keep_their_slots():
    net, flat, opt = net_and_optimizer()
    net[0].weight.requires_grad_(False)
    net(torch.randn(4, 8, device='cuda')).square().sum().backward()
    opt.step()
    assert opt.t == 1
