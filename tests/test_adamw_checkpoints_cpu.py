"""What AdamW takes from checkpoints, and that a refused one changes nothing."""
import copy

import pytest
import torch

from semseg_amd.engine import AdamW, FlatParams


def nets():
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(4, 4), torch.nn.LayerNorm(4), torch.nn.Linear(4, 4))
    for p in net.parameters():
        p.grad = torch.randn_like(p)
    return net


def vectors(p):
    return {'weight_decay': 0.0, 'lr_scale': 0.5} if p.dim() == 1 else {}


def torch_checkpoint(net, lr=2e-3, vector_lr=1e-3, decay=0.1, vector_decay=0.0, **kw):
    """the usual two groups; -> checkpoint, parameters in the order torch numbers them"""
    big, small = [p for p in net.parameters() if p.dim() > 1], [p for p in net.parameters() if p.dim() == 1]
    ref = torch.optim.AdamW([{'params': small, 'lr': vector_lr, 'weight_decay': vector_decay}, {'params': big, 'lr': lr, 'weight_decay': decay, **kw}], betas=(0.8, 0.95))
    ref.step()
    return copy.deepcopy(ref.state_dict()), small + big, ref


def everything(opt):
    return [opt.exp_avg.clone(), opt.exp_avg_sq.clone()] + [x.clone() for x in (opt.exp_avg_scale, opt.exp_avg_sq_scale) if x is not None], \
        (opt.lr, opt.wd, opt.betas, opt.eps, opt.seed, opt.t)


def same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a[0], b[0])) and a[1] == b[1]


def refused(opt, sd, match, **kw):
    before = everything(opt)
    with pytest.raises(ValueError, match=match):
        opt.load_state_dict(sd, **kw)
    assert same(everything(opt), before)


@pytest.mark.parametrize('flat', [False, True])
def test_torch_groups_need_an_order_and_then_reach_their_parameters(flat):
    net = nets()
    sd, order, ref = torch_checkpoint(net)
    opt = AdamW(FlatParams(net) if flat else net.parameters(), per_param=vectors)
    refused(opt, sd, 'order')
    opt.load_state_dict(sd, order=order)
    assert (opt.t, opt.betas) == (1, (0.8, 0.95)) and opt.lr == pytest.approx(2e-3) and opt.wd == pytest.approx(0.1)
    back = opt.state_dict()
    for i, p in enumerate(net.parameters()):
        st = ref.state[p]
        assert torch.equal(back['state'][i]['exp_avg'], st['exp_avg']) and torch.equal(back['state'][i]['exp_avg_sq'], st['exp_avg_sq'])
    again = AdamW(FlatParams(net) if flat else net.parameters(), per_param=vectors)
    again.load_state_dict(back)
    assert same(everything(again), everything(opt))


def test_wrong_orders_are_refused():
    net = nets()
    sd, order, _ = torch_checkpoint(net)
    opt = AdamW(net.parameters(), per_param=vectors)
    refused(opt, sd, 'order', order=order[:-1])
    refused(opt, sd, 'order', order=order[:-1] + order[:1])
    refused(opt, sd, 'order', order=order[:-1] + [torch.zeros(4, 4)])
    refused(opt, sd, 'state|parameter', order=list(net.parameters()))


def test_groups_trained_otherwise_are_refused():
    net = nets()
    for kw, match in ((dict(vector_lr=2e-3), 'rate'), (dict(vector_decay=0.05), 'decay'), (dict(betas=(0.9, 0.95)), 'betas'), (dict(eps=1e-6), 'eps'),
                      (dict(amsgrad=True), 'amsgrad')):
        sd, order, _ = torch_checkpoint(net, **kw)
        refused(AdamW(net.parameters(), per_param=vectors), sd, match, order=order)
    own = AdamW(net.parameters(), per_param=vectors).state_dict()
    refused(AdamW(net.parameters()), own, 'rate')
    refused(AdamW(net.parameters(), per_param=lambda p: {'lr_scale': 0.5, 'weight_decay': 0.02} if p.dim() == 1 else {}), own, 'decay')


@pytest.mark.parametrize('bits', [8, 32])
def test_a_refused_checkpoint_changes_nothing(bits):
    net = nets()
    params = list(net.parameters())
    opt = AdamW(params, state_bits=bits, betas=(0.7, 0.8), seed=5, lr=0.5)
    opt.exp_avg.fill_(3), opt.exp_avg_sq.fill_(4)
    good = AdamW(params, state_bits=bits, seed=9).state_dict()
    last = len(params) - 1

    def spoil(f):
        sd = copy.deepcopy(good)
        f(sd)
        return sd
    for f, match in ((lambda sd: sd['state'][last].update(exp_avg_sq=torch.zeros(5)), 'exp_avg_sq'), (lambda sd: sd['state'][last].pop('exp_avg'), 'exp_avg'),
                     (lambda sd: sd['state'][last].update(step=7), 'steps'), (lambda sd: sd['param_groups'][0].update(betas=(1.0, 0.9)), 'betas'),
                     (lambda sd: sd['param_groups'][0]['params'].pop(), 'parameters'), (lambda sd: sd['state'].update({99: sd['state'][0]}), 'state'),
                     (lambda sd: sd.update(lr=-1.0), 'lr'), (lambda sd: sd['state'][0].update(exp_avg=sd['state'][0]['exp_avg'].to(torch.float32 if bits == 8 else torch.int32)), 'exp_avg')):
        refused(opt, spoil(f), match)
    opt.load_state_dict(good)
    assert (opt.lr, opt.betas, opt.seed, opt.t) == (1e-3, (0.9, 0.999), 9, 0) and not opt.exp_avg[:16].any()


def test_a_checkpoint_with_parameters_that_are_frozen_here():
    """torch was given all parameters, the first of them frozen: its numbers are not those of the trainable ones"""
    net = nets()
    net[0].weight.requires_grad_(False)
    net[0].weight.grad = None
    ref = torch.optim.AdamW(net.parameters(), lr=2e-3, weight_decay=0.1)
    ref.step()
    trainable = [p for p in net.parameters() if p.requires_grad]
    opt = AdamW(trainable)
    refused(opt, ref.state_dict(), 'order')
    opt.load_state_dict(ref.state_dict(), order=net.parameters())
    for i, p in enumerate(trainable):
        assert torch.equal(opt.state_dict()['state'][i]['exp_avg'], ref.state[p]['exp_avg'])


def test_codes_of_another_type_are_refused():
    net = nets()
    opt = AdamW(net.parameters(), state_bits=8)
    sd = opt.state_dict()
    sd['state'][2]['exp_avg_sq'] = sd['state'][2]['exp_avg_sq'].to(torch.int8)
    refused(opt, sd, 'exp_avg_sq')
