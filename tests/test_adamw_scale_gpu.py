"""A negative gradient scale climbs: the norm that clips and skips is a length whatever the sign."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('bits', [8, 32])
@pytest.mark.parametrize('skip', [False, True])                # joined inside the update, and by a launch of its own
@pytest.mark.parametrize('max_norm', [0.5, 1e9])
def test_a_negative_scale_is_the_positive_one_of_the_negative_gradients(bits, skip, max_norm):
    from semseg_amd.engine import AdamW
    torch.manual_seed(0)
    a, b = ([torch.nn.Parameter(torch.linspace(-1, 1, n, device='cuda')) for n in (1000, 33)] for _ in range(2))
    kw = dict(lr=1e-2, max_grad_norm=max_norm, state_bits=bits, skip_nonfinite=skip)
    up, down = AdamW(a, **kw), AdamW(b, **kw)
    for _ in range(3):
        for p, q in zip(a, b):
            p.grad = torch.randn_like(p)
            q.grad = -p.grad
        n, m = up.step(grad_scale=-0.25), down.step(grad_scale=0.25)
        assert float(n) > 0 and torch.equal(n, m)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert torch.equal(up.exp_avg, down.exp_avg) and torch.equal(up.exp_avg_sq, down.exp_avg_sq)


def test_a_negative_scale_skips_an_infinite_norm():
    from semseg_amd.engine import AdamW
    p = torch.nn.Parameter(torch.ones(300, device='cuda'))
    opt = AdamW([p], max_grad_norm=1.0, skip_nonfinite=True)
    p.grad = torch.full_like(p, float('inf'))
    norm = opt.step(grad_scale=-1.0)
    assert float(norm) == float('inf') and (p == 1).all() and opt.t == 0
