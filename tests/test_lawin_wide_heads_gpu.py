"""Lawin window attention backward at head widths 32 and 64 on the vector kernels (f32, and bf16 rows that the matrix kernels do not take because they
are not aligned): the widest need more registers than a lane has, each form against the 64-bit formula.

f32: a score sums 64 products of values below 5 (at most 64 2^-24 of their magnitudes, some 1e-5 in the exponent), a gradient 64 terms of it: 1e-4 of
the largest gradient.  bf16: half a step of the output, and of y (which delta sums), 2^-8 each: 2e-2 of the largest."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('lead', [0, 1, 3])
@pytest.mark.parametrize('inter,heads', [(64, 2), (64, 1), (128, 2), (192, 3)])
def test_each_gradient_of_wide_heads(dtype, lead, inter, heads):
    from semseg_amd import ops
    B, H, W, d = 2, 8, 16, inter // heads
    g = torch.Generator().manual_seed(inter + lead)
    theta, pg, dy = (torch.randn(B * H * W, n, generator=g).to(dtype) for n in (inter, 2 * inter, inter))

    def inside(v):
        wide = torch.full((v.shape[0], inter + 5), float('nan'), dtype=dtype, device='cuda')
        wide[:, lead:lead + inter] = v.cuda()
        return wide[:, lead:lead + inter]
    t, p = theta.double().requires_grad_(), pg.double().requires_grad_()
    windows = lambda v: v.view(B, H // 8, 8, W // 8, 8, heads, d).permute(0, 1, 3, 5, 2, 4, 6).reshape(-1, heads, 64, d)  # noqa: E731
    phi, gg = (v.reshape(-1, 64, heads, d).transpose(1, 2) for v in (p[:, :inter], p[:, inter:]))
    y64 = torch.softmax(windows(t) @ phi.transpose(-1, -2).contiguous() / math.sqrt(d), -1) @ gg
    y64 = y64.view(B, H // 8, W // 8, heads, 8, 8, d).permute(0, 1, 4, 2, 5, 3, 6).reshape(B * H * W, inter)
    y64.backward(dy.double())
    y, lse = ops.lawin_attn_fwd(inside(theta), pg.cuda(), B, H, W, heads)
    dt, dp = ops.lawin_attn_bwd(inside(theta), pg.cuda(), inside(y.cpu()), inside(dy), lse, B, H, W, heads)
    for got, want in ((y, y64.detach()), (dt, t.grad), (dp[:, :inter], p.grad[:, :inter]), (dp[:, inter:], p.grad[:, inter:])):
        error = (got.double().cpu() - want).abs().max() / want.abs().max()
        assert error < (1e-4 if dtype == torch.float32 else 2e-2), float(error)
