"""The residual update without a norm behind the block (``post='none'``, what a block without a sandwich norm uses) where a row takes two, four
and eight waves: kernels of their own, forward and backward, against the 64-bit restatement with the tolerances of test_resnorm_gpu.py."""
import pytest
import torch

from test_resnorm_gpu import TYPES, make, run_and_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('types', TYPES)
@pytest.mark.parametrize('gate,act', [('none', 'none'), ('sample', 'sigmoid'), ('sample', 'none'), ('row', 'sigmoid')])
@pytest.mark.parametrize('C', [513, 640, 768, 769, 800, 1000, 1024, 1025, 1280, 1537, 1600, 2048, 2049, 3000, 4095, 4096])
def test_wide_rows_without_a_post_norm(C, gate, act, types):
    for rows, samples, pre, keep in ((7, 1, 'layer', False), (1200, 4, 'rms', True), (66, 66, 'layer', True), (9, 3, 'none', True)):
        run_and_check(*make(rows, C, *types, seed=C + rows, samples=samples, pre=pre, gate=gate, act=act, keep=keep, alpha=0.75))


@pytest.mark.parametrize('types', TYPES)
@pytest.mark.parametrize('C', [800, 1000, 1600, 2048])
def test_many_samples_without_a_post_norm(C, types):
    """more samples than workgroups, each gate's gradient written by the workgroup that walks the sample; and a plain join without scale"""
    run_and_check(*make(2400, C, *types, seed=1, samples=1200, pre='rms', gate='sample', act='sigmoid', keep=True))
    run_and_check(*make(2400, C, *types, seed=2, samples=2, gate='sample', scale=False))
