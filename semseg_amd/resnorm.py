"""The residual update between two blocks with a norm on either side of it, as one launch forward and two backward:

    n = post(branch);   h = alpha * x + keep[s] * scale * act(gate) * n;   y = pre(h)

The reference writes the plain form of it, ``x + drop_path(gamma * branch)`` followed by the next block's LayerNorm
(modules/convnext.py:38-51, modules/segformer.py:94-98).  ``post`` normalises what a block hands over before it joins the stream (sandwich
norm), ``pre`` is the norm that the next block starts with, ``scale`` is LayerScale, ``gate`` modulates per sample (conditioned
blocks) or per element (gated blocks), ``keep`` is DropPath's multiplier (``runtime.drop_path_keep``) and ``alpha`` the weight of the
residual (DeepNorm).  Activations are token matrices, fp32 or bf16, or an fp32 stream around bf16 blocks; statistics, sums and all
parameters are fp32.  ``y`` is the norm of ``h`` as it is stored, so that it is what any other reader of ``h`` would compute.
"""
import torch
from torch import nn, Tensor

from . import ops
from .runtime import GradAwareFunction, deliver_grads, drop_path_keep, expect_grads

_VECTORS = ('pre_w', 'pre_b', 'post_w', 'post_b', 'scale')


def _rows(t, C):
    """[..., C] -> [rows, C] with unit inner stride; a copy only where the layout asks for one (a broadcast gradient, split strides)"""
    t = t.reshape(-1, C)
    return t if t.stride(1) == 1 else t.contiguous().as_strided(t.shape, (C, 1))


class _ResnormFn(GradAwareFunction):
    @staticmethod
    def forward(ctx, x, b, gate, keep, meta, *vectors):
        C = x.shape[-1]
        h, y, stats = ops.resnorm_fwd(_rows(x.detach(), C), _rows(b.detach(), C), gate=None if gate is None else _rows(gate.detach(), C), keep=keep,
                                      **meta, **dict(zip(_VECTORS, vectors)))
        h = h.view(x.shape)
        ctx.meta = {k: v for k, v in meta.items() if k != 'eps'}
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h, b, gate, keep, stats, *vectors)
        expect_grads(ctx, vectors, 5)
        return h, None if y is None else y.view(x.shape)

    @staticmethod
    def backward(ctx, dh, dy):
        h, b, gate, keep, stats, *vectors = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dh is None and dy is None:
            return (None,) * (5 + len(vectors))
        C = h.shape[-1]
        V = {k: v for k, v in zip(_VECTORS, vectors) if k != 'pre_b'}
        dx, db, dgate, G = ops.resnorm_bwd(None if dh is None else _rows(dh, C), None if dy is None else _rows(dy, C), _rows(h, C), _rows(b, C), stats,
                                           gate=None if gate is None else _rows(gate, C), keep=keep, **ctx.meta, **V)
        grads = deliver_grads(vectors, [G[k].view(v.shape) if v is not None and need[5 + i] else None for i, (k, v) in enumerate(zip(_VECTORS, vectors))])
        return (dx.view(h.shape) if need[0] else None, db.view(b.shape) if need[1] else None,
                dgate.view(gate.shape) if gate is not None and need[2] else None, None, None, *grads)


def gated_residual_norm(x: Tensor, branch: Tensor, *, post='none', post_weight=None, post_bias=None, gate=None, gate_act='none', scale=None, keep=None,
                        alpha=1.0, pre='none', pre_weight=None, pre_bias=None, eps=1e-6, samples=None):
    """-> (h, y): ``h = alpha * x + keep * scale * act(gate) * post(branch)`` in x's type, ``y = pre(h)`` in branch's type (None without a norm).

    x, branch: [..., C], alike; float32 / float32, bfloat16 / bfloat16 or a float32 stream around a bfloat16 branch.  post, pre: 'none', 'layer'
    (weight, optionally bias) or 'rms' (weight).  gate (branch's type): per sample [samples, C] or per element, shaped like x; gate_act:
    'none' or 'sigmoid'.  scale, weights, biases: float32 [C].  keep: float32 [samples].  A sample is an index of x's first dimension (a 2-D
    x is one sample) unless ``samples`` says into how many equal runs of rows x divides.  Differentiable in everything but keep."""
    if x.dim() < 2 or x.shape != branch.shape:
        raise ValueError(f'gated_residual_norm: x {tuple(x.shape)} and branch {tuple(branch.shape)} must be alike, [..., C]')
    C, rows = x.shape[-1], x.numel() // max(x.shape[-1], 1)
    if samples is None:
        samples = x.shape[0] if x.dim() > 2 else 1
    if samples < 1 or rows % samples:
        raise ValueError(f'gated_residual_norm: {rows} rows do not divide into {samples} samples')
    if gate is not None and gate.shape != x.shape and gate.shape != (samples, C):
        raise ValueError(f'gated_residual_norm: gate must be [{samples}, {C}] or like x, got {tuple(gate.shape)}')
    meta = {'rows_per_sample': rows // samples, 'gate_act': gate_act, 'alpha': float(alpha), 'post': post, 'pre': pre, 'eps': float(eps)}
    vectors = (pre_weight, pre_bias, post_weight, post_bias, scale)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, branch, gate) + vectors):
        return _ResnormFn.apply(x, branch, gate, keep, meta, *vectors)
    h, y, _ = ops.resnorm_fwd(_rows(x, C), _rows(branch, C), gate=None if gate is None else _rows(gate, C), keep=keep, want_stats=False, **meta,
                              **dict(zip(_VECTORS, vectors)))
    return h.view(x.shape), None if y is None else y.view(x.shape)


class GatedResidualNorm(nn.Module):
    """``forward(x, branch, gate=None) -> (h, y)``: the join of a residual block and the norm that starts the next one (``gated_residual_norm``
    with this module's parameters).  ``layer_scale``: initial value of LayerScale (modules/convnext.py:35), None for none;
    ``drop_path``: DropPath's rate, drawn per sample in training as modules/helpers.py:20-24 draws it."""

    def __init__(self, dim, post='none', pre='layer', layer_scale=None, gate_act='none', alpha=1.0, drop_path=0.0, eps=1e-6):
        super().__init__()
        for name, kind in (('post', post), ('pre', pre)):
            if kind not in ('none', 'layer', 'rms'):
                raise ValueError(f"GatedResidualNorm: {name} must be 'none', 'layer' or 'rms', got {kind!r}")
            self.register_parameter(name + '_weight', nn.Parameter(torch.ones(dim)) if kind != 'none' else None)
            self.register_parameter(name + '_bias', nn.Parameter(torch.zeros(dim)) if kind == 'layer' else None)
        if gate_act not in ('none', 'sigmoid'):
            raise ValueError(f"GatedResidualNorm: gate_act must be 'none' or 'sigmoid', got {gate_act!r}")
        self.scale = nn.Parameter(torch.full((dim,), float(layer_scale))) if layer_scale is not None else None
        self.post, self.pre, self.gate_act, self.alpha, self.drop_path, self.eps = post, pre, gate_act, alpha, drop_path, eps

    def forward(self, x: Tensor, branch: Tensor, gate=None, samples=None):
        n = samples if samples is not None else (x.shape[0] if x.dim() > 2 else 1)
        keep = drop_path_keep(n, self.drop_path, branch.dtype, x.device) if self.training and self.drop_path > 0. else None
        return gated_residual_norm(x, branch, post=self.post, post_weight=self.post_weight, post_bias=self.post_bias, gate=gate, gate_act=self.gate_act,
                                   scale=self.scale, keep=keep, alpha=self.alpha, pre=self.pre, pre_weight=self.pre_weight, pre_bias=self.pre_bias,
                                   eps=self.eps, samples=samples)
