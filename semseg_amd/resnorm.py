"""The residual update between two blocks with a norm on either side of it, as one launch forward and two backward:

    n = post(branch);   h = alpha * x + keep[s] * scale * act(gate) * n;   y = pre(h)

The reference's MiT blocks write the plain form of it, ``x + drop_path(branch)`` followed by the next norm (modules/segformer.py:94-98); its
ConvNeXt blocks end in ``x + drop_path(gamma * branch)`` and no norm, the next block's comes behind its depthwise convolution
(modules/convnext.py:38-51): ``pre='none'``.  This package's own MiT and ConvNeXt have residual, LayerScale and DropPath in the epilogue of the product
that makes the branch; the operator is for blocks put together by hand, where the branch comes from anything else.
``post`` normalises what a block hands over before it joins the stream (sandwich
norm), ``pre`` is the norm that the next block starts with, ``scale`` is LayerScale, ``gate`` modulates per sample (conditioned
blocks) or per element (gated blocks), ``keep`` is DropPath's multiplier (``runtime.drop_path_keep``) and ``alpha`` the weight of the
residual (DeepNorm).  Activations are token matrices, fp32 or bf16, or an fp32 stream around bf16 blocks; statistics, sums and all
parameters are fp32.  ``y`` is the norm of ``h`` as it is stored, so that it is what any other reader of ``h`` would compute.
"""
import torch
from torch import nn, Tensor

from . import _lib, ops
from .runtime import GradAwareFunction, deliver_grads, drop_path_keep, expect_grads

_VECTORS = ('pre_w', 'pre_b', 'post_w', 'post_b', 'scale')


def _rows(t, C):
    """[..., C] -> (tensor, elements between rows) with unit inner stride; a view or a copy only where the layout asks for one (a broadcast
    gradient, split strides)"""
    if t.is_contiguous():
        return t, C
    if t.dim() != 2:
        t = t.reshape(-1, C)
    if t.stride(1) != 1 or t.stride(0) >= 1 << 23:             # 32-bit lane offsets in the kernels
        t = t.contiguous()
        return t, C
    return t, t.stride(0)


class _ResnormFn(GradAwareFunction):
    """``cfg``: what ``gated_residual_norm`` checked -- rows, rows of a sample, C, gate mode, codes of post, pre and the activation, alpha, eps"""

    @staticmethod
    def forward(ctx, x, b, gate, keep, cfg, *vectors):
        rows, n, C, mode, post, pre, act, alpha, eps = cfg
        pre_w, pre_b, post_w, post_b, scale = vectors
        xs, ldx = _rows(x, C)
        bs, ldb = _rows(b, C)
        gs, ldg = _rows(gate, C) if mode else (None, 0)
        h, y, stats = ops._resnorm_launch_fwd(xs, ldx, bs, ldb, gs, ldg, mode, act, scale, keep, alpha, post, post_w, post_b, pre, pre_w, pre_b, eps, True,
                                              rows, n, C, x.shape)
        ctx.cfg = cfg
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h, b, gate, keep, stats, *vectors)
        expect_grads(ctx, vectors, 5)
        return h, y

    @staticmethod
    def backward(ctx, dh, dy):
        if torch.is_grad_enabled():
            raise RuntimeError('gated_residual_norm: no gradients of gradients (create_graph=True) are built')
        if dh is None and dy is None:
            return (None,) * 10
        _lib.native().refuse_captured_leaves()
        rows, n, C, mode, post, pre, act, alpha, _ = ctx.cfg
        h, b, gate, keep, stats, *vectors = ctx.saved_tensors
        _, _, post_w, post_b, scale = vectors
        need = ctx.needs_input_grad
        dhs, lddh = (None, 0) if dh is None else _rows(dh, C)
        dys, lddy = (None, 0) if dy is None else _rows(dy, C)
        bs, ldb = _rows(b, C)
        gs, ldg = _rows(gate, C) if mode else (None, 0)
        dx, db, dgate, dvec = ops._resnorm_launch_bwd(dhs, lddh, dys, lddy, h, C, bs, ldb, stats, gs, ldg, mode, act, scale, keep, alpha, post, post_w, post_b,
                                                      pre, vectors[0], rows, n, C, h.shape)
        made = dict(zip(ops._resnorm_slots(post, pre, scale), dvec.unbind(0)))
        grads = deliver_grads(vectors, [made[k] if v is not None and need[5 + i] else None for i, (k, v) in enumerate(zip(_VECTORS, vectors))])
        return (dx if need[0] else None, db if need[1] else None, dgate.view(gate.shape) if mode and need[2] else None, None, None, *grads)


def gated_residual_norm(x: Tensor, branch: Tensor, *, post='none', post_weight=None, post_bias=None, gate=None, gate_act='none', scale=None, keep=None,
                        alpha=1.0, pre='none', pre_weight=None, pre_bias=None, eps=1e-6, samples=None):
    """-> (h, y): ``h = alpha * x + keep * scale * act(gate) * post(branch)`` in x's type, ``y = pre(h)`` in branch's type (None without a norm).

    x, branch: [..., C], alike; float32 / float32, bfloat16 / bfloat16 or a float32 stream around a bfloat16 branch.  post, pre: 'none', 'layer'
    (weight, optionally bias) or 'rms' (weight).  gate (branch's type): per sample [samples, C] or per element, shaped like x; gate_act:
    'none' or 'sigmoid'.  scale, weights, biases: float32 [C].  keep: float32 [samples].  A sample is an index of x's first dimension (a 2-D
    x is one sample) unless ``samples`` says into how many equal runs of rows x divides.  Differentiable in everything but keep,
    by backward only: forward-mode derivatives are refused, and so is tracing (torch.jit.trace, make_fx, export)."""
    vectors = (pre_weight, pre_bias, post_weight, post_bias, scale)
    if _lib.TRACE is None and not any(hasattr(v, '_ss_grad_ready') for v in vectors):
        if post not in ops._NORM or pre not in ops._NORM or gate_act not in ops._GATE_ACT:
            raise ValueError(f'gated_residual_norm: unknown norm or gate activation in {post!r}, {pre!r}, {gate_act!r}')
        if samples is not None and samples < 1:
            raise ValueError(f'gated_residual_norm: rows do not divide into {samples} samples')
        sinks = [getattr(v, '_ss_grad_sink', None) for v in vectors]            # slots in engine.FlatParams' gradient buffer
        return _lib.native().gated_residual_norm(x, branch, ops._NORM[post], post_weight, post_bias, gate, ops._GATE_ACT[gate_act], scale, keep, alpha,
                                                 ops._NORM[pre], pre_weight, pre_bias, eps, samples or 0,
                                                 sinks if any(s is not None for s in sinks) else [])
    # parameters whose gradients an engine.GradReducer waits for (its callbacks are Python), and traced calls: the same node in Python
    _lib.native().refuse_watchers([x, branch, gate, keep, *vectors])
    shape = x.shape
    if len(shape) < 2 or branch.shape != shape:
        raise ValueError(f'gated_residual_norm: x {tuple(shape)} and branch {tuple(branch.shape)} must be alike, [..., C]')
    C, total, device = shape[-1], x.numel(), x.device
    if total == 0:
        raise ValueError(f'gated_residual_norm: nothing in x {tuple(shape)}')
    rows = total // C
    if samples is None:
        samples = shape[0] if len(shape) > 2 else 1
    if samples < 1 or rows % samples:
        raise ValueError(f'gated_residual_norm: {rows} rows do not divide into {samples} samples')
    mode = 0
    if gate is not None:
        mode = 2 if gate.shape == shape else 1 if gate.shape == (samples, C) else 0
        if mode == 0 or gate.dtype != branch.dtype:
            raise ValueError(f'gated_residual_norm: gate must be {branch.dtype} [{samples}, {C}] or like x, got {gate.dtype} {tuple(gate.shape)}')
    ops._dev(x)
    if branch.device != device or (mode and gate.device != device):
        raise ValueError('gated_residual_norm: x, branch and gate must be on one device')
    if (x.dtype, branch.dtype) not in ops._STREAMS:
        raise TypeError(f'gated_residual_norm: stream / branch types must be f32 / f32, bf16 / bf16 or f32 / bf16, got {x.dtype} / {branch.dtype}')
    post_k, pre_k, act = ops._resnorm_vectors(C, samples, device, gate_act, scale, keep, post, post_weight, post_bias, pre, pre_weight, pre_bias,
                                              'gated_residual_norm')
    if torch.is_grad_enabled() and (x.requires_grad or branch.requires_grad or (mode and gate.requires_grad) or
                                    any(t is not None and t.requires_grad for t in vectors)):
        return _ResnormFn.apply(x, branch, gate, keep, (rows, rows // samples, C, mode, post_k, pre_k, act, float(alpha), float(eps)), *vectors)
    xs, ldx = _rows(x, C)
    bs, ldb = _rows(branch, C)
    gs, ldg = _rows(gate, C) if mode else (None, 0)
    return ops._resnorm_launch_fwd(xs, ldx, bs, ldb, gs, ldg, mode, act, scale, keep, alpha, post_k, post_weight, post_bias, pre_k, pre_weight, pre_bias, eps,
                                   False, rows, rows // samples, C, shape)[:2]


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
