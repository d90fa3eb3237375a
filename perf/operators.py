"""The operators of a transformer block's training step around its matrix products, as they are measured.

Two families, each with its plain form (elementary torch operations), its definition in 64 bits (``exact``) and, where ``own`` is
true, the calls that a user of this package makes:

``resnorm``   the residual update between two blocks with a norm on either side of it.  For rows r of a stream x and a block's output b
              (sample s = r // N):

                  n = post(b)                                        no norm, LayerNorm or RMSNorm over the C channels
                  h = alpha x + keep[s] scale act(gate) n            LayerScale, a gate per sample or per row, DropPath, residual scale
                  y = pre(h)                                         the next block's norm, over the STORED h (rounded to x's type)

              ``infer``: h and y.  ``train``: h and y, and from their gradients dh and dy those of x, b, gate, scale and both norms.
``adamw``     one AdamW step over a model's tensors with the gradient clipped by its global norm.  The two moments are held in 32 bits
              or in 8.  In 8 bits each run of 256 elements of a tensor has one scale q per moment and

                  first moment  = sign(c) c^2 q    with -127 <= c <= 127
                  second moment = c^4 q            with    0 <= c <= 255, never 0 for a positive moment

              and a moment is stored on one of the two neighbouring codes, drawn so that its expectation is the moment itself (a moving
              average with weight 0.999 moves by far less than one step of any 8-bit code; rounding to nearest would hold it still).
              The draws are a hash of (seed, step, run, element), so the seed is an input and a step repeats itself exactly.
"""
import math

import torch

own = False

RUN = 256                    # elements of a tensor that share one scale
M32 = 0xFFFFFFFF
DT = {'f32': torch.float32, 'bf16': torch.bfloat16}


# ------------------------------------------------------------------ the cases
def _rn(name, mode, B, N, C, stream, branch, post, pre, gate='none', act='none', scale=True, keep=False, alpha=1.0):
    return {'name': name, 'op': 'resnorm', 'mode': mode, 'B': B, 'N': N, 'C': C, 'stream': stream, 'branch': branch, 'post': post, 'pre': pre,
            'gate': gate, 'act': act, 'scale': scale, 'keep': keep, 'alpha': alpha}


def _opt(name, bits, model, dtype, clip=1.0, step=100):
    return {'name': name, 'op': 'adamw', 'bits': bits, 'model': model, 'dtype': dtype, 'clip': clip, 'step': step}


def listed():
    return [
        # one token through a 512-wide block, gated and normed on both sides: the launch is the cost
        _rn('token_512_bf16', 'infer', 1, 1, 512, 'bf16', 'bf16', 'rms', 'rms', gate='row'),
        # a batch of single tokens at a generic large width
        _rn('tokens_64x4096_bf16', 'infer', 64, 1, 4096, 'bf16', 'bf16', 'rms', 'rms'),
        # MiT stage 1 of the default benchmark (16 tiles of 1024 x 1024): 256 x 256 tokens a tile, 64 channels, DropPath, LayerScale
        _rn('mit_stage1_train_bf16', 'train', 16, 65536, 64, 'bf16', 'bf16', 'none', 'layer', keep=True),
        # ConvNeXt-T stage 3 of the same tiles with norms on both sides and a gate per tile (conditioned blocks)
        _rn('convnext_stage3_train_bf16', 'train', 16, 4096, 384, 'bf16', 'bf16', 'layer', 'layer', gate='sample', keep=True),
        # odd channel and row counts in single precision, a sigmoid gate for every element, a weighted residual
        _rn('odd_97_train_f32', 'train', 3, 1741, 97, 'f32', 'f32', 'rms', 'layer', gate='row', act='sigmoid', alpha=1.25),
        # a wide model that keeps its stream in 32 bits and its blocks in bf16
        _rn('wide_4096_train_mixed', 'train', 4, 2048, 4096, 'f32', 'bf16', 'rms', 'rms', gate='row', act='sigmoid'),
        # a classifier head fine-tuned alone: few small tensors, the launches are the cost
        _opt('adamw_head_f32', 32, 'head', 'f32'),
        # the encoder of the default benchmark
        _opt('adamw_mit_b2_f32', 32, 'mit_B2', 'f32'),
        # a model held in bf16 altogether, moments in 32 bits
        _opt('adamw_convnext_t_bf16', 32, 'convnext_T', 'bf16'),
        # the smallest encoder with moments in 8 bits
        _opt('adamw8_mit_b0_f32', 8, 'mit_B0', 'f32'),
        # tensors of ragged sizes, from one element on, in bf16
        _opt('adamw8_ragged_bf16', 8, 'ragged_40', 'bf16', step=7),
        # the largest encoder, where 8-bit moments save the most
        _opt('adamw8_mit_b5_f32', 8, 'mit_B5', 'f32'),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.6:
        C = _log_int(rng, 8, 4096)
        if rng.random() < 0.5:
            C = max(8, C // 8 * 8)
        mode = rng.choice(['infer', 'train', 'train'])
        B = rng.randint(1, 16)
        N = max(1, _log_int(rng, 1, 30e6 / C) // B)
        stream, branch = rng.choice([('f32', 'f32'), ('bf16', 'bf16'), ('f32', 'bf16')])
        gate = rng.choice(['none', 'sample', 'row'])
        # a sigmoid is drawn for streams in 32 bits: on a bf16 stream the last bit of exp() decides which way some h round, and with
        # them the weight gradient of the norm behind it, in 32 bits, changes by more than 32 bits say
        act = rng.choice(['none', 'sigmoid']) if gate != 'none' and stream == 'f32' else 'none'
        c = _rn('', mode, B, N, C, stream, branch, rng.choice(['none', 'layer', 'rms']), rng.choice(['layer', 'rms']), gate, act,
                rng.random() < 0.7, rng.random() < 0.4, rng.choice([1.0, 1.0, 0.5, 1.4142]))
    else:
        model = rng.choice(['mit_B0', 'mit_B1', 'mit_B2', 'mit_B3', 'convnext_T', 'convnext_S', 'ragged_%d' % rng.randint(1, 400),
                            'ragged_%d' % rng.randint(1, 400)])
        c = _opt('', rng.choice([32, 8]), model, rng.choice(['f32', 'f32', 'bf16']), rng.choice([1.0, 0.0]), _log_int(rng, 1, 100000))
    del c['name']
    return c


# ------------------------------------------------------------------ tensor sizes of the models this package has
def _mit_sizes(variant):
    dims, depths = {'B0': ((32, 64, 160, 256), (2, 2, 2, 2)), 'B1': ((64, 128, 320, 512), (2, 2, 2, 2)), 'B2': ((64, 128, 320, 512), (3, 4, 6, 3)),
                    'B3': ((64, 128, 320, 512), (3, 4, 18, 3)), 'B5': ((64, 128, 320, 512), (3, 6, 40, 3))}[variant]
    out, cin = [], 3
    for c, depth, sr, k in zip(dims, depths, (8, 4, 2, 1), (7, 3, 3, 3)):
        out += [(c, cin * k * k), (c,), (c,), (c,)]
        for _ in range(depth):
            out += [(c,), (c,), (c, c), (c,), (2 * c, c), (2 * c,), (c, c), (c,)]
            out += [(c, c * sr * sr), (c,), (c,), (c,)] if sr > 1 else []
            out += [(c,), (c,), (4 * c, c), (4 * c,), (4 * c, 9), (4 * c,), (c, 4 * c), (c,)]
        out += [(c,), (c,)]
        cin = c
    return out


def _convnext_sizes(variant):
    depths, dims = {'T': ((3, 3, 9, 3), (96, 192, 384, 768)), 'S': ((3, 3, 27, 3), (96, 192, 384, 768))}[variant]
    out, cin = [], 3
    for c, depth, k in zip(dims, depths, (4, 2, 2, 2)):
        out += [(c, cin * k * k), (c,), (c,), (c,)]
        for _ in range(depth):
            out += [(c,), (c, 49), (c,), (c,), (c,), (4 * c, c), (4 * c,), (c, 4 * c), (c,)]
        out += [(c,), (c,)]
        cin = c
    return out


def _sizes(model):
    """Shapes of the tensors: matrices decay, vectors do not."""
    kind, _, what = model.partition('_')
    if kind == 'head':
        return [(256, 256), (256,), (256,), (6, 256), (6,)]
    if kind == 'mit':
        return _mit_sizes(what)
    if kind == 'convnext':
        return _convnext_sizes(what)
    return [(1 + (i * i * 7919) % 8191, 1 + (i * 131) % 67) if i % 3 else (1 + (i * 977) % 1500,) for i in range(int(what))]


class _Layout:
    """Every tensor in a slot of whole runs of one flat buffer, last tensor first (the order in which a backward pass makes gradients)."""

    def __init__(self, model):
        self.shapes = _sizes(model)
        self.slots, at, decays = [], 0, []
        for shape in reversed(self.shapes):
            n = math.prod(shape)
            runs = -(-n // RUN)
            self.slots.append((at, n, shape))
            decays += [1.0 if len(shape) > 1 else 0.0] * runs
            at += runs * RUN
        self.total, self.used, self.decays = at, sum(n for _, n, _ in self.slots), decays


HYPER = {'lr': 6e-4, 'b1': 0.9, 'b2': 0.999, 'eps': 1e-8, 'wd': 0.05, 'seed': 12345}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(int(seed) * 2 + 1)


def _prepare_resnorm(case, seed):
    g = _gen(seed)
    B, N, C = case['B'], case['N'], case['C']
    tx, tb = DT[case['stream']], DT[case['branch']]

    def rnd(*shape, dtype=torch.float32, scale=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device='cuda') * scale + mean).to(dtype)

    s = {'case': case, 'x': rnd(B, N, C, dtype=tx, scale=2.0, mean=0.3), 'b': rnd(B, N, C, dtype=tb, mean=-0.2)}
    s['gate'] = None if case['gate'] == 'none' else rnd(B, C, dtype=tb) if case['gate'] == 'sample' else rnd(B, N, C, dtype=tb)
    s['scale'] = rnd(C, scale=0.05, mean=0.1) if case['scale'] else None
    # DropPath as it is drawn: dropped, or divided by the probability of being kept
    s['keep'] = (torch.rand(B, generator=g, device='cuda') < 0.9).float() / 0.9 if case['keep'] else None
    for k in ('post', 'pre'):
        s[k + '_w'] = rnd(C, scale=0.2, mean=1.0) if case[k] != 'none' else None
        s[k + '_b'] = rnd(C, scale=0.2) if case[k] == 'layer' else None
    if case['mode'] == 'train':
        s['dh'], s['dy'] = rnd(B, N, C, dtype=tx), rnd(B, N, C, dtype=tb)
        if own:                                                # leaves of the user's graph
            for k in ('x', 'b', 'gate', 'scale', 'post_w', 'post_b', 'pre_w', 'pre_b'):
                if s[k] is not None:
                    s[k].requires_grad_()
    return s


def _prepare_adamw(case, seed):
    g = _gen(seed)
    lay = _Layout(case['model'])
    T = DT[case['dtype']]
    live = torch.zeros(lay.total, dtype=torch.bool, device='cuda')
    for at, n, _ in lay.slots:
        live[at:at + n] = True

    def rnd(scale):
        return torch.randn(lay.total, generator=g, device='cuda').mul_(live).mul_(scale)

    # gradients whose size differs from run to run by a few powers of ten, some rows all zero
    size = torch.exp(torch.randn(lay.total // RUN, 1, generator=g, device='cuda') * 1.5 - 6.0)
    size = size * (torch.rand(lay.total // RUN, 1, generator=g, device='cuda') > 0.02)
    s = {'case': case, 'layout': lay, 't': case['step']}
    s['p'] = rnd(0.05).to(T)
    s['g'] = (rnd(1.0).view(-1, RUN) * size).view(-1).to(T)
    m = (rnd(0.3).view(-1, RUN) * size).view(-1)
    v = (rnd(1.0).view(-1, RUN) * size).square().view(-1).mul_(0.9).add_(size.square().mul(0.1).expand(-1, RUN).reshape(-1) * live)
    if case['bits'] == 32:
        s['m'], s['v'] = m, v
    else:
        for k, x, top, power in (('m', m, 127.0, 2), ('v', v, 255.0, 4)):
            x = x.view(-1, RUN)
            q = x.abs().amax(1, keepdim=True) / top ** power
            c = (x.abs() / q.clamp_min(1e-38)).pow(1.0 / power).round().clamp(max=top)
            c = torch.where((x > 0) & (c == 0), torch.ones_like(c), c) if k == 'v' else c * x.sign()
            s[k] = c.to(torch.int8 if k == 'm' else torch.uint8).view(-1)
            s['q' + k] = q.view(-1)
    s['decays'] = torch.tensor(lay.decays, device='cuda')[:, None]
    if own:
        from semseg_amd.engine import AdamW, FlatParams
        opts = dict(lr=HYPER['lr'], betas=(HYPER['b1'], HYPER['b2']), eps=HYPER['eps'], weight_decay=HYPER['wd'], max_grad_norm=case['clip'] or None,
                    state_bits=case['bits'], seed=HYPER['seed'], per_param=lambda p: {'weight_decay': 0.0} if p.dim() <= 1 else {})
        if T == torch.float32:                                 # the trainer's flat parameters
            net = torch.nn.ParameterList([torch.nn.Parameter(torch.empty(shape, device='cuda')) for shape in lay.shapes])
            flat = FlatParams(net, align=RUN)
            flat.data.copy_(s['p']), flat.grad.copy_(s['g'])
            s['p'], s['opt'] = flat.data, AdamW(flat, **opts)
        else:                                                  # a list of tensors of their own
            params = []
            for at, n, shape in lay.slots:
                params.append(torch.nn.Parameter(s['p'][at:at + n].view(shape)))
                params[-1].grad = s['g'][at:at + n].view(shape)
            s['opt'] = AdamW(params, **opts)
        opt = s['opt']
        opt.exp_avg.copy_(s['m']), opt.exp_avg_sq.copy_(s['v'])
        if case['bits'] == 8:
            opt.exp_avg_scale.copy_(s['qm']), opt.exp_avg_sq_scale.copy_(s['qv'])
        opt.t = case['step']
    return s


def prepare(case, seed):
    return (_prepare_resnorm if case['op'] == 'resnorm' else _prepare_adamw)(case, seed)


# ------------------------------------------------------------------ resnorm, plain
def _stats(v, kind, eps):
    """Row mean and 1 / deviation.  The sums are taken in 64 bits: h is rounded to the stream's type, and an h next to the border of two
    values must not change sides with the order of a sum."""
    d = v.double()
    mu = d.mean(-1, keepdim=True) if kind == 'layer' else torch.zeros_like(d[..., :1])
    var = d.square().mean(-1, keepdim=True) - mu.square()
    return mu.float(), (1.0 / (var.clamp_min(0) + eps).sqrt()).float()


def _norm(v, kind, w, b):
    if kind == 'none':
        return v, None, None
    mu, r = _stats(v, kind, 1e-6)
    hat = (v - mu) * r if kind == 'layer' else v * r
    n = hat * w
    return (n if b is None else n + b), hat, r


def _norm_back(dn, hat, r, kind, w):
    """-> gradient of the norm's input, of its weight, of its bias"""
    if kind == 'none':
        return dn, None, None
    g = dn * w
    s2 = (g * hat).mean(-1, keepdim=True)
    dv = r * (g - hat * s2 - g.mean(-1, keepdim=True)) if kind == 'layer' else r * (g - hat * s2)
    rows = tuple(range(dn.dim() - 1))
    return dv, (dn * hat).sum(rows), dn.sum(rows) if kind == 'layer' else None


def _resnorm_plain(s):
    case = s['case']
    tx, tb = s['x'].dtype, s['b'].dtype
    per = lambda t: t[:, None, :] if case['gate'] == 'sample' else t  # noqa: E731
    gate = None if s['gate'] is None else per(s['gate'].float())
    a = None if gate is None else 1.0 / (1.0 + torch.exp(-gate)) if case['act'] == 'sigmoid' else gate
    keep = None if s['keep'] is None else s['keep'][:, None, None]
    n, nhat, rn = _norm(s['b'].float(), case['post'], s['post_w'], s['post_b'])
    f = n if a is None else n * a
    f = f if s['scale'] is None else f * s['scale']
    f = f if keep is None else f * keep
    h = (s['x'].float() * case['alpha'] + f).to(tx)
    y, hhat, rh = _norm(h.float(), case['pre'], s['pre_w'], s['pre_b'])
    out = {'h': h, 'y': y.to(tb)}
    if case['mode'] == 'infer':
        return out
    dH, out['pre_w'], out['pre_b'] = _norm_back(s['dy'].float(), hhat, rh, case['pre'], s['pre_w'])
    dH = dH + s['dh'].float()
    out['x'] = (dH * case['alpha']).to(tx)
    dk = dH if keep is None else dH * keep
    if s['scale'] is not None:
        out['scale'] = (dk * n if a is None else dk * n * a).sum((0, 1))
        dk = dk * s['scale']
    if a is not None:
        da = dk * n
        da = da * a * (1.0 - a) if case['act'] == 'sigmoid' else da
        out['gate'] = (da.sum(1) if case['gate'] == 'sample' else da).to(tb)
        dk = dk * a
    db, out['post_w'], out['post_b'] = _norm_back(dk, nhat, rn, case['post'], s['post_w'])
    out['b'] = db.to(tb)
    return {k: v for k, v in out.items() if v is not None}


def _resnorm_own(s):
    from semseg_amd.resnorm import gated_residual_norm
    case = s['case']
    h, y = gated_residual_norm(s['x'], s['b'], post=case['post'], post_weight=s['post_w'], post_bias=s['post_b'], gate=s['gate'],
                               gate_act=case['act'], scale=s['scale'], keep=s['keep'], alpha=case['alpha'], pre=case['pre'],
                               pre_weight=s['pre_w'], pre_bias=s['pre_b'], eps=1e-6)
    if case['mode'] == 'infer':
        return {'h': h, 'y': y}
    names = [k for k in ('x', 'b', 'gate', 'scale', 'post_w', 'post_b', 'pre_w', 'pre_b') if s[k] is not None]
    grads = torch.autograd.grad((h, y), [s[k] for k in names], (s['dh'], s['dy']))
    return {'h': h.detach(), 'y': y.detach(), **dict(zip(names, grads))}


# ------------------------------------------------------------------ adamw, plain
def _mix(x):
    """32 bits to 32 bits, every bit of the input in every bit of the result (multipliers: the fractions of the golden ratio and of the root of 3)."""
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B9) & M32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & M32
    return x ^ (x >> 16)


def _draws(total, t, seed):
    """Two 16-bit numbers for every element."""
    key = _mix((seed & M32) ^ _mix(t & M32))
    runs = torch.arange(total // RUN, dtype=torch.int64, device='cuda')[:, None]
    lane = torch.arange(RUN, dtype=torch.int64, device='cuda')[None, :]
    r = _mix((_mix((key + runs * 0xBB67AE85) & M32) + lane * 0x9E3779B9) & M32)
    return (r & 0xFFFF).float() / 65536.0, (r >> 16).float() / 65536.0


def _store(x, top, power, u, q_of):
    """x >= 0 [runs, RUN] -> (codes, scales): the code below x or the one above it, above with the chance that makes the mean x."""
    big = x.amax(1, keepdim=True)
    q = torch.where(big >= 1e-28, big * q_of, torch.zeros_like(big))     # what is smaller is held as zero
    inv = torch.where(q > 0, torch.ones_like(q) / q, torch.zeros_like(q))
    t = x * inv
    c = torch.arange(int(top) + 1, dtype=torch.float32, device=x.device)
    grid = (c * c) if power == 2 else (c * c) * (c * c)
    lo = (torch.bucketize(t, grid, right=True) - 1).clamp_(0, int(top) - 1)
    below, above = grid[lo], grid[lo + 1]
    return lo + ((t - below) > u * (above - below)), q, t


def _adamw_plain(s):
    case, lay, hy = s['case'], s['layout'], HYPER
    s['t'] += 1
    t = s['t']
    g = s['g'].float()
    if case['clip']:
        norm = g.double().square().sum().sqrt()
        g = g * (case['clip'] / (norm + 1e-6)).clamp(max=1.0).float()
    if case['bits'] == 8:
        cm, cv = s['m'].float().view(-1, RUN), s['v'].float().view(-1, RUN)
        m, v = (cm * cm.abs() * s['qm'][:, None]).view(-1), ((cv * cv) * (cv * cv) * s['qv'][:, None]).view(-1)
    else:
        m, v = s['m'], s['v']
    m = m * hy['b1'] + g * (1 - hy['b1'])
    v = v * hy['b2'] + (g * g) * (1 - hy['b2'])
    denom = v.sqrt() / math.sqrt(1 - hy['b2'] ** t) + hy['eps']
    p = s['p'].float().view(-1, RUN) * (1 - hy['lr'] * hy['wd'] * s['decays'])
    s['p'].copy_(p.view(-1) - (hy['lr'] / (1 - hy['b1'] ** t)) * m / denom)
    if case['bits'] == 32:
        s['m'], s['v'] = m, v
    else:
        um, uv = _draws(lay.total, t, hy['seed'])
        m, v = m.view(-1, RUN), v.view(-1, RUN)
        c, q, _ = _store(m.abs(), 127, 2, um, 1.0 / 16129.0)
        cm, s['qm'] = c * m.sign(), q.view(-1)
        s['m'] = cm.to(torch.int8).view(-1)
        c, q, x = _store(v, 255, 4, uv, 1.0 / 65025.0 ** 2)
        cv, s['qv'] = torch.where((x > 0) & (c == 0), torch.ones_like(c), c), q.view(-1)
        s['v'] = cv.to(torch.uint8).view(-1)
        cm, cv = cm.float(), cv.float()
        m, v = (cm * cm.abs() * s['qm'][:, None]).view(-1), ((cv * cv) * (cv * cv) * s['qv'][:, None]).view(-1)
    return {'p': s['p'], 'm': m, 'v': v, **({'norm': norm.float()} if case['clip'] else {})}


def _adamw_own(s):
    norm = s['opt'].step()
    m, v = (s['opt'].exp_avg, s['opt'].exp_avg_sq) if s['case']['bits'] == 32 else s['opt'].state_values()
    return {'p': s['p'], 'm': m, 'v': v, **({'norm': norm} if s['case']['clip'] else {})}


def run(state):
    if state['case']['op'] == 'resnorm':
        return _resnorm_own(state) if own else _resnorm_plain(state)
    return _adamw_own(state) if own else _adamw_plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case['op'] == 'resnorm':
        rows, C = case['B'] * case['N'], case['C']
        sx, sb = (4 if case[k] == 'f32' else 2 for k in ('stream', 'branch'))
        gate = sb * {'none': 0, 'sample': case['B'] * C, 'row': rows * C}[case['gate']]
        vectors = 4 * C * (bool(case['scale']) + sum({'none': 0, 'rms': 1, 'layer': 2}[case[k]] for k in ('post', 'pre')))
        once = rows * C * (2 * sx + 2 * sb) + gate + vectors               # x, b, the gate and the vectors in; h and y out
        train = case['mode'] == 'train'                                    # the same again: dh, dy in; dx, db and the other gradients out
        return {'bytes': once * (2 if train else 1), 'flops': rows * C * (60 if train else 20)}
    n, size = _Layout(case['model']).used, 4 if case['dtype'] == 'f32' else 2
    if case['bits'] == 32:
        return {'bytes': n * (3 * size + 16), 'flops': 16 * n}             # p and g in, p out; both moments in and out
    return {'bytes': n * (3 * size + 2 + 2 + 8) + n // RUN * 16, 'flops': 60 * n}   # 8-bit moments in and out, and the values they stand for out


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_norm(v, kind, w, b):
    if kind == 'none':
        return v
    c = v - v.mean(-1, keepdim=True) if kind == 'layer' else v
    n = c / (c.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w
    return n if b is None else n + b


def _exact_resnorm(case, seed):
    s = _prepare_resnorm(case, seed)
    L = {k: s[k].detach().double().requires_grad_() for k in ('x', 'b', 'gate', 'scale', 'post_w', 'post_b', 'pre_w', 'pre_b') if s[k] is not None}
    with torch.enable_grad():
        f = _exact_norm(L['b'], case['post'], L.get('post_w'), L.get('post_b'))
        if 'gate' in L:
            a = torch.sigmoid(L['gate']) if case['act'] == 'sigmoid' else L['gate']
            f = f * (a.unsqueeze(1) if case['gate'] == 'sample' else a)
        if 'scale' in L:
            f = f * L['scale']
        if s['keep'] is not None:
            f = f * s['keep'].double().view(-1, 1, 1)
        h = case['alpha'] * L['x'] + f
        held = h.detach().to(s['x'].dtype).double().requires_grad_()       # the stream as it is stored
        y = _exact_norm(held, case['pre'], L.get('pre_w'), L.get('pre_b'))
    out = {'h': held.detach(), 'y': y.detach()}
    if case['mode'] == 'train':
        behind = [k for k in ('pre_w', 'pre_b') if k in L]
        got = torch.autograd.grad(y, [held] + [L[k] for k in behind], s['dy'].double())
        out.update(zip(behind, got[1:]))
        front = [k for k in L if k not in behind]
        out.update(zip(front, torch.autograd.grad(h, front and [L[k] for k in front], got[0] + s['dh'].double())))
        if case['stream'] == 'bf16':
            # an h next to the border of two bf16 values goes to one side in 32 bits and to the other in 64; this gradient multiplies
            # each by a gradient of its own and has 32 bits itself, which say less than that
            out['pre_w'] = None
    return out


def _exact_adamw(case, seed):
    s = _prepare_adamw(case, seed)
    p, g = (s[k].detach().double() for k in ('p', 'g'))
    t = case['step'] + 1
    b1, b2 = HYPER['b1'], HYPER['b2']
    norm = torch.linalg.vector_norm(g)
    if case['clip']:
        g = g * min(1.0, case['clip'] / (float(norm) + 1e-6))
    m, v = s['m'].double(), s['v'].double()
    if case['bits'] == 8:
        m = m.sign() * m ** 2 * s['qm'].double().repeat_interleave(RUN)
        v = v ** 4 * s['qv'].double().repeat_interleave(RUN)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    decay = 1 - HYPER['lr'] * HYPER['wd'] * s['decays'].double().view(-1).repeat_interleave(RUN)
    p = p * decay - HYPER['lr'] * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + HYPER['eps'])
    # which of two codes a moment takes is a comparison: 32 and 64 bits decide differently for a few, which are then a whole step apart
    eight = case['bits'] == 8
    return {'p': p, 'm': None if eight else m, 'v': None if eight else v, **({'norm': norm} if case['clip'] else {})}


def exact(case, seed):
    return (_exact_resnorm if case['op'] == 'resnorm' else _exact_adamw)(case, seed)
