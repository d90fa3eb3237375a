"""The residual update between two norms (semseg_amd/resnorm.py) restated in 64 bits, formulas written out.  Next to every value stands its
``mag``: the sum of the absolute values of the terms it is made of, which is what rounding errors of its computation are relative to."""
import torch


def _norm(v, kind, w, b, eps):
    """-> (n, mag), normalised rows (hat, mag), 1 / deviation"""
    if kind == 'none':
        return (v, v.abs()), (v, v.abs()), torch.ones_like(v[:, :1])
    mu = v.mean(1, keepdim=True) if kind == 'layer' else torch.zeros_like(v[:, :1])
    r = ((v - mu).pow(2).mean(1, keepdim=True) + eps).rsqrt()
    hat, mag = (v - mu) * r, (v.abs() + mu.abs()) * r
    n, nmag = hat * w, mag * w.abs()
    return (n, nmag) if b is None else (n + b, nmag + b.abs()), (hat, mag), r


def _norm_back(dn, dmag, hat, hmag, r, kind, w):
    if kind == 'none':
        return (dn, dmag), None, None
    g, gmag = dn * w, dmag * w.abs()
    dv = g - hat * (g * hat).mean(1, keepdim=True)
    mag = gmag + hmag * (gmag * hmag).mean(1, keepdim=True)
    if kind == 'layer':
        dv, mag = dv - g.mean(1, keepdim=True), mag + gmag.mean(1, keepdim=True)
    weight = (dn * hat).sum(0), (dmag * hmag).sum(0)
    return (r * dv, r * mag), weight, (dn.sum(0), dmag.sum(0)) if kind == 'layer' else None


def resnorm(x, b, h_stored=None, dh=None, dy=None, rows_per_sample=0, gate=None, gate_act='none', scale=None, keep=None, alpha=1.0, post='none', post_w=None,
            post_b=None, pre='none', pre_w=None, pre_b=None, eps=1e-6):
    """Tensors as the entry points take them (CPU).  ``h_stored``: the stream as it was stored, which everything behind h is computed from.
    -> {name: (value, mag)} for h, y and, with dh or dy, x, b, gate, pre_w, pre_b, post_w, post_b, scale."""
    D = lambda t: None if t is None else t.detach().double()  # noqa: E731
    x, b, gate, scale, keep, post_w, post_b, pre_w, pre_b, dh, dy = map(D, (x, b, gate, scale, keep, post_w, post_b, pre_w, pre_b, dh, dy))
    rows, C = x.shape
    n_rows = rows_per_sample or rows
    of = torch.arange(rows) // n_rows
    per_row = gate is not None and gate.shape[0] == rows
    a = torch.ones_like(x) if gate is None else gate if per_row else gate[of]
    slope, amag = torch.ones_like(a), a.abs()
    if gate_act == 'sigmoid':
        a = torch.sigmoid(a)
        slope, amag = a * (1 - a), a
    s = (torch.ones(C, dtype=torch.float64) if scale is None else scale) * (torch.ones(rows, 1, dtype=torch.float64) if keep is None else keep[of, None])
    (n, nmag), (nhat, nhmag), rn = _norm(b, post, post_w, post_b, eps)
    out = {'h': (alpha * x + s * a * n, abs(alpha) * x.abs() + s.abs() * amag * nmag)}
    hs = out['h'][0] if h_stored is None else h_stored.detach().double()
    (y, ymag), (hhat, hhmag), rh = _norm(hs, pre, pre_w, pre_b, eps)
    if pre != 'none':
        out['y'] = (y, ymag)
    if dh is None and dy is None:
        return out
    d, dmag = torch.zeros_like(x), torch.zeros_like(x)
    if pre != 'none':
        g = torch.zeros_like(x) if dy is None else dy
        (d, dmag), out['pre_w'], out['pre_b'] = _norm_back(g, g.abs(), hhat, hhmag, rh, pre, pre_w)
    if dh is not None:
        d, dmag = d + dh, dmag + dh.abs()
    out['x'] = (alpha * d, abs(alpha) * dmag)
    k = torch.ones(rows, 1, dtype=torch.float64) if keep is None else keep[of, None]
    if scale is not None:
        out['scale'] = ((d * k * a * n).sum(0), (dmag * k.abs() * amag * nmag).sum(0))
    if gate is not None:
        dg, gmag = d * s * n * slope, dmag * s.abs() * nmag * (amag if gate_act == 'sigmoid' else 1.0)
        if not per_row:
            dg, gmag = (t.view(-1, n_rows, C).sum(1) for t in (dg, gmag))
        out['gate'] = (dg, gmag)
    out['b'], out['post_w'], out['post_b'] = _norm_back(d * s * a, dmag * s.abs() * amag, nhat, nhmag, rn, post, post_w)
    return {k_: v for k_, v in out.items() if v is not None}
