"""AdamW restated twice: in 64 bits, and its 8-bit moments operation by operation in IEEE single precision (numpy rounds each product and
sum once, as the definition of the code asks), so that codes can be compared for equality."""
import math

import numpy as np

RUN = 256
F = np.float32


def step64(p, g, m, v, t, lr, betas, eps, wd, coef=1.0):
    """numpy float64 arrays -> p, m, v after step t (t counted from 1)"""
    b1, b2 = betas
    g = g * coef
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * (1 - lr * wd) - lr / (1 - b1 ** t) * m / (np.sqrt(v) / math.sqrt(1 - b2 ** t) + eps), m, v


def clip_coef(grads, max_norm, grad_scale=1.0):
    """-> norm after grad_scale, what each gradient is multiplied by"""
    norm = math.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in grads)) * grad_scale
    return norm, grad_scale * (min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0)


def mix32(x):
    x = np.asarray(x, dtype=np.uint64)
    for shift, mul in ((16, 0x9E3779B9), (15, 0xBB67AE85)):
        x = x ^ (x >> np.uint64(shift))
        x = (x * np.uint64(mul)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def draws(runs, t, seed):
    """-> two [len(runs), 256] arrays of 0..65535"""
    low = np.uint64(0xFFFFFFFF)
    key = mix32(np.uint64(seed) ^ mix32(np.uint64(t) & low))
    rk = mix32((key + np.asarray(runs, dtype=np.uint64) * np.uint64(0xBB67AE85)) & low)[:, None]
    h = mix32((rk + np.arange(RUN, dtype=np.uint64) * np.uint64(0x9E3779B9)) & low)
    return (h & np.uint64(0xFFFF)).astype(F), (h >> np.uint64(16)).astype(F)


def grid(power):
    c = np.arange(128 if power == 2 else 256, dtype=F)
    return c * c if power == 2 else (c * c) * (c * c)


def decode(codes, scale, power):
    """[runs, 256] codes, [runs] scales -> moments (float32)"""
    c = codes.astype(F)
    return (c * np.abs(c) if power == 2 else (c * c) * (c * c)) * scale.astype(F)[:, None]


def encode(x, u16, power):
    """x >= 0 [runs, 256] float32 -> codes, scales"""
    table = grid(power)
    big = x.max(1)
    with np.errstate(all='ignore'):
        big = np.where(np.isnan(x).any(1), F(np.nan), big).astype(F)
        q = np.where(big < F(1e-28), F(0), big * F(1.0 / 16129.0 if power == 2 else 1.0 / 65025.0 ** 2)).astype(F)
        inv = np.where(q > 0, F(1) / q, F(0)).astype(F)
        t = x * inv[:, None]
        lo = np.clip(np.searchsorted(table, np.nan_to_num(t, nan=0.0), side='right') - 1, 0, len(table) - 2)
        gap = table[lo + 1] - table[lo]
        code = lo + ((t - table[lo]) * F(65536) > u16 * gap)
        if power == 4:
            code = np.where((code == 0) & (t > 0), 1, code)
    return code, q


def moments8(g, cm, qm, cv, qv, t, seed, runs, betas, coef):
    """One tensor's run-padded [runs, 256] gradient (float32) and 8-bit state -> new state, and the moments before they were rounded"""
    b1, b2 = betas
    um, uv = draws(runs, t, seed)
    g = g.astype(F) * F(coef)
    m = decode(cm, qm, 2) * F(b1) + g * F(1 - b1)
    v = decode(cv, qv, 4) * F(b2) + (g * g) * F(1 - b2)
    nm, nqm = encode(np.abs(m), um, 2)
    nv, nqv = encode(v, uv, 4)
    return (nm * np.where(m < 0, -1, 1)).astype(np.int8), nqm, nv.astype(np.uint8), nqv, m, v
