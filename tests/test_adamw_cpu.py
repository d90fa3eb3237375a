"""AdamW over many tensors: the plan, what is refused, and what the 8-bit code of the moments does (on its bit-exact restatement)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import adamw as oracle


def test_plan_covers_every_element_once():
    from semseg_amd.ops import ADAMW_RUN, TensorPlan
    for numels in ([1], [0, 5, 0], [255, 256, 257, 1023, 1024, 1025, 5000], [3_000_000, 7, 8192 * 3]):
        for offsets in (None, np.concatenate([[0], np.cumsum([-(-n // 64) * 64 for n in numels])])[:-1].tolist()):
            groups = [i % 3 for i in range(len(numels))]
            p = TensorPlan(numels, 'cpu', groups, offsets)
            rows = p.table.numpy()
            assert p.chunks == len(rows) and p.count == (1 if offsets is not None else len(numels))
            assert list(p.first_chunk)[0] == 0 and list(p.first_chunk)[-1] == len(rows)
            assert p.runs == sum(-(-n // ADAMW_RUN) for n in numels)
            k = 0
            for i, n in enumerate(numels):
                at = 0
                while at < n:
                    start, word, who, _ = (int(v) for v in rows[k])
                    count, run = word & 0xFFFFFFFF, word >> 32
                    assert start - (offsets[i] if offsets is not None else 0) == at and run == p.first_run[i] + at // ADAMW_RUN
                    assert who & 0xFFFFFFFF == (0 if offsets is not None else i) and who >> 32 == groups[i]
                    assert count % ADAMW_RUN == 0 or at + count == n
                    at, k = at + count, k + 1
                assert at == n
            assert k == len(rows)


def _lib():
    from semseg_amd._lib import lib
    return lib()


def _err():
    return _lib().ss_last_error().decode()


def _step(**kw):
    one = (ctypes.c_void_p * 1)(64)
    d = (ctypes.c_double * 1)(0.1)
    a = dict(pd=0, gd=0, bits=32, count=1, p=one, g=one, first=(ctypes.c_int64 * 2)(0, 1), plan=64, m=64, v=64, ms=None, vs=None, b1=0.9, b2=0.999, eps=1e-8,
             scale=1.0, t=1, groups=1, lr=d, wd=d, seed=0, dyn=None, stream=None)
    a.update(kw)
    return _lib().ss_adamw_step(*a.values())


@pytest.mark.parametrize('bad,text', [
    (dict(pd=2), 'dtype'), (dict(gd=-1), 'dtype'), (dict(bits=4), 'bits'), (dict(groups=0), 'groups'), (dict(groups=65), 'groups'), (dict(b1=1.0), 'betas'),
    (dict(b2=-0.1), 'betas'), (dict(scale=float('nan')), 'grad_scale'), (dict(count=-1), 'list'), (dict(first=(ctypes.c_int64 * 2)(1, 1)), 'list'),
    (dict(first=(ctypes.c_int64 * 2)(0, -1)), 'ranges'), (dict(p=(ctypes.c_void_p * 1)(None)), 'null'), (dict(p=(ctypes.c_void_p * 1)(66)), 'misaligned'),
    (dict(g=(ctypes.c_void_p * 1)(65), gd=1), 'misaligned'), (dict(plan=None), 'plan'), (dict(t=0), 'step count'), (dict(eps=-1.0), 'eps'), (dict(m=None), 'state'),
    (dict(v=72), 'state'), (dict(bits=8), 'state')])
def test_step_refusals_at_the_c_entry(bad, text):
    assert _step(**bad) != 0 and 'ss_adamw_step' in _err() and text in _err()


def test_other_refusals_at_the_c_entry():
    d = (ctypes.c_double * 1)(0.1)
    L = _lib()
    assert L.ss_multi_sqnorm(3, 0, None, None, None, None, None) != 0
    assert L.ss_multi_sqnorm(0, 1, (ctypes.c_void_p * 1)(64), (ctypes.c_int64 * 2)(0, 1), 64, None, None) != 0 and 'partial' in _err()
    assert L.ss_adamw_prepare(None, 3, 1.0, 1.0, 0.9, 0.999, 1, None, 1, d, d, None, 0, 0, None, 64, None) != 0
    assert L.ss_adamw_prepare(None, 0, 1.0, 1.0, 0.9, 0.999, 0, None, 1, d, d, None, 0, 0, None, 64, None) != 0
    assert L.ss_adamw_prepare(None, 0, 1.0, 1.0, 0.9, 0.999, 1, None, 1, d, d, None, 0, 0, None, None, None) != 0
    assert L.ss_adamw8_values(None, None, None, None, None, None, 1, None) != 0 and L.ss_adamw8_values(None, None, None, None, None, None, 0, None) == 0
    # nothing to do is not an error
    assert _step(first=(ctypes.c_int64 * 2)(0, 0), m=None, v=None) == 0 and _step(count=0) == 0


def test_python_refusals():
    from semseg_amd.engine import AdamW, FlatParams
    P = lambda *s, **k: torch.nn.Parameter(torch.zeros(*s, **k))  # noqa: E731
    a, b = P(4), P(5)
    for params, kw in (([], {}), ([a, a], {}), ([a, P(3, dtype=torch.float64)], {}), ([a, P(3, dtype=torch.bfloat16)], {}), ([torch.zeros(3, 4).t()], {}),
                       ([a], dict(state_bits=16)), ([a], dict(betas=(1.0, 0.9))), ([a], dict(lr=-1)), ([a], dict(max_grad_norm=0.0)),
                       ([a], dict(per_param=lambda p: {'momentum': 1})), ([P(1) for _ in range(65)], dict(per_param=lambda p, n=iter(range(99)): {'lr_scale': next(n)}))):
        with pytest.raises(ValueError):
            AdamW(params, **kw)
    with pytest.raises(RuntimeError, match='HIP device'):
        AdamW([a, b]).step()
    with pytest.raises(RuntimeError, match='HIP device'):
        AdamW(FlatParams(torch.nn.Linear(3, 4))).step()
    with pytest.raises(RuntimeError, match='capturable'):
        AdamW([a]).push_lr()
    bits8 = AdamW([a, b], state_bits=8)
    with pytest.raises(ValueError, match='bits'):
        bits8.load_state_dict(AdamW([a, b]).state_dict())


def test_state_dict_layout_and_torch_checkpoint():
    from semseg_amd.engine import AdamW, FlatParams
    net = torch.nn.Sequential(torch.nn.Linear(7, 5), torch.nn.Linear(5, 3))
    ref = torch.optim.AdamW(net.parameters(), lr=2e-3, weight_decay=0.1)
    for p in net.parameters():
        p.grad = torch.randn_like(p)
    ref.step()
    saved = ref.state_dict()
    for params in (list(net.parameters()), FlatParams(net)):
        opt = AdamW(params, per_param=lambda p: {'weight_decay': 0.0} if p.dim() == 1 else {})
        opt.load_state_dict(saved)
        assert (opt.t, opt.lr, opt.wd) == (1, 2e-3, 0.1)
        sd = opt.state_dict()
        for i, st in saved['state'].items():
            assert torch.equal(sd['state'][i]['exp_avg'], st['exp_avg']) and torch.equal(sd['state'][i]['exp_avg_sq'], st['exp_avg_sq'])
        assert sorted(i for g in sd['param_groups'] for i in g['params']) == [0, 1, 2, 3]
        again = AdamW(params, per_param=lambda p: {'weight_decay': 0.0} if p.dim() == 1 else {})
        again.load_state_dict(sd)
        assert torch.equal(again.exp_avg, opt.exp_avg) and again.t == 1


# ---------------------------------------------------------------------------------- the 8-bit code
@pytest.mark.parametrize('power', [2, 4])
def test_code_takes_a_neighbour_and_is_right_on_average(power):
    rng = np.random.default_rng(0)
    x = np.exp(rng.normal(0, 3, (8, 256))).astype(np.float32)
    x[:, 0] = 0
    table = oracle.grid(power).astype(np.float64)
    n, total = 4096, 0.0
    for k in range(n):
        code, q = oracle.encode(x, np.full(x.shape, (k * 16 + 7) % 65536, dtype=np.float32), power)
        v = table[code] * q[:, None]
        total = total + v
        if k % 512 == 0:
            t = x.astype(np.float64) / np.where(q[:, None] > 0, q[:, None], 1)
            lo = np.clip(np.searchsorted(table, t * (1 + 1e-6), side='right') - 1, 0, len(table) - 2)
            assert ((code == lo) | (code == lo + 1) | (code == lo - 1)).all()
    t = x / q[:, None].astype(np.float64)
    gap = (table[np.clip(np.searchsorted(table, t, side='right'), 1, len(table) - 1)] - table[np.clip(np.searchsorted(table, t, side='right') - 1, 0, len(table) - 2)]) * q[:, None]
    free = np.ones(x.shape, bool) if power == 2 else t > 1                     # a positive second moment never takes code 0
    assert (np.abs(total / n - x)[free] <= (gap / 2048 + 1e-6 * x)[free]).all()   # 4096 draws, evenly spread: the mean to 1 / 2048 of a gap


def test_zero_tiny_and_bad_runs():
    x = np.zeros((4, 256), np.float32)
    x[1] = 9e-29
    x[2, 5] = np.nan
    x[3, 5] = np.inf
    for power in (2, 4):
        code, q = oracle.encode(x, np.zeros(x.shape, np.float32), power)
        assert q[0] == 0 and q[1] == 0 and (code[:2] == 0).all() and np.isnan(q[2]) and np.isinf(q[3])
        with np.errstate(all='ignore'):
            assert np.isnan(oracle.decode(code, q, power)[2:]).all()


def test_moving_averages_in_8_bits_follow_those_in_64():
    """500 steps of gradients whose size jumps by 10 half way.  The draws leave a second moment (weight 0.999) and a first one (0.9) right on
    average; rounding to nearest would leave the second where it was: its largest step is (1 - b2) (g^2 - v), far below half a code."""
    rng = np.random.default_rng(1)
    b = (0.9, 0.999)
    runs = np.arange(16)
    cm, qm, cv, qv = np.zeros((16, 256), np.int8), np.zeros(16, np.float32), np.zeros((16, 256), np.uint8), np.zeros(16, np.float32)
    m, v = np.zeros((16, 256)), np.zeros((16, 256))
    size = np.exp(rng.normal(0, 1, (16, 256)))
    for t in range(1, 501):
        g = (rng.normal(0, 1, (16, 256)) * size * (10.0 if t > 250 else 1.0)).astype(np.float32)
        cm, qm, cv, qv, _, _ = oracle.moments8(g, cm, qm, cv, qv, t, 7, runs, b, 1.0)
        m, v = b[0] * m + (1 - b[0]) * g, b[1] * v + (1 - b[1]) * g.astype(np.float64) ** 2
    v8, m8 = oracle.decode(cv, qv, 4).astype(np.float64), oracle.decode(cm, qm, 2).astype(np.float64)
    assert abs((v8 / v).mean() - 1) < 0.02 and (v8 / v).std() < 0.2 and (v8 > 0).all()
    assert abs((m8 * np.sign(m)).sum() / np.abs(m).sum() - 1) < 0.02


def test_draws_are_spread_and_independent():
    um, uv = oracle.draws(np.arange(1000), 11, 3)
    u2, _ = oracle.draws(np.arange(1000), 12, 3)
    u3, _ = oracle.draws(np.arange(1000), 11, 4)
    n = um.size
    for a in (um, uv):
        assert abs(a.mean() / 65535 - 0.5) < 4 * 0.29 / n ** 0.5 and abs(a.std() / 65535 - 12 ** -0.5) < 0.005
    for a, b in ((um, uv), (um, u2), (um, u3), (um[:, 1:], um[:, :-1]), (um[1:], um[:-1])):
        assert abs(np.corrcoef(a.ravel(), b.ravel())[0, 1]) < 5 / n ** 0.5


def test_shared_memory_and_hyperparameters_that_are_no_numbers_are_refused():
    from semseg_amd.engine import AdamW
    base = torch.zeros(12)
    with pytest.raises(ValueError, match='share memory'):
        AdamW([base[:8], base[7:]])
    AdamW([base[:7], base[7:], torch.zeros(0)])
    for kw in (dict(lr=float('nan')), dict(eps=float('nan')), dict(weight_decay=-0.1), dict(per_param=lambda p: {'weight_decay': -0.1}),
               dict(per_param=lambda p: {'lr_scale': float('nan')})):
        with pytest.raises(ValueError, match='negative|betas'):
            AdamW([torch.zeros(3)], **kw)
