"""The operators on a policy's action scores (magical_amd/policy.py, include/mgx_policy.h) against their formulas in 64 bits.

Tolerances.  u = 2^-24 is fp32's largest relative rounding error.  With d = (x - m) / T, s = sum e^d, L = log n:
  * d has three roundings (the difference, 1 / T, the product): |err d| <= 3 u |d|;
  * e^d: 2 ulp of the exponential and err d: relative 4 u + 3 u |d|; a sum of n of them by lanes and trees of at most
    A = 40 + n / 256 additions in a row: relative A u.  sum |d| e^d / s <= L + 1, so err(log s) <= u (A + 4 + 3 (L + 1) + L);
  * log p = d - log s: u (4 |d| + A + 8 + 4 L);
  * H = log s - t / s with t = sum d e^d: |t / s| <= L + 1, sum d^2 e^d / s <= (L + 2)^2, so err H <= u (2 A (L + 2) + 4 (L + 2)^2 + 16);
  * the gradient's p = e^(log p): relative err(log p) + 4 u; the rest is the product rule, and one rounding to the logits' type (half a
    step, eps / 2 relative, in float16 at least 2^-25)."""
import math
import os
import re

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24


# ------------------------------------------------------------------------------------------------ the formulas, in 64 bits, on the CPU
def oracle(x, mask=None, temperature=1.0):
    """(open, log p, H, undefined rows) of logits [rows, n] (float64 numpy)."""
    x = np.asarray(x, dtype=np.float64)
    is_open = ~np.isneginf(x)
    if mask is not None:
        is_open &= np.broadcast_to(np.asarray(mask), x.shape)
    bad = (is_open & (np.isnan(x) | np.isposinf(x))).any(1)
    z = np.where(is_open, x, -np.inf)
    z[bad] = 0.0
    with np.errstate(all='ignore'):
        m = z.max(1, keepdims=True)
        m = np.where(np.isneginf(m), 0.0, m)
        d = (z - m) / temperature
        s = np.exp(d).sum(1, keepdims=True)
        lp = np.where(is_open, d - np.log(s), -np.inf)
        h = np.where(is_open.any(1), -(np.where(np.isneginf(lp), 0.0, np.exp(lp)) * np.where(np.isneginf(lp), 0.0, lp)).sum(1), 0.0)
    lp[bad] = np.nan
    h[bad] = np.nan
    return is_open, lp, h, bad


def oracle_top(x, is_open, bad, k):
    out = np.full((x.shape[0], k), -1, dtype=np.int32)
    for r in range(x.shape[0]):
        if not bad[r]:
            idx = np.nonzero(is_open[r])[0]
            best = idx[np.argsort(-x[r, idx], kind='stable')][:k]
            out[r, :len(best)] = best
    return out


def oracle_grad(is_open, lp, h, actions, g_lp, g_h, temperature):
    p = np.where(is_open, np.exp(lp), 0.0)
    safe = np.where(is_open & ~np.isneginf(lp), lp, 0.0)
    given = actions >= 0
    gl = np.where(given, g_lp, 0.0)[:, None]
    g = -p * (gl + g_h[:, None] * (safe + h[:, None]))
    rows = np.nonzero(given & (actions < lp.shape[1]))[0]
    rows = rows[is_open[rows, actions[rows]]]
    g[rows, actions[rows]] += g_lp[rows]
    return np.where(is_open, g / temperature, 0.0)


def oracle_draw(is_open, lp, u):
    """(action, smallest distance of u to a border of the distribution) per row."""
    p = np.where(is_open, np.exp(lp), 0.0)
    c = np.cumsum(p, 1)
    c /= np.where(c[:, -1:] > 0, c[:, -1:], 1.0)
    a = np.minimum((c <= u[:, None]).sum(1), p.shape[1] - 1)
    inner = np.where(p > 0, np.abs(c - u[:, None]), np.inf)
    return np.where(is_open.any(1), a, -1), np.minimum(inner.min(1), np.where(is_open.any(1), 1.0, np.inf))


def in_f32(v):
    """Values outside fp32's range round to the infinities (the type's lowest value over a temperature below 1 does)."""
    return np.where(np.abs(v) > np.finfo(np.float32).max, np.where(v > 0, np.inf, -np.inf), v)


def err_log_prob(d, n):
    L, A = math.log(n), 40 + n / 256
    return U * (4 * np.abs(d) + A + 8 + 4 * L)


def err_entropy(n):
    L, A = math.log(n), 40 + n / 256
    return U * (2 * A * (L + 2) + 4 * (L + 2) ** 2 + 16)


def err_grad(is_open, lp, h, g_lp, g_h, want, temperature, eps, tiny):
    n = lp.shape[1]
    lpz = np.where(is_open & ~np.isneginf(lp), lp, 0.0)
    p = np.where(is_open, np.exp(lp), 0.0)
    rel = err_log_prob(np.abs(lpz) + math.log(n), n) + 4 * U
    size = np.abs(g_lp)[:, None] + np.abs(g_h)[:, None] * (np.abs(lpz) + h[:, None])
    e = p * (rel * size + np.abs(g_h)[:, None] * (rel + err_entropy(n)) + 4 * U * size) / temperature + 4 * U * np.abs(want)
    return e + np.maximum(np.abs(want) * (1 + 1e-3) * eps / 2, tiny) + 2.0 ** -126


# ------------------------------------------------------------------------------------------------ no GPU needed
def test_the_library_exports_the_policy_header():
    from magical_amd import _native
    L = _native.lib()
    header = open(os.path.join(ROOT, 'include', 'mgx_policy.h')).read()
    header = re.sub(r'/\*.*?\*/', '', header, flags=re.S)
    declared = set(re.findall(r'\b(mgx_policy_[a-z_]+)\s*\(', header))
    assert declared == set(_native.POLICY_SYMBOLS)
    for name in declared:
        getattr(L, name)


def _c_args(**kw):
    a = dict(dtype=0, logits=64, rows=1, n=18, row_stride=18, mask=None, mask_row_stride=0, temperature=1.0)
    a.update(kw)
    return [a[k] for k in ('dtype', 'logits', 'rows', 'n', 'row_stride', 'mask', 'mask_row_stride', 'temperature')]


@pytest.mark.parametrize('kw', [dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(n=0), dict(n=(1 << 30) + 1), dict(row_stride=-1),
                                dict(mask=64, mask_row_stride=-1), dict(temperature=0.0), dict(temperature=-1.0),
                                dict(temperature=float('nan')), dict(temperature=float('inf')), dict(temperature=1e-60),
                                dict(temperature=1e300), dict(logits=None)])
def test_the_c_entries_refuse_bad_scores_before_any_device_work(kw):
    from magical_amd import _native
    L = _native.lib()
    args = _c_args(**kw)
    assert L.mgx_policy_log_probs(0, *args, 64, 4, 0, 64, 64, None, None, None, None, 0, None) == -1
    assert L.mgx_policy_last_error()
    assert L.mgx_policy_log_probs_backward(0, *args, 64, 4, 64, 64, None, 0, None, 0, 64, None) == -1
    assert L.mgx_policy_sample(0, *args, 64, 4, 64, None, None, None, 0, None) == -1


def test_the_c_entries_refuse_other_bad_arguments_before_any_device_work():
    from magical_amd import _native
    L = _native.lib()
    a = _c_args()
    for action_bytes, top in ((2, 0), (4, -1), (4, 19), (4, 65)):
        assert L.mgx_policy_log_probs(0, *a, 64, action_bytes, top, 64, 64, None, 64, 64, None, 0, None) == -1
    assert L.mgx_policy_log_probs(0, *_c_args(n=100, row_stride=100), 64, 4, 65, 64, 64, None, 64, 64, None, 0, None) == -1
    assert L.mgx_policy_log_probs(0, *a, None, 4, 0, 64, 64, None, None, None, None, 0, None) == -1
    assert L.mgx_policy_log_probs(0, *a, 64, 4, 0, None, 64, None, None, None, None, 0, None) == -1
    assert L.mgx_policy_log_probs(0, *a, 64, 4, 2, 64, 64, None, None, 64, None, 0, None) == -1
    assert L.mgx_policy_log_probs_backward(0, *a, 64, 2, 64, 64, None, 0, None, 0, 64, None) == -1
    assert L.mgx_policy_log_probs_backward(0, *_c_args(n=5000, row_stride=5000), 64, 4, None, 64, None, 0, None, 0, 64, None) == -1
    assert L.mgx_policy_log_probs_backward(0, *a, 64, 4, None, None, None, 0, None, 0, 64, None) == -1
    assert L.mgx_policy_log_probs_backward(0, *a, 64, 4, 64, 64, 64, -1, None, 0, 64, None) == -1
    assert L.mgx_policy_log_probs_backward(0, *a, 64, 4, 64, 64, None, 0, None, 0, None, None) == -1
    assert L.mgx_policy_sample(0, *a, 64, 2, 64, None, None, None, 0, None) == -1
    assert L.mgx_policy_sample(0, *a, None, 4, 64, None, None, None, 0, None) == -1
    assert L.mgx_policy_sample(0, *a, 64, 4, None, None, None, None, 0, None) == -1
    # nothing to do is no error, whatever the pointers
    empty = _c_args(rows=0, logits=None)
    assert L.mgx_policy_log_probs(0, *empty, None, 4, 0, None, None, None, None, None, None, 0, None) == 0
    assert L.mgx_policy_log_probs_backward(0, *empty, None, 4, None, None, None, 0, None, 0, None, None) == 0
    assert L.mgx_policy_sample(0, *empty, None, 4, None, None, None, None, 0, None) == 0


def test_the_python_entries_refuse_bad_arguments():
    import torch
    import magical_amd as m
    from magical_amd._native import MgxError
    x, a, u = torch.zeros(3, 18), torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    with pytest.raises(MgxError, match='no CPU fallback'):
        m.action_log_probs(x, a)
    with pytest.raises(MgxError, match='no CPU fallback'):
        m.sample_actions(x, u)
    for bad in (np.zeros((3, 18)), x.double(), x.int(), x.to(torch.complex64)):
        with pytest.raises(TypeError):
            m.action_log_probs(bad, a)
        with pytest.raises(TypeError):
            m.sample_actions(bad, u)
    for bad in (torch.zeros(()), torch.zeros(3, 0)):
        with pytest.raises(ValueError):
            m.action_log_probs(bad, a)
    for bad in (a.float(), a.to(torch.int16), a.bool(), [0, 0, 0]):
        with pytest.raises(TypeError):
            m.action_log_probs(x, bad)
    for bad in (a[:2], a[:, None], torch.zeros((), dtype=torch.int64)):
        with pytest.raises(ValueError):
            m.action_log_probs(x, bad)
    for bad in (torch.ones(18), torch.ones(18, dtype=torch.uint8), np.ones(18, bool)):
        with pytest.raises(TypeError):
            m.action_log_probs(x, a, mask=bad)
        with pytest.raises(TypeError):
            m.sample_actions(x, u, mask=bad)
    for bad in (torch.ones(17, dtype=torch.bool), torch.ones(2, 18, dtype=torch.bool), torch.ones(1, 3, 18, dtype=torch.bool)):
        with pytest.raises(ValueError):
            m.action_log_probs(x, a, mask=bad)
    for bad in (0.0, -1.0, float('nan'), float('inf'), 1e-38, 1e38):
        with pytest.raises(ValueError):
            m.action_log_probs(x, a, temperature=bad)
        with pytest.raises(ValueError):
            m.sample_actions(x, u, temperature=bad)
    for bad in (-1, 19):
        with pytest.raises(ValueError):
            m.action_log_probs(x, a, top=bad)
    with pytest.raises(ValueError):
        m.action_log_probs(torch.zeros(3, 100), a, top=65)
    with pytest.raises(TypeError):
        m.sample_actions(x, u.half())
    with pytest.raises(ValueError):
        m.sample_actions(x, u[:2])


# ------------------------------------------------------------------------------------------------ on the GPU
NS = [1, 2, 3, 4, 5, 8, 9, 16, 17, 18, 19, 20, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 324, 511, 512, 513,
      1000, 1024, 1025, 2047, 2048, 2049, 4097, 5832, 8191, 20011]
DTYPES = ['f32', 'f16', 'bf16']


def _torch_type(name):
    import torch
    return {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}[name]


def _case(n, dtype, seed, rows=None, masked=None):
    """Logits with the values that masks and policies bring: spread scores, one far ahead, ties, -inf, the type's lowest value; in row 0 (of
    several) nothing is open, in row 1 only one action, row 2 is all equal, row 3 all the type's lowest value."""
    import torch
    rng = np.random.RandomState(seed)
    rows = rows if rows is not None else (13 if n < 3000 else 6)
    t = _torch_type(dtype)
    x = rng.randn(rows, n) * 3
    x[rng.rand(rows) < 0.3] *= 0.01
    ahead = rng.rand(rows) < 0.4
    x[ahead, rng.randint(0, n, rows)[ahead]] += 12
    x[rng.rand(rows, n) < 0.05] = -np.inf
    x[rng.rand(rows, n) < 0.05] = float(torch.finfo(t).min)
    mask = None
    if masked == 'rows':
        mask = rng.rand(rows, n) < 0.7
    elif masked == 'shared':
        mask = rng.rand(n) < 0.7
    if rows > 4:
        x[0] = -np.inf
        x[1] = -np.inf
        x[1, rng.randint(n)] = -1.5
        x[2] = 0.75
        x[3] = float(torch.finfo(t).min)
    if masked == 'rows' and rows > 5:
        mask[5] = False
    x = torch.tensor(x, dtype=torch.float64).to(t)
    actions = rng.randint(0, n, rows)
    actions[rng.rand(rows) < 0.2] = -1
    return x, mask, actions, rng


def _check_forward(out, x64, mask, actions, temperature, top, what):
    is_open, lp, h, bad = oracle(x64, mask, temperature)
    n = x64.shape[1]
    got_lp, got_h = out.log_prob.detach().double().cpu().numpy(), out.entropy.detach().double().cpu().numpy()
    with np.errstate(invalid='ignore'):
        d = np.where(is_open, (x64 - np.where(is_open, x64, -np.inf).max(1, keepdims=True)) / temperature, 0.0)
    for r in range(len(actions)):
        a = int(actions[r])
        want = 0.0 if a < 0 else (np.nan if a >= n or bad[r] else float(in_f32(lp[r, a])))
        if np.isfinite(want):
            assert abs(got_lp[r] - want) <= (0 if a < 0 else err_log_prob(d[r, a], n)), (what, r, got_lp[r], want)
        else:
            assert got_lp[r] == want or (np.isnan(want) and np.isnan(got_lp[r])), (what, r, got_lp[r], want)
    assert np.array_equal(np.isnan(got_h), bad), what
    assert np.all(np.abs(got_h - h)[~bad] <= err_entropy(n)), (what, np.abs(got_h - h)[~bad].max())
    if top:
        want_a = oracle_top(x64, is_open, bad, top)
        got_a, got_t = out.top_actions.cpu().numpy(), out.top_log_probs.double().cpu().numpy()
        assert np.array_equal(got_a, want_a), what
        there = want_a >= 0
        rows = np.nonzero(there)[0]
        want_t = in_f32(lp[rows, want_a[there]])
        fine = np.isfinite(want_t)
        assert np.all(np.abs(got_t[there][fine] - want_t[fine]) <= err_log_prob(d[rows, want_a[there]][fine], n)), what
        assert np.all(np.isneginf(got_t[there][~fine])) and np.all(np.isneginf(got_t[~there])), what
    return is_open, lp, h, bad


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('n', NS)
def test_log_probs_gradient_and_draws_against_64_bits(n, dtype):
    import torch
    import magical_amd as m
    for k, (masked, temperature) in enumerate([(None, 1.0), ('shared', 1.0), ('rows', 0.7), ('rows', 2.5)]):
        x, mask, actions, rng = _case(n, dtype, 1000 * n + k, masked=masked)
        rows = x.shape[0]
        x64 = x.double().numpy()
        top = min(n, (0, 1, 5, 64)[k])
        leaf = x.cuda().requires_grad_(True)
        m_dev = None if mask is None else torch.tensor(mask).cuda()
        a_dev = torch.tensor(actions, dtype=(torch.int32, torch.int64)[k % 2]).cuda()
        out = m.action_log_probs(leaf, a_dev, mask=m_dev, temperature=temperature, top=top)
        what = (n, dtype, masked, temperature)
        is_open, lp, h, bad = _check_forward(out, x64, mask, actions, temperature, top, what)
        # the gradient
        g_lp, g_h = rng.randn(rows).astype(np.float32), (rng.randn(rows) * 0.1).astype(np.float32)
        torch.autograd.backward((out.log_prob, out.entropy), (torch.tensor(g_lp).cuda(), torch.tensor(g_h).cuda()))
        assert leaf.grad.dtype == x.dtype
        got = leaf.grad.double().cpu().numpy()
        want = oracle_grad(is_open, lp, h, actions, g_lp.astype(np.float64), g_h.astype(np.float64), temperature)
        eps, tiny = torch.finfo(x.dtype).eps, 2.0 ** -25 if dtype == 'f16' else 0.0
        bound = err_grad(is_open, lp, h, g_lp.astype(np.float64), g_h.astype(np.float64), want, temperature, eps, tiny)
        assert np.all(np.abs(got - want) <= bound), (what, np.max(np.abs(got - want) / bound))
        assert np.all(got[~is_open] == 0), what
        # without a graph: the same bits
        again = m.action_log_probs(leaf.detach(), a_dev, mask=m_dev, temperature=temperature, top=top)
        assert torch.equal(again.log_prob, out.log_prob) and torch.equal(again.entropy, out.entropy), what
        # draws
        u = rng.rand(rows)
        u[-1] = 0.0
        u = u.astype(np.float32) if k % 2 else u
        drawn = m.sample_actions(leaf.detach(), torch.tensor(u).cuda(), mask=m_dev, temperature=temperature)
        want_a, gap = oracle_draw(is_open, lp, u.astype(np.float64))
        clear = gap > 1e-11
        clear[-1] = True                      # u = 0: the first action of non-zero probability, exactly
        if is_open[-1].any():
            want_a[-1] = np.nonzero(is_open[-1] & (np.exp(lp[-1]) > 0))[0][0]
        assert clear.sum() >= rows - 1
        got_a = drawn.action.cpu().numpy()
        assert np.array_equal(got_a[clear], want_a[clear]), (what, got_a, want_a)
        rows_open = np.nonzero(got_a >= 0)[0]
        want_lp = in_f32(lp[rows_open, got_a[rows_open]])
        assert np.all(np.abs(drawn.log_prob.double().cpu().numpy()[rows_open] - want_lp) <= U * (np.abs(want_lp) + 1e-6)), what
        assert np.all(np.isneginf(drawn.log_prob.cpu().numpy()[got_a < 0])), what
        assert np.all(np.abs(drawn.entropy.double().cpu().numpy() - h) <= U * (h + 1e-6) + 1e-12), what


@pytest.mark.gpu
@pytest.mark.parametrize('n', [1, 18, 300, 1500, 6000, 70000])
def test_rows_that_nothing_or_nonsense_is_left_in(n):
    """NaN and infinities among the open scores, behind the mask, and everywhere."""
    import torch
    import magical_amd as m
    nan, inf = float('nan'), float('inf')
    x = torch.randn(8, n, generator=torch.Generator().manual_seed(n))
    mask = torch.ones(8, n, dtype=torch.bool)
    k = n // 2
    x[0, k] = nan
    x[1, k] = inf
    x[2, k] = nan
    mask[2, k] = False
    x[3, k] = inf
    mask[3, k] = False
    x[4] = nan
    x[5] = nan
    mask[5] = False
    x[6] = -inf
    x[7, k] = -inf
    actions = torch.full((8,), n - 1, dtype=torch.int64)
    leaf = x.cuda().requires_grad_(True)
    top = min(n, 3)
    out = m.action_log_probs(leaf, actions.cuda(), mask=mask.cuda(), top=top)
    is_open, lp, h, bad = _check_forward(out, x.double().numpy(), mask.numpy(), actions.numpy(), 1.0, top, n)
    assert bad.tolist() == [True, True, False, False, True, False, False, False]
    (out.log_prob.nan_to_num(0, 0, 0).sum() * 0 + out.log_prob.sum() + out.entropy.sum()).backward()
    grad = leaf.grad.cpu().numpy()
    assert np.all(np.isnan(grad[bad][is_open[bad]])) and np.all(grad[~is_open] == 0) and np.all(np.isfinite(grad[~bad]))
    drawn = m.sample_actions(leaf.detach(), torch.full((8,), 0.5).cuda(), mask=mask.cuda())
    assert np.all((drawn.action.cpu().numpy() == -1) == (bad | ~is_open.any(1)))
    assert np.all(np.isnan(drawn.log_prob.cpu().numpy()) == bad) and np.all(np.isnan(drawn.entropy.cpu().numpy()) == bad)
    # padded rows keep log probability 0 even so; an action behind the last one is NaN
    out = m.action_log_probs(leaf.detach(), torch.tensor([-1, -7, n, n + 5, -1, -1, -1, n]).cuda(), mask=mask.cuda())
    got = out.log_prob.cpu().numpy()
    assert np.all(got[[0, 1, 4, 5, 6]] == 0) and np.all(np.isnan(got[[2, 3, 7]]))


@pytest.mark.gpu
@pytest.mark.parametrize('n', [140001, 300000, 1200007])
def test_very_long_rows(n):
    """Rows of more segments than a workgroup keeps together (512), and of more than 64 a lane."""
    import torch
    import magical_amd as m
    rng = np.random.RandomState(n)
    x = (rng.randn(2, n) * 2).astype(np.float32)
    x[1] = 0.5
    u = rng.rand(2)
    is_open, lp, h, bad = oracle(x)
    actions = rng.randint(0, n, 2)
    out = m.action_log_probs(torch.tensor(x).cuda(), torch.tensor(actions).cuda(), top=33)
    _check_forward(out, x.astype(np.float64), None, actions, 1.0, 33, n)
    want, gap = oracle_draw(is_open, lp, u)
    assert (gap > 1e-11).all()
    drawn = m.sample_actions(torch.tensor(x).cuda(), torch.tensor(u).cuda())
    assert np.array_equal(drawn.action.cpu().numpy(), want)
    assert np.all(np.abs(drawn.entropy.double().cpu().numpy() - h) <= U * h + 1e-10)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('n', [18, 500, 5000])
def test_any_byte_but_zero_in_a_mask_is_open(n, dtype):
    import torch
    import magical_amd as m
    g = torch.Generator().manual_seed(n)
    x = torch.randn(9, n, generator=g).to(_torch_type(dtype)).cuda()
    a = torch.randint(0, n, (9,), generator=g).cuda()
    u = torch.rand(9, generator=g).cuda()
    raw = (torch.randint(0, 256, (9, n), generator=g) * (torch.rand(9, n, generator=g) < 0.7)).to(torch.uint8).cuda()
    leaf = x.clone().requires_grad_(True)
    got = [*m.action_log_probs(leaf, a, mask=raw.view(torch.bool), top=4), *m.sample_actions(x, u, mask=raw.view(torch.bool))]
    got.append(torch.autograd.grad(got[0].sum(), leaf)[0])
    want = [*m.action_log_probs(leaf, a, mask=raw != 0, top=4), *m.sample_actions(x, u, mask=raw != 0)]
    want.append(torch.autograd.grad(want[0].sum(), leaf)[0])
    for p, q in zip(got, want):
        assert torch.equal(p, q)


@pytest.mark.gpu
@pytest.mark.parametrize('temperature', [1e-37, 1e-20, 1e20, 1e37])
@pytest.mark.parametrize('n', [18, 600, 5000])
def test_temperatures_at_the_ends(n, temperature):
    """Towards 0 only the best action is left (all of them, if several are equal), towards infinity all are alike."""
    import torch
    import magical_amd as m
    x = torch.randn(5, n, generator=torch.Generator().manual_seed(n))
    x[1, 3] = x[1, 9] = 8.0
    x[2, 4] = float('-inf')
    best = x.argmax(1)
    out = m.action_log_probs(x.cuda().requires_grad_(True), best.cuda(), temperature=temperature, top=2)
    drawn = m.sample_actions(x.cuda(), torch.full((5,), 0.25).cuda(), temperature=temperature)
    is_open, lp, h, _ = oracle(x.double().numpy(), None, temperature)
    want = lp[np.arange(5), best.numpy()]
    assert np.all(np.abs(out.log_prob.detach().cpu().numpy() - want) <= err_log_prob(0, n))
    assert np.all(np.abs(out.entropy.detach().cpu().numpy() - h) <= err_entropy(n))
    # (5000 equal probabilities have a border at exactly 0.25 = 1250 / 5000, where sums of 1250 terms, each rounded by up to 2^-53, lie on either
    # side: within that, 1250 x 2^-53 < 1e-11, the action on either side of the border is the formula's)
    got_a, (want_a, gap) = drawn.action.cpu().numpy(), oracle_draw(is_open, lp, np.full(5, 0.25))
    assert np.all((got_a == want_a) | ((gap < 1e-11) & (np.abs(got_a - want_a) == 1)))
    if temperature < 1:
        assert np.array_equal(drawn.action.cpu().numpy(), [int(b) for b in x.argmax(1)])


@pytest.mark.gpu
@pytest.mark.parametrize('n', [18, 700, 6000])
def test_random_numbers_at_and_outside_the_ends(n):
    import torch
    import magical_amd as m
    x = torch.randn(7, n, generator=torch.Generator().manual_seed(n))
    x[:, 0] = x[:, -1] = float('-inf')
    u = torch.tensor([0.0, -3.0, float('nan'), 1.0, 5.0, float('inf'), 1 - 2.0 ** -53], dtype=torch.float64)
    a = m.sample_actions(x.cuda(), u.cuda()).action.cpu().tolist()
    assert a == [1, 1, 1, n - 2, n - 2, n - 2, n - 2]
    a = m.sample_actions(x.cuda(), u.float().cuda()).action.cpu().tolist()
    assert a == [1, 1, 1, n - 2, n - 2, n - 2, n - 2]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('n', [18, 19, 300, 1500, 5000, 40000])
def test_strides_offsets_and_orders_change_no_bit(n, dtype):
    """Views of a wider head, odd offsets, transposed, expanded and higher-dimensional tensors: the results of the dense copy."""
    import torch
    import magical_amd as m
    g = torch.Generator(device='cuda').manual_seed(n)
    rows = 24
    base = torch.randn(rows, n, generator=g, device='cuda').to(_torch_type(dtype))
    mask = torch.rand(rows, n, generator=g, device='cuda') < 0.8
    actions = torch.randint(0, n, (rows,), generator=g, device='cuda')
    u = torch.rand(rows, generator=g, device='cuda')
    g_lp, g_h = torch.randn(rows, generator=g, device='cuda'), torch.randn(rows, generator=g, device='cuda')

    def all_of(x, msk, acts=actions, uu=u, gl=g_lp, gh=g_h):
        x = x.detach().requires_grad_(True)
        out = m.action_log_probs(x, acts, mask=msk, top=3)
        grad, = torch.autograd.grad((out.log_prob, out.entropy), (x,), (gl, gh))
        return list(out) + [grad] + list(m.sample_actions(x.detach(), uu, mask=msk))

    want = all_of(base, mask)

    def same(got, shape=None):
        for a, b in zip(got, want):
            a = a.reshape(b.shape)
            assert torch.equal(a, b)

    wide = torch.full((rows, n + 3), 7.0, device='cuda', dtype=base.dtype)
    wide[:, 1:n + 1] = base
    wide_mask = torch.zeros((rows, n + 5), device='cuda', dtype=torch.bool)
    wide_mask[:, 3:n + 3] = mask
    same(all_of(wide[:, 1:n + 1], wide_mask[:, 3:n + 3]))
    flat = torch.zeros(rows * n + 1, device='cuda', dtype=base.dtype)
    flat[1:] = base.reshape(-1)
    same(all_of(flat[1:].view(rows, n), mask))
    same(all_of(base.t().contiguous().t(), mask.t().contiguous().t()))
    cube = lambda t: t.view(2, 3, 4, *t.shape[1:])      # noqa: E731
    same(all_of(cube(base), cube(mask), cube(actions), cube(u), cube(g_lp), cube(g_h)))
    same(all_of(base, mask, actions.int()))
    # one row for all, one mask for all
    row = base[:1].expand(rows, n)
    got, dense = all_of(row, mask[0]), all_of(row.contiguous(), mask[:1].expand(rows, n).contiguous())
    for a, b in zip(got, dense):
        assert torch.equal(a, b)
    # ... and the gradient of the one row is the sum over its uses
    leaf = base[0].float().clone().requires_grad_(True)
    out = m.action_log_probs(leaf.expand(rows, n), actions, mask=mask[0])
    (out.log_prob * g_lp).sum().backward()
    grads = all_of(leaf.detach().expand(rows, n).contiguous(), mask[0], gh=torch.zeros_like(g_h))[4]
    assert torch.allclose(leaf.grad.double(), grads.double().sum(0), rtol=rows * 2.0 ** -23, atol=rows * 2.0 ** -23)
    # a single row without a batch dimension
    one = m.action_log_probs(base[5], actions[5], mask=mask[5], top=3)
    assert one.log_prob.shape == () and one.top_actions.shape == (3,)
    assert torch.allclose(one.log_prob, want[0][5], rtol=0, atol=float(err_log_prob(30, n)))
    assert m.sample_actions(base[5], u[5], mask=mask[5]).action.shape == ()
    # none at all
    none = m.action_log_probs(base[:0].requires_grad_(True), actions[:0], top=2)
    assert none.log_prob.shape == (0,) and none.top_actions.shape == (0, 2)
    none.log_prob.sum().backward()
    assert m.sample_actions(base[:0], u[:0]).action.shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,n', [((1 << 20) + 3, 18), (2000003, 31), (300007, 5), (200003, 324), (5003, 2500), (40009, 1700), (1031, 40000)])
def test_many_rows(rows, n):
    """Every row of a large batch is worked on: the results of row subsets equal those of the whole."""
    import torch
    import magical_amd as m
    g = torch.Generator(device='cuda').manual_seed(rows)
    x = (torch.randn(rows, n, generator=g, device='cuda') * 2).bfloat16()
    a = torch.randint(0, n, (rows,), generator=g, device='cuda')
    u = torch.rand(rows, generator=g, device='cuda')
    xr = x.clone().requires_grad_(True)
    out = m.action_log_probs(xr, a, top=2)
    out.log_prob.sum().backward()
    x32 = x.float()
    lse = torch.logsumexp(x32, 1)
    tol = float(err_log_prob(40, n)) + 40 * 2.0 ** -23
    assert (out.log_prob - (x32.gather(1, a[:, None])[:, 0] - lse)).abs().max() <= tol
    p = torch.exp(x32 - lse[:, None])
    want = -p
    want.scatter_add_(1, a[:, None], torch.ones_like(want[:, :1]))
    assert (xr.grad.float() - want).abs().max() <= 2.0 ** -8 + 1e-5
    assert (x.gather(1, out.top_actions[:, :1].long())[:, 0] == x.amax(1)).all()
    drawn = m.sample_actions(x, u)
    assert ((drawn.action >= 0) & (drawn.action < n)).all()
    cut = rows - 1234
    part = m.sample_actions(x[cut:], u[cut:])
    assert torch.equal(part.action, drawn.action[cut:])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('n,rows', [(18, 5000), (40, 700), (700, 3000), (3000, 600), (3000, 4200), (9000, 40), (9000, 2100), (9000, 4100), (30011, 700),
                                    (30011, 2100)])
def test_every_row_alike_in_every_launch_shape(n, rows, dtype):
    """The special rows (nothing open, one action, all equal, the lowest value, ties, masks), repeated to many: how rows are shared out over lanes,
    wavefronts and workgroups goes by their number and length.  One copy against 64 bits, the others the same bits."""
    import torch
    import magical_amd as m
    x, mask, actions, rng = _case(n, dtype, n + rows, rows=13, masked='rows')
    copies = -(-rows // 13)
    rep = lambda t: torch.as_tensor(t).repeat((copies,) + (1,) * (torch.as_tensor(t).dim() - 1))[:rows].cuda()      # noqa: E731
    u = rng.rand(13)
    g_lp, g_h = rng.randn(13).astype(np.float32), (rng.randn(13) * 0.1).astype(np.float32)
    leaf = rep(x).requires_grad_(True)
    for top in (0, 5, 40):
        top = min(top, n)
        out = m.action_log_probs(leaf, rep(actions), mask=rep(mask), temperature=1.3, top=top)
        first = m.policy.ActionLogProbs(*(None if t is None else t[:13] for t in out))
        is_open, lp, h, bad = _check_forward(first, x.double().numpy(), mask, actions, 1.3, top, (n, rows, dtype, top))
        for t in out:
            assert t is None or torch.equal(t, rep(t[:13]))
    grad, = torch.autograd.grad((out.log_prob, out.entropy), (leaf,), (rep(g_lp), rep(g_h)))
    want = oracle_grad(is_open, lp, h, actions, g_lp.astype(np.float64), g_h.astype(np.float64), 1.3)
    bound = err_grad(is_open, lp, h, g_lp.astype(np.float64), g_h.astype(np.float64), want, 1.3, torch.finfo(x.dtype).eps, 0.0)
    assert np.all(np.abs(grad[:13].double().cpu().numpy() - want) <= bound)
    assert torch.equal(grad, rep(grad[:13]))
    drawn = m.sample_actions(leaf.detach(), rep(u), mask=rep(mask), temperature=1.3)
    want_a, gap = oracle_draw(*oracle(x.double().numpy(), mask, 1.3)[:2], u)
    assert (gap > 1e-11).all() and np.array_equal(drawn.action[:13].cpu().numpy(), want_a)
    for t in drawn:
        assert torch.equal(t, rep(t[:13]))


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [1, 2, 63, 64, 65, 190, 257])
def test_alternatives_of_a_few_rows_more_or_less_than_a_wavefront_holds(rows):
    import torch
    import magical_amd as m
    for n, dtype in ((2, 'f32'), (7, 'bf16'), (18, 'f16'), (32, 'f32')):
        x, mask, actions, _ = _case(n, dtype, rows * n, rows=rows, masked='rows')
        for top in sorted({1, 2, 3, n}):
            if top <= n:
                out = m.action_log_probs(x.cuda(), torch.tensor(actions).cuda(), mask=torch.tensor(mask).cuda(), top=top)
                _check_forward(out, x.double().numpy(), mask, actions, 1.0, top, (rows, n, top))


@pytest.mark.gpu
@pytest.mark.parametrize('n', [70, 190, 385, 511, 513, 616, 768, 769, 1023])
def test_draws_of_rows_in_a_few_lanes(n):
    import torch
    import magical_amd as m
    for dtype in DTYPES:
        x, mask, _, rng = _case(n, dtype, n, rows=37, masked='rows')
        u = rng.rand(37)
        want_a, gap = oracle_draw(*oracle(x.double().numpy(), mask, 0.8)[:2], u)
        assert (gap > 1e-11).all()
        got = m.sample_actions(x.cuda(), torch.tensor(u).cuda(), mask=torch.tensor(mask).cuda(), temperature=0.8)
        assert np.array_equal(got.action.cpu().numpy(), want_a), dtype


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [16, 4096])
@pytest.mark.parametrize('n', [18, 900, 2500, 5832, 20000, 104976])
def test_draws_next_to_long_closed_stretches(n, rows):
    """The first and the last that is open, with everything before and behind it ruled out: numbers of 0 and 1 have to reach them."""
    import torch
    import magical_amd as m
    if rows * n > 1 << 27:
        rows = 1100
    x = torch.zeros(rows, n, dtype=torch.bfloat16, device='cuda')
    u = (torch.arange(rows, device='cuda') % 2).float()
    for first in sorted({0, 1, n // 9, min(2048, n // 2), n // 2}):
        mask = torch.zeros(n, dtype=torch.bool, device='cuda')
        last = n - 1 - first // 2
        mask[first:last + 1] = True
        old = torch.full((rows,), -7, dtype=torch.int32, device='cuda')          # (what the result's memory holds before, most likely)
        del old
        got = m.sample_actions(x, u, mask=mask)
        assert torch.equal(got.action, torch.where(u == 0, first, last).int()), (first, last)
        want = -np.log(last + 1 - first)
        assert (got.log_prob.double() - want).abs().max() <= U * abs(want) + 1e-12


@pytest.mark.gpu
@pytest.mark.parametrize('n', [18, 200, 900, 5832, 104976])
def test_draws_among_probabilities_that_are_next_to_nothing(n):
    """Each below 2^-990, their sum above it: still an action that is open."""
    import torch
    import magical_amd as m
    for rows in (3, 4096):
        for bits in (985, 991, 994, 998, 1200):
            x = torch.full((1, n), -bits * float(np.log(2)), device='cuda')
            x[0, n // 3 * 2:] = 0
            x[0, :n // 9] = -float('inf')
            x = x.expand(rows, n)
            got = m.sample_actions(x, torch.zeros(rows, device='cuda'))
            assert (got.action >= n // 9).all() and (got.action <= n // 3 * 2).all(), (rows, bits)
            if bits < 990:
                assert (got.action == n // 9).all()
            if bits > 1100:
                assert (got.action == n // 3 * 2).all()


@pytest.mark.gpu
@pytest.mark.parametrize('n', [257, 1025, 5832, 20011, 104976])
def test_alternatives_among_equal_extreme_and_few_scores(n):
    """Rows of the lowest value, of zeros of both signs, of the smallest numbers around zero, with less open than asked for, with the best far back."""
    import torch
    import magical_amd as m
    for dtype in DTYPES:
        t = _torch_type(dtype)
        low, tiny = float(torch.finfo(t).min), float(torch.finfo(t).smallest_normal)
        x = torch.full((9, n), -float('inf'), dtype=torch.float64)
        x[0] = low
        x[1, n // 2:] = low
        x[2, ::97] = low
        x[3] = torch.where(torch.arange(n) % 3 == 0, -0.0, 0.0)
        x[4] = torch.where(torch.arange(n) % 5 == 0, -tiny, 0.0)
        x[4, n - 2] = tiny
        x[5, n - 3:] = low
        x[6] = low
        x[6, n - 1] = 0.0
        x[7] = torch.linspace(-3, 3, n, dtype=torch.float64)
        x[8] = torch.linspace(3, -3, n, dtype=torch.float64)
        x = x.to(t)
        actions = np.full(9, n - 1)
        for top in (1, 5, 9, 64):
            out = m.action_log_probs(x.cuda(), torch.tensor(actions).cuda(), top=top)
            is_open, _, _, bad = oracle(x.double().numpy())
            want = oracle_top(x.double().numpy(), is_open, bad, top)
            assert np.array_equal(out.top_actions.cpu().numpy(), want), (dtype, top)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows that lie further than 2^32 bytes and 2^31 elements from the first one."""
    import torch
    import magical_amd as m
    far = (1 << 31) + 64
    buf = torch.empty(far + 40000, dtype=torch.float16, device='cuda')
    for n in (18, 1000, 30000):
        g = torch.Generator(device='cuda').manual_seed(n)
        x = torch.randn(2, n, generator=g, device='cuda').half()
        buf[:n], buf[far:far + n] = x[0], x[1]
        view = buf.as_strided((2, n), (far, 1)).requires_grad_(True)
        a = torch.tensor([0, n - 1], device='cuda')
        u = torch.tensor([0.3, 0.6], device='cuda')
        dense = x.clone().requires_grad_(True)
        got, want = m.action_log_probs(view, a, top=4), m.action_log_probs(dense, a, top=4)
        for p, q in zip(got, want):
            assert torch.equal(p, q)
        # (the gradient as the kernel hands it out: autograd would lay a view's gradient out over the whole buffer)
        out = m.action_log_probs(view.detach(), a)
        assert torch.equal(out.log_prob, want.log_prob)
        assert torch.equal(m.sample_actions(view.detach(), u).action, m.sample_actions(x, u).action)
    del buf, view
    rows = (1 << 31) // 18 + 1000                       # results and gradient of more than 2^31 elements in all
    x = torch.zeros(1, 18, device='cuda', dtype=torch.bfloat16)
    x[0, 3] = 2.0
    a = torch.full((rows,), 3, dtype=torch.int32, device='cuda')
    leaf = x.expand(rows, 18).requires_grad_(True)
    out = m.action_log_probs(leaf, a)
    assert (out.log_prob == out.log_prob[0]).all()
    grad, = torch.autograd.grad(out.log_prob, leaf, torch.ones((), device='cuda').expand(rows))
    assert torch.equal(grad[-1000:], grad[:1000]) and (grad[-1] != 0).all()


@pytest.mark.gpu
def test_gradient_against_differences():
    """The kernels' gradient (fp32) against central differences of the formula in 64 bits: (f(x + h) - f(x - h)) / 2h, h = 1e-4, is off by
    h^2 / 6 x the third derivative (of log p and H: below 10 + L) and by rounding 2^-52 |f| / h."""
    import torch
    import magical_amd as m
    rng = np.random.RandomState(0)
    for n, temperature in ((2, 1.0), (18, 0.5), (70, 3.0)):
        x = rng.randn(4, n).astype(np.float32)
        actions, gl, gh = rng.randint(0, n, 4), rng.randn(4), rng.randn(4)
        leaf = torch.tensor(x).cuda().requires_grad_(True)
        out = m.action_log_probs(leaf, torch.tensor(actions).cuda(), temperature=temperature)
        torch.autograd.backward((out.log_prob, out.entropy), (torch.tensor(gl).float().cuda(), torch.tensor(gh).float().cuda()))

        def f(z):
            _, lp, h, _ = oracle(z, None, temperature)
            return gl.astype(np.float32) * lp[np.arange(4), actions] + gh.astype(np.float32) * h
        step, want = 1e-4, np.zeros((4, n))
        for j in range(n):
            e = np.zeros((1, n))
            e[0, j] = step
            want[:, j] = (f(x.astype(np.float64) + e) - f(x.astype(np.float64) - e)) / (2 * step)
        L = math.log(n)
        tol = (np.abs(gl) + np.abs(gh)) * (step ** 2 / 6 * (10 + L) / temperature ** 3 + 2.0 ** -52 * (10 / temperature + L) / step)
        tol = tol[:, None] + (np.abs(gl) + np.abs(gh) * (L + 1))[:, None] * 2 * err_entropy(n) / temperature
        assert np.all(np.abs(leaf.grad.cpu().numpy() - want) <= tol)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,n', [(64, 18), (300, 324), (9, 5832), (2, 104976)])
def test_captured_calls_replay(rows, n):
    """Forward, backward and draws in one captured graph, replayed on new inputs with eager calls of other sizes in between."""
    import torch
    import magical_amd as m
    g = torch.Generator(device='cuda').manual_seed(1)

    def new():
        return (torch.randn(rows, n, generator=g, device='cuda'), torch.randint(0, n, (rows,), generator=g, device='cuda'),
                torch.rand(rows, generator=g, device='cuda'))

    gl, gh = torch.randn(rows, generator=g, device='cuda'), torch.full((rows,), -0.01, device='cuda')

    def work(x, a, u):
        out = m.action_log_probs(x, a, top=4)
        grad, = torch.autograd.grad((out.log_prob, out.entropy), (x,), (gl, gh))
        drawn = m.sample_actions(x.detach(), u, temperature=0.8)
        return [out.log_prob.detach(), out.entropy.detach(), out.top_actions, out.top_log_probs, grad, *drawn]

    sx, sa, su = (t.clone() for t in new())
    sx.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(sx, sa, su)
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work(sx, sa, su)
    with torch.cuda.graph(other):
        held2 = work(sx, sa, su)
    for _ in range(4):
        x, a, u = new()
        with torch.no_grad():
            sx.copy_(x)
        sa.copy_(a)
        su.copy_(u)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        want = work(x.requires_grad_(True), a, u)
        for p, p2, q in zip(held, held2, want):
            assert torch.equal(p, q) and torch.equal(p2, q)
        m.action_log_probs(torch.randn(3, 50000, device='cuda'), torch.zeros(3, dtype=torch.int64, device='cuda'), top=8)


@pytest.mark.gpu
def test_calls_on_other_streams_and_interleaved():
    """Two streams at once, each with its own inputs: the results of one after the other."""
    import torch
    import magical_amd as m
    torch.cuda.synchronize()
    sets = []
    for k, (rows, n) in enumerate([(3, 60000), (5, 90000), (4096, 18), (2, 104976)]):
        g = torch.Generator(device='cuda').manual_seed(k)
        sets.append((torch.randn(rows, n, generator=g, device='cuda'), torch.randint(0, n, (rows,), generator=g, device='cuda'),
                     torch.rand(rows, generator=g, device='cuda')))
    want = [(m.action_log_probs(x, a, top=7), m.sample_actions(x, u)) for x, a, u in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(5):
        for s, (x, a, u) in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append((m.action_log_probs(x, a, top=7), m.sample_actions(x, u)))
    torch.cuda.synchronize()
    for k, (p, q) in enumerate(got):
        for t, w in zip(list(p) + list(q), list(want[k % 4][0]) + list(want[k % 4][1])):
            assert torch.equal(t, w)


@pytest.mark.gpu
def test_a_capture_beside_an_eager_graph_of_the_same_leaf_is_refused():
    import torch
    import magical_amd as m
    x, a = torch.randn(9, 18, device='cuda', requires_grad=True), torch.arange(9, device='cuda')
    alive = m.action_log_probs(x, a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(m._native.MgxError, match='earlier calls'):
            m.action_log_probs(x, a)
        detached = m.action_log_probs(x.detach(), a)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(detached.log_prob, alive.log_prob.detach())
    want, = torch.autograd.grad(alive.log_prob.sum(), x)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(m.action_log_probs(x, a).log_prob.sum(), x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_a_capture_beside_a_warm_up_on_a_side_stream():
    """The usual way to a captured training step: warmed up on a side stream, its results freed."""
    import torch
    import magical_amd as m
    x, a = torch.randn(9, 18, device='cuda', requires_grad=True), torch.arange(9, device='cuda')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            x.grad = None
            loss = m.action_log_probs(x, a).log_prob.sum()
            loss.backward()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    want = x.grad.clone()
    del loss
    x.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        m.action_log_probs(x, a).log_prob.sum().backward()
    for _ in range(3):
        x.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x.grad, want)


@pytest.mark.gpu
def test_negations_that_torch_has_put_off_are_taken():
    import torch
    import magical_amd as m
    z = torch.complex(torch.zeros(9, 18), torch.randn(9, 18)).cuda()
    x, a, u = z.conj().imag, torch.arange(9, device='cuda'), torch.rand(9, device='cuda')
    assert x.is_neg()
    for got, want in zip(m.action_log_probs(x, a, top=3) + m.sample_actions(x, u),
                         m.action_log_probs(x.resolve_neg().clone(), a, top=3) + m.sample_actions(x.resolve_neg().clone(), u)):
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    import torch
    import magical_amd as m
    x, a = torch.zeros(3, 18, device='cuda'), torch.zeros(3, dtype=torch.int32, device='cuda')
    with pytest.raises(ValueError):
        m.action_log_probs(x, a.cpu())
    with pytest.raises(ValueError):
        m.action_log_probs(x, a, mask=torch.ones(18, dtype=torch.bool))
    with pytest.raises(ValueError):
        m.sample_actions(x, torch.zeros(3))
    # twice differentiable it is not, and it says so
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(m.action_log_probs(leaf, a).entropy.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match='differentiable once'):
        g.sum().backward()
    # a graph is there for one backward pass unless it is kept, and holds no memory afterwards
    out = m.action_log_probs(leaf, a)
    first, = torch.autograd.grad(out.log_prob.sum(), leaf, retain_graph=True)
    assert torch.equal(first, torch.autograd.grad(out.log_prob.sum(), leaf)[0])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out.entropy.sum(), leaf)
    del out, first
    big = torch.randn(64, 100000, device='cuda').requires_grad_(True)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    for _ in range(3):
        out = m.action_log_probs(big, torch.zeros(64, dtype=torch.int64, device='cuda'), top=3)
        (out.log_prob.sum() + out.entropy.sum()).backward()
        big.grad = None
        unused = m.action_log_probs(big, torch.zeros(64, dtype=torch.int64, device='cuda'))
    del out, unused
    assert torch.cuda.memory_allocated() == held
    # one of the two upstream gradients, or neither
    out = m.action_log_probs(leaf, a)
    g_lp, = torch.autograd.grad(out.log_prob.sum(), leaf, retain_graph=True)
    g_h, = torch.autograd.grad(out.entropy.sum(), leaf, retain_graph=True)
    both, = torch.autograd.grad(out.log_prob.sum() + out.entropy.sum(), leaf)
    assert torch.allclose(g_lp + g_h, both, rtol=0, atol=2.0 ** -20)
    assert torch.autograd.grad((leaf * 0).sum() + m.action_log_probs(leaf, a, top=1).top_log_probs.sum(), leaf)[0].abs().max() == 0
    # inputs changed in between are noticed
    y = (leaf * 1.0)
    out = m.action_log_probs(y, a)
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError):
        out.log_prob.sum().backward()


@pytest.mark.gpu
def test_a_rollout_and_its_learning_step():
    """As they are used together: actions drawn per env-step by step_policy, the same bits as sample_actions + step; the rollout's log
    probabilities again from action_log_probs; one ascent step along the gradient makes the drawn actions likelier."""
    import torch
    import magical_amd as m
    n_envs, T = 64, 6
    env = m.make('MoveToCorner-Demo-LoRes4E-v0', n_envs=n_envs, device='cuda:0')
    twin = m.make('MoveToCorner-Demo-LoRes4E-v0', n_envs=n_envs, device='cuda:0')
    g = torch.Generator(device='cuda').manual_seed(5)
    weights = (torch.randn(12, 18, generator=g, device='cuda') * 0.05).requires_grad_(True)
    obs, _ = env.reset(), twin.reset()
    feats, acts, lps, ents = [], [], [], []
    for t in range(T):
        feat = obs.float().mean((1, 2)) / 32
        feats.append(feat)
        u = torch.rand(n_envs, generator=g, device='cuda')
        with torch.no_grad():
            logits = feat @ weights
        obs, rew, done, info = env.step_policy(logits, u)
        drawn = m.sample_actions(logits, u)
        want, _, _, _ = twin.step(drawn.action)
        assert torch.equal(obs, want)
        assert torch.equal(info['action'], drawn.action) and torch.equal(info['action_log_prob'], drawn.log_prob)
        acts.append(info['action'])
        lps.append(info['action_log_prob'])
        ents.append(info['action_entropy'])
    feats, acts, lps, ents = torch.stack(feats), torch.stack(acts), torch.stack(lps), torch.stack(ents)
    out = m.action_log_probs(feats @ weights, acts)
    tol = float(err_log_prob(30, 18)) + 60 * 2.0 ** -23             # (+ the two matrix products' own rounding of scores below 8)
    assert (out.log_prob - lps).abs().max() <= tol and (out.entropy - ents).abs().max() <= tol + float(err_entropy(18))
    (out.log_prob.mean() + 0.01 * out.entropy.mean()).backward()
    # the gradient to the weights, from the formula in 64 bits
    z = (feats.double() @ weights.detach().double()).requires_grad_(True)
    lp = torch.log_softmax(z, 2)
    ref = lp.gather(2, acts.long()[..., None]).mean() - 0.01 * (lp.exp() * lp).sum(2).mean()
    gz, = torch.autograd.grad(ref, z)
    gw = feats.double().flatten(0, 1).t() @ gz.flatten(0, 1)
    assert (weights.grad.double() - gw).abs().max() <= 1e-5 * gw.abs().max() + 1e-7
    # no action is open: the env idles
    obs, _, _, info = env.step_policy(torch.full((n_envs, 18), float('-inf'), device='cuda'))
    want, _, _, _ = twin.step(np.zeros(n_envs, dtype=np.int32))
    assert torch.equal(obs, want) and (info['action'] == -1).all()
    with pytest.raises(ValueError):
        env.step_policy(torch.zeros(n_envs, 17, device='cuda'))
    with pytest.raises(ValueError):
        env.step_policy(torch.zeros(n_envs, 18))
    env.close()
    twin.close()


@pytest.mark.gpu
def test_replay_scores_a_policy_on_demonstrations():
    """replay_demos(policy=...): per demo, the log probability of every recorded action, the entropies and the policy's own choice; demos
    that are over take no part."""
    import torch
    from magical_amd import saved_trajectories as st
    rng = np.random.RandomState(3)
    lengths = (5, 9, 2)
    demos = [{'env_name': 'MoveToCorner-Demo-v0', 'score': 0.0,
              'trajectory': st.MAGICALTrajectory(acts=rng.randint(0, 18, T), obs={}, rews=np.zeros(T), infos=None)} for T in lengths]
    seen = []
    w = torch.randn(12, 18, generator=torch.Generator().manual_seed(0)).cuda() * 0.05

    def policy(obs):
        logits = (obs.float().mean((1, 2)) / 32) @ w
        seen.append(logits.double().cpu().numpy())
        return logits

    plain = st.replay_demos(demos, preproc='LoRes4E')
    out = st.replay_demos(demos, preproc='LoRes4E', policy=policy)
    assert np.array_equal(out['scores'], plain['scores']) and torch.equal(out['final_obs'], plain['final_obs'])
    assert set(plain) == {'scores', 'recorded_scores', 'final_obs'} and len(seen) == max(lengths)
    for k, demo in enumerate(demos):
        T = lengths[k]
        assert len(out['log_probs'][k]) == len(out['entropies'][k]) == len(out['best_actions'][k]) == T
        for t in range(T):
            is_open, lp, h, _ = oracle(seen[t][k:k + 1])
            assert abs(out['log_probs'][k][t] - lp[0, demo['trajectory'].acts[t]]) <= err_log_prob(60, 18)
            assert abs(out['entropies'][k][t] - h[0]) <= err_entropy(18)
            assert out['best_actions'][k][t] == seen[t][k].argmax()
