"""The operators on a policy's action scores at the ends of what is documented, and beside torch's own machinery: each test fails for a fault that
was there once.  The oracle and the counting of roundings are test_policy_ops.py's; where a bound differs, it is derived beside the test."""
import math

import numpy as np
import pytest

from tests.test_policy_ops import U, _torch_type, err_entropy, err_log_prob, oracle, oracle_grad


def grad_bound(is_open, lp, h, g_lp, g_h, want, temperature, eps, tiny):
    """dx = p (g_lp' + g_H (log p + H)) / T: p is off by err(log p) + 4 u relative, the factor by the roundings of its terms; one rounding to the
    logits' type.  As in test_policy_ops.py but for two things.  An exponential below 2^-126 may be taken as none: times a factor of at most
    2^40 (1 + 160 ln 2), beyond which the kernels work in 64 bits, that is below 2^-79.  And nothing is added for the least number the result's type
    holds where the type is fp32: results here go down to 1e-37, and what is below the normal numbers, 2^-126, counts as nothing."""
    n = lp.shape[1]
    lpz = np.where(is_open & ~np.isneginf(lp), lp, 0.0)
    p = np.where(is_open, np.exp(lp), 0.0)
    rel = err_log_prob(np.abs(lpz) + math.log(n), n) + 4 * U
    size = np.abs(g_lp)[:, None] + np.abs(g_h)[:, None] * (np.abs(lpz) + h[:, None])
    e = p * (rel * size + np.abs(g_h)[:, None] * (rel + err_entropy(n)) + 4 * U * size) / temperature + 4 * U * np.abs(want)
    scale = (np.abs(g_lp) + np.abs(g_h) * (h + 1))[:, None] / temperature
    return e + np.maximum(np.abs(want) * (1 + 1e-3) * eps / 2, tiny) + 2.0 ** -126 * (1 + 160 * np.minimum(scale, 2.0 ** 40))


# (n, rows): a lane a row, 4 ... 64 lanes, a wavefront a row by halves of tiles (16-bit) and by whole ones, a workgroup a row
GRADIENT_SHAPES = [(18, 13), (40, 13), (324, 13), (1500, 13), (2500, 13), (6000, 13), (60000, 7)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('n,rows', GRADIENT_SHAPES)
def test_gradients_at_every_temperature_and_scale(n, rows, dtype):
    """Places that are not open, and open ones of no probability, have gradient 0 whatever the temperature and the upstream gradients: in products
    with what overflows they would be NaN."""
    import torch
    import magical_amd as m
    t = _torch_type(dtype)
    rng = np.random.RandomState(n)
    x = rng.randn(rows, n) * 3
    x[rng.rand(rows, n) < 0.1] = -np.inf
    x[rng.rand(rows, n) < 0.1] = float(torch.finfo(t).min)
    x[0] = -np.inf
    x[1] = 0.75
    x[2] = float(torch.finfo(t).min)
    x[3, : n // 2] = 2.0
    x[4] = rng.randn(n) * 1e-3
    x = torch.tensor(x).to(t)
    x64 = x.double().numpy()
    mask = rng.rand(rows, n) < 0.8
    mask[5] = False
    actions = rng.randint(0, n, rows)
    actions[6] = -1
    base_lp, base_h = rng.randn(rows), rng.randn(rows)
    for temperature, scale in [(1e-37, 1.0), (1e-37, 1e-30), (1e-30, 1.0), (1e-20, 1.0), (1e-20, 1e-18), (1e-10, 1.0), (1e-9, 1.0), (1e-4, 65536.0),
                               (1e-4, 1.0), (1.0, 1e9), (1.0, 1e30), (1.0, 2.0 ** 24), (1.0, 1e-30), (1e4, 1.0), (1e10, 1e10), (1e20, 1e30), (1e37, 1e37)]:
        for use_mask in (None, mask):
            g_lp, g_h = (base_lp * scale).astype(np.float32), (base_h * scale).astype(np.float32)
            if scale == 2.0 ** 24:
                g_lp[:] = 0
            leaf = x.cuda().requires_grad_(True)
            out = m.action_log_probs(leaf, torch.tensor(actions).cuda(), mask=None if use_mask is None else torch.tensor(mask).cuda(), temperature=temperature)
            torch.autograd.backward((out.log_prob, out.entropy), (torch.tensor(g_lp).cuda(), torch.tensor(g_h).cuda()))
            got = leaf.grad.double().cpu().numpy()
            is_open, lp, h, bad = oracle(x64, use_mask, temperature)
            gl64, gh64 = g_lp.astype(np.float64), g_h.astype(np.float64)
            want = oracle_grad(is_open, lp, h, actions, gl64, gh64, temperature)
            bound = grad_bound(is_open, lp, h, gl64, gh64, want, temperature, torch.finfo(t).eps, 2.0 ** -25 if dtype == 'f16' else 0.0)
            what = (n, dtype, temperature, scale, use_mask is not None)
            assert not np.isnan(got).any(), what
            assert np.all(got[~is_open] == 0), what
            big = float(torch.finfo(t).max)
            huge = np.isinf(got)          # (beyond the type's range)
            assert np.all(np.sign(got[huge]) == np.sign(want[huge])) and np.all(np.abs(want[huge]) + bound[huge] >= big), what
            err = np.abs(got - want)[~huge]
            assert np.all(err <= bound[~huge]), (what, np.max(err / bound[~huge]))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('n,rows', [(18, 13), (40, 13), (324, 13), (1500, 13), (2500, 13), (6000, 13), (60000, 7)])
def test_an_action_behind_the_last_one_has_no_finite_gradient(n, rows, dtype):
    """Its log probability is NaN, and so is what flows back through it -- unless nothing does.  The entropy's gradient and other rows are not
    touched."""
    import torch
    import magical_amd as m
    g = torch.Generator().manual_seed(n)
    x = torch.randn(rows, n, generator=g).to(_torch_type(dtype))
    x[:, 1] = float('-inf')
    mask = torch.rand(rows, n, generator=g) < 0.8
    mask[:, 0] = True
    mask[4] = False
    is_open = (mask & (x > float('-inf'))).numpy()
    actions = torch.randint(0, n, (rows,), generator=g)
    bad = actions.clone()
    bad[0], bad[2], bad[3], bad[4] = n, n + 7, n, n
    g_lp, g_h = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    g_lp[3] = 0.0
    leaf = x.cuda().requires_grad_(True)

    def grads(acts, gl, gh):
        out = m.action_log_probs(leaf, acts.cuda(), mask=mask.cuda())
        outs, ups = zip(*[(o, u.cuda()) for o, u in ((out.log_prob, gl), (out.entropy, gh)) if u is not None])
        return torch.autograd.grad(outs, leaf, ups)[0].float().cpu().numpy()

    for kind in (torch.int64, torch.int32):
        for gh in (g_h, None):
            got, fine = grads(bad.to(kind), g_lp, gh), grads(actions.to(kind), g_lp, gh)
            for r in range(rows):
                if r in (0, 2):
                    assert np.all(np.isnan(got[r][is_open[r]])) and np.all(got[r][~is_open[r]] == 0), r
                elif r == 4:
                    assert np.all(got[r] == 0)
                elif r != 3:
                    assert np.array_equal(got[r], fine[r]), r
            assert np.array_equal(got[3], grads(torch.full_like(actions, -1).to(kind), g_lp, gh)[3])
    # (against rows without an action: the place of a given one is worked out with a rounding less than its neighbours)
    entropy_only, none = grads(bad, None, g_h), grads(torch.where(bad >= n, -1, bad), None, g_h)
    assert np.array_equal(entropy_only, none) and np.all(np.isfinite(none))


def additions(n, rows, dtype):
    """The longest chain of additions behind a row's sums: a tile's scores of a lane, its tiles, the 6 steps over a wavefront's lanes, 3 over a
    workgroup's wavefronts, 16 parts of a lane and 6 steps over the lanes that join them.  Tiles are 4 vectors of 16 bytes a lane."""
    in_tile = 16 if dtype == 'f32' else 32
    tiles = -(-n // (64 * in_tile)) if rows >= 2048 else -(-n // (256 * in_tile))          # (fewer where a row is shared out further)
    return in_tile + tiles + 6 + 3 + 16 + 6


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('n,rows', [(2500, 5), (5832, 4096), (20000, 1), (20000, 4096), (104976, 3), (104976, 1100), (104976, 4096), (1200007, 2), (1200007, 4096)])
def test_sums_of_long_rows_are_as_close_as_their_additions(n, rows, dtype):
    """One score ahead of all others, so far that each of these is next to nothing beside it and all together are not: a sum that takes them one
    by one loses them.  log p = d - log s: 3 roundings of d, a relative error of A u of the sum of A additions in a row, 4 u d of the others'
    exponentials, 8 u for the exponential, the logarithm and the difference, 2 u |log s|; H = log s - t / s with t / s, d times the others' share,
    off by twice as much relative (t and s)."""
    import torch
    import magical_amd as m
    L = math.log(n)
    for ahead in (17.5, 15.0, 12.0, L):
        row = torch.zeros(n, dtype=_torch_type(dtype))
        row[n // 3] = ahead
        x64 = row.double().numpy()[None]
        _, lp, h, _ = oracle(x64)
        d = float(x64.max())
        A = additions(n, rows, dtype)
        share = float(np.exp(lp[0, 0]) * (n - 1))          # of the sum, the others'
        tol_lp = lambda dist: U * (4 * dist + A + 8 + 4 * d * share + 2 * abs(lp[0, n // 3]))      # noqa: E731
        tol_h = tol_lp(0.0) + U * (2 * A + 16 + 8 * d) * d * share
        actions = torch.full((rows,), n // 3, device='cuda')
        actions[1::2] = n - 1
        for top in (0, 3):
            out = m.action_log_probs(row.cuda().expand(rows, n), actions, top=top)
            got_lp, got_h = out.log_prob.double().cpu().numpy(), out.entropy.double().cpu().numpy()
            assert np.abs(got_lp[::2] - lp[0, n // 3]).max() <= tol_lp(0.0), (ahead, np.abs(got_lp[::2] - lp[0, n // 3]).max() / U, A)
            if rows > 1:
                assert np.abs(got_lp[1::2] - lp[0, n - 1]).max() <= tol_lp(d), (ahead, np.abs(got_lp[1::2] - lp[0, n - 1]).max() / U, A)
            assert np.abs(got_h - h[0]).max() <= tol_h, (ahead, np.abs(got_h - h[0]).max(), tol_h)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('n,rows', [(18, 13), (324, 13), (1500, 13), (2500, 13), (6000, 13), (9000, 2100), (60000, 7), (20000, 4096)])
def test_scores_further_apart_than_the_largest_number(n, rows, dtype):
    """3e38 and -3e38 are 6e38 apart, which fp32 does not hold; over a temperature of 1e37 they are 60 apart, and both are open."""
    import torch
    import magical_amd as m
    temperature = 1e37
    rng = np.random.RandomState(n)
    base = (rng.rand(13, n) * 2 - 1) * 3.3e38
    base[0, : n // 2], base[0, n // 2:] = -3.3e38, 3.3e38
    base[1] = -3.3e38
    base[1, n // 3] = 3.3e38
    x = torch.tensor(base).to(_torch_type(dtype))
    x64 = x.double().numpy()
    is_open, lp, h, _ = oracle(x64, None, temperature)
    actions = rng.randint(0, n, 13)
    actions[:2] = 0
    g_lp, g_h = (rng.randn(13) * 1e37).astype(np.float32), (rng.randn(13) * 1e36).astype(np.float32)
    rep = lambda v: torch.as_tensor(v)[torch.arange(rows) % 13].cuda()      # noqa: E731
    k = min(rows, 13)
    leaf = rep(x).requires_grad_(True)
    top = min(n, 9)
    out = m.action_log_probs(leaf, rep(actions), temperature=temperature, top=top)
    d = (x64.max(1, keepdims=True) - x64) / temperature
    got = out.log_prob.detach().double().cpu().numpy()[:k]
    at = np.arange(k)
    assert np.all(np.abs(got - lp[at, actions[:k]]) <= err_log_prob(d[at, actions[:k]], n))
    assert np.all(np.abs(out.entropy.detach().double().cpu().numpy()[:k] - h[:k]) <= err_entropy(n))
    best = np.argsort(-x64, axis=1, kind='stable')[:k, :top]
    assert np.array_equal(out.top_actions.cpu().numpy()[:k], best)
    want = np.take_along_axis(lp[:k], best, 1)
    assert np.all(np.abs(out.top_log_probs.double().cpu().numpy()[:k] - want) <= err_log_prob(np.take_along_axis(d[:k], best, 1), n))
    grad, = torch.autograd.grad((out.log_prob, out.entropy), leaf, (rep(g_lp), rep(g_h)))
    gl64, gh64 = g_lp.astype(np.float64), g_h.astype(np.float64)
    want = oracle_grad(is_open, lp, h, actions, gl64, gh64, temperature)
    bound = grad_bound(is_open, lp, h, gl64, gh64, want, temperature, torch.finfo(x.dtype).eps, 0.0)
    assert np.all(np.abs(grad.double().cpu().numpy()[:k] - want[:k]) <= bound[:k])
    drawn = m.sample_actions(leaf.detach(), torch.full((rows,), 0.5, device='cuda'), temperature=temperature)
    a = drawn.action.cpu().numpy()[:k]
    assert np.all(np.abs(drawn.log_prob.double().cpu().numpy()[:k] - lp[at, a]) <= U * np.abs(lp[at, a]) + 1e-6 * U)
    if rows > 13:
        for t in list(out) + [grad, drawn.action]:
            assert torch.equal(t, t[:13][torch.arange(rows, device='cuda') % 13])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,n,top', [(0, 1000, 0), (0, 2048, 3), (2, 400, 20), (1, 1500, 0)])
def test_statistics_that_the_backward_call_does_not_need_are_not_written(dtype, n, top):
    """mgx_policy_stats_bytes() is 0 for these rows: whatever pointer is given, nothing belongs to the call behind it."""
    import ctypes
    import torch
    from magical_amd import _native
    L = _native.lib()
    rows = 6
    assert L.mgx_policy_stats_bytes(rows, n) == 0
    x = torch.randn(rows, n, device='cuda').to([torch.float32, torch.float16, torch.bfloat16][dtype])
    a = torch.zeros(rows, dtype=torch.int32, device='cuda')
    lp, h = torch.empty(rows, device='cuda'), torch.empty(rows, device='cuda')
    t_lp, t_a = torch.empty(rows * max(top, 1), device='cuda'), torch.empty(rows * max(top, 1), dtype=torch.int32, device='cuda')
    ws = torch.empty(max(16, L.mgx_policy_workspace_bytes(0, dtype, rows, n, top)), dtype=torch.uint8, device='cuda')
    guard = torch.full((2 * rows,), 7.0, device='cuda')          # (another's memory)
    p = lambda t: ctypes.c_void_p(t.data_ptr())      # noqa: E731
    rc = L.mgx_policy_log_probs(0, dtype, p(x), rows, n, n, None, 0, 1.0, p(a), 4, top, p(lp), p(h), p(guard), p(t_lp), p(t_a), p(ws), ws.numel(),
                                ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    torch.cuda.synchronize()
    assert torch.isfinite(lp).all() and torch.isfinite(h).all()
    assert (guard == 7).all()


@pytest.mark.gpu
def test_a_policy_scored_on_demonstrations_without_actions():
    import torch
    from magical_amd import saved_trajectories as st
    demos = [{'env_name': 'MoveToCorner-Demo-v0', 'score': 0.0,
              'trajectory': st.MAGICALTrajectory(acts=np.zeros(0, dtype=np.int64), obs={}, rews=np.zeros(0), infos=None)} for _ in range(2)]
    plain = st.replay_demos(demos, preproc='LoRes4E')
    out = st.replay_demos(demos, preproc='LoRes4E', policy=lambda obs: torch.zeros(2, 18, device='cuda'))
    assert np.array_equal(out['scores'], plain['scores'])
    for key, kind in (('log_probs', np.float32), ('entropies', np.float32), ('best_actions', np.int32)):
        assert [v.shape for v in out[key]] == [(0,), (0,)] and all(v.dtype == kind for v in out[key])


@pytest.mark.gpu
def test_a_refused_device_is_no_error_of_the_next_call():
    """The C call says what it could not do; nothing of it is left for somebody else's call to report."""
    import ctypes
    import torch
    from magical_amd import _native
    L = _native.lib()
    x, a = torch.randn(6, 18, device='cuda'), torch.zeros(6, dtype=torch.int32, device='cuda')
    lp, h = torch.empty(6, device='cuda'), torch.empty(6, device='cuda')
    torch.cuda.synchronize()
    p = lambda t: ctypes.c_void_p(t.data_ptr())      # noqa: E731
    scores = [99, 0, p(x), 6, 18, 18, None, 0, 1.0]          # (there is no device 99)
    for call in (lambda: L.mgx_policy_log_probs(*scores, p(a), 4, 0, p(lp), p(h), None, None, None, None, 0, None),
                 lambda: L.mgx_policy_log_probs_backward(*scores, p(a), 4, None, p(h), None, 0, None, 0, p(x), None),
                 lambda: L.mgx_policy_sample(*scores, p(lp), 4, p(a), None, None, None, 0, None)):
        assert call() == -4          # MGX_ERR_HIP
        assert L.mgx_policy_last_error() == b'hipSetDevice failed'
        before = x.sum()
        y = x + 1
        torch.cuda.synchronize()
        assert torch.equal((y - x).round(), torch.ones_like(x)) and torch.equal(x.sum(), before) and torch.cuda.current_device() == 0


def test_what_would_drop_a_derivative_or_bake_a_result_in_is_refused():
    """Forward-mode tangents do not come out at the other end; traced, the results would be constants."""
    import torch
    import torch.autograd.forward_ad as fwd
    import magical_amd as m
    x, a, u = torch.zeros(3, 18), torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match='forward'):
            m.action_log_probs(dual, a)
        with pytest.raises(NotImplementedError, match='forward'):
            m.action_log_probs(dual.requires_grad_(True), a)
    for call in (lambda x: m.action_log_probs(x, a).log_prob, lambda x: m.sample_actions(x, u).log_prob):
        with pytest.raises(NotImplementedError, match='trac'):
            torch.jit.trace(call, (x,))


@pytest.mark.gpu
def test_forward_mode_on_the_gpu():
    import torch
    import torch.autograd.forward_ad as fwd
    import magical_amd as m
    x, a = torch.randn(3, 18, device='cuda'), torch.zeros(3, dtype=torch.int64, device='cuda')
    want = m.action_log_probs(x, a).log_prob
    leaf = x.clone().requires_grad_(True)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match='forward'):
            m.action_log_probs(dual, a)
        # tangents of the upstream gradients would be lost just so
        out = m.action_log_probs(leaf, a).log_prob
        with pytest.raises(NotImplementedError, match='forward'):
            torch.autograd.grad(out, leaf, fwd.make_dual(torch.ones(3, device='cuda'), torch.ones(3, device='cuda')))
        # a draw has no derivative, of any mode; where tangents are switched off there is none to lose
        assert (m.sample_actions(dual, torch.zeros(3, device='cuda')).action >= 0).all()
        with fwd._set_fwd_grad_enabled(False):
            assert torch.equal(m.action_log_probs(dual, a).log_prob, want)
    assert torch.equal(m.action_log_probs(x, a).log_prob, want)


def test_a_star_import_needs_neither_torch_nor_the_library():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ('from magical_amd import *\nimport sys, magical_amd\nassert "torch" not in sys.modules\nmake, register_envs\n'
            'assert action_log_probs is magical_amd.action_log_probs is magical_amd.policy.action_log_probs and SampledActions and sample_actions\n'
            'import torch\n'
            'try:\n    action_log_probs(torch.zeros(2, 18), torch.zeros(2, dtype=torch.int64))\n'
            'except magical_amd._native.MgxError as e:\n    assert "not built" in str(e) or "not found" in str(e), e\n'
            'else:\n    raise AssertionError\n')
    env = dict(os.environ, MGX_LIB_PATH='/nonexistent/libmagical_hip.so')
    run = subprocess.run([sys.executable, '-c', code], cwd=root, env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr


def test_a_development_builds_flags_reach_the_compiler_and_the_linker(monkeypatch, tmp_path):
    from magical_amd import _native
    commands = []

    class Done:
        def __init__(self, cmd, **kw):
            commands.append(cmd)

        def wait(self):
            return 0
    monkeypatch.setattr(_native.subprocess, 'Popen', Done)
    monkeypatch.setattr(_native.subprocess, 'check_call', lambda cmd, **kw: commands.append(cmd))
    _native.build(defines=['MGX_SOME'], out=str(tmp_path / 'lib.so'), extra=['-some-flag'])
    assert len(commands) == len(_native._SOURCES) + 1
    assert all('-some-flag' in cmd for cmd in commands)
    assert all('-DMGX_SOME' in cmd for cmd in commands if '-c' in cmd)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('n,rows', GRADIENT_SHAPES)
def test_padded_rows_of_nonsense_have_no_gradient(n, rows, dtype):
    """A row into which nothing flows back -- a padded step whose entropy is not asked for, a row that a loss leaves out -- has gradient 0, whatever its
    logits: NaN there would reach every weight behind them."""
    import torch
    import magical_amd as m
    g = torch.Generator().manual_seed(n)
    x = torch.randn(rows, n, generator=g)
    x[0] = float('nan')
    x[1, n // 2] = float('nan')
    x[2, 0] = float('inf')
    x[3, n - 1] = float('nan')
    x[4, n - 1] = float('nan')
    actions = torch.randint(0, n, (rows,), generator=g)
    actions[:3] = -1
    used = torch.ones(rows, dtype=torch.bool)
    used[3] = False
    leaf = x.to(_torch_type(dtype)).cuda().requires_grad_(True)
    out = m.action_log_probs(leaf, actions.cuda())
    assert torch.equal(out.log_prob[:3], torch.zeros(3, device='cuda')) and torch.isnan(out.log_prob[3:5]).all() and torch.isnan(out.entropy[:5]).all()
    used, zero = used.cuda(), torch.zeros((), device='cuda')
    for with_entropy in (False, True):
        loss = torch.where(used, out.log_prob, zero).sum()
        if with_entropy:
            loss = loss + torch.where(used & (torch.arange(rows, device='cuda') > 2), out.entropy, zero).sum()
        grad, = torch.autograd.grad(loss, leaf, retain_graph=True)
        assert (grad[:4] == 0).all() and torch.isnan(grad[4]).all() and torch.isfinite(grad[5:]).all()
    grad, = torch.autograd.grad(out.log_prob.sum() + out.entropy.sum(), leaf)
    assert torch.isnan(grad[:5]).all() and torch.isfinite(grad[5:]).all()


@pytest.mark.gpu
def test_a_captured_backward_pass_beside_an_eager_graph_of_the_weights_is_refused():
    """Torch would end the process where it comes to a weight that an eager graph still holds; what does not come there goes on."""
    import gc
    import torch
    import magical_amd as m
    refused = m._native.MgxError
    g = torch.Generator(device='cuda').manual_seed(0)
    feats, weight = torch.randn(9, 12, generator=g, device='cuda'), torch.randn(12, 18, generator=g, device='cuda').requires_grad_(True)
    a = torch.arange(9, device='cuda')
    alive = m.action_log_probs(feats @ weight, a)
    logits = feats @ weight
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(refused, match='default stream'):
            m.action_log_probs(feats @ weight, a).log_prob.sum().backward()
        with pytest.raises(refused, match='default stream'):
            torch.autograd.grad(m.action_log_probs(feats @ weight, a).entropy.sum(), weight)
        with pytest.raises(refused, match='default stream'):          # (a graph whose first half is an eager one)
            torch.autograd.grad(m.action_log_probs(logits, a).log_prob.sum(), weight)
        inner = feats @ weight
        to_logits, = torch.autograd.grad(m.action_log_probs(inner, a).log_prob.sum(), inner)
    assert weight.grad is None
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
    want, = torch.autograd.grad(alive.log_prob.sum(), weight)
    leaf = logits.detach().requires_grad_(True)
    assert torch.equal(to_logits, torch.autograd.grad(m.action_log_probs(leaf, a).log_prob.sum(), leaf)[0])
    del alive, logits, inner, to_logits
    gc.collect()          # (what the refusals' tracebacks still hold)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(m.action_log_probs(feats @ weight, a).log_prob.sum(), weight)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_step_policy_with_masks_temperatures_and_generators():
    import torch
    import magical_amd as m
    n_envs = 64
    env, twin = (m.make('MoveToCorner-Demo-LoRes4E-v0', n_envs=n_envs, device='cuda:0') for _ in range(2))
    env.reset(), twin.reset()
    g = torch.Generator(device='cuda').manual_seed(5)
    logits = torch.randn(n_envs, 18, generator=g, device='cuda') * 2
    per_env = torch.rand(n_envs, 18, generator=g, device='cuda') < 0.5
    per_env[3] = False
    for mask in (None, per_env, per_env[0], per_env.any(1, keepdim=True)):
        for temperature in (1.0, 0.3, 5.0):
            for x in (logits, logits.half(), logits.clone().requires_grad_(True)):
                ours, theirs = torch.Generator(device='cuda').manual_seed(9), torch.Generator(device='cuda').manual_seed(9)
                obs, _, _, info = env.step_policy(x, mask=mask, temperature=temperature, generator=ours)
                u = torch.rand(n_envs, generator=theirs, device='cuda')
                want = m.sample_actions(x, u, mask=mask, temperature=temperature)
                assert torch.equal(info['action'], want.action) and torch.equal(info['action_log_prob'], want.log_prob)
                assert torch.equal(info['action_entropy'], want.entropy) and not info['action_log_prob'].requires_grad
                twin_obs, _, _, _ = twin.step(want.action.clamp(min=0))
                assert torch.equal(obs, twin_obs)
                if mask is not None:
                    full = mask.expand(n_envs, 18)
                    assert ((info['action'] == -1) == ~full.any(1)).all()
                    assert full[info['action'] >= 0].gather(1, info['action'][info['action'] >= 0, None].long()).all()
    for bad in (dict(mask=per_env[:5]), dict(temperature=0.0), dict(uniforms=torch.rand(3, device='cuda'))):
        with pytest.raises(ValueError):
            env.step_policy(logits, **bad)
    with pytest.raises(TypeError):
        env.step_policy(logits, mask=per_env.float())
    env.close()
    twin.close()
