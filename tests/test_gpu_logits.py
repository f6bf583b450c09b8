"""ops.logits_sample and ops.logits_log_prob: policies over action sets of any size, against plain implementations in 64
bits.  -m gpu."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _logits(rows, A, dtype, dev, seed, spread=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(rows, A, generator=g, device=dev) * spread).to(dtype)


# ---------------------------------------------------------------------------------------------------- drawing


def draw_row(x, u, t, k, p, min_p):
    """one row in float64: (action, log_prob)"""
    x = np.asarray(x, np.float64)
    if np.isnan(x).any() or (x == np.inf).any():
        return -1, math.nan
    if (x == -np.inf).all():
        return -1, 0.0
    if t == 0:
        return int(np.argmax(x)), 0.0
    m = x.max()
    with np.errstate(over='ignore'):
        w = np.exp((x - m) / t)
    w[w < 2.0**-42] = 0.0
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[x[order] > -np.inf]
    if 0 < k < len(order):
        order = order[:k]
    total_k = w[order].sum()
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[order])[:-1]])
        keep = before < p * total_k
        keep[0] = True
        order = order[keep]
    order = np.concatenate([order[:1], order[1:][w[order[1:]] >= min_p]])
    kept = np.zeros_like(w)
    kept[order] = w[order]
    c = np.cumsum(kept)
    a = int(np.searchsorted(c, u * c[-1], side='right'))
    a = min(a, int(np.flatnonzero(kept)[-1]))
    return a, (x[a] - m) / t - math.log(w.sum())


def check_draw(logits, u, actions, log_probs, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = logits.shape[0]
    xs, us = logits.float().cpu().numpy(), u.cpu().numpy()
    col = lambda v, dt: np.broadcast_to(v.cpu().numpy() if torch.is_tensor(v) else np.asarray(v, dt), (rows, ))  # noqa: E731
    t, k, p, mp = col(temperature, np.float32), col(top_k, np.int64), col(top_p, np.float32), col(min_p, np.float32)
    got_a, got_l = actions.cpu().numpy(), log_probs.cpu().numpy()
    for r in range(rows):
        a, lp = draw_row(xs[r], us[r], float(t[r]), int(k[r]), float(p[r]), float(mp[r]))
        assert got_a[r] == a, 'row %d: %d, not %d' % (r, got_a[r], a)
        # rounded once to float32 from float64: half a step, and the float64 sums' own error far below it
        assert got_l[r] == pytest.approx(lp, rel=2.0**-23, abs=1e-12, nan_ok=True), 'row %d' % r


SETTINGS = [
    dict(),
    dict(temperature=0.7, top_k=5),
    dict(top_p=0.9),
    dict(min_p=0.05),
    dict(temperature=1.3, top_k=40, top_p=0.8, min_p=0.01),
    dict(temperature=0.0),
    dict(top_k=1),
    dict(top_p=0.0),
    dict(min_p=1.0),
    dict(temperature=50.0, top_k=1000, top_p=0.999),
]


@pytest.mark.parametrize('settings', SETTINGS, ids=lambda s: ','.join('%s=%s' % kv for kv in s.items()) or 'plain')
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,A', [(3, 1), (70, 2), (300, 6), (257, 18), (33, 63), (33, 64), (20, 65), (20, 257),
                                    (9, 1000), (5, 1025), (4, 4099), (3, 20000)])
def test_draw_matches_float64(rows, A, dtype, settings, dev):
    from parl_amd import ops
    x = _logits(rows, A, dtype, dev, rows + A)
    u = torch.rand(rows, generator=torch.Generator(device=dev).manual_seed(A), dtype=torch.float64, device=dev)
    a, lp = ops.logits_sample(x, u, **settings)
    assert a.dtype == torch.int64 and lp.dtype == torch.float32 and a.shape == (rows, )
    check_draw(x, u, a, lp, **settings)


@pytest.mark.parametrize('settings', [dict(), dict(top_k=50, top_p=0.9, temperature=0.7), dict(top_p=0.97), dict(min_p=0.001),
                                      dict(top_k=30000), dict(top_k=60000, top_p=0.5, temperature=3.0)],
                         ids=lambda s: ','.join('%s=%s' % kv for kv in s.items()) or 'plain')
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,A', [(2, 65537), (1, 131072), (3, 262144), (1, 1 << 20)])
def test_draw_of_long_rows_matches_float64(rows, A, dtype, settings, dev):
    from parl_amd import ops
    x = _logits(rows, A, dtype, dev, 7 + A, spread=2.0)
    u = torch.rand(rows, generator=torch.Generator(device=dev).manual_seed(A + 1), dtype=torch.float64, device=dev)
    check_draw(x, u, *ops.logits_sample(x, u, **settings), **settings)


@pytest.mark.parametrize('rows,A,dtype', [(2, 1 << 20, torch.bfloat16), (2, 300000, torch.float32), (36, 250000, torch.bfloat16),
                                          (3, 3500, torch.float32), (600, 17000, torch.bfloat16)])
def test_draw_from_flat_rows(rows, A, dtype, dev):
    """an untrained policy: many thousand values in the class that holds the border"""
    from parl_amd import ops
    x = _logits(rows, A, dtype, dev, 3, spread=0.3)
    u = torch.rand(rows, generator=torch.Generator(device=dev).manual_seed(4), dtype=torch.float64, device=dev)
    for s in (dict(top_p=0.6), dict(top_k=A // 3, top_p=0.99), dict(min_p=0.4)):
        check_draw(x, u, *ops.logits_sample(x, u, **s), **s)


@pytest.mark.parametrize('settings', [dict(), dict(top_k=20, top_p=0.8), dict(top_p=0.9, min_p=0.02), dict(temperature=0.0)])
@pytest.mark.parametrize('A', [18, 300, 4097, 40000])
def test_a_row_is_drawn_alike_in_any_batch(A, settings, dev):
    """alone, in a few, in many (other kernels, other splits), with settings as numbers or for each row: the same bits"""
    from parl_amd import ops
    rows = 1200
    x = _logits(rows, A, torch.bfloat16, dev, A)
    u = torch.rand(rows, generator=torch.Generator(device=dev).manual_seed(4), dtype=torch.float64, device=dev)
    a, lp = ops.logits_sample(x, u, **settings)
    for part in (slice(0, 1), slice(5, 20), slice(100, 400)):
        b, lq = ops.logits_sample(x[part], u[part], **settings)
        assert torch.equal(a[part], b) and torch.equal(lp[part], lq)
    each = {k: torch.full((rows, ), v, device=dev, dtype=torch.int32 if k == 'top_k' else torch.float32)
            for k, v in settings.items()}
    b, lq = ops.logits_sample(x, u, **each)
    assert torch.equal(a, b) and torch.equal(lp, lq)


def test_draw_from_more_rows_than_go_through_the_launches_together(dev):
    from parl_amd import ops
    rows, A = 66000, 4097
    x = _logits(rows, A, torch.bfloat16, dev, 1)
    u = torch.rand(rows, generator=torch.Generator(device=dev).manual_seed(4), dtype=torch.float64, device=dev)
    for s in (dict(), dict(top_p=0.7)):
        a, lp = ops.logits_sample(x, u, **s)
        for part in (slice(0, 700), slice(65000, 66000)):
            b, lq = ops.logits_sample(x[part], u[part], **s)
            assert torch.equal(a[part], b) and torch.equal(lp[part], lq)
    check_draw(x[-3:], u[-3:], a[-3:], lp[-3:], **s)


@pytest.mark.parametrize('A', [20, 3000, 5000])
def test_rows_whose_offsets_pass_32_bits(A, dev):
    from parl_amd import ops
    base = torch.empty(2**31 + 2 * A, dtype=torch.bfloat16, device=dev)
    x = base.as_strided((3, A), (2**30, 1))
    x.copy_(_logits(3, A, torch.bfloat16, dev, 8))
    u = torch.rand(3, generator=torch.Generator(device=dev).manual_seed(4), dtype=torch.float64, device=dev)
    for s in (dict(), dict(top_k=9, top_p=0.9)):
        a, lp = ops.logits_sample(x, u, **s)
        check_draw(x, u, a, lp, **s)
    check_logp(x, a, 1.0, dev)


@pytest.mark.parametrize('A', [18, 700, 5000, 70000])
def test_draw_with_settings_for_each_row(A, dev):
    from parl_amd import ops
    rows = 48 if A < 60000 else 12
    g = torch.Generator(device=dev).manual_seed(A)
    x = _logits(rows, A, torch.bfloat16, dev, A)
    u = torch.rand(rows, generator=g, dtype=torch.float64, device=dev)
    r = torch.rand(rows, 4, generator=g, device=dev)
    s = dict(temperature=torch.where(r[:, 0] < 0.2, 0.0, r[:, 0] * 2), top_k=(r[:, 1] * 60 - 10).to(torch.int32),
             top_p=r[:, 2] * 1.3, min_p=torch.where(r[:, 3] < 0.5, 0.0, r[:, 3] * 0.3))
    a, lp = ops.logits_sample(x, u, **s)
    check_draw(x, u, a, lp, **s)
    # a leading shape of its own
    a3, lp3 = ops.logits_sample(x.view(4, -1, A), u.view(4, -1), **{k: v.view(4, -1) for k, v in s.items()})
    assert a3.shape == (4, rows // 4) and torch.equal(a3.view(-1), a) and torch.equal(lp3.view(-1), lp)


@pytest.mark.parametrize('A', [6, 300, 9000, 40000])
@pytest.mark.parametrize('settings', [dict(), dict(top_k=7, top_p=0.7), dict(top_p=0.5), dict(min_p=0.5)])
def test_draw_among_ties_takes_the_lowest_indices(A, settings, dev):
    """rows of one value, of two, of a few: whole borders of equal logits"""
    from parl_amd import ops
    g = torch.Generator(device=dev).manual_seed(A)
    rows = 16
    x = torch.zeros(rows, A, device=dev)
    x[4:8] = torch.randint(0, 2, (4, A), generator=g, device=dev).float()
    x[8:12] = torch.randint(-3, 3, (4, A), generator=g, device=dev).float()
    x[12:] = torch.where(torch.rand(4, A, generator=g, device=dev) < 0.5, -0.0, 0.0)   # -0 equals 0
    u = torch.rand(rows, generator=g, dtype=torch.float64, device=dev)
    u[0], u[1], u[2] = 0.0, 0.5, 1.0 - 2.0**-53
    check_draw(x, u, *ops.logits_sample(x, u, **settings), **settings)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('A', [6, 500, 20000])
@pytest.mark.parametrize('settings', [dict(), dict(top_k=3), dict(top_p=0.6, temperature=0.5), dict(temperature=0.0)])
def test_draw_of_masked_and_bad_rows(A, dtype, settings, dev):
    from parl_amd import ops
    ops.consume_device_errors()
    x = _logits(12, A, dtype, dev, A)
    u = torch.rand(12, generator=torch.Generator(device=dev).manual_seed(3), dtype=torch.float64, device=dev)
    low = torch.finfo(dtype).min
    x[0] = float('-inf')                       # nothing legal
    x[1, 1:] = float('-inf')                   # one action left
    x[2, :-1] = float('-inf')
    x[3] = low                                 # the type's lowest value everywhere
    x[4, :A // 2] = low
    x[5, ::2] = float('-inf')
    x[6] = torch.finfo(dtype).max
    a, lp = ops.logits_sample(x, u, **settings)
    check_draw(x, u, a, lp, **settings)
    assert ops.consume_device_errors() == 0
    x[7, A // 2] = float('nan')
    x[8, 0] = float('inf')
    x[9] = float('nan')
    x[10, -1] = -float('nan')
    b, lpb = ops.logits_sample(x, u, **settings)
    check_draw(x, u, b, lpb, **settings)
    assert ops.consume_device_errors() > 0 and ops.consume_device_errors() == 0
    assert torch.equal(b[:7], a[:7]) and torch.equal(b[11:], a[11:])


@pytest.mark.parametrize('A', [50, 3000, 9000])
def test_draw_at_the_ends_of_the_uniforms(A, dev):
    """u = 0 takes the first kept action, the largest u the last; what lies outside [0, 1) counts as its nearest end"""
    from parl_amd import ops
    x = _logits(6, A, torch.float32, dev, 1)
    x[:, :5] = float('-inf')
    u = torch.tensor([0.0, 1.0 - 2.0**-53, -3.0, 1.0, 7.0, float('nan')], dtype=torch.float64, device=dev)
    for s in (dict(), dict(top_k=20), dict(top_p=0.4)):
        a, lp = ops.logits_sample(x, u, **s)
        v = torch.tensor([0.0, 1 - 2.0**-53, 0.0, 1 - 2.0**-53, 1 - 2.0**-53, 0.0], dtype=torch.float64)
        check_draw(x, v, a, lp, **s)


@pytest.mark.parametrize('A', [40, 800, 9000])
def test_settings_out_of_range_in_tensors_count_as_the_nearest_end(A, dev):
    from parl_amd import ops
    x = _logits(6, A, torch.float32, dev, 2)
    u = torch.rand(6, generator=torch.Generator(device=dev).manual_seed(3), dtype=torch.float64, device=dev)
    f = lambda *v: torch.tensor(v, device=dev)  # noqa: E731
    nan, inf = float('nan'), float('inf')
    a, lp = ops.logits_sample(x, u, temperature=f(-1.0, nan, 1.0, 1.0, 1.0, 1.0),
                              top_p=f(1.0, 1.0, nan, -2.0, 9.0, 1.0), min_p=f(0.0, 0.0, 0.0, 0.0, -1.0, 4.0))
    check_draw(x, u, a, lp, temperature=f(0.0, 0.0, 1.0, 1.0, 1.0, 1.0), top_p=f(1.0, 1.0, 0.0, 0.0, 9.0, 1.0),
               min_p=f(0.0, 0.0, 0.0, 0.0, 0.0, 1.0))
    # an endless temperature: every legal action alike
    x[:, 3] = -inf
    a, lp = ops.logits_sample(x, u, temperature=torch.full((6, ), inf, device=dev))
    legal = [i for i in range(A) if i != 3]
    for r in range(6):
        assert int(a[r]) == legal[int(float(u[r]) * (A - 1))]
        assert float(lp[r]) == pytest.approx(-math.log(A - 1), rel=1e-6)


@pytest.mark.parametrize('dtype', DTYPES)
def test_draw_reads_rows_of_a_wider_buffer_and_other_layouts(dtype, dev):
    from parl_amd import ops
    wide = _logits(20, 1013, dtype, dev, 4)
    u = torch.rand(20, generator=torch.Generator(device=dev).manual_seed(5), dtype=torch.float64, device=dev)
    for x in (wide[:, :1000], wide[:, 13:], wide[:, 1:400], wide[:, ::2], wide[:1].expand(20, 1013), wide[:, 5:6]):
        a, lp = ops.logits_sample(x, u, top_k=30)
        check_draw(x, u, a, lp, top_k=30)
    y = wide[:, :20].t()
    a, lp = ops.logits_sample(y, u, top_p=0.9)
    check_draw(y, u, a, lp, top_p=0.9)
    a, lp = ops.logits_sample(wide[3], u[3], temperature=0.5)   # one row without a leading axis
    assert a.shape == () and lp.shape == ()
    check_draw(wide[3:4], u[3:4], a.view(1), lp.view(1), temperature=0.5)


def test_draw_of_no_rows(dev):
    from parl_amd import ops
    a, lp = ops.logits_sample(torch.empty(0, 7, device=dev), torch.empty(0, dtype=torch.float64, device=dev), top_k=3)
    assert a.shape == (0, ) and lp.shape == (0, )


def test_draw_refusals(dev):
    from parl_amd import ops
    from parl_amd._native import ParlHipError
    x = torch.zeros(4, 10, device=dev)
    u = torch.zeros(4, dtype=torch.float64, device=dev)
    bad = [
        (x.double(), u, {}), (x.long(), u, {}), (x.cpu(), u, {}), (x, u.cpu(), {}), (x, u.float(), {}), (x, u[:3], {}),
        (torch.zeros(4, 0, device=dev), u, {}), (torch.tensor(1.0, device=dev), u, {}),
        (x, u, dict(temperature=-1.0)), (x, u, dict(temperature=float('nan'))), (x, u, dict(temperature=float('inf'))),
        (x, u, dict(temperature=1e39)), (x, u, dict(top_p=-0.1)), (x, u, dict(top_p=float('nan'))),
        (x, u, dict(min_p=-0.1)), (x, u, dict(min_p=1.1)), (x, u, dict(min_p=float('nan'))), (x, u, dict(top_k=2.5)),
        (x, u, dict(top_k=2**31)), (x, u, dict(top_k=torch.zeros(4, device=dev))),
        (x, u, dict(top_k=torch.zeros(4, dtype=torch.int64, device=dev))),
        (x, u, dict(top_p=torch.ones(4, dtype=torch.float64, device=dev))), (x, u, dict(top_p=torch.ones(3, device=dev))),
        (x, u, dict(temperature=torch.ones(4))),
        (torch.zeros(1, (1 << 20) + 1, device=dev), u[:1], {}),
    ]
    for logits, uniforms, settings in bad:
        with pytest.raises(ParlHipError):
            ops.logits_sample(logits, uniforms, **settings)


# ------------------------------------------------------------------------------------- log-probability and gradient


def logp_f64(logits, actions, g_logp, g_ent, T):
    """log-probability, entropy and gradient in float64, by the formulas; row by row independent"""
    z = logits.detach().to(torch.float64).cpu() / T
    rows, A = z.shape
    a = actions.cpu()
    live = (a >= 0) & ~(z == -math.inf).all(1)
    zl = torch.where(live.view(-1, 1), z, torch.zeros_like(z))
    lp = torch.log_softmax(zl, 1)
    p = lp.exp()
    lp0 = torch.where(p > 0, lp, torch.zeros_like(lp))
    lp0 = torch.where(torch.isnan(p), p, lp0)
    ent = -(p * lp0).sum(1)
    taken = lp.gather(1, a.clamp(min=0).view(-1, 1)).view(-1)
    grad = torch.zeros_like(p)
    grad.scatter_(1, a.clamp(min=0).view(-1, 1), g_logp.double().cpu().view(-1, 1))
    grad = grad - p * (g_logp.double().cpu().view(-1, 1) + g_ent.double().cpu().view(-1, 1) * (lp0 + ent.view(-1, 1)))
    zero = torch.zeros_like(taken)
    grad = torch.where(live.view(-1, 1), grad / T, torch.zeros_like(grad))
    return torch.where(live, taken, zero), torch.where(live, ent, zero), grad


def check_logp(logits, actions, T, dev, seed=0, use=(True, True)):
    from parl_amd import ops
    rows, A = logits.shape
    g = torch.Generator(device=dev).manual_seed(seed)
    g_logp = torch.randn(rows, generator=g, device=dev) * use[0]
    g_ent = torch.randn(rows, generator=g, device=dev) * 0.1 * use[1]
    x = logits.detach().requires_grad_(True)
    lp, ent = ops.logits_log_prob(x, actions, temperature=T)
    assert lp.dtype == torch.float32 and ent.dtype == torch.float32 and lp.shape == (rows, )
    outs = [(o, gg) for o, gg, on in ((lp, g_logp, use[0]), (ent, g_ent, use[1])) if on]
    grad, = torch.autograd.grad([o for o, _ in outs], [x], [gg for _, gg in outs])
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    r_lp, r_ent, r_grad = logp_f64(logits, actions, g_logp, g_ent, T)
    # float32 sums of up to A terms in chains of n = A / 256 (a thread's part), pairwise behind that: relative error of s
    # and t at most (n + 24) 2^-24; a logit's distance d from the maximum is rounded at |d| 2^-24 and 2^x / log2 at
    # 2^-23; |t / s| and |log s| are at most the entropy's scale log A + 1
    n = max(8, A / 256) + 24
    scale = math.log(A) + 1
    tol = 2.0**-24 * (n + 8) * scale
    fin = torch.isfinite(r_lp)
    d = (lp.detach().cpu().double() - r_lp)[fin].abs()
    assert (d <= tol + 4 * 2.0**-24 * r_lp[fin].abs()).all(), float(d.max())
    assert torch.equal(lp.detach().cpu()[~fin].double().nan_to_num(nan=7.0), r_lp[~fin].nan_to_num(nan=7.0))
    fin = torch.isfinite(r_ent)
    d = (ent.detach().cpu().double() - r_ent)[fin].abs()
    assert (d <= 2 * tol).all(), float(d.max())
    assert torch.isnan(ent.detach().cpu()[~fin]).all()
    # the gradient: p (relative 2^-24 (n + |d| + 8)) times g_l + g_h (log p + H), rounded once to the logits' type; at the
    # taken action the difference of two numbers of at most `size`, each rounded a few times: 2^-22 size, also where
    # they cancel (p near 1)
    half = torch.finfo(logits.dtype).eps / 2
    size = (g_logp.abs().cpu().double() + g_ent.abs().cpu().double() * 2 * scale).view(-1, 1) / T
    fin = torch.isfinite(r_grad)
    d = (grad.cpu().double() - r_grad).abs()
    zl = (logits.detach().double().cpu() / T)
    p = torch.softmax(zl.masked_fill((zl == -math.inf).all(1, keepdim=True), 0.0), 1)
    dist = (-torch.log(p)).clamp(max=200.0)
    bound = half * r_grad.abs() + 2.0**-24 * (n + 8 + 4 * dist) * size * p * 4 + torch.finfo(logits.dtype).smallest_normal
    bound.scatter_add_(1, actions.cpu().clamp(min=0).view(-1, 1), 2.0**-22 * size)
    if not (d <= bound)[fin].all():
        r, i = divmod(int(torch.where(fin, d / bound, torch.zeros_like(d)).argmax()), A)
        print('row', r, 'index', i, 'action', int(actions[r]), 'got', float(grad[r, i]), 'want', float(r_grad[r, i]), 'p', float(p[r, i]))
    assert (d <= bound)[fin].all(), float((d / bound)[fin].max())
    assert torch.isnan(grad.cpu()[~fin]).all()
    return lp, ent, grad


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('T', [1.0, 0.7])
@pytest.mark.parametrize('rows,A', [(3, 1), (700, 2), (1000, 6), (515, 18), (70, 32), (70, 33), (65, 128), (65, 129), (31, 512),
                                    (31, 513), (17, 1000), (9, 4096), (9, 4097), (5, 20003), (2, 131072), (1100, 600)])
def test_log_prob_entropy_and_gradient_match_float64(rows, A, T, dtype, dev):
    x = _logits(rows, A, dtype, dev, rows * 7 + A)
    a = torch.randint(0, A, (rows, ), generator=torch.Generator(device=dev).manual_seed(A), device=dev)
    a[::5] = -1
    lp, ent, grad = check_logp(x, a, T, dev)
    assert (lp[::5] == 0).all() and (ent[::5] == 0).all() and (grad[::5] == 0).all()


@pytest.mark.parametrize('use', [(True, False), (False, True)])
@pytest.mark.parametrize('rows,A', [(40, 18), (6, 3000), (2, 70001)])
def test_log_prob_gradient_of_one_output_only(rows, A, use, dev):
    x = _logits(rows, A, torch.float32, dev, A)
    a = torch.randint(0, A, (rows, ), generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    check_logp(x, a, 1.0, dev, use=use)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('A', [6, 100, 500, 3000, 50000])
def test_log_prob_of_masked_and_bad_rows(A, dtype, dev):
    from parl_amd import ops
    ops.consume_device_errors()
    x = _logits(10, A, dtype, dev, A)
    low = torch.finfo(dtype).min
    a = torch.randint(0, A, (10, ), generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    x[0] = float('-inf')                       # nothing legal: ignored
    x[1, 1:] = float('-inf')                   # one action left, and it is taken
    a[1] = 0
    x[2, :A - 2] = float('-inf')
    a[2] = 0                                   # an action that could not have been taken
    x[3] = low
    x[4, ::2] = low
    x[5] = -1000.0
    clean = check_logp(x, a, 1.0, dev)
    assert float(clean[0][0]) == 0 and float(clean[1][0]) == 0 and (clean[2][0] == 0).all()
    assert float(clean[0][1]) == 0 and float(clean[0][2]) == -math.inf
    y = x.clone()
    y[6, A // 2] = float('nan')
    y[7, 0] = float('inf')
    bad = check_logp(y, a, 1.0, dev)
    for c, b in zip(clean, bad):
        assert torch.equal(c[:6], b[:6]) and torch.equal(c[8:], b[8:]) and torch.isnan(b[6:8]).all()
    assert ops.consume_device_errors() == 0


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('A', [1, 6, 100, 500, 3000, 50000])
def test_log_prob_of_rows_without_any_number_but_nan_is_nan(A, dtype, dev):
    """a network that has diverged: no maximum, as in an empty row, but not ignored as one"""
    from parl_amd import ops
    x = _logits(4, A, dtype, dev, A)
    x[1] = float('nan')
    x[2, 1:] = float('-inf')
    x[2, 0] = float('nan')
    x[3] = float('-inf')
    x = x.requires_grad_(True)
    lp, ent = ops.logits_log_prob(x, torch.zeros(4, dtype=torch.int64, device=dev))
    grad, = torch.autograd.grad((lp, ent), (x, ), (torch.ones_like(lp), torch.ones_like(ent)))
    for t in (lp, ent, grad):
        assert torch.isfinite(t[0]).all() and torch.isnan(t[1:3]).all() and (t[3] == 0).all()


@pytest.mark.parametrize('A', [6, 3000])
def test_log_prob_of_an_action_outside_the_set_is_clamped_and_flagged(A, dev):
    from parl_amd import ops
    ops.consume_device_errors()
    x = _logits(4, A, torch.float32, dev, A)
    a = torch.tensor([-2, A, 1, 2**40], device=dev)
    lp, ent = ops.logits_log_prob(x, a)
    want, _ = ops.logits_log_prob(x, torch.tensor([0, A - 1, 1, A - 1], device=dev))
    assert torch.equal(lp, want)
    assert ops.consume_device_errors() > 0 and ops.consume_device_errors() == 0


@pytest.mark.parametrize('dtype', DTYPES)
def test_log_prob_reads_other_layouts(dtype, dev):
    from parl_amd import ops
    wide = _logits(24, 1013, dtype, dev, 4)
    for x in (wide[:, :1000], wide[:, 13:], wide[:, 1:30], wide[:, ::2], wide[:, :24].t(), wide[:1].expand(24, 1013)):
        A = x.shape[1]
        a = torch.randint(0, A, (x.shape[0], ), generator=torch.Generator(device=dev).manual_seed(2), device=dev)
        check_logp(x, a, 0.9, dev)
        lp, ent = ops.logits_log_prob(x, a, 0.9)
        lc, ec = ops.logits_log_prob(x.contiguous().view(4, -1, A), a.view(4, -1), 0.9)
        assert lc.shape == (4, x.shape[0] // 4) and torch.equal(lc.view(-1), lp) and torch.equal(ec.view(-1), ent)
    one = wide[0].detach().requires_grad_(True)
    lp, ent = ops.logits_log_prob(one, torch.tensor(5, device=dev))
    assert lp.shape == ()
    (lp + ent).backward()
    assert one.grad.shape == one.shape
    # the gradient of a view reaches its base: the padded columns get zeros
    base = wide.detach().clone().requires_grad_(True)
    lp, _ = ops.logits_log_prob(base[:, :1000], torch.zeros(24, dtype=torch.int64, device=dev))
    lp.sum().backward()
    assert (base.grad[:, 1000:] == 0).all() and (base.grad[:, 0] != 0).any()


def test_log_prob_of_no_rows(dev):
    from parl_amd import ops
    x = torch.empty(0, 9, device=dev, requires_grad=True)
    lp, ent = ops.logits_log_prob(x, torch.empty(0, dtype=torch.int64, device=dev))
    (lp.sum() + ent.sum()).backward()
    assert lp.shape == (0, ) and x.grad.shape == (0, 9)


def test_lazily_negated_views_are_read_as_what_they_are(dev):
    """the imaginary part of a conjugate: a view whose memory holds the values with the other sign"""
    from parl_amd import ops

    def pair(*shape, dtype=torch.float32):
        t = torch.randn(*shape, 2, dtype=dtype, device=dev)
        v = torch.view_as_complex(t).conj().imag
        assert v.is_neg()
        return v, -t[..., 1]

    x, x0 = pair(20, 33)
    y, y0 = pair(20, 33, 1)
    u, u0 = pair(20, dtype=torch.float64)
    a = torch.randint(0, 33, (20, ), device=dev)
    for v, v0 in ((x, x0), (y[..., 0], y0[..., 0])):
        for got, want in zip(ops.logits_sample(v, u), ops.logits_sample(v0.contiguous(), u0.contiguous())):
            assert torch.equal(got, want)
    leaf, leaf0 = x.detach().requires_grad_(True), x0.contiguous().requires_grad_(True)
    g, g0 = pair(20)
    out, out0 = ops.logits_log_prob(leaf, a), ops.logits_log_prob(leaf0, a)
    assert torch.equal(out[0], out0[0]) and torch.equal(out[1], out0[1])
    assert torch.equal(torch.autograd.grad(out, (leaf, ), (g, g))[0],
                       torch.autograd.grad(out0, (leaf0, ), (g0.contiguous(), g0.contiguous()))[0])


@pytest.mark.parametrize('lead', [(0, ), (3, 0)])
@pytest.mark.parametrize('A', [1, 9, 600, 5000, 131072])
def test_no_rows_of_any_length(A, lead, dev):
    from parl_amd import ops
    x = torch.empty(*lead, A, device=dev, requires_grad=True)
    a, lp0 = ops.logits_sample(x, torch.empty(lead, dtype=torch.float64, device=dev), top_p=0.9)
    assert a.shape == lead and lp0.shape == lead
    lp, ent = ops.logits_log_prob(x, a)
    (lp.sum() + ent.sum()).backward()
    assert lp.shape == lead and ent.shape == lead and x.grad.shape == x.shape


def test_log_prob_gradient_matches_differences(dev):
    """central differences of the float64 formula at the kernel's own gradient"""
    x = _logits(3, 11, torch.float32, dev, 5, spread=1.0)
    a = torch.tensor([0, 10, 4], device=dev)
    from parl_amd import ops
    y = x.detach().requires_grad_(True)
    lp, ent = ops.logits_log_prob(y, a, 0.8)
    (1.5 * lp - 0.3 * ent).sum().backward()
    h = 1e-5

    def value(z):
        q = torch.log_softmax(z / 0.8, 1)
        return (1.5 * q.gather(1, a.cpu().view(-1, 1)).view(-1) + 0.3 * (q.exp() * q).sum(1)).sum()

    z = x.double().cpu()
    for r in range(3):
        for i in range(11):
            e = torch.zeros_like(z)
            e[r, i] = h
            want = float((value(z + e) - value(z - e)) / (2 * h))
            # differences: h^2 / 6 times a third derivative of at most ~10, rounding 1e-16 / h; the kernel: float32
            assert float(y.grad[r, i]) == pytest.approx(want, abs=1e-6)


def test_log_prob_refusals(dev):
    from parl_amd import ops
    from parl_amd._native import ParlHipError
    x = torch.zeros(4, 10, device=dev)
    a = torch.zeros(4, dtype=torch.int64, device=dev)
    for logits, actions, T in [(x.double(), a, 1.0), (x.cpu(), a.cpu(), 1.0), (x, a.cpu(), 1.0), (x, a.int(), 1.0),
                               (x, a[:3], 1.0), (x, a, 0.0), (x, a, -1.0), (x, a, float('nan')), (x, a, float('inf')),
                               (x, a, 1e-39), (torch.zeros(4, 0, device=dev), a, 1.0)]:
        with pytest.raises(ParlHipError):
            ops.logits_log_prob(logits, actions, T)


# ------------------------------------------------------------------------------------------------- used together


@pytest.mark.parametrize('dtype,A', [(torch.float32, 18), (torch.bfloat16, 5000), (torch.float32, 40000)])
def test_the_learner_finds_the_log_prob_that_the_actor_drew_with(dtype, A, dev):
    """logits_sample's log_probs are logits_log_prob's at the same temperature, empty rows (action -1) included"""
    from parl_amd import ops
    x = _logits(64, A, dtype, dev, 9)
    x[:, ::3] = float('-inf')
    x[7] = float('-inf')
    u = torch.rand(64, generator=torch.Generator(device=dev).manual_seed(1), dtype=torch.float64, device=dev)
    a, lp = ops.logits_sample(x, u, temperature=0.8, top_k=200)
    assert int(a[7]) == -1 and (a[:7] % 3 != 0).all()
    lp2, ent = ops.logits_log_prob(x, a, temperature=0.8)
    torch.testing.assert_close(lp, lp2, rtol=2e-6, atol=2.0**-24 * (A / 256 + 40) * 12)
    assert float(lp2[7]) == 0 and float(ent[7]) == 0


@pytest.mark.parametrize('A', [18, 5000, 70000])
def test_calls_on_two_streams_and_in_a_replayed_graph(A, dev):
    from parl_amd import ops
    xs = [_logits(8, A, torch.bfloat16, dev, s) for s in (1, 2)]
    us = [torch.rand(8, generator=torch.Generator(device=dev).manual_seed(s), dtype=torch.float64, device=dev) for s in (3, 4)]
    s = dict(temperature=0.9, top_p=0.9)
    want = [ops.logits_sample(x, u, **s) for x, u in zip(xs, us)]

    def step(x, u):
        y = x.detach().requires_grad_(True)
        a, lp = ops.logits_sample(x, u, **s)
        l2, e2 = ops.logits_log_prob(y, a, 0.9)
        g, = torch.autograd.grad([l2, e2], [y], [torch.ones_like(l2), torch.ones_like(e2)])
        return a, lp, l2.detach(), e2.detach(), g

    full = [step(x, u) for x, u in zip(xs, us)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for st, x, u in zip(streams, xs, us):
            with torch.cuda.stream(st):
                got.append(step(x, u))
        torch.cuda.synchronize()
        for w, f, o in zip(want, full, got):
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])
            assert all(torch.equal(p, q) for p, q in zip(f, o))
    # two graphs, replayed in turn with eager work between, on new inputs
    bufs = [(x.clone(), u.clone()) for x, u in zip(xs, us)]
    graphs, outs = [], []
    for x, u in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(streams[0]):
            step(x, u)
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            outs.append(step(x, u))
        graphs.append(g)
    for k in range(4):
        for i in (0, 1):
            j = (i + k) % 2
            bufs[i][0].copy_(xs[j])
            bufs[i][1].copy_(us[j])
            graphs[i].replay()
            step(xs[0], us[0])
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(full[j], outs[i]))


# -------------------------------------------------------------------------------- one definition in every form


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('A', [600, 4096, 5000, 20000, 131072, 1 << 20])
def test_a_weight_under_the_floor_counts_nothing(A, dtype, dev):
    """Rows full of values just under 2^-42 of the largest, one just above it in every thousand: those under it are no choice
    and no part of the mass, with a filter that keeps everything, without one, and in any type."""
    from parl_amd import ops
    x = torch.full((12, A), -29.125, dtype=dtype, device=dev)   # 2^-42.08; exact in every type
    x[:, ::1000] = -29.0                                         # 2^-41.9
    x[8:, ::1000] = -29.125                                      # nothing but the largest
    x[:4, -1], x[4:8, 0], x[8:, A // 2] = 0.0, 0.0, 0.0
    t = float(np.float32(29.0 / math.log(2.0) / 41.9))
    few = A * 2.0**-42.08                                        # what the values under the floor would add up to
    u = torch.tensor([0.0, 0.2 * few, 0.5 * few, 0.5] * 3, dtype=torch.float64, device=dev)
    a, lp = ops.logits_sample(x, u, temperature=t)
    xs, us = x.double().cpu().numpy(), u.cpu().numpy()
    bits = math.ceil(math.log2(A))
    for r in range(12):
        want, want_lp = draw_row(xs[r], us[r], t, 0, 1.0, 0.0)
        assert int(a[r]) == want, 'row %d' % r
        # each of the n weights is off by at most half a unit of 2^-min(51, 62 - bits), the logarithm rounded once
        n = -(-A // 1000)
        assert float(lp[r]) == pytest.approx(want_lp, rel=2.0**-23, abs=n * 2.0**-(min(51, 62 - bits) + 1) + 1e-15), 'row %d' % r
    k = torch.zeros(12, dtype=torch.int32, device=dev)
    k[::2] = A
    for y, kw in ((x, dict(top_k=A)), (x, dict(top_k=k)), (x.float(), dict()), (x.float(), dict(top_k=A))):
        b, lq = ops.logits_sample(y, u, temperature=t, **kw)
        assert torch.equal(a, b) and torch.equal(lp, lq), kw


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('A', [18, 64, 300, 700, 4096, 4097, 40000, 131072])
def test_a_filter_that_keeps_everything_changes_nothing(A, dtype, dev):
    """top-k of all actions, a minimum that none is under, float32 copies of 16-bit rows: the same bits"""
    from parl_amd import ops
    rows = 48
    x = _logits(rows, A, dtype, dev, A, spread=4.0)
    x[::5, ::3] = float('-inf')
    x[7] = float('-inf')
    u = torch.rand(rows, generator=torch.Generator(device=dev).manual_seed(A), dtype=torch.float64, device=dev)
    a, lp = ops.logits_sample(x, u, temperature=0.8)
    k = torch.zeros(rows, dtype=torch.int32, device=dev)
    k[::2] = A
    for y, kw in ((x, dict(top_k=A)), (x, dict(top_k=k)), (x, dict(min_p=2.0**-44)), (x.float(), dict()), (x.float(), dict(top_k=A))):
        b, lq = ops.logits_sample(y, u, temperature=0.8, **kw)
        assert torch.equal(a, b) and torch.equal(lp, lq), kw


@pytest.mark.parametrize('times', [190, 6000])
def test_draw_from_any_number_of_long_rows(times, dev):
    """133,000 rows, and more than four million (34 GB): each block of 700 is drawn as it is alone"""
    from parl_amd import ops
    A = 4097
    block = _logits(700, A, torch.bfloat16, dev, 1)
    u = torch.rand(700, generator=torch.Generator(device=dev).manual_seed(4), dtype=torch.float64, device=dev)
    x, us = block.repeat(times, 1), u.repeat(times)
    for s in (dict(), dict(temperature=0.0), dict(top_p=0.7)):
        a, lp = ops.logits_sample(block, u, **s)
        b, lq = ops.logits_sample(x, us, **s)
        assert (b.view(times, 700) == a).all() and (lq.view(times, 700) == lp).all(), s


def test_log_prob_with_a_temperature_for_each_row(dev):
    """is refused by its name; the logits divided by it are the same policy, which the draw's log_probs agree with"""
    from parl_amd import ops
    from parl_amd._native import ParlHipError
    rows, A = 24, 5000
    x = _logits(rows, A, torch.bfloat16, dev, 3)
    g = torch.Generator(device=dev).manual_seed(1)
    u, t = torch.rand(rows, generator=g, dtype=torch.float64, device=dev), torch.rand(rows, generator=g, device=dev) + 0.3
    a, lp = ops.logits_sample(x, u, temperature=t)
    with pytest.raises(ParlHipError, match='divide the logits'):
        ops.logits_log_prob(x, a, temperature=t)
    got, _ = ops.logits_log_prob(x.float() / t.unsqueeze(-1), a)
    # float32 logits of up to 45, divided: half a step each of the row's largest and the action's; sums as in check_logp
    torch.testing.assert_close(got, lp, rtol=2.0**-22, atol=2.0**-24 * (2 * 45 + (A / 256 + 32) * (math.log(A) + 1)))
    one, _ = ops.logits_log_prob(x, a, temperature=torch.tensor(0.7))
    assert torch.equal(one, ops.logits_log_prob(x, a, temperature=float(torch.tensor(0.7)))[0])
