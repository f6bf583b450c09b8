"""ops.grad_norm and ops.clip_grad_norm_: the global norm over many tensors, and clipping, against 64-bit sums.  -m gpu."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _grads(shapes, dtypes, dev, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(torch.randn(s, generator=g, device=dev) * scale).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


def _params(grads):
    ps = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(ps, grads):
        p.grad = g
    return ps


def _norm64(tensors):
    return math.sqrt(math.fsum(float(t.detach().double().square().sum()) for t in tensors))


def _check(before, after, norm, max_norm):
    want = _norm64(before)
    # sums in float64 and one rounding to float32
    assert float(norm) == pytest.approx(want, rel=2.0**-23)
    clip = min(1.0, max_norm / (want + 1e-6))
    for b, a in zip(before, after):
        # the factor rounded to float32, the product in float32, then to the tensor's type
        half = torch.finfo(a.dtype).eps / 2
        w = b.double() * clip
        assert ((a.double() - w).abs() <= w.abs() * (half + 2.0**-22) + torch.finfo(a.dtype).smallest_normal * half * 2).all()


SHAPES = [
    [(1, )],
    [(16, 4, 4, 4), (16, ), (32, 16, 4, 4), (32, ), (256, 3872), (256, ), (6, 256), (6, ), (1, 256), (1, )],
    [(3, 5), (0, 7), (16384, ), (16385, ), (16383, ), (1, ), (2, ), (7, 11, 13)],
    [(17 * (i % 9) + 1, ) for i in range(97)],
    [(1 + (i * 37) % 301, ) for i in range(400)],
    [(5000003, ), (3, )],
    [(40000001, )],
]


@pytest.mark.parametrize('shapes', SHAPES, ids=lambda s: '%dx%s' % (len(s), s[0]))
@pytest.mark.parametrize('dtypes', [[d] for d in DTYPES] + [DTYPES], ids=lambda d: '+'.join(str(x)[6:] for x in d))
@pytest.mark.parametrize('ratio', [0.3, 5.0])
def test_clip_in_place_matches_float64(shapes, dtypes, ratio, dev):
    from parl_amd import ops
    grads = _grads(shapes, dtypes, dev, len(shapes))
    before = [g.clone() for g in grads]
    max_norm = ratio * _norm64(before)
    versions = [g._version for g in grads]
    norm = ops.clip_grad_norm_(_params(grads), max_norm)
    assert norm.shape == () and norm.dtype == torch.float32 and norm.is_cuda
    _check(before, grads, norm, max_norm)
    if ratio > 1:
        assert all(torch.equal(a, b) for a, b in zip(before, grads))
    assert all(g._version > v for g, v in zip(grads, versions))
    assert float(ops.grad_norm(before)) == float(norm)
    again = [b.clone() for b in before]
    assert float(ops.clip_grad_norm_(_params(again), max_norm)) == float(norm)
    assert all(torch.equal(a, b) for a, b in zip(again, grads))      # the same bits in every call


@pytest.mark.parametrize('src', DTYPES)
@pytest.mark.parametrize('dst', DTYPES)
@pytest.mark.parametrize('ratio', [0.3, 5.0])
def test_clip_into_other_tensors(src, dst, ratio, dev):
    """the views of one flat buffer start at any element"""
    from parl_amd import ops
    sizes = [1, 7, 4096, 16384, 16391, 3, 100001, 0, 5]
    flat = torch.randn(sum(sizes), generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(src)
    grads = list(flat.split(sizes))
    keep = flat.clone()
    out_flat = torch.full((sum(sizes) + 2, ), 7.0, dtype=dst, device=dev)
    out = list(out_flat[1:-1].split(sizes))
    max_norm = ratio * _norm64(grads)
    norm = ops.clip_grad_norm_(_params(grads), max_norm, out=out)
    assert torch.equal(flat, keep)
    _check(grads, out, norm, max_norm)
    assert float(out_flat[0]) == 7 and float(out_flat[-1]) == 7       # the neighbours are as they were


def test_a_tensor_of_more_than_32_bits_of_elements(dev):
    from parl_amd import ops
    n = 2**31 + 19
    g = torch.full((n, ), 0.5, dtype=torch.bfloat16, device=dev)
    g[-1] = 2.0
    norm = ops.clip_grad_norm_(_params([g]), 0.25 * math.sqrt(n))
    want = math.sqrt((n - 1) * 0.25 + 4.0)
    assert float(norm) == pytest.approx(want, rel=2.0**-23)
    c = 0.25 * math.sqrt(n) / (want + 1e-6)
    for i in (0, 1, 2**30, 2**31 - 1, 2**31, n - 2):
        assert float(g[i]) == pytest.approx(0.5 * c, rel=2.0**-8)
    assert float(g[-1]) == pytest.approx(2.0 * c, rel=2.0**-8)
    assert int((g[:-1] != g[0]).sum()) == 0


def test_clip_of_other_layouts(dev):
    from parl_amd import ops
    g = torch.Generator(device=dev).manual_seed(1)
    a = torch.randn(8, 16, 5, 5, generator=g, device=dev).to(memory_format=torch.channels_last)
    b = torch.randn(40, 30, generator=g, device=dev).t()
    before = [a.clone(), b.clone()]
    norm = ops.clip_grad_norm_(_params([a, b]), 1.0)
    _check(before, [a, b], norm, 1.0)
    o = [torch.empty_like(a), torch.empty_like(b)]
    ops.clip_grad_norm_(_params(before), 1.0, out=o)
    assert torch.equal(o[0], a) and torch.equal(o[1], b)


def test_clip_takes_what_torch_takes(dev):
    """one tensor, an iterator, parameters without a gradient, none at all; torch's own result"""
    from parl_amd import ops
    ps = _params(_grads([(100, 3), (7, )], [torch.float32], dev, 3))
    ps.insert(1, torch.nn.Parameter(torch.zeros(5, device=dev)))
    qs = [torch.nn.Parameter(torch.zeros_like(p)) for p in ps]
    for p, q in zip(ps, qs):
        q.grad = None if p.grad is None else p.grad.clone()
    want = torch.nn.utils.clip_grad_norm_(qs, 2.0)
    got = ops.clip_grad_norm_(iter(ps), 2.0)
    torch.testing.assert_close(got, want, rtol=2e-6, atol=0)
    for p, q in zip(ps, qs):
        assert p.grad is None and q.grad is None or torch.allclose(p.grad, q.grad, rtol=4e-6, atol=0)
    one = _params(_grads([(33, )], [torch.float32], dev, 4))[0]
    assert float(ops.clip_grad_norm_(one, 1e9)) == pytest.approx(_norm64([one.grad]), rel=1e-6)
    assert float(ops.clip_grad_norm_([], 1.0)) == 0 and float(ops.grad_norm([])) == 0
    assert float(ops.clip_grad_norm_([torch.nn.Parameter(torch.zeros(5, device=dev))], 1.0)) == 0
    assert float(ops.grad_norm([torch.zeros(0, device=dev)])) == 0
    z = _params([torch.zeros(9, device=dev)])
    assert float(ops.clip_grad_norm_(z, 1.0)) == 0 and (z[0].grad == 0).all()
    h = _params([torch.ones(9, device=dev)])
    assert float(ops.clip_grad_norm_(h, 0.0)) == 3 and (h[0].grad == 0).all()
    i = _params([torch.ones(9, device=dev)])
    assert float(ops.clip_grad_norm_(i, float('inf'))) == 3 and (i[0].grad == 1).all()


def test_norm_of_values_whose_squares_leave_the_float_range(dev):
    from parl_amd import ops
    for v in (1e30, 1e-30):
        g = torch.full((1000, ), v, device=dev)
        assert float(ops.grad_norm([g])) == pytest.approx(float(g[0]) * math.sqrt(1000), rel=1e-6)


def test_non_finite_norms(dev):
    from parl_amd import ops
    for v, other in ((float('nan'), float('nan')), (float('inf'), 0.0)):
        grads = [torch.ones(5000, device=dev), torch.ones(20, device=dev)]
        grads[1][3] = v
        keep = [g.clone() for g in grads]
        with pytest.raises(RuntimeError):
            ops.clip_grad_norm_(_params(grads), 1.0, error_if_nonfinite=True)
        assert torch.equal(grads[0], keep[0])
        norm = ops.clip_grad_norm_(_params(grads), 1.0)
        assert not math.isfinite(float(norm))
        # as torch: a NaN norm turns everything NaN, an endless one takes the finite values to 0
        torch.testing.assert_close(grads[0], torch.full_like(grads[0], other), equal_nan=True)
        assert math.isnan(float(grads[1][3]))


def test_refusals(dev):
    from parl_amd import ops
    from parl_amd._native import ParlHipError
    ones = lambda *s, **k: torch.ones(*s, device=dev, **k)  # noqa: E731
    shared = ones(100)
    cases = [
        ([torch.ones(3)], {}), ([ones(3, dtype=torch.float64)], {}), ([ones(3), torch.ones(3)], {}),
        ([ones(4, 6)[:, ::2]], {}), ([ones(1).expand(5)], {}), ([shared, shared], {}), ([shared[:60], shared[40:]], {}),
        ([ones(3)], dict(out=[])), ([ones(3)], dict(out=[ones(4)])), ([ones(3)], dict(out=[torch.ones(3)])),
        ([ones(3)], dict(out=[ones(3, dtype=torch.float64)])), ([ones(4, 6)], dict(out=[ones(6, 4).t()])),
        ([shared[:50], shared[50:]], dict(out=[shared[50:], ones(50)])),
        ([shared[:50]], dict(out=[shared[10:60]])), ([ones(50), ones(50)], dict(out=[shared[:50], shared[20:70]])),
        ([shared], dict(out=[shared.view(torch.int32).view(torch.bfloat16)[:100]])),
    ]
    for grads, kw in cases:
        ps = [torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype, device=g.device)) for g in grads]
        for p, g in zip(ps, grads):
            p.grad = g
        with pytest.raises(ParlHipError):
            ops.clip_grad_norm_(ps, 1.0, **kw)
        assert all((g == 1).all() for g in grads)
    for m in (-1.0, float('nan')):
        with pytest.raises(ParlHipError):
            ops.clip_grad_norm_(_params([ones(3)]), m)
    with pytest.raises(ParlHipError):
        ops.grad_norm([torch.ones(3)])
    with pytest.raises(ParlHipError):
        ops.grad_norm([torch.sparse_coo_tensor([[0]], [1.0], (3, ), device=dev)])
    assert float(ops.grad_norm([shared, shared])) == pytest.approx(math.sqrt(200))   # reading twice is no conflict


def test_a_lazily_negated_view_is_refused(dev):
    from parl_amd import ops
    from parl_amd._native import ParlHipError
    v = torch.view_as_complex(torch.ones(1, 2, device=dev)).conj().imag   # one element: dense for all its stride of two
    assert v.is_neg()
    with pytest.raises(ParlHipError, match='negated'):
        ops.grad_norm([v])


@pytest.mark.parametrize('n', [10, 200])
def test_clip_in_replayed_graphs_and_on_two_streams(n, dev):
    from parl_amd import ops
    sets = [_grads([(1000 + 7 * i, ) for i in range(n)], DTYPES, dev, s) for s in (1, 2)]
    work = [[g.clone() for g in s] for s in sets]
    params = [_params(w) for w in work]
    limit = [0.1 * _norm64(s) for s in sets]
    want = []
    for s, m in zip(sets, limit):
        c = [g.clone() for g in s]
        want.append((ops.clip_grad_norm_(_params(c), m), c))
    graphs, norms = [], []
    for p, m in zip(params, limit):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            norms.append(ops.clip_grad_norm_(p, m))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(4):
        for w, s in zip(work, sets):
            torch._foreach_copy_(w, s)
        torch.cuda.synchronize()
        for i in (0, 1):
            with torch.cuda.stream(streams[(i + k) % 2]):
                graphs[i].replay()
        ops.grad_norm(sets[0])
        torch.cuda.synchronize()
        for i in (0, 1):
            assert float(norms[i]) == float(want[i][0])
            assert all(torch.equal(a, b) for a, b in zip(work[i], want[i][1]))
