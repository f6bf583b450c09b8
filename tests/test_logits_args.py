"""The C entries of the operators over logits and of the gradient norm refuse what they cannot do before they touch the device, and
the Python entries refuse host tensors.  CPU only."""
import ctypes

import pytest
import torch

INVALID, NOSUP, NOMEM = -1, -3, -4


@pytest.fixture(scope='module')
def lib():
    from parl_amd import _native
    return _native.lib()


def _sample(lib, logits=16, dtype=0, stride=8, u=16, t=None, k=None, p=None, mp=None, ta=1.0, ka=0, pa=1.0, ma=0.0, a=16, lp=16,
            B=2, A=8, ws=16, wsb=1 << 40):
    return lib.parlhip_logits_sample(logits, dtype, stride, u, t, k, p, mp, ta, ka, pa, ma, a, lp, B, A, ws, wsb, None)


def test_sample_arguments(lib):
    nan, inf = float('nan'), float('inf')
    for kw in (dict(logits=None), dict(u=None), dict(a=None), dict(lp=None), dict(B=-1), dict(A=0), dict(stride=7), dict(ta=-1.0),
               dict(ta=nan), dict(ta=inf), dict(pa=-0.5), dict(pa=nan), dict(ma=-0.5), dict(ma=2.0), dict(ma=nan),
               dict(logits=18), dict(logits=17, dtype=1)):
        assert _sample(lib, **kw) == INVALID, kw
    assert _sample(lib, dtype=3) == NOSUP and _sample(lib, dtype=-1) == NOSUP
    assert _sample(lib, A=(1 << 20) + 1, stride=1 << 21) == NOSUP
    assert _sample(lib, B=1 << 40) == NOSUP
    assert _sample(lib, B=0, logits=None, u=None, a=None, lp=None) == 0


def test_sample_workspace(lib):
    f = lib.parlhip_logits_sample_workspace_bytes
    for A in (1, 64, 65, 2048):
        assert f(1000, A) == 0
    assert f(0, 100000) == 0 and f(5, 0) == 0 and f(5, (1 << 20) + 1) == 0
    for A in (4097, 5000, 6143, 6145, 8191, 8193, 16385, 50000, 131072, 262143, 1 << 20):
        for B in (1, 2, 63, 300, 5000, 262143):
            n = f(B, A)
            # the pieces' sums of every row, and no more than a few times the logits behind that
            assert B * (A // 1024) * 12 <= n <= B * (A // 1024 + 1) * 12 + 8 * B * (A + 2048) + (1 << 20), (A, B)
    need = f(3, 5000)
    assert _sample(lib, B=3, A=5000, stride=5000, wsb=need - 1) == NOMEM
    assert _sample(lib, B=3, A=5000, stride=5000, ws=None) == INVALID
    assert _sample(lib, B=3, A=5000, stride=5000, ws=20) == INVALID


def test_log_prob_arguments(lib):
    def f(x=16, dtype=0, stride=8, a=16, lp=16, h=16, st=16, N=2, A=8, T=1.0, ws=16, wsb=1 << 40):
        return lib.parlhip_logits_log_prob(x, dtype, stride, a, lp, h, st, N, A, T, ws, wsb, None)

    def b(x=16, dtype=0, stride=8, a=16, st=16, h=16, gl=16, gh=16, g=16, N=2, A=8, T=1.0):
        return lib.parlhip_logits_log_prob_backward(x, dtype, stride, a, st, h, gl, gh, g, N, A, T, None)

    nan, inf = float('nan'), float('inf')
    for kw in (dict(x=None), dict(a=None), dict(N=-1), dict(A=0), dict(stride=7), dict(T=0.0), dict(T=-1.0), dict(T=nan),
               dict(T=inf), dict(T=1e-39), dict(x=18), dict(x=17, dtype=2), dict(st=20)):
        assert f(**kw) == INVALID, kw
        assert b(**kw) == INVALID, kw
    assert f(lp=None) == INVALID and f(h=None) == INVALID
    assert b(st=None) == INVALID and b(h=None) == INVALID and b(g=None) == INVALID and b(g=18) == INVALID
    assert f(dtype=7) == NOSUP and b(dtype=7) == NOSUP
    assert f(N=1 << 39, A=1000, stride=1000) == NOSUP
    assert f(N=0, x=None, a=None, lp=None, h=None) == 0 and b(N=0, x=None, a=None, st=None, h=None, g=None) == 0
    need = lib.parlhip_logits_log_prob_workspace_bytes(1, 131072)
    assert need > 0
    assert f(N=1, A=131072, stride=131072, wsb=need - 1) == NOMEM
    assert f(N=1, A=131072, stride=131072, ws=None) == INVALID
    assert lib.parlhip_logits_log_prob_workspace_bytes(100000, 131072) == 0
    assert lib.parlhip_logits_log_prob_workspace_bytes(5, 6) == 0


@pytest.mark.parametrize('A', [1, 512, 513, 4096, 5000, 131072])
def test_log_prob_of_no_rows_and_of_more_than_a_launch_takes(lib, A):
    f = lambda N: lib.parlhip_logits_log_prob(None, 0, A, None, None, None, None, N, A, 1.0, None, 0, None)  # noqa: E731
    b = lambda N: lib.parlhip_logits_log_prob_backward(None, 0, A, None, None, None, None, None, None, N, A, 1.0,  # noqa: E731
                                                       None)
    assert f(0) == 0 and b(0) == 0
    # a launch has fewer than 2^32 threads; up to 512 actions it walks over the rows
    threads = None if A <= 512 else 64 if A <= 4096 else 256 if A < 16384 else 1024
    if threads:
        most = 0xffffffff // threads
        assert f(most + 1) == NOSUP and b(most + 1) == NOSUP
        if most * A <= 1 << 40:
            assert f(most) == INVALID and b(most) == INVALID   # the NULL pointers


def test_log_prob_of_more_rows_than_a_launch_of_512_threads_takes(lib):
    f = lambda N: lib.parlhip_logits_log_prob(None, 0, 16384, None, None, None, None, N, 16384, 1.0, None, 0, None)  # noqa: E731
    assert f(0xffffffff // 512) == INVALID and f(0xffffffff // 512 + 1) == NOSUP


def test_grad_norm_arguments(lib):
    def arr(t, *v):
        return (t * len(v))(*v)

    P, I, T = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
    at, n, ty = arr(P, 4096, 8192), arr(I, 100, 200), arr(T, 0, 1)
    assert lib.parlhip_grad_norm_workspace_bytes(2, n) == 16
    assert lib.parlhip_grad_norm_workspace_bytes(2, arr(I, 0, 0)) == 8
    assert lib.parlhip_grad_norm_workspace_bytes(2, arr(I, -1, 5)) == 0
    assert lib.parlhip_grad_norm(-1, at, n, ty, 16, 1 << 30, 16, None) == INVALID
    assert lib.parlhip_grad_norm(2, None, n, ty, 16, 1 << 30, 16, None) == INVALID
    assert lib.parlhip_grad_norm(2, at, None, ty, 16, 1 << 30, 16, None) == INVALID
    assert lib.parlhip_grad_norm(2, at, n, None, 16, 1 << 30, 16, None) == INVALID
    assert lib.parlhip_grad_norm(2, at, n, ty, None, 1 << 30, 16, None) == INVALID
    assert lib.parlhip_grad_norm(2, at, n, ty, 20, 1 << 30, 16, None) == INVALID
    assert lib.parlhip_grad_norm(2, at, n, ty, 16, 1 << 30, None, None) == INVALID
    assert lib.parlhip_grad_norm(2, at, n, ty, 16, 15, 16, None) == NOMEM
    assert lib.parlhip_grad_norm(2, at, n, arr(T, 0, 3), 16, 1 << 30, 16, None) == NOSUP
    assert lib.parlhip_grad_norm(2, at, arr(I, -1, 2), ty, 16, 1 << 30, 16, None) == INVALID
    assert lib.parlhip_grad_norm(2, arr(P, None, 8192), n, ty, 16, 1 << 30, 16, None) == INVALID
    assert lib.parlhip_grad_norm(2, arr(P, 4098, 8192), n, ty, 16, 1 << 30, 16, None) == INVALID

    def c(at=at, out=None, n=n, ty=ty, oty=None, m=1.0):
        return lib.parlhip_clip_grad_norm(2, at, out, n, ty, oty, m, 16, 1 << 30, 16, None)

    assert c(m=-1.0) == INVALID and c(m=float('nan')) == INVALID
    assert c(at=arr(P, 4096, 4096)) == INVALID and c(at=arr(P, 4096, 4096 + 396)) == INVALID      # the same memory twice
    assert c(out=arr(P, 65536, 70000)) == INVALID and c(oty=ty) == INVALID
    assert c(out=arr(P, 65536, None), oty=ty) == INVALID and c(out=arr(P, 65537, 70000), oty=ty) == INVALID
    assert c(out=arr(P, 65536, 65600), oty=ty) == INVALID                                           # outputs overlap
    assert c(out=arr(P, 8192, 70000), oty=ty) == INVALID                                            # ... another gradient
    assert c(out=arr(P, 4100, 70000), oty=ty) == INVALID                                            # ... its own, shifted
    assert c(out=arr(P, 4096, 8192), oty=arr(T, 1, 1)) == INVALID                                   # in place, another type


def test_host_tensors_are_refused(lib):
    from parl_amd import ops
    from parl_amd._native import ParlHipError
    x = torch.zeros(3, 5)
    with pytest.raises(ParlHipError):
        ops.logits_sample(x, torch.zeros(3, dtype=torch.float64))
    with pytest.raises(ParlHipError):
        ops.logits_log_prob(x, torch.zeros(3, dtype=torch.int64))
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(ParlHipError):
        ops.clip_grad_norm_([p], 1.0)
    with pytest.raises(ParlHipError):
        ops.grad_norm([p.grad])


def test_rows_that_a_draw_takes(lib):
    """what a launch of at most 2^32 - 1 threads takes, a wave for each row, up to 4,096 actions; above, launches follow each other"""
    n = lambda B, A: _sample(lib, logits=None, B=B, A=A, stride=A)  # noqa: E731
    for A in (1, 64, 65, 512, 513, 4096):
        assert n((1 << 26) - 4, A) == INVALID          # the NULL pointer
        for over in (3, 2, 1):
            assert n((1 << 26) - over, A) == NOSUP     # four rows to a workgroup, rounded up
    for A in (4097, 5000, 131072, 1 << 20):
        assert n((1 << 40) // A, A) == INVALID
        assert n((1 << 40) // A + 1, A) == NOSUP
    assert n(131072, 5000) == n(200000, 5000) == INVALID


def test_scratch_memory_apart_from_the_tensors(lib):
    """the partial sums and the norm are written while the gradients are still read"""
    def arr(t, *v):
        return (t * len(v))(*v)

    P, I, T = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
    at, n, ty = arr(P, 4096, 8192), arr(I, 100, 200), arr(T, 0, 1)   # 4096..4495, 8192..8591
    out = arr(P, 65536, 70000)                                       # 65536..65935, 70000..70399
    for ws, norm in ((4096, 1024), (4488, 1024), (4088, 1024), (8584, 1024), (512, 4492), (512, 8192), (512, 512), (512, 524)):
        assert lib.parlhip_grad_norm(2, at, n, ty, ws, 1 << 30, norm, None) == INVALID, (ws, norm)
        assert lib.parlhip_clip_grad_norm(2, at, None, n, ty, None, 1.0, ws, 1 << 30, norm, None) == INVALID, (ws, norm)
    for ws, norm in ((65536, 1024), (70392, 1024), (512, 65932), (512, 70396)):
        assert lib.parlhip_clip_grad_norm(2, at, out, n, ty, ty, 1.0, ws, 1 << 30, norm, None) == INVALID, (ws, norm)
    assert lib.parlhip_grad_norm(0, None, None, None, 512, 8, 516, None) == INVALID
