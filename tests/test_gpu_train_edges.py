"""Where the training operators can go wrong: dz's bits in the bf16 backward.

Tolerances are those of test_gpu_train, whose helpers these tests use.
"""
import math

import pytest
import torch

import test_gpu_train as tt
from vibecheck_amd import train

pytestmark = pytest.mark.gpu
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


# ------------------------------------------------------------------- fc layer

# one row, odd and even widths, products by 64 x 64 and by larger tiles, slices of k
BACKWARD = [(1, 5, 50), (3, 64, 64), (17, 333, 65), (64, 128, 256), (131, 203, 117), (257, 1031, 40),
            (1021, 333, 777), (520, 784, 1024), (2050, 512, 1030), (1, 4096, 130), (257, 15872, 117),
            (4100, 1031, 513)]


@pytest.mark.parametrize('act', ['gelu', 'silu'])
@pytest.mark.parametrize('M,K,N', BACKWARD)
def test_bf16_backward_keeps_dz(gpu, M, K, N, act):
    """bf16 gradients are the exact ones rounded once.  dz in two parts, the first cut: what the
    cut leaves is under 2^-7 of it, the rounding of that 2^-9, so 2^-16 of |dz| |W| besides the
    sums (over two parts) and the slope's own few units."""
    f = tt._randn(gpu, M + K + 3 * N)
    x, W, dy, z = f(M, K, to=BF16), f(N, K, to=BF16, std=K ** -0.5), f(M, N, to=BF16), f(M, N, to=BF16)
    dx, dW, db = train.linear_backward(dy, x, W, z=z, act=act)
    xd, Wd = x.double(), W.double()
    dz = dy.double() * tt._slope(z.double(), act)
    e = dy.double().abs() * 2.0 ** -20 * (1 + z.double().abs()) + 2.0 ** -16 * dz.abs()
    for got, want, a, b, ea, n in ((dx, dz @ Wd, dz.abs(), Wd.abs(), e @ Wd.abs(), 2 * N),
                                   (dW, dz.t() @ xd, dz.abs().t(), xd.abs(), e.t() @ xd.abs(), 2 * M)):
        tt._within(got, want, tt._sum_tol(a, b, n) + ea + 2.0 ** -8 * want.abs() + 1e-30, 'product')
    for need in (('x',), ('W',), ('x', 'bias')):
        part = train.linear_backward(dy, x, W, z=z, act=act, need=need)
        for p, q, name in zip(part, (dx, dW, db), ('x', 'W', 'bias')):
            assert p is None if name not in need else torch.equal(p, q)
    # rounded where the caller asks for it: 2^-8 of |dz| |W| more, db as it was
    rx, rW, rb = train.linear_backward(dy, x, W, z=z, act=act, round_dz=True)
    e = e + 2.0 ** -8 * dz.abs()
    for got, want, a, b, ea, n in ((rx, dz @ Wd, dz.abs(), Wd.abs(), e @ Wd.abs(), N),
                                   (rW, dz.t() @ xd, dz.abs().t(), xd.abs(), e.t() @ xd.abs(), M)):
        tt._within(got, want, tt._sum_tol(a, b, n) + ea + 2.0 ** -8 * want.abs() + 1e-30, 'rounded')
    assert torch.equal(rb, db)


@pytest.mark.parametrize('act', [None, 'relu'])
def test_round_dz_leaves_exact_ones(gpu, act):
    f = tt._randn(gpu, 8)
    for to in (F32, BF16):
        x, W, dy, z = f(70, 130, to=to), f(90, 130, to=to), f(70, 90, to=to), f(70, 90, to=to)
        z = z if act else None
        got = train.linear_backward(dy, x, W, z=z, act=act, round_dz=True)
        assert all(map(torch.equal, got, train.linear_backward(dy, x, W, z=z, act=act)))


def test_round_dz_through_autograd(gpu):
    f = tt._randn(gpu, 9)
    x, W, up = f(40, 30, to=BF16).requires_grad_(), f(50, 30, to=BF16).requires_grad_(), f(40, 50, to=BF16)
    z = train.linear(x.detach(), W.detach(), act='gelu', save=True)[1]
    for rounded in (False, True):
        y = train.linear(x, W, act='gelu', round_dz=rounded)
        got = torch.autograd.grad(y, (x, W), up)
        want = train.linear_backward(up, x.detach(), W.detach(), z=z, act='gelu', round_dz=rounded)
        assert all(map(torch.equal, got, want[:2]))


@pytest.mark.parametrize('rounded', [False, True])
@pytest.mark.parametrize('M,K,N', [(40, 30, 50), (1030, 520, 777)])
def test_bf16_backward_infinities_and_nan_behind_an_activation(gpu, M, K, N, rounded):
    """What is not finite in dy, x or W reaches its own rows and columns, and what they reach in
    the plain products; the largest finite gradient stays finite."""
    f = tt._randn(gpu, 12)
    x, W, dy, z = f(M, K, to=BF16), f(N, K, to=BF16, std=0.05), f(M, N, to=BF16), f(M, N, to=BF16)
    z[5, 7], z[30, 8], z[31, 9] = 0.5, 0.5, 40.0
    dy[5, 7], dy[30, 8] = math.inf, math.nan
    dy[31] = 0
    dy[31, 9] = torch.finfo(BF16).max
    W[9], W[9, 0] = 0, 0.5
    x[31] = 0.25
    x[20, 9], W[11, 3] = -math.inf, math.inf
    got = train.linear_backward(dy, x, W, z=z, act='silu', round_dz=rounded)
    d, xd = dy.double() * tt._slope(z.double(), 'silu'), x.double()
    for p, q in zip(got, (d @ W.double(), d.t() @ xd, d.sum(0))):
        assert torch.equal(p.isnan(), q.isnan()) and torch.equal(p.isinf(), q.isinf())
        assert torch.equal(p[p.isinf()].double(), q[q.isinf()])
