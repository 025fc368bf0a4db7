"""Where the training operators can go wrong: dz's bits in the bf16 backward, fp32 activations'
last places, NaN and infinities behind them, masks by large finite values and logits far from
zero, second derivatives and what is written in place, sizes near a launch's limit, the 8-bit
step's parameter to the bit.

Tolerances are those of test_gpu_train, whose helpers these tests use, where a test does not
derive its own.
"""
import math
from array import array

import pytest
import torch

import test_gpu_train as tt
from vibecheck_amd import _lib, train

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


@pytest.mark.parametrize('to', [F32, BF16])
@pytest.mark.parametrize('M,K,N', [(7, 20, 50), (300, 333, 203), (1030, 520, 776)])
def test_relu_chooses(gpu, to, M, K, N):
    """An infinite or NaN gradient where a ReLU is closed adds nothing, at zero too: the results
    are those of zeros there, to the bit."""
    f = tt._randn(gpu, 31)
    x, W, dy, z = f(M, K, to=to), f(N, K, to=to), f(M, N, to=to), f(M, N, to=to)
    z[2, 5], z[3, 6], z[4], z[5, 7] = -1.0, -0.0, 0.0, -math.inf
    clean = dy.clone()
    dy[2, 5], dy[3, 6], dy[4], dy[5, 7] = math.inf, math.nan, -math.inf, math.nan
    clean[2, 5], clean[3, 6], clean[4], clean[5, 7] = 0, 0, 0, 0
    got = train.linear_backward(dy, x, W, z=z, act='relu')
    assert all(map(torch.equal, got, train.linear_backward(clean, x, W, z=z, act='relu')))
    assert all(bool(t.isfinite().all()) for t in got)
    z[2, 5] = 1.0  # open: it passes
    dx, _, db = train.linear_backward(dy, x, W, z=z, act='relu')
    assert db[5] == math.inf and not bool(dx[2].isfinite().any())


@pytest.mark.parametrize('act', ['gelu', 'silu'])
@pytest.mark.parametrize('M,K,N', [(1, 64, 4096), (300, 100, 51), (512, 784, 1024), (2050, 785, 2051)])
def test_fp32_activations_to_a_few_units(gpu, act, M, K, N):
    """fp32 results to a few units in the last place of each result, small ones beside negative
    arguments among them.  gelu: (8 + 2 z^2) units of 2^-24 (the argument of erfc, of exp is rounded,
    which 2 z^2 / 2 multiplies), silu eight units; slopes the same of their terms' magnitudes,
    and 2^-22 for what the product of parts leaves out.  The oracle's normal integral is by erfc:
    by 1 + erf it would lose what is measured here."""
    def side(z):
        return torch.special.erfc(-z / math.sqrt(2)) / 2 if act == 'gelu' else torch.sigmoid(z)

    f = tt._randn(gpu, 41 + M)
    x, W = f(M, K), f(N, K, std=3 * K ** -0.5)
    y, z = train.linear(x, W, f(N), act=act, save=True)
    zd = z.double()
    assert float(zd.min()) < -4
    unit = (8 + 2 * zd.square() if act == 'gelu' else 8) * 2.0 ** -24
    tt._within(y, zd * side(zd), unit * (zd * side(zd)).abs() + 1e-37, act)
    # one column: dx is dz itself
    z = zd.flatten()[:100_000].float().unsqueeze(1)
    dy, one = f(len(z), 1), torch.ones(1, 1, device=gpu)
    dx, _, _ = train.linear_backward(dy, torch.zeros_like(z), one, z=z, act=act, need=('x',))
    zd = z.double()
    q = side(zd)
    other = torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi) if act == 'gelu' else q * side(-zd)
    unit = (8 + 2 * zd.square() if act == 'gelu' else 8) * 2.0 ** -24
    tol = (unit * (q + zd.abs() * other) + 2.0 ** -22 * (q + zd * other).abs()) * dy.double().abs()
    tt._within(dx, dy.double() * (q + zd * other), tol + 1e-37, 'slope')


@pytest.mark.parametrize('M,K,N', [(1, 64, 40), (17, 333, 65), (300, 203, 117), (520, 784, 1024), (1021, 1031, 1030)])
def test_any_nan_stays_one(gpu, M, K, N):
    """A NaN whose bits differ from an infinity's in the last sixteen alone, of either sign, in
    each of the operands."""
    def nan(t, i, j, bits):
        t.view(torch.int32)[i, j] = bits

    f = tt._randn(gpu, 61)
    for bits in (0x7f800001, 0xff808000 - (1 << 32), 0x7f80ffff):
        x, W, dy = f(M, K), f(N, K), f(M, N)
        nan(x, M - 1, 5, bits)
        nan(W, 7, K - 1, bits)
        y = train.linear(x, W)
        want = torch.zeros(M, N, dtype=torch.bool, device=gpu)
        want[M - 1], want[:, 7] = True, True
        assert torch.equal(y.isnan(), want) and not y.isinf().any()
        nan(dy, 0, 3, bits)
        dx, dW, db = train.linear_backward(dy, x, W)
        wx, ww, wb = (torch.zeros(t.shape, dtype=torch.bool, device=gpu) for t in (dx, dW, db))
        wx[0], wx[:, K - 1], ww[3], ww[:, 5], wb[3] = True, True, True, True, True
        for got, nans in ((dx, wx), (dW, ww), (db, wb)):
            assert torch.equal(got.isnan(), nans) and not got.isinf().any()


# ----------------------------------------------------------------------- loss

FILLS = [-1e9, -1e10, -1e20, -1e30, -1e35, 'lowest']
VS = [300, 5003, 140001]  # a wave, a workgroup, a row that registers do not hold


def _fill(fill, to):
    return torch.finfo(to).min if fill == 'lowest' else fill


def _loss_and_grad(z, t, **kw):
    return train.cross_entropy(z, torch.tensor(t, device=z.device), reduction='none', **kw)


@pytest.mark.parametrize('to', [F32, BF16])
@pytest.mark.parametrize('V', VS)
@pytest.mark.parametrize('fill', FILLS)
def test_cross_entropy_masked_by_large_values(gpu, to, V, fill):
    """Classes masked by a large finite value in front, behind, in whole chunks, at odd places, all
    but one: the loss and the gradient of what is left, whose values are within 30 of each other.
    2^-18 of the loss: (32 + V / 64 + 4 * 30) units of 2^-24 at V 5003, 2^-12 at V 140001."""
    live = torch.ones(6, V, dtype=torch.bool, device=gpu)
    live[0, :V // 2] = False
    live[1, V // 2:] = False
    live[2, 8:64] = False
    live[2, V - 70:] = False
    live[3, ::2] = False
    live[4] = False
    live[4, V // 3] = True
    live[5, 1:] = False
    z = tt._randn(gpu, V)(6, V, to=to, std=3.0)
    t = [int(r.nonzero()[len(r.nonzero()) // 2]) for r in live]
    masked = torch.where(live, z, torch.full_like(z, _fill(fill, to)))
    want = torch.where(live, z.double(), -math.inf)
    want_l = torch.logsumexp(want, 1) - want[range(6), t]
    want_d = torch.softmax(want, 1)
    want_d[range(6), t] -= 1
    for h in (0, 1):  # rows at even and odd places
        buf = torch.zeros(6, V + 3, dtype=to, device=gpu)
        buf[:, h:h + V] = masked
        loss, d = _loss_and_grad(buf[:, h:h + V], t)
        rel = (32 + V / 64 + 120) * 2.0 ** -24
        tt._within(loss, want_l, rel * (1 + want_l.abs()), 'loss')
        half = 2.0 ** -8 if to == BF16 else 0.0
        tt._within(d, want_d, (rel + half) * want_d.abs() + rel * 2.0 ** -24 + 1e-37, 'gradient')
        assert not d[~live].any()


@pytest.mark.parametrize('to', [F32, BF16])
@pytest.mark.parametrize('V', VS)
@pytest.mark.parametrize('at', [3e6, 1e7, 1e10, 1e20, 1e30, -3e6, -1e7, -1e10, -1e20, -1e30, -2e37])
def test_cross_entropy_uniform_rows_far_from_zero(gpu, to, V, at):
    """log V and 1 / V, whatever the value; of the two halves' values the larger alone counts."""
    z = torch.full((3, V), at, dtype=to, device=gpu)
    z[1, :V // 2] -= abs(at) / 2
    z[2, V // 2:] -= abs(at) / 2
    t = [V - 1, V - 1, 1]
    n = torch.tensor([V, V - V // 2, V // 2], dtype=F64, device=gpu)
    loss, d = _loss_and_grad(z, t)
    rel = (32 + V / 64) * 2.0 ** -24
    tt._within(loss, n.log(), rel * (1 + n.log()), 'loss')
    want = torch.where(z == z.amax(1, keepdim=True), 1 / n.unsqueeze(1), 0.0)
    want[range(3), t] -= 1
    half = 2.0 ** -8 if to == BF16 else 0.0
    tt._within(d, want, (rel + half) * want.abs() + 1e-37, 'gradient')


@pytest.mark.parametrize('to', [F32, BF16])
@pytest.mark.parametrize('V', VS)
@pytest.mark.parametrize('e', [0.0, 0.1])
@pytest.mark.parametrize('by', [1e6, 1e9, 1e13, 1e20, 1e30])
def test_cross_entropy_large_logits(gpu, to, V, e, by):
    """Logits so large that the softmax is one class: the loss is a difference of logits, to a few
    units of the largest; the gradient the chosen class's less the target's."""
    z = tt._randn(gpu, V + 1)(5, V, std=by).to(to)
    z[0, 7] = 6 * by
    t = [7, 8, V - 1, 0, V // 2]
    tgt = torch.tensor(t, device=gpu)
    lw, dw = tt._loss64(z, tgt, e, -100)
    loss, d = _loss_and_grad(z, t, smoothing=e)
    tt._within(loss, lw, 2.0 ** -18 * z.double().abs().amax(1), 'loss')
    # where two classes are within some 100 of each other the exponentials show it
    top = z.double().topk(2, dim=1).values
    clear = (top[:, 0] - top[:, 1]) > 200
    half = 2.0 ** -8 if to == BF16 else 2.0 ** -18
    tt._within(d[clear], dw[clear], half * dw[clear].abs() + 2.0 ** -40, 'gradient')


@pytest.mark.parametrize('to', [F32, BF16])
@pytest.mark.parametrize('V', [20] + VS)
@pytest.mark.parametrize('at', [0, 1, 299, -1])
def test_cross_entropy_nan_beside_large_values(gpu, to, V, at):
    """A NaN anywhere makes its row's loss NaN, in front of, behind or among large values; the
    target's own counts, and one masked by a large value costs that value."""
    at = min(at, V - 1)
    for v in (1e10, -1e10, 2e38, -math.inf):
        z = torch.full((2, V), v, dtype=to, device=gpu)
        z[0, at] = math.nan
        z[1] = 1.0
        z[1, 2] = v
        loss, _ = _loss_and_grad(z, [3, 2])
        assert loss[0].isnan()
        want = z[1].double()
        want = torch.logsumexp(want, 0) - want[2]
        if v > 0:
            assert abs(float(loss[1])) < 1e-6
        else:
            assert float(loss[1]) == pytest.approx(float(want), rel=1e-6)


# ------------------------------------------------------------------- autograd

def test_second_derivatives_raise(gpu):
    """What create_graph=True returns has the first derivative's values, and a penalty on it does
    not lose its gradient without a word: alone, beside another loss, through either operator."""
    f = tt._randn(gpu, 21)
    x, W, b = (t.requires_grad_() for t in (f(8, 20), f(40, 20), f(40)))
    t = torch.arange(8, device=gpu)
    for make in (lambda: train.linear(x, W, b, act='gelu').square().sum(),
                 lambda: train.linear(x, W, b).sum(),
                 lambda: train.cross_entropy(x, t)[0],
                 lambda: train.cross_entropy(x, t, reduction='none')[0].sum(),
                 lambda: train.cross_entropy(train.linear(x, W, b, act='silu'), t)[0]):
        want, = torch.autograd.grad(make(), x)
        for also in (0.0, 1.0):
            g, = torch.autograd.grad(make(), x, create_graph=True)
            assert torch.equal(g, want) and g.requires_grad
            with pytest.raises(NotImplementedError, match='second derivative'):
                (g.square().sum() + also * x.square().sum()).backward()
    # the gradients of a bias and a weight alike; what the upstream gradient itself carries passes
    gW, gb = torch.autograd.grad(train.linear(x, W, b, act='gelu').square().sum(), (W, b), create_graph=True)
    for g in (gW, gb):
        for of in (x, W, b):
            with pytest.raises(NotImplementedError, match='second derivative'):
                torch.autograd.grad(g.sum(), of, retain_graph=True, allow_unused=True)
    # one that requires none of the others' gradients
    for i in range(3):
        ts = [u if j == i else u.detach() for j, u in enumerate((x, W, b))]
        g, = torch.autograd.grad(train.linear(*ts, act='silu').sum(), ts[i], create_graph=True)
        with pytest.raises(NotImplementedError, match='second derivative'):
            torch.autograd.grad(g.sum(), ts[i], allow_unused=True)
    with pytest.raises(NotImplementedError, match='second derivative'):
        torch.autograd.functional.hessian(lambda u: train.cross_entropy(u, t)[0], x.detach())
    r, up = f(8, 40).requires_grad_(), f(8, 40).requires_grad_()
    g, = torch.autograd.grad(train.linear(x, W, b, residual=r), r, up, create_graph=True)
    assert torch.equal(torch.autograd.grad(g.sum(), up)[0], torch.ones_like(up))
    g, = torch.autograd.grad(train.cross_entropy(x, t, reduction='none')[0], x, f(8).requires_grad_(),
                             create_graph=True)
    assert g.requires_grad


def test_forward_mode_raises(gpu):
    f = tt._randn(gpu, 22)
    x, W, t = f(8, 20), f(40, 20), torch.arange(8, device=gpu)
    y, z = train.linear(x, W, act='gelu', save=True)
    with torch.autograd.forward_ad.dual_level():
        def dual(t):
            return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: train.linear(dual(x), W), lambda: train.linear(x, dual(W), save=True),
                     lambda: train.linear(x, W, residual=dual(y)),
                     lambda: train.linear(dual(x), W.clone().requires_grad_()),
                     lambda: train.linear_backward(dual(y), x, W, z=z, act='gelu'),
                     lambda: train.cross_entropy(dual(x), t)):
            with pytest.raises(NotImplementedError, match='forward-mode'):
                call()
        assert torch.equal(train.linear(x, W, act='gelu'), y)


def test_written_tensors_count_as_written(gpu):
    """A graph that saved a parameter, a working copy or an output that is written in place
    raises, as it does behind torch's own in-place operations."""
    f = tt._randn(gpu, 23)
    x, up = f(8, 20), f(8, 40)
    for bits in (32, 8):
        W, c = f(40, 20).requires_grad_(), f(40, 20, to=BF16).requires_grad_()
        state = train.adamw_state([W], bits)
        before = {k: t._version for k, t in state.items() if k != 'bits'}
        x.requires_grad_()
        ys = [train.linear(x, W, act='gelu').sum(), train.linear(x.to(BF16), c).sum()]
        train.adamw_step([W], [f(40, 20)], state, 1, copies=[c])
        for y in ys:
            with pytest.raises(RuntimeError, match='modified by an inplace operation'):
                y.backward()
        assert all(state[k]._version > v for k, v in before.items())
    # relu's output is what its backward needs; the gradient has taken its place
    y = train.linear(x, f(40, 20), act='relu')
    loss, d = train.cross_entropy(y.detach(), torch.arange(8, device=gpu), out=y.detach())
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward(d)
    # where nothing that is needed was overwritten all goes on
    y = train.linear(x, f(40, 20))
    loss, d = train.cross_entropy(y.detach(), torch.arange(8, device=gpu), out=y.detach())
    y.backward(d)
    with torch.inference_mode():
        W = f(40, 20)
        train.adamw_step([W], [f(40, 20)], train.adamw_state([W]), 1)
        z = f(8, 20)
        train.cross_entropy(z, torch.arange(8, device=gpu), out=z)


@pytest.mark.parametrize('to', [F32, BF16])
@pytest.mark.parametrize('V', [10, 300])
def test_loss_without_its_gradient_is_differentiable(gpu, to, V):
    """grad=False leaves the gradient out of the answer, not out of the graph."""
    f = tt._randn(gpu, 24)
    z, t = f(4, 5, V, to=to).requires_grad_(), torch.arange(20, device=gpu).view(4, 5) % V
    t[0, 1] = -100
    for red, up in (('none', f(4, 5)), ('sum', f(1)[0]), ('mean', None)):
        kw = dict(reduction=red, smoothing=0.1)
        loss, d = train.cross_entropy(z, t, **kw)
        only, none = train.cross_entropy(z, t, grad=False, **kw)
        assert none is None and torch.equal(only, loss)
        got, = torch.autograd.grad(only, z, up)
        assert torch.equal(got, torch.autograd.grad(loss, z, up)[0])
    g, = torch.autograd.grad(train.cross_entropy(z, t, grad=False)[0], z, create_graph=True)
    with pytest.raises(NotImplementedError, match='second derivative'):
        g.sum().backward()
    with torch.no_grad():
        assert not train.cross_entropy(z, t, grad=False)[0].requires_grad
    # with out the caller passes the gradient on
    loss, d = train.cross_entropy(z, t, out=torch.empty_like(z, requires_grad=False))
    assert not loss.requires_grad and torch.equal(d, train.cross_entropy(z, t)[1])


def test_cross_entropy_more_rows_than_a_launch_has_threads(gpu):
    """2^26 rows and some by a wavefront each, 4.4 GB: every sixty-fourth row alike."""
    V, n = 33, (1 << 20) + 3
    f = tt._randn(gpu, 25)
    z, t = f(64, V, to=BF16, std=3.0), torch.arange(64, device=gpu) % V
    t[5] = -100
    many = torch.empty(n, 64, V, dtype=BF16, device=gpu)
    many[:] = z
    want, dw = train.cross_entropy(z, t, reduction='none')
    loss, d = train.cross_entropy(many, t.expand(n, 64), reduction='none')
    assert torch.equal(loss, want.expand(n, 64)) and bool((d == dw).all())
    loss, d = train.cross_entropy(many, t.expand(n, 64), out=d)
    mean, dm = train.cross_entropy(z, t)
    assert float(loss) == pytest.approx(float(mean), rel=1e-6)
    tt._within(d[-1] * 1024.0, dm.double() * 1024.0 / n, 2.0 ** -7 * dm.double().abs() * 1024.0 / n + 1e-30, 'd')


# ------------------------------------------------- sizes near a launch's limit

@pytest.mark.parametrize('to', [F32, BF16])
@pytest.mark.parametrize('M', [40_000_003, 140_000_003])
def test_linear_many_rows(gpu, to, M):
    """More rows than the kernel that would be the fastest has workgroups for in a launch: rows in
    a period of 61, whole numbers, so that every sum is exact."""
    K = N = 8
    g = torch.Generator(device=gpu).manual_seed(3)
    x = torch.randint(-1, 2, (61, K), generator=g, device=gpu).to(to)
    dy = torch.randint(-1, 2, (61, N), generator=g, device=gpu).to(to)
    x[60] = -x[:60].sum(0)  # a period adds nothing to dW or db: no sum grows
    dy[:] = dy[0]
    W = torch.randint(-2, 3, (N, K), generator=g, device=gpu).to(to)
    times, rest = divmod(M, 61)

    def rows(t):
        out = torch.empty(M, 8, dtype=to, device=gpu)
        out[:times * 61].view(times, 61, 8)[:] = t
        out[times * 61:] = t[:rest]
        return out

    def whole(got, want):
        return torch.equal(got[:61], want) and bool((got[:times * 61].view(times, 61, 8) == want).all()) \
            and torch.equal(got[times * 61:], want[:rest])

    big = rows(x)
    assert whole(train.linear(big, W), (x.double() @ W.double().t()).to(to))
    dx, dW, db = train.linear_backward(rows(dy), big, W)
    assert whole(dx, (dy.double() @ W.double()).to(to))
    want = times * (dy.double().t() @ x.double()) + dy[:rest].double().t() @ x[:rest].double()
    assert torch.equal(dW.double(), want.to(to).double())
    want = times * dy.double().sum(0) + dy[:rest].double().sum(0)
    tt._within(db, want, 2.0 ** -7 * want.abs(), 'db')


def test_backward_of_many_columns(gpu):
    """The columns' sums where there are more of them than workgroups: 10 million."""
    N = 10_000_019
    dy = (torch.arange(3 * N, device=gpu).view(3, N) % 7).float()
    x, W = torch.ones(3, 1, device=gpu), torch.ones(N, 1, device=gpu)
    _, dW, db = train.linear_backward(dy, x, W, need=('W', 'bias'))
    assert torch.equal(db, dy.sum(0)) and torch.equal(dW[:, 0], db)
    assert torch.equal(train.linear_backward(dy, x, W, need=('bias',))[2], db)


def test_bf16_backward_long_offsets(gpu):
    """dz's parts past 2^32 values: a gradient in the last rows alone."""
    M, K, N = (1 << 19) + 61, 64, 4096
    f = tt._randn(gpu, 81)
    x, W = f(M, K, to=BF16), f(N, K, to=BF16)
    dy, z = torch.zeros(M, N, dtype=BF16, device=gpu), torch.zeros(M, N, dtype=BF16, device=gpu)
    dy[-3:], z[-3:] = f(3, N, to=BF16), f(3, N, to=BF16)
    dx, dW, db = train.linear_backward(dy, x, W, z=z, act='silu')
    wx, ww, wb = train.linear_backward(dy[-3:], x[-3:], W, z=z[-3:], act='silu')
    assert not dx[:-3].any()
    for got, want in ((dx[-3:], wx), (dW, ww), (db, wb)):
        tt._close(got, want)


# ------------------------------------------------------------------ optimiser

def test_adamw_8_parameter_to_the_bit(gpu):
    """The parameter of a step with 8-bit states: every operation rounded to 32 bits by itself
    (in 64 bits and rounded again, which for these is the same)."""
    n, (b1, b2), lr, eps, wd = 1 << 20, (0.9, 0.999), 1e-3, 1e-8, 0.1
    f = tt._randn(gpu, 51)
    one = tt._single
    p, state = f(n, std=1e-3), train.adamw_state([f(n)], bits=8)
    p[::3] = 0  # the step itself
    w = [float(torch.tensor(v, dtype=F32)) for v in (b1, 1 - b1, b2, 1 - b2)]
    for k in range(1, 4):
        g = f(n) * torch.exp(3 * f(n))
        m, u = (one(state[s].view(torch.float8_e4m3fn).double()
                    * state[s + '_scale'].double().repeat_interleave(256)) for s in ('m', 'v'))
        gd = g.double()
        m = one(one(w[0] * m) + one(w[1] * gd))
        u = one(one(one(w[2] * one(u * u)) + one(one(w[3] * gd) * gd)).sqrt())
        c = [float(torch.tensor(v, dtype=F32)) for v in
             (1 - lr * wd, -lr / (1 - b1 ** k), math.sqrt(1 - b2 ** k), eps)]
        want = one(one(p.double() * c[0]) + one(one(c[1] * m) / one(one(u / c[2]) + c[3])))
        train.adamw_step([p], [g], state, k, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd)
        assert torch.equal(p.double(), want)


def test_adamw_refuses_before_it_changes_anything(gpu):
    """A tensor larger than a launch takes, behind more small ones than one launch has."""
    n = array('q', [256] * 99 + [1 << 36])
    p, g = torch.ones(99, 256, device=gpu), torch.ones(99, 256, device=gpu)
    state = train.adamw_state([p])
    at = [t.data_ptr() for t in (*p, p[0])]
    ptrs, grads = array('Q', at), array('Q', [t.data_ptr() for t in (*g, g[0])])
    with pytest.raises(NotImplementedError):
        _lib.call('vc_adamw_step', ptrs.buffer_info()[0], grads.buffer_info()[0], None,
                  n.buffer_info()[0], len(n), 0, 0, 32, state['m'].data_ptr(),
                  state['v'].data_ptr(), None, None, 0.1, 0.9, 0.999, 1e-8, 0.0, 1, None, _lib.stream())
    assert bool((p == 1).all()) and not state['m'].any()


def test_cross_entropy_out_over_the_logits(gpu):
    """The logits' own place, or none of it: shifted or with rows closer together a row would be
    read after another's gradient was written there."""
    f, t = tt._randn(gpu, 71), torch.arange(6, device=gpu)
    buf = f(4000)
    z = buf[:3000].view(6, 500)
    for out in (buf[4:3004], buf[500:3500]):
        with pytest.raises(ValueError, match='overlaps'):
            train.cross_entropy(z, t, out=out.view(6, 500))
    with pytest.raises(ValueError, match='overlaps'):
        train.cross_entropy(buf[:3600].view(6, 600)[:, :500], t, out=z)
    want = train.cross_entropy(z, t)
    for zz, out in ((z, buf[1000:1000].new_empty(6, 500)), (buf.clone()[:3000].view(6, 500),) * 2,
                    (z[:2], buf[1000:2000].view(2, 500))):
        loss, d = train.cross_entropy(zz, t[:len(zz)], out=out)
        if len(zz) == 6:
            assert torch.equal(loss, want[0]) and torch.equal(d, want[1])
    loss, d = train.cross_entropy(buf[:600].view(1, 600)[:, :500], t[:1], out=buf[:500].view(1, 500))
    assert bool(loss.isfinite())
