"""The operators together: an fc / ReLU classifier is trained and its CROWN bounds taken.
The step's gradients against 64-bit autograd, the point forward against the oracle's, what
certified says against sampled points, every form of the step against its own repetition."""
import pytest
import torch

from oracle import ref_bound as rb
from vibecheck_amd import train_mlp as tm
from vibecheck_amd import workloads as wk

import _util

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize('widths,B', [([20, 64, 64, 10], 300), ([5, 50, 50, 50, 5], 77),
                                      ([33, 117, 203, 75, 7], 131)])
def test_gradients(gpu, widths, B):
    """Every parameter's gradient of the mean loss against autograd in 64 bits.  The products carry
    under 2^-18 of their magnitudes' sums through at most five layers, and no pre-activation of
    these seeds lies within 1e-7 of zero (checked), so every relu takes the same side."""
    net = tm.Mlp(widths, seed=B, device=gpu)
    x, t = tm.prototype_points(B, widths[0], widths[-1], seed=1, device=gpu)
    logits, saved = net.forward(x, save=True)
    loss, d = tm.train.cross_entropy(logits, t)
    grads = net.gradients(d, saved)
    ps = [p.double().requires_grad_() for p in net.params]
    a = x.double()
    for i in range(0, len(ps), 2):
        a = a @ ps[i].t() + ps[i + 1]
        if i + 2 < len(ps):
            assert float(a.detach().abs().min()) > 1e-7
            a = a.clamp(min=0)
    want = torch.nn.functional.cross_entropy(a, t)
    want.backward()
    assert abs(float(loss) - float(want)) < 1e-5 * (1 + float(want))
    for g, p in zip(grads, ps):
        assert float((g.double() - p.grad).norm()) <= 1e-4 * float(p.grad.norm())


@pytest.mark.parametrize('make', [lambda d: wk.acas_gg(device=d, dtype=F32),
                                  lambda d: wk.mlp_gg(*wk.mlp_params([33, 117, 203, 75, 7], 3, 0.1),
                                                      device=d)])
def test_point_forward(gpu, make):
    """Against the oracle in 64 bits, layer sums of up to 203 products deep: 2^-18 of the scale."""
    gg = make(gpu)
    n_in = gg['input_n']
    x = torch.rand(257, n_in, device=gpu, generator=torch.Generator(device=gpu).manual_seed(2))
    got = tm.point_forward(gg, x).double().cpu()
    want, _ = rb.point_forward(x.double().cpu(), _util.to_dev(gg, 'cpu', torch.float64))
    assert float((got - want).abs().max()) <= 2.0 ** -16 * float(want.abs().max())


@pytest.mark.parametrize('compute', [F32, BF16])
@pytest.mark.parametrize('bits', [32, 8])
def test_training_learns_and_holds(gpu, compute, bits):
    """Well separated classes are learnt in every form; a class that is said to hold on a box holds
    at 200 points of it and at the box's corners' signs of the input gradient; the same seeds give
    the same bits."""
    eps = 0.02
    runs = []
    for _ in range(2):
        net = tm.Mlp([12, 64, 64, 5], seed=4, device=gpu, compute=compute, bits=bits)
        x, t = tm.prototype_points(1024, 12, 5, seed=3, spread=0.05, device=gpu)
        losses = tm.fit(net, x, t, 150, batch=256, lr=5e-3)
        runs.append((net, losses))
    (net, losses), (other, again) = runs
    assert torch.equal(losses, again)
    assert all(torch.equal(p, q) for p, q in zip(net.params, other.params))
    assert float(losses[-10:].mean()) < 0.2 * float(losses[0])
    gg = net.gg()
    assert float((tm.point_forward(gg, x).argmax(1) == t).float().mean()) > 0.97
    held = tm.certified(gg, x[:200], t[:200], eps)
    assert float(held.float().mean()) > 0.5
    xs, ts = x[:200][held], t[:200][held]
    g = torch.Generator(device=gpu).manual_seed(5)
    for _ in range(200):
        p = xs + eps * (2 * torch.rand(xs.shape, device=gpu, generator=g) - 1)
        assert bool((tm.point_forward(gg, p).argmax(1) == ts).all())
        p = xs + eps * torch.sign(torch.randn(xs.shape, device=gpu, generator=g))
        assert bool((tm.point_forward(gg, p).argmax(1) == ts).all())
    if compute == BF16:
        assert all(torch.equal(c, p.to(BF16)) for c, p in zip(net.copies, net.params))


def test_snapshot(gpu):
    """A net's op graph is of the weights as they were: training on leaves it."""
    net = tm.Mlp([5, 50, 50, 5], device=gpu)
    x, t = tm.prototype_points(64, 5, 5, device=gpu)
    gg = net.gg()
    before = tm.point_forward(gg, x)
    net.step(x, t, lr=0.1)
    assert torch.equal(tm.point_forward(gg, x), before)
    assert not torch.equal(tm.point_forward(net.gg(), x), before)


def test_command(gpu, capsys):
    tm.main(['--widths', '8-32-4', '--steps', '20', '--batch', '64', '--bf16', '--bits', '8'])
    out = capsys.readouterr().out
    assert out.startswith('before: loss') and 'after 20 steps' in out


def test_point_forward_refusals(gpu):
    gg = wk.residual_mlp_gg(6, 16, 3, device=gpu)
    with pytest.raises(NotImplementedError):
        tm.point_forward(gg, torch.zeros(2, 6, device=gpu))
    with pytest.raises(ValueError):
        tm.point_forward(wk.acas_gg(device=gpu), torch.zeros(2, 6, device=gpu))
