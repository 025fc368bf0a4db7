"""The training operators' refusals that need no GPU: CPU tensors, the C entry
points' argument checks, workspace sizes."""
import ctypes

import pytest
import torch

from vibecheck_amd import _lib, train

CALLS = {
    'linear': lambda x: train.linear(x, x),
    'linear_backward': lambda x: train.linear_backward(x, x, x),
    'cross_entropy': lambda x: train.cross_entropy(x, torch.zeros(4, dtype=torch.int64)),
    'adamw_step': lambda x: train.adamw_step([x], [x], train.adamw_state([x]), 1),
}


@pytest.mark.parametrize('name', CALLS)
def test_cpu_tensors_are_refused(name):
    with pytest.raises(RuntimeError, match='not on the GPU'):
        CALLS[name](torch.zeros(4, 4))


def test_unknown_names_are_refused():
    x = torch.zeros(4, 4)
    with pytest.raises(ValueError, match='activation'):
        train.linear(x, x, act='tanh')
    with pytest.raises(ValueError, match='bits'):
        train.adamw_state([x], bits=16)


BUF = ctypes.create_string_buffer(64)
P = ctypes.addressof(BUF)  # host memory: these calls return before any launch


@pytest.mark.parametrize('args', [
    dict(type=2), dict(M=-1), dict(ldx=3), dict(act=4), dict(x=None), dict(W=None), dict(y=None),
    dict(res=P, ldr=4)])
def test_linear_arguments(args):
    a = dict(type=0, x=P, M=4, K=4, ldx=4, W=P, N=5, bias=None, act=0, res=None, ldr=0, y=P, z=None,
             work=None, bytes=0, stream=None)
    a.update(args)
    with pytest.raises(ValueError):
        _lib.call('vc_linear', *a.values())


@pytest.mark.parametrize('args', [
    dict(type=7), dict(N=-1), dict(ldy=3), dict(act=-1), dict(act=1), dict(act=1, z=P, ldz=3),
    dict(dy=None), dict(W=None), dict(x=None), dict(ldx=2)])
def test_linear_backward_arguments(args):
    a = dict(type=0, dy=P, ldy=5, x=P, ldx=4, W=P, z=None, ldz=0, act=0, M=4, K=4, N=5, dx=P, dW=P,
             db=None, work=None, bytes=0, stream=None)
    a.update(args)
    with pytest.raises(ValueError):
        _lib.call('vc_linear_backward', *a.values())


@pytest.mark.parametrize('args', [
    dict(type=3), dict(R=-1), dict(V=0), dict(ld=9), dict(smooth=1.5), dict(smooth=float('nan')),
    dict(red=3), dict(loss=None), dict(ldd=9), dict(z=None), dict(t=None)])
def test_cross_entropy_arguments(args):
    a = dict(type=0, z=P, R=4, V=10, ld=10, t=P, ignore=-100, smooth=0.0, red=0, loss=P, d=P, ldd=10,
             work=None, bytes=0, stream=None)
    a.update(args)
    with pytest.raises(ValueError):
        _lib.call('vc_cross_entropy', *a.values())


@pytest.mark.parametrize('args', [
    dict(count=-1), dict(ptype=2), dict(gtype=2), dict(bits=16), dict(step=0), dict(b1=1.0),
    dict(b2=-0.1), dict(eps=-1.0), dict(p=None), dict(m=None), dict(m=P + 4), dict(bits=8)])
def test_adamw_arguments(args):
    ptrs, sizes = (ctypes.c_void_p * 1)(P), (ctypes.c_int64 * 1)(4)
    at = ctypes.addressof(ptrs)
    a = dict(p=at, g=at, copy=None, n=ctypes.addressof(sizes), count=1, ptype=0, gtype=0, bits=32,
             m=P, v=P, ms=None, vs=None, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, step=1,
             scale=None, stream=None)
    a.update(args)
    with pytest.raises(ValueError):
        _lib.call('vc_adamw_step', *a.values())


def test_workspaces():
    lib = _lib.load()
    assert lib.vc_linear_workspace(0, 0, 7, 7) == 0
    assert lib.vc_linear_workspace(0, -1, 7, 7) < 0
    assert lib.vc_linear_backward_workspace(1, 4, 4, 4, 9, 7) < 0
    assert lib.vc_linear_backward_workspace(1, 64, 64, 64, 3, 7) >= 2 * 64 * 64 + 4 * 64
    assert lib.vc_cross_entropy_workspace(-1, 1) < 0
    # a workspace too small is refused, not overrun
    with pytest.raises(torch.cuda.OutOfMemoryError):
        _lib.call('vc_cross_entropy', 0, P, 4, 10, 10, P, -100, 0.0, 2, P, None, 0, P, 8, None)


def test_backward_of_a_rounded_dz():
    """The flag belongs to the backward's activation; a dz in two parts needs the more room."""
    lib = _lib.load()
    for act in (2, 3):
        assert lib.vc_linear_backward_workspace(1, 64, 64, 64, act | 16, 7) < \
            lib.vc_linear_backward_workspace(1, 64, 64, 64, act, 7)
    for act in (0, 1):
        assert lib.vc_linear_backward_workspace(1, 64, 64, 64, act | 16, 7) == \
            lib.vc_linear_backward_workspace(1, 64, 64, 64, act, 7)
    assert lib.vc_linear_backward_workspace(1, 64, 64, 64, 32, 7) < 0
    assert lib.vc_linear_backward_workspace(1, 64, 64, 64, 4 | 16, 7) < 0
    with pytest.raises(ValueError):
        _lib.call('vc_linear', 0, P, 4, 4, 4, P, 5, None, 1 | 16, None, 0, P, None, None, 0, None)


def test_sizes_that_no_launch_holds():
    """Refused by the workspace, before anything is launched; whatever some cut can hold is not."""
    lib = _lib.load()
    top = 0x7fffff00
    for k in (0, 1):
        assert lib.vc_linear_workspace(k, top, 64, 1 << 30) < 0
        assert lib.vc_linear_backward_workspace(k, top, 64, 1 << 30, 0, 7) < 0
        for M in (40_000_003, 140_000_003, 400_000_000):
            assert lib.vc_linear_workspace(k, M, 8, 8) >= 0
            assert lib.vc_linear_backward_workspace(k, M, 8, 8, 0, 7) >= 0
    for need in (1, 2, 7):
        assert lib.vc_linear_backward_workspace(1, 1 << 29, 8, 8, 2, need) < 0
        assert lib.vc_linear_backward_workspace(1, (1 << 29) - 512, 8, 8, 2, need) > 0
    assert lib.vc_linear_backward_workspace(1, top, 8, 8, 2, 4) > 0  # db alone has no product
    with pytest.raises(NotImplementedError):
        _lib.call('vc_linear', 1, P, top, 64, 64, P, 1 << 30, None, 0, None, 0, P, None, None, 0, None)
