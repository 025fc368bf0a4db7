"""Train an fc / ReLU classifier, then bound it: the operators of ``train`` in one
training step, and the engine's CROWN bounds of the net that comes out (no
reference counterpart).

  python -m vibecheck_amd.train_mlp --widths 20-256-256-10 --steps 300 --eps 0.01

trains on points around ten seeded prototypes and prints, before and after, the
loss, the accuracy and the share of points whose class holds on the whole box of
half-width eps.
"""
import argparse

import torch

from . import train, workloads
from .verify_zono_bnb import _bound_crown_spec, _op_params, validate_gg


class Mlp:
    """An fc / ReLU chain on the GPU with its optimiser state: fp32 weights, and with
    ``compute`` bf16 their working copies, which forward and backward then use."""

    def __init__(self, widths, seed=0, device='cuda', compute=torch.float32, bits=32):
        Ws, bs = workloads.mlp_params(widths, seed=seed, bias_std=0.01)
        self.params = [t.to(device=device, dtype=torch.float32).contiguous()
                       for pair in zip(Ws, bs) for t in pair]
        self.copies = None if compute == torch.float32 else [p.to(compute) for p in self.params]
        self.state = train.adamw_state(self.params, bits)
        self.steps, self.compute = 0, compute

    def layers(self):
        """(W, bias) of each fc layer, as the products read them."""
        p = self.copies or self.params
        return list(zip(p[::2], p[1::2]))

    def forward(self, x, save=False):
        """Logits of x (B, n_in); with ``save`` also what gradients needs."""
        saved, layers = [], self.layers()
        for i, (W, b) in enumerate(layers):
            act = 'relu' if i + 1 < len(layers) else None
            y, z = train.linear(x, W, b, act=act, save=True)
            saved.append((x, z))
            x = y
        return (x, saved) if save else x

    def gradients(self, d, saved):
        """Gradients of every parameter, in their order, from that of the logits."""
        out, layers = [], self.layers()
        for i in reversed(range(len(layers))):
            x, z = saved[i]
            need = ('x', 'W', 'bias') if i else ('W', 'bias')
            d, dW, db = train.linear_backward(d, x, layers[i][0], z=z,
                                              act='relu' if z is not None else None, need=need)
            out[:0] = [dW, db]
        return out

    def step(self, x, target, lr=1e-3, weight_decay=0.01, smoothing=0.0):
        """One training step; the mean loss before it, on the GPU."""
        logits, saved = self.forward(x.to(self.compute), save=True)
        loss, d = train.cross_entropy(logits, target, smoothing=smoothing, out=logits)
        grads = self.gradients(d, saved)
        self.steps += 1
        train.adamw_step(self.params, grads, self.state, self.steps, lr=lr,
                         weight_decay=weight_decay, copies=self.copies)
        return loss

    def gg(self):
        """The net as it is now as the bound engine's op graph (fp32 copies: the engine keeps
        layouts of the weights it has seen)."""
        p = [t.clone() for t in self.params]
        return workloads.mlp_gg(p[::2], p[1::2], device=p[0].device)


def point_forward(gg, x):
    """The answers of an fc / ReLU / reshape net at points x (B, n_in), fp32 on the GPU."""
    validate_gg(gg, x.shape[1])
    ops, act = gg['ops'], {gg['input_name']: x}
    readers = [i for op in ops for i in op['inputs']]
    for op, after in zip(ops, ops[1:] + [None]):
        if op['name'] in act:  # a relu that its fc has applied
            continue
        a, kind = act[op['inputs'][0]], op['type']
        if kind == 'fc':
            p = _op_params(op, x.device)
            if a.shape[-1] != p['n_in']:
                raise NotImplementedError('vibecheck_amd: the N-D fc form has no point forward')
            relu = after is not None and after['type'] == 'relu' and \
                after['inputs'] == [op['name']] and readers.count(op['name']) == 1
            y = train.linear(a, p['W'], p['b'], act='relu' if relu else None)
            act[after['name'] if relu else op['name']] = y
        elif kind == 'relu':
            act[op['name']] = a.clamp(min=0)
        elif kind == 'reshape':
            act[op['name']] = a
        else:
            raise NotImplementedError(f'vibecheck_amd: {kind} has no point forward')
    return act[ops[-1]['name']]


def class_rows(n_classes, c):
    """spec_ew of y_c - y_j for every other class j."""
    out = {}
    for i, k in enumerate(j for j in range(n_classes) if j != c):
        w = torch.zeros(n_classes)
        w[c], w[k] = 1.0, -1.0
        out[i] = (w, 0.0)
    return out


def certified(gg, x, target, eps, chunk=512):
    """Whether each point's class holds on its whole box of half-width ``eps``: CROWN lower
    bounds of y_t - y_j above zero for every j."""
    ok = torch.zeros(x.shape[0], dtype=torch.bool, device=x.device)
    n = gg['ops'][-1]['W'].shape[0]
    for c in range(n):
        rows = {i: (w.to(x.device), b) for i, (w, b) in class_rows(n, c).items()}
        of_c = (target == c).nonzero()[:, 0]
        for at in of_c.split(chunk):
            xl, xh = (x[at] - eps).contiguous(), (x[at] + eps).contiguous()
            _, lb = _bound_crown_spec(gg, xl, xh, rows, x.device, torch.float32)
            ok[at] = (lb > 0).all(1)
    return ok


def prototype_points(n, n_in, n_classes, seed=0, spread=0.08, device='cuda'):
    """Points around one seeded prototype in [0, 1]^n_in per class, and their classes."""
    g = torch.Generator(device='cpu').manual_seed(seed)
    proto = torch.rand(n_classes, n_in, generator=g)
    t = torch.randint(0, n_classes, (n,), generator=g)
    x = proto[t] + spread * torch.randn(n, n_in, generator=g)
    return x.to(device), t.to(device)


def fit(net, x, target, steps, batch=512, seed=0, **hyper):
    """``steps`` training steps on seeded batches; their losses, (steps,) on the GPU."""
    g = torch.Generator(device='cpu').manual_seed(seed)
    losses = []
    for _ in range(steps):
        at = torch.randint(0, x.shape[0], (batch,), generator=g).to(x.device)
        losses.append(net.step(x[at], target[at], **hyper))
    return torch.stack(losses)


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split('\n\n')[0])
    p.add_argument('--widths', default='20-256-256-10')
    p.add_argument('--steps', type=int, default=300)
    p.add_argument('--batch', type=int, default=512)
    p.add_argument('--eps', type=float, default=0.01)
    p.add_argument('--lr', type=float, default=2e-3)
    p.add_argument('--bf16', action='store_true', help='products in bf16, weights kept in fp32')
    p.add_argument('--bits', type=int, default=32, choices=(8, 32), help='of the optimiser state')
    a = p.parse_args(argv)
    widths = [int(w) for w in a.widths.split('-')]
    net = Mlp(widths, compute=torch.bfloat16 if a.bf16 else torch.float32, bits=a.bits)
    x, t = prototype_points(4096, widths[0], widths[-1])

    def report(when):
        gg = net.gg()
        y = point_forward(gg, x)
        loss, _ = train.cross_entropy(y, t, grad=False)
        right = y.argmax(1) == t
        held = certified(gg, x[:512], t[:512], a.eps)
        print(f'{when}: loss {float(loss):.4f}, accuracy {float(right.float().mean()):.4f}, '
              f'class holds within {a.eps} for {float(held.float().mean()):.4f} of 512 points')

    report('before')
    fit(net, x, t, a.steps, a.batch, lr=a.lr)
    report(f'after {a.steps} steps')


if __name__ == '__main__':
    main()
