"""Definitions of the token-row operators in 64 bits and how far a float32 evaluation with one rounding at the end may be from them.

u(t) = finfo(t).eps / 2 is the largest relative error of one rounding to t. A float32 sum of K products, in whatever order and with additions that
may truncate instead of rounding, is off by at most K * 2^-23 * sum |products| (first order; the products of 16- and 8-bit values are exact in
float32, those of float32 values add u per product, which the +2 covers)."""

import torch

F32_ULP = 2.0 ** -23
ACTS = ('linear', 'relu', 'lrelu', 'tanh', 'sigmoid', 'elu', 'selu', 'softplus', 'swish')
# largest |act'| and |act''| away from the kinks (swish' <= 1.1, swish'' <= 0.5; selu' <= 1.7581, selu'' <= 1.7581)
STEEP = {'linear': 1, 'relu': 1, 'lrelu': 1, 'tanh': 1, 'sigmoid': 0.25, 'elu': 1, 'selu': 1.7581, 'softplus': 1, 'swish': 1.1}
BEND = {'linear': 0, 'relu': 0, 'lrelu': 0, 'tanh': 0.77, 'sigmoid': 0.1, 'elu': 1, 'selu': 1.7581, 'softplus': 0.25, 'swish': 0.5}
# jump of act' at zero
JUMP = {'relu': 1.0, 'lrelu': 0.8, 'selu': 0.71}


def u(dtype):
    return torch.finfo(dtype).eps / 2


def act64(v, act, alpha):
    F = torch.nn.functional
    return {'linear': lambda: v, 'relu': lambda: F.relu(v), 'lrelu': lambda: torch.where(v > 0, v, v * alpha), 'tanh': lambda: torch.tanh(v),
            'sigmoid': lambda: torch.sigmoid(v), 'elu': lambda: F.elu(v), 'selu': lambda: F.selu(v), 'softplus': lambda: torch.logaddexp(v, torch.zeros_like(v)),
            'swish': lambda: v * torch.sigmoid(v)}[act]()


def sums64(x, w, b, xs=None, ws=None):
    """(x w^T + b, its float32 error bound) from tensors of any dtype."""
    x, w = x.double(), w.double()
    if xs is not None:
        x, w = x * xs.double().unsqueeze(-1), w * ws.double().unsqueeze(-1)
    k = x.shape[-1]
    v, big = x @ w.t(), x.abs() @ w.abs().t()
    off = (k + 2 + (2 if xs is not None else 0)) * F32_ULP * big
    if xs is not None:
        # The matrix unit adds the products of eight neighbouring 8-bit values at the largest one's exponent and cuts 13 bits below it: seven others
        # lose less than 2^-13 of it each. The largest product of a group is at most the product of the two groups' largest values.
        top = [torch.nn.functional.pad(t.abs(), (0, -k % 8)).reshape(t.shape[0], -1, 8).amax(dim=2) for t in (x.reshape(-1, k), w)]
        off = off + 7 * 2.0 ** -13 * (top[0] @ top[1].t()).reshape(off.shape)
    if b is not None:
        v = v + b.double()
        off = off + F32_ULP * v.abs()
    return v, off


def slopes64(v, off, act, alpha, gain, clamp):
    """act(v) * gain clamped, d/dv of it, and the error bounds of both when v is off by `off`."""
    a = act64(v, act, alpha)
    t = v.detach().clone().requires_grad_(True)
    with torch.enable_grad():
        d = torch.autograd.grad(act64(t, act, alpha).sum(), t)[0]
    # values: the sum's error times the slope, and the function's own float32 error (a few units of its result; tanh and the exponentials of ocml
    # are within 2 units, the quotients and products around them add 3)
    a_off = STEEP[act] * max(1.0, abs(alpha) if act == 'lrelu' else 1.0) * off + 6 * F32_ULP * a.abs()
    d_off = BEND[act] * off + 8 * F32_ULP * (d.abs() + 0.1)
    if act in JUMP:
        jump = abs(1 - alpha) if act == 'lrelu' else JUMP[act]
        d_off = d_off + torch.where(v.abs() <= off, jump, 0.0)
    if act == 'elu':
        d_off = d_off + torch.where(v.abs() <= off, off, torch.zeros_like(off))
    a, d, a_off, d_off = a * gain, d * gain, a_off * abs(gain) + F32_ULP * (a * gain).abs(), d_off * abs(gain) + F32_ULP * (d * gain).abs()
    if clamp is not None:
        edge = (a.abs() - clamp).abs() <= a_off
        d_off = torch.where(edge, d.abs() + d_off, d_off)
        out = a.abs() >= clamp
        d, d_off = torch.where(out, 0.0, d), torch.where(out & ~edge, 0.0, d_off)
        a = a.clamp(-clamp, clamp)
    return a, d, a_off, d_off


def rounded(value, off, dtype):
    """Bound of a value that is off by `off` and then rounded to dtype (its subnormals included)."""
    return off + u(dtype) * (value.abs() + off) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def assert_within(got, want, bound, what):
    got = got.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), what
    over = (got - want).abs() - bound
    if over.numel() and float(over.max()) > 0:
        i = int(over.argmax())
        raise AssertionError(f'{what}: {float(got.reshape(-1)[i])} for {float(want.reshape(-1)[i])}, allowed {float(bound.reshape(-1)[i])}')


def product64(a, b, a_off, dtype):
    """a @ b for a in 64 bits that is rounded to dtype first (off by a_off before), b exact: (value, bound after the result's rounding)."""
    k = a.shape[1]
    ra = rounded(a, a_off, dtype)
    v = a @ b
    off = ra @ b.abs() + (k + 2) * F32_ULP * ((a.abs() + ra) @ b.abs())
    return v, rounded(v, off, dtype)
