"""Measured cases of the token-row operators: `linear_act`, `gated_ff`, `rms_norm` and `quantize_rows`.

All four work on matrices of rows (a row is one token, one frame's latent or one sample):

  linear      y = clamp(act(x w^T + b) * gain) + residual
  gated       h = gain * act(x wg^T + bg) * (x wu^T + bu), w = [wg; wu] stacked
  norm        s = x + residual, y = weight * s / sqrt(mean(s^2) + eps); or y in 8 bits with one scale a row
  quantize    q = x / scale in e4m3, scale = max |x| of the row / 448

`run` computes the plain form in float32 (`own` False) or calls the operators (`own` True). Training cases return the result
and every gradient; cases of type e4m3 multiply 8-bit rows by 8-bit weights, each with its scales."""

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32, 'e4m3': torch.float8_e4m3fn}
_BYTES = {'bf16': 2, 'f16': 2, 'f32': 4, 'e4m3': 1}
_E4M3_MAX = 448.0
_SCALE_MIN = 2.0 ** -64
_EPS = 1e-6
_GAINS = {'linear': 1.0, 'lrelu': math.sqrt(2), 'relu': math.sqrt(2), 'swish': math.sqrt(2), 'tanh': 1.0, 'sigmoid': 1.0, 'softplus': 1.0}


def _ops():
    package = os.path.join(_ROOT, 'long-video-gan_amd')
    if package not in sys.path:
        sys.path.insert(0, package)
    from torch_utils.ops import gated_ff, linear_act, rms_norm
    return linear_act.linear_act, gated_ff.gated_ff, rms_norm.rms_norm, rms_norm.quantize_rows


# ------------------------------------------------------------------------------------------------------------------------------
# Cases.

def listed():
    return [
        # the style projection of one layer for a single clip while a video is sampled: latency
        dict(name='linear one latent', op='linear', train=False, type='bf16', rows=1, inner=1024, outer=512, act='linear', bias=True, residual=False, clamp=-1.0),
        # the discriminator head's first layer (16 frames of 1024 features a sample, 32 samples), training in float32
        dict(name='linear head f32 train', op='linear', train=True, type='f32', rows=32, inner=16384, outer=1024, act='swish', bias=True, residual=False, clamp=-1.0),
        # a ragged batch of token rows through a layer of odd widths, training
        dict(name='linear ragged f16 train', op='linear', train=True, type='f16', rows=1237, inner=771, outer=515, act='lrelu', bias=True, residual=True, clamp=256.0),
        # the projection back into the residual stream for a long prompt
        dict(name='linear residual long', op='linear', train=False, type='bf16', rows=16384, inner=8192, outer=2048, act='linear', bias=True, residual=True, clamp=-1.0),
        # the same serving layer with 8-bit rows and weights
        dict(name='linear 8 bit', op='linear', train=False, type='e4m3', rows=8192, inner=4096, outer=4096, act='linear', bias=True, residual=True, clamp=-1.0),
        # one token through the gated block
        dict(name='gated one token', op='gated', train=False, type='bf16', rows=1, inner=2048, outer=8192, act='swish', bias=False, residual=False, clamp=-1.0),
        # a training step of the gated block over a full batch of tokens
        dict(name='gated train', op='gated', train=True, type='bf16', rows=8192, inner=2048, outer=8192, act='swish', bias=True, residual=False, clamp=-1.0),
        # a batch of prompts through the 8-bit gated block
        dict(name='gated 8 bit', op='gated', train=False, type='e4m3', rows=4096, inner=4096, outer=8192, act='swish', bias=False, residual=False, clamp=-1.0),
        # one token: residual addition, norm and 8-bit rows for the products that follow
        dict(name='norm one token 8 bit', op='norm', train=False, type='bf16', rows=1, inner=2048, residual=True, out8=True),
        # a training step of the norm with its residual stream
        dict(name='norm train', op='norm', train=True, type='bf16', rows=16384, inner=4096, residual=True, out8=False),
        # a few decoded tokens' hidden features to 8 bits
        dict(name='quantize few', op='quantize', train=False, type='f16', rows=8, inner=8192),
        # a prompt batch's hidden features to 8 bits
        dict(name='quantize many', op='quantize', train=False, type='bf16', rows=8192, inner=8192),
    ]


_MOST_FLOPS = 1.6e12
_MOST_VALUES = 130e6      # rows x widest row


def _log(rng, low, high):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(['linear', 'linear', 'linear', 'gated', 'gated', 'norm', 'norm', 'quantize'])
    while True:
        rows, inner, outer = _log(rng, 1, 16384), _log(rng, 64, 16384), _log(rng, 16, 8192)
        if rng.random() < 0.5:              # half of the widths are those of aligned layers
            inner, outer = -(-inner // 64) * 64, -(-outer // 64) * 64
        if op in ('norm', 'quantize'):
            if rows * inner <= _MOST_VALUES / 2:
                break
        else:
            products = 6.0 * rows * inner * outer * (2 if op == 'gated' else 1)
            if products <= _MOST_FLOPS and max(rows * inner, rows * outer, inner * outer) <= _MOST_VALUES / 2:
                break
    if op == 'quantize':
        return dict(op=op, train=False, type=rng.choice(['bf16', 'f16', 'f32']), rows=rows, inner=inner)
    if op == 'norm':
        train = rng.random() < 0.5
        return dict(op=op, train=train, type=rng.choice(['bf16', 'f16', 'f32']), rows=rows, inner=inner, residual=rng.random() < 0.6,
                    out8=not train and rng.random() < 0.5)
    kind = rng.choice(['bf16', 'bf16', 'f16', 'f32', 'e4m3'])
    train = kind != 'e4m3' and rng.random() < 0.5
    # the derivative of lrelu and of the clamp jumps: a sum that lies on the jump within float32's rounding has two right answers, so float32
    # training cases are drawn with smooth activations
    smooth = kind == 'f32' and train
    act = rng.choice(['swish', 'tanh', 'sigmoid'] + ([] if smooth else ['lrelu', 'relu']) + (['linear', 'softplus'] if op == 'linear' else []))
    return dict(op=op, train=train, type=kind, rows=rows, inner=inner, outer=outer, act=act, bias=rng.random() < 0.6,
                residual=op == 'linear' and rng.random() < 0.5, clamp=2.5 if op == 'linear' and not smooth and rng.random() < 0.25 else -1.0)


def work(case):
    rows, inner, e = case['rows'], case['inner'], _BYTES[case['type']]
    x = rows * inner * e
    if case['op'] == 'quantize':
        return {'bytes': x + rows * inner + 4 * rows, 'flops': 3.0 * rows * inner}
    if case['op'] == 'norm':
        stream = x * (3 if case['residual'] else 1) + inner * e         # x, residual, their sum written
        out = rows * inner + 4 * rows if case['out8'] else x
        back = x * (4 if case['residual'] else 2) + inner * e if case['train'] else 0      # gradients of both results read, of both inputs written
        return {'bytes': stream + out + back, 'flops': (16.0 if case['train'] else 5.0) * rows * inner}
    both = 2 if case['op'] == 'gated' else 1
    outer, o = case['outer'], max(2, e)
    w = both * inner * outer * e
    y = rows * outer * o
    scales = 4 * (rows + both * outer) if case['type'] == 'e4m3' else 0
    forward = x + w + y * (2 if case['residual'] else 1) + (both * outer * o if case['bias'] else 0) + scales
    # the backward pass reads the gradient of the result and writes those of the rows, the weight, the bias; x and w count once
    back = y + x + w + (both * outer * o if case['bias'] else 0) if case['train'] else 0
    return {'bytes': forward + back, 'flops': (6.0 if case['train'] else 2.0) * rows * inner * outer * both}


# ------------------------------------------------------------------------------------------------------------------------------
# Inputs.

def _rows_to_8bit(v):
    """Rows of float32 -> e4m3 rows and their scales: what a program keeps for its weights."""
    scale = (v.abs().amax(dim=1) / _E4M3_MAX).clamp(min=_SCALE_MIN)
    return (v / scale[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn), scale


def _features(rows, width, g):
    """Feature rows as networks have them: unit normal with a spread of channel magnitudes, a few channels ten times the others."""
    x = torch.randn(rows, width, generator=g, device='cuda')
    size = torch.exp(0.4 * torch.randn(width, generator=g, device='cuda'))
    size = torch.where(torch.rand(width, generator=g, device='cuda') < 0.003, size * 10, size)
    return x.mul_(size)


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(int(seed))
    kind, rows, inner, train = _DTYPES[case['type']], case['rows'], case['inner'], case['train']
    s = {'case': case, 'out': torch.bfloat16 if case['type'] == 'e4m3' else kind}
    x = _features(rows, inner, g)
    if case['op'] in ('linear', 'gated'):
        total = case['outer'] * (2 if case['op'] == 'gated' else 1)
        w = torch.randn(total, inner, generator=g, device='cuda') / math.sqrt(inner)
        s['xs'] = s['ws'] = s['b'] = s['r'] = None
        if case['type'] == 'e4m3':
            (s['x'], s['xs']), (s['w'], s['ws']) = _rows_to_8bit(x), _rows_to_8bit(w)
        else:
            s['x'], s['w'] = x.to(kind).requires_grad_(train), w.to(kind).requires_grad_(train)
        if case['bias']:
            s['b'] = (0.2 * torch.randn(total, generator=g, device='cuda')).to(s['out']).requires_grad_(train)
        if case['residual']:
            s['r'] = torch.randn(rows, case['outer'], generator=g, device='cuda').to(s['out']).requires_grad_(train)
        if train:
            s['dy'] = (0.05 * torch.randn(rows, case['outer'], generator=g, device='cuda')).to(kind)
        return s
    s['x'] = x.to(kind).requires_grad_(train)
    if case['op'] == 'norm':
        s['w'] = (1 + 0.2 * torch.randn(inner, generator=g, device='cuda')).to(kind).requires_grad_(train)
        s['r'] = torch.randn(rows, inner, generator=g, device='cuda').to(kind).requires_grad_(train) if case['residual'] else None
        if train:
            s['dy'] = (0.05 * torch.randn(rows, inner, generator=g, device='cuda')).to(kind)
            s['ds'] = (0.05 * torch.randn(rows, inner, generator=g, device='cuda')).to(kind) if case['residual'] else None
    return s


# ------------------------------------------------------------------------------------------------------------------------------
# One pass.

def run(s):
    if own:
        return _call(s)
    with torch.no_grad():
        return {'linear': _plain_linear, 'gated': _plain_gated, 'norm': _plain_norm, 'quantize': _plain_quantize}[s['case']['op']](s)


def _call(s):
    linear_act, gated_ff, rms_norm, quantize_rows = _ops()
    c = s['case']
    if c['op'] == 'quantize':
        q, scale = quantize_rows(s['x'])
        return {'q': q, 'scale': scale}
    if c['op'] == 'norm':
        got = rms_norm(s['x'], s['w'], residual=s['r'], eps=_EPS, quantize=c['out8'])
        names = (['q', 'scale'] if c['out8'] else ['y']) + (['sum'] if c['residual'] else [])
        out = dict(zip(names, got if isinstance(got, tuple) else (got,)))
        if c['train']:
            wrt = {k: s[k] for k in ('x', 'w', 'r') if s[k] is not None}
            given = [s['dy']] + ([s['ds']] if c['residual'] else [])
            out.update(zip(['d' + k for k in wrt], torch.autograd.grad(list(out.values()), list(wrt.values()), given)))
        return out
    if c['op'] == 'linear':
        y = linear_act(s['x'], s['w'], s['b'], residual=s['r'], act=c['act'], clamp=c['clamp'] if c['clamp'] >= 0 else None,
                       x_scale=s['xs'], weight_scale=s['ws'], out_dtype=s['out'])
    else:
        y = gated_ff(s['x'], s['w'], s['b'], act=c['act'], x_scale=s['xs'], weight_scale=s['ws'], out_dtype=s['out'])
    out = {'y': y}
    if c['train']:
        wrt = {k: s[k] for k in ('x', 'w', 'b', 'r') if s[k] is not None}
        out.update(zip(['d' + k for k in wrt], torch.autograd.grad(y, list(wrt.values()), s['dy'])))
    return out


def _act(v, name):
    """The activation of float32 sums, and its derivative."""
    if name == 'linear':
        return v, torch.ones_like(v)
    if name in ('relu', 'lrelu'):
        slope = torch.where(v > 0, 1.0, 0.2 if name == 'lrelu' else 0.0)
        return v * slope, slope
    if name == 'tanh':
        t = torch.tanh(v)
        return t, 1 - t * t
    sig = 1 / (1 + torch.exp(-v))
    if name == 'sigmoid':
        return sig, sig * (1 - sig)
    if name == 'swish':
        return v * sig, sig * (1 + v * (1 - sig))
    if name == 'softplus':
        return v.clamp(min=0) + torch.log1p(torch.exp(-v.abs())), sig
    raise ValueError(name)


def _sums(s):
    """x w^T + b in float32; 8-bit operands at the values they stand for."""
    x, w = s['x'].float(), s['w'].float()
    if s['xs'] is not None:
        x, w = x * s['xs'][:, None], w * s['ws'][:, None]
    v = x @ w.t()
    return v if s['b'] is None else v + s['b'].float()


def _back(s, dv, out):
    """Gradients of the rows, the weight and the bias from the gradient of the sums."""
    x, w = s['x'].float(), s['w'].float()
    out['dx'], out['dw'] = (dv @ w).to(s['out']), (dv.t() @ x).to(s['out'])
    if s['b'] is not None:
        out['db'] = dv.sum(dim=0).to(s['out'])


def _plain_linear(s):
    c = s['case']
    a, slope = _act(_sums(s), c['act'])
    a, slope = a * _GAINS[c['act']], slope * _GAINS[c['act']]
    if c['clamp'] >= 0:
        slope = torch.where(a.abs() < c['clamp'], slope, 0.0)
        a = a.clamp(-c['clamp'], c['clamp'])
    if s['r'] is not None:
        a = a + s['r'].float()
    out = {'y': a.to(s['out'])}
    if c['train']:
        _back(s, s['dy'].float() * slope, out)
        if s['r'] is not None:
            out['dr'] = s['dy']
    return out


def _plain_gated(s):
    c = s['case']
    gate, up = _sums(s).chunk(2, dim=1)
    a, slope = _act(gate, c['act'])
    out = {'y': (a * up).to(s['out'])}
    if c['train']:
        dy = s['dy'].float()
        _back(s, torch.cat([dy * up * slope, dy * a], dim=1), out)
    return out


def _plain_norm(s):
    c, out = s['case'], {}
    total = s['x'].float()
    if s['r'] is not None:
        total = total + s['r'].float()
    w = s['w'].float()
    inv = torch.rsqrt(total.square().mean(dim=1, keepdim=True) + _EPS)
    y = total * inv * w
    if c['out8']:
        out['q'], out['scale'] = _rows_to_8bit(y)
    else:
        out['y'] = y.to(s['out'])
    if s['r'] is not None:
        out['sum'] = total.to(s['out'])
    if c['train']:
        dy = s['dy'].float()
        dn = dy * w
        dt = inv * dn - total * inv ** 3 * (dn * total).mean(dim=1, keepdim=True)
        if s['r'] is not None:
            dt = dt + s['ds'].float()
            out['dr'] = dt.to(s['out'])
        out['dx'] = dt.to(s['out'])
        out['dw'] = (dy * total * inv).sum(dim=0).to(s['out'])
    return out


def _plain_quantize(s):
    q, scale = _rows_to_8bit(s['x'].float())
    return {'q': q, 'scale': scale}


# ------------------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits; gradients by differentiation of the definition.

def exact(case, seed):
    s = prepare(case, seed)
    v = {k: t.detach().double() for k, t in s.items() if isinstance(t, torch.Tensor)}
    F = torch.nn.functional
    acts = {'linear': lambda t: t, 'relu': F.relu, 'lrelu': lambda t: F.leaky_relu(t, 0.2), 'tanh': torch.tanh, 'sigmoid': torch.sigmoid,
            'swish': F.silu, 'softplus': F.softplus}
    if case['op'] == 'quantize':
        scale = torch.clamp(v['x'].abs().max(dim=1).values / 448, min=2.0 ** -64)
        return {'q': v['x'] / scale.unsqueeze(1), 'scale': scale}
    leaves = {k: v[k].requires_grad_(case['train']) for k in ('x', 'w', 'b', 'r') if k in v}
    if case['op'] == 'norm':
        total = v['x'] + v['r'] if 'r' in v else v['x'] * 1
        y = F.rms_norm(total, (case['inner'],), v['w'], _EPS)
        if case['out8']:
            scale = torch.clamp(y.abs().max(dim=1).values / 448, min=2.0 ** -64)
            out = {'q': y / scale.unsqueeze(1), 'scale': scale}
        else:
            out = {'y': y}
        if 'r' in v:
            out['sum'] = total
        given = [v.get('dy'), v.get('ds')]
    else:
        if 'xs' in v:
            sums = F.linear(v['x'] * v['xs'].unsqueeze(1), v['w'] * v['ws'].unsqueeze(1), v.get('b'))
        else:
            sums = F.linear(v['x'], v['w'], v.get('b'))
        if case['op'] == 'gated':
            y = acts[case['act']](sums[:, :case['outer']]) * sums[:, case['outer']:]
        else:
            y = acts[case['act']](sums) * (2 ** 0.5 if case['act'] in ('relu', 'lrelu', 'swish') else 1)
            if case['clamp'] >= 0:
                y = torch.clamp(y, -case['clamp'], case['clamp'])
            if 'r' in v:
                y = y + v['r']
        out, given = {'y': y}, [v.get('dy')]
    if case['train']:
        ys = [out[k] for k in ('y', 'sum') if k in out]
        grads = torch.autograd.grad(ys, list(leaves.values()), given[:len(ys)])
        out = {k: t.detach() for k, t in out.items()}
        out.update(zip(['d' + k for k in leaves], grads))
    return out
