"""Operators on token rows (torch_utils/ops/linear_act.py, gated_ff.py, rms_norm.py) against their definitions in 64 bits; every bound is derived in
tests/helpers/token_rows.py. CPU: the plain definitions, refusals of the Python and of the C entry points. GPU: the kernels."""

import ctypes
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), 'helpers'))
import token_rows as tr  # noqa: E402

from torch_utils.ops import _hip, bias_act
from torch_utils.ops import gated_ff as gf
from torch_utils.ops import linear_act as la
from torch_utils.ops import rms_norm as rn

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
DTYPES = [F32, F16, BF16]


def rand(*shape, seed, dtype=F32, scale=1.0, device='cuda'):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype).to(device)


# --------------------------------------------------------------------------------------------------------------------
# Checks shared by the cases.

def kept(dtype, act, gated):
    """Relative error of the derivatives that the forward pass keeps: the bfloat16 ones of smooth activations are rounded to 18 bits, two more than
    bfloat16 has, so to a quarter of its largest rounding error; all others are float32 or exact."""
    return tr.u(BF16) / 4 if dtype == BF16 and (gated or act not in ('linear', 'relu', 'lrelu')) else 0.0


def check_linear(x, w, b, r, act='linear', alpha=None, gain=None, clamp=None, dy=None):
    spec = bias_act.activation_funcs[act]
    al, ga = float(spec.def_alpha if alpha is None else alpha), float(spec.def_gain if gain is None else gain)
    leaves = [t for t in (x, w, b, r) if t is not None]
    if dy is not None:
        for t in leaves:
            t.requires_grad_(True)
    y = la.linear_act(x, w, b, residual=r, act=act, alpha=alpha, gain=gain, clamp=clamp)
    dt, k, n = x.dtype, w.shape[1], w.shape[0]
    x2, w2 = x.detach().double().reshape(-1, k), w.detach().double()
    v, off = tr.sums64(x2, w2, None if b is None else b.detach())
    a, d, a_off, d_off = tr.slopes64(v, off, act, al, ga, clamp)
    want = a if r is None else a + r.detach().double().reshape(-1, n)
    tr.assert_within(y.reshape(-1, n), want, tr.rounded(want, a_off + tr.F32_ULP * want.abs(), dt), 'y')
    assert y.dtype == dt and y.shape == x.shape[:-1] + (n,)
    if dy is None:
        return y
    grads = dict(zip([i for i, t in enumerate((x, w, b, r)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    g = dy.double().reshape(-1, n)
    dz, dz_off = g * d, g.abs() * d_off + (tr.F32_ULP + kept(dt, act, False)) * (g * d).abs()
    check_sums_gradients(grads, dz, dz_off, x2, w2, dt, x.shape)
    if r is not None:
        assert torch.equal(grads[3], dy)
    return y


def check_sums_gradients(grads, dz, dz_off, x2, w2, dt, x_shape):
    want, bound = tr.product64(dz, w2, dz_off, dt)
    tr.assert_within(grads[0].reshape(-1, w2.shape[1]), want, bound, 'dx')
    assert grads[0].shape == x_shape and grads[0].dtype == dt
    want, bound = tr.product64(dz.t(), x2, dz_off.t(), dt)
    tr.assert_within(grads[1], want, bound, 'dw')
    if 2 in grads:
        want = dz.sum(dim=0)
        off = dz_off.sum(dim=0) + (dz.shape[0] + 2) * tr.F32_ULP * dz.abs().sum(dim=0)
        tr.assert_within(grads[2], want, tr.rounded(want, off, dt), 'db')


def check_gated(x, w, b, act='swish', gain=1.0, dy=None):
    spec = bias_act.activation_funcs[act]
    al = float(spec.def_alpha)
    leaves = [t for t in (x, w, b) if t is not None]
    if dy is not None:
        for t in leaves:
            t.requires_grad_(True)
    h = gf.gated_ff(x, w, b, act=act, gain=gain)
    dt, k, n = x.dtype, w.shape[1], w.shape[0] // 2
    x2, w2 = x.detach().double().reshape(-1, k), w.detach().double()
    v, off = tr.sums64(x2, w2, None if b is None else b.detach())
    a, d, a_off, d_off = tr.slopes64(v[:, :n], off[:, :n], act, al, gain, None)
    up, up_off = v[:, n:], off[:, n:]
    want = a * up
    want_off = a.abs() * up_off + up.abs() * a_off + a_off * up_off + tr.F32_ULP * want.abs()
    tr.assert_within(h.reshape(-1, n), want, tr.rounded(want, want_off, dt), 'h')
    assert h.dtype == dt and h.shape == x.shape[:-1] + (n,)
    if dy is None:
        return
    grads = dict(enumerate(torch.autograd.grad(h, leaves, dy)))
    g = dy.double().reshape(-1, n)
    dz = torch.cat([g * d * up, g * a], dim=1)
    dz_off = torch.cat([g.abs() * (d_off * (up.abs() + up_off) + d.abs() * up_off), g.abs() * a_off], dim=1) + (3 * tr.F32_ULP + kept(dt, act, True)) * dz.abs()
    check_sums_gradients(grads, dz, dz_off, x2, w2, dt, x.shape)


def norm64(x, w, r, eps):
    s = x.detach().double() + (0 if r is None else r.detach().double())
    inv = (s.square().mean(dim=-1, keepdim=True) + eps).rsqrt()
    return s, inv, s * inv * (1 if w is None else w.detach().double())


def check_norm(x, w, r, eps=1e-6, dy=None, ds=None):
    leaves = [t for t in (x, w, r) if t is not None]
    if dy is not None:
        for t in leaves:
            t.requires_grad_(True)
    got = rn.rms_norm(x, w, residual=r, eps=eps)
    y, total = (got, None) if r is None else got
    dt, width = x.dtype, x.shape[-1]
    s, inv, want = norm64(x, w, r, eps)
    # the mean square: width float32 terms of one sign, halved by the root; then root, quotient and two products
    rel = (width / 2 + 8) * tr.F32_ULP
    tr.assert_within(y, want, tr.rounded(want, rel * want.abs(), dt), 'y')
    assert y.dtype == dt and y.shape == x.shape
    if r is not None:
        tr.assert_within(total, s, tr.rounded(s, tr.F32_ULP * s.abs(), dt), 'sum')
    if dy is None:
        return
    outs, given = ([y], [dy]) if r is None or ds is None else ([y, total], [dy, ds])
    grads = torch.autograd.grad(outs, leaves, given)
    g = dy.double() * (1 if w is None else w.detach().double())
    dot = (g * s).mean(dim=-1, keepdim=True)
    big = (g * s).abs().mean(dim=-1, keepdim=True)
    want = inv * g - s * inv ** 3 * dot + (0 if ds is None or r is None else ds.double())
    # the kernel reads the sum as it was stored, rounded once, with two bits of what the rounding left: within a third of half a step
    su = (tr.u(dt) / 3 if r is not None and x.is_cuda else tr.u(dt) if r is not None else 0) + 3 * tr.F32_ULP
    off = rel * (inv * g).abs() * 2 + (s * inv ** 3).abs() * big * (2 * su + 4 * rel) + 4 * tr.F32_ULP * want.abs()
    bound = tr.rounded(want, off, dt)
    tr.assert_within(grads[0], want, bound, 'dx')
    if r is not None:
        tr.assert_within(grads[-1], want, bound, 'dr')
    if w is not None:
        terms = (dy.double() * s * inv).reshape(-1, width)
        want = terms.sum(dim=0)
        off = terms.abs().sum(dim=0) * (su + rel + (terms.shape[0] + 3) * tr.F32_ULP)
        tr.assert_within(grads[1], want, tr.rounded(want, off, dt), 'dw')


def check_8bit_rows(q, scale, want, rel):
    """q, scale against the rows `want` in 64 bits, whose float32 evaluation is off by `rel` relative to each value."""
    assert q.dtype == E4M3 and scale.dtype == F32 and scale.shape == want.shape[:-1] and q.shape == want.shape
    top = (want.abs().amax(dim=-1) / 448).clamp(min=2.0 ** -64)
    tr.assert_within(scale, top, (rel + 4 * tr.F32_ULP) * top, 'scale')
    v = want / top.unsqueeze(-1)
    # e4m3: half a step is 2^-4 of the value, and 2^-10 below its smallest normal number 2^-6
    bound = torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + 4 * (rel + 4 * tr.F32_ULP) * v.abs()
    tr.assert_within(q.float(), v, bound, 'q')


# --------------------------------------------------------------------------------------------------------------------
# CPU: plain definitions and refusals.

@pytest.mark.parametrize('act', tr.ACTS)
def test_plain_linear_is_the_definition_cpu(act):
    x, w, b, r = (rand(*s, seed=i, device='cpu') for i, s in enumerate([(3, 4, 7), (5, 7), (5,), (3, 4, 5)]))
    check_linear(x, w, b, r, act=act, clamp=0.9, dy=rand(3, 4, 5, seed=9, device='cpu'))


@pytest.mark.parametrize('act', ['swish', 'tanh', 'relu'])
def test_plain_gated_is_the_definition_cpu(act):
    check_gated(rand(6, 7, seed=0, device='cpu'), rand(10, 7, seed=1, device='cpu'), rand(10, seed=2, device='cpu'), act=act, gain=1.5, dy=rand(6, 5, seed=3, device='cpu'))


def test_plain_norm_is_the_definition_cpu():
    x, w, r, dy, ds = (rand(*s, seed=i, device='cpu') for i, s in enumerate([(4, 9), (9,), (4, 9), (4, 9), (4, 9)]))
    check_norm(x, w, r, dy=dy, ds=ds)
    q, scale, total = rn.rms_norm(x.detach(), w.detach(), residual=r.detach(), quantize=True)
    check_8bit_rows(q, scale, norm64(x, w, r, 1e-8)[2], 20 * tr.F32_ULP)
    q, scale = rn.quantize_rows(torch.zeros(2, 5))
    assert float(scale.max()) == 2.0 ** -64 and not q.float().any()


def test_chained_plain_forms_have_gradients_by_differences_cpu():
    """The whole row-wise block in float64-free plain form: its gradients against central differences of the 64-bit definition."""
    x, r, nw, w1, w2 = (rand(*s, seed=i, device='cpu', scale=0.5) for i, s in enumerate([(3, 6), (3, 6), (6,), (8, 6), (6, 4)]))
    dy = rand(3, 6, seed=9, device='cpu')

    def block(x, r, nw, w1, w2):
        y, s = rn.rms_norm(x, nw, residual=r, eps=1e-6, impl='ref')
        return la.linear_act(gf.gated_ff(y, w1, impl='ref'), w2, residual=s, impl='ref')

    def value64(args):
        x, r, nw, w1, w2 = (t.double() for t in args)
        s = x + r
        y = s * (s.square().mean(dim=1, keepdim=True) + 1e-6).rsqrt() * nw
        g, up = (y @ w1.t()).chunk(2, dim=1)
        return float((((g * torch.sigmoid(g) * up) @ w2.t() + s) * dy.double()).sum())

    args = [x, r, nw, w1, w2]
    leaves = [t.clone().requires_grad_(True) for t in args]
    grads = torch.autograd.grad(block(*leaves), leaves, dy)
    h = 1e-5
    for i, t in enumerate(args):
        for at in range(t.numel()):
            moved = [[a.double().clone() for a in args] for _ in range(2)]
            moved[0][i].view(-1)[at] += h
            moved[1][i].view(-1)[at] -= h
            diff = (value64(moved[0]) - value64(moved[1])) / (2 * h)
            # differences are exact to h^2 * third derivative (order 10 here) + 64-bit rounding / h; the gradient is float32
            assert abs(float(grads[i].view(-1)[at]) - diff) <= 1e-8 + 100 * tr.F32_ULP * max(1.0, abs(diff)), (i, at)


def test_refusals_python_cpu():
    x, w = torch.randn(4, 8), torch.randn(6, 8)
    q, s = rn.quantize_rows(x)
    qw, sw = rn.quantize_rows(w)
    for call in (lambda: la.linear_act(x, torch.randn(6, 7)), lambda: la.linear_act(x, w.half()), lambda: la.linear_act(x, w, torch.randn(5)),
                 lambda: la.linear_act(x, w, torch.randn(6).half()), lambda: la.linear_act(x, w, residual=torch.randn(4, 5)),
                 lambda: la.linear_act(x, w, residual=torch.randn(4, 6).half()), lambda: la.linear_act(x, w, act='gelu'), lambda: la.linear_act(x, w, clamp=-1),
                 lambda: la.linear_act(x.double(), w.double()), lambda: la.linear_act(x, w, x_scale=s, weight_scale=sw), lambda: la.linear_act(x, w, out_dtype=BF16),
                 lambda: la.linear_act(q, qw), lambda: la.linear_act(q, qw, x_scale=s), lambda: la.linear_act(q, qw, x_scale=s, weight_scale=s),
                 lambda: la.linear_act(q, qw, x_scale=s.half(), weight_scale=sw.half()), lambda: la.linear_act(q, qw, x_scale=s, weight_scale=sw, out_dtype=F32),
                 lambda: la.linear_act(q, qw, torch.randn(6, dtype=BF16, requires_grad=True), x_scale=s, weight_scale=sw),
                 lambda: la.linear_act(q, qw, residual=torch.randn(4, 6, dtype=BF16, requires_grad=True), x_scale=s, weight_scale=sw),
                 lambda: la.linear_act(q.clone().requires_grad_(True), qw, x_scale=s, weight_scale=sw), lambda: gf.gated_ff(q, qw.clone().requires_grad_(True), x_scale=s, weight_scale=sw),
                 lambda: la.linear_act(x, w.unsqueeze(0)), lambda: la.linear_act(x, w, impl='fast'),
                 lambda: gf.gated_ff(x, torch.randn(5, 8)), lambda: gf.gated_ff(x, w, torch.randn(3)), lambda: gf.gated_ff(x, w, act='silu'),
                 lambda: rn.rms_norm(x, torch.randn(7)), lambda: rn.rms_norm(x, torch.randn(8).half()), lambda: rn.rms_norm(x, residual=torch.randn(8)),
                 lambda: rn.rms_norm(x, eps=-1.0), lambda: rn.rms_norm(x.double()), lambda: rn.rms_norm(torch.randn(3, 0)), lambda: rn.rms_norm(torch.randint(3, (2, 2))),
                 lambda: rn.rms_norm(x.clone().requires_grad_(True), quantize=True), lambda: rn.quantize_rows(q), lambda: rn.quantize_rows(x.clone().requires_grad_(True)),
                 lambda: rn.quantize_rows(torch.randn(2, 0))):
        with pytest.raises(AssertionError):
            call()


def test_refusals_of_the_c_entries_cpu():
    """Bad arguments come back as LVG_ERR_INVALID before anything is launched (no device is touched)."""
    lib = _hip.lib()
    p = ctypes.addressof((ctypes.c_char * 4096)()) & ~15
    good = dict(x=p, w=p, b=None, r=None, xs=None, ws=None, y=p, s=None, work=None, size=0, rows=4, outer=4, inner=4, ldx=4, ldw=4, ldr=0, ldy=4,
                dtype=2, out=2, gated=0, act=1, kind=0, alpha=0.0, gain=1.0, clamp=-1.0)

    def linear(**kw):
        return lib.lvg_linear_act(*{**good, **kw}.values(), None)

    for kw in (dict(dtype=3), dict(dtype=7), dict(out=0), dict(dtype=4), dict(dtype=4, xs=p), dict(dtype=4, xs=p, ws=p, out=0), dict(xs=p, ws=p), dict(rows=-1), dict(outer=1 << 31),
               dict(inner=-4), dict(act=0), dict(act=10), dict(y=None), dict(x=None), dict(w=None), dict(ldx=-4), dict(ldy=3), dict(gated=1, r=p), dict(gated=1, clamp=1.0),
               dict(kind=1), dict(kind=3, s=p), dict(kind=2, s=p, act=4), dict(kind=2, s=p, gated=1), dict(inner=1 << 20, ldx=1 << 20, ldw=1 << 20),
               dict(inner=1 << 20, ldx=1 << 20, ldw=1 << 20, work=p + 8, size=1 << 40)):
        assert linear(**kw) == -1, kw
        assert lib.lvg_last_error()
    assert linear(rows=0) == 0 and linear(outer=0) == 0
    assert lib.lvg_linear_act_work(-1, 4, 4, 2, 0) == -1 and lib.lvg_linear_act_work(4, 4, 4, 3, 0) == -1
    assert lib.lvg_linear_slope_bytes(4, 5, 2, 1, 2) == 4 * 2 * (10 + 2) and lib.lvg_linear_slope_bytes(4, 5, 1, 1, 0) == 80 and lib.lvg_linear_slope_bytes(4, 5, 1, 2, 2) == 20
    assert lib.lvg_linear_slope_bytes(4, 5, 3, 1, 2) == -1 and lib.lvg_linear_slope_bytes(4, 5, 1, 3, 2) == -1 and lib.lvg_linear_slope_bytes(4, 5, 1, 1, 4) == -1
    for bad in ((-1, 4, 4, 1, 0, 7, 2), (4, 4, 4, 3, 0, 7, 2), (4, 4, 4, 1, 3, 7, 2), (4, 4, 4, 2, 2, 7, 2), (4, 4, 4, 1, 0, 7, 4), (4, 1 << 30, 4, 2, 1, 7, 2)):
        assert lib.lvg_linear_backward_work(*bad) == -1, bad
    size = lib.lvg_linear_backward_work(4, 4, 4, 1, 1, 7, 2)
    back = dict(dy=p, s=p, x=p, w=p, dx=p, dw=p, db=p, work=p, size=size, rows=4, outer=4, inner=4, ldy=4, ldx=4, ldw=4, halves=1, kind=1, alpha=0.0, gain=1.0, dtype=2)
    for kw in (dict(dtype=4), dict(dy=None), dict(s=None), dict(x=None), dict(w=None), dict(work=None), dict(work=p + 8), dict(size=size - 1), dict(rows=-1), dict(halves=3),
               dict(halves=2, kind=0), dict(halves=2, kind=2), dict(kind=5), dict(ldy=-1), dict(ldx=-1), dict(ldw=-1)):
        assert lib.lvg_linear_backward(*{**back, **kw}.values(), None) == -1, kw
    assert lib.lvg_linear_backward(*{**back, 'rows': 0, 'outer': 0}.values(), None) == 0
    norm = dict(x=p, r=None, w=None, y=p, s=None, rest=None, rstd=None, scale=None, rows=4, width=4, ldx=4, ldr=0, eps=0.0, dtype=2, quant=0)
    for kw in (dict(dtype=3), dict(x=None), dict(y=None), dict(quant=1), dict(s=p), dict(rest=p), dict(rows=-1), dict(width=0), dict(ldx=-1), dict(eps=-1.0), dict(eps=math.nan)):
        assert lib.lvg_rms_norm(*{**norm, **kw}.values(), None) == -1, kw
    assert lib.lvg_rms_norm_backward_work(4, 0, 1, 2) == -1 and lib.lvg_rms_norm_backward_work(-1, 4, 1, 2) == -1 and lib.lvg_rms_norm_backward_work(4, 4, 1, 4) == -1
    size = lib.lvg_rms_norm_backward_work(4, 4, 1, 2)
    back = dict(dy=p, ds=None, s=p, rest=None, w=None, rstd=p, dx=p, dw=p, work=p, size=size, rows=4, width=4, lddy=4, ldds=0, lds=4, dtype=2)
    for kw in (dict(dtype=4), dict(dy=None), dict(rstd=None), dict(dx=None), dict(s=None), dict(work=None), dict(work=p + 4), dict(size=size - 1), dict(lds=-1), dict(lddy=-1)):
        assert lib.lvg_rms_norm_backward(*{**back, **kw}.values(), None) == -1, kw
    assert lib.lvg_quantize_rows(p, p, None, 4, 4, 4, 2, None) == -1 and lib.lvg_quantize_rows(p, p, p, 4, 0, 4, 2, None) == -1


# --------------------------------------------------------------------------------------------------------------------
# GPU: products.

# rows, inner, outer: single values, less than a fragment, odd widths, one more than a tile, a summed index of one and of many steps (split over
# the chip), and results of several tiles of every size
SIZES = [(1, 1, 1), (1, 64, 64), (2, 7, 3), (3, 515, 5), (16, 1024, 96), (17, 130, 67), (33, 256, 128), (64, 2048, 16), (65, 63, 129), (129, 257, 515), (300, 64, 1000), (20, 9000, 40), (40, 9000, 40)]
BIG = [(2100, 192, 2304), (1025, 200, 4113), (2100, 1021, 2311)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('size', SIZES + BIG)
def test_linear_forward_and_gradients_gpu(size, dtype):
    m, k, n = size
    x, w = rand(m, k, seed=1, dtype=dtype), rand(n, k, seed=2, dtype=dtype, scale=k ** -0.5)
    b, r, dy = rand(n, seed=3, dtype=dtype), rand(m, n, seed=4, dtype=dtype), rand(m, n, seed=5, dtype=dtype)
    check_linear(x, w, b, r, act='lrelu', dy=dy)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('act', tr.ACTS)
def test_linear_activations_gpu(act, dtype):
    x, w, b = rand(37, 40, seed=1, dtype=dtype), rand(29, 40, seed=2, dtype=dtype, scale=0.3), rand(29, seed=3, dtype=dtype)
    dy = rand(37, 29, seed=5, dtype=dtype)
    check_linear(x.clone(), w.clone(), b.clone(), None, act=act, dy=dy)
    check_linear(x.clone(), w.clone(), None, None, act=act, gain=-1.7, clamp=0.8, alpha=0.3 if act == 'lrelu' else None, dy=dy)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('size', [(1, 1, 1), (1, 64, 64), (3, 515, 5), (17, 130, 67), (33, 256, 128), (129, 257, 260), (20, 9000, 40), (40, 9000, 40), (1030, 136, 2100), (1530, 1037, 1301)])
def test_gated_forward_and_gradients_gpu(size, dtype):
    m, k, n = size
    x, w = rand(m, k, seed=1, dtype=dtype), rand(2 * n, k, seed=2, dtype=dtype, scale=k ** -0.5)
    check_gated(x, w, rand(2 * n, seed=3, dtype=dtype), dy=rand(m, n, seed=5, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('act', tr.ACTS)
def test_gated_activations_gpu(act):
    check_gated(rand(37, 40, seed=1, dtype=F16), rand(58, 40, seed=2, dtype=F16, scale=0.3), None, act=act, gain=-1.3, dy=rand(37, 29, seed=5, dtype=F16))


def odd_views(dtype):
    """x [.., 48], w [40, 48]: contiguous, rows that start at odd places, wide row strides, columns of a matrix, rows that are all the same one."""
    base = rand(70, 111, seed=7, dtype=dtype, scale=0.5)
    return {'offset': (base.reshape(-1)[1:1 + 30 * 48].view(30, 48), base.reshape(-1)[3:3 + 40 * 48].view(40, 48)),
            'stride': (base[:30, 5:53], base[30:70, 8:56]),
            'columns': (base[:48, :30].t(), base[:48, 60:100].t()),
            'expanded': (base[:1, :48].expand(30, 48), base[1:2, :48].expand(40, 48)),
            'three': (base[:30, :96].reshape(5, 6, 2, 48)[:, :, 1], base[30:70, :48]),
            'permuted': (base[:30, :48].reshape(5, 6, 48).transpose(0, 1), base[30:70, :48])}


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('view', ['offset', 'stride', 'columns', 'expanded', 'three', 'permuted'])
def test_layouts_gpu(view, dtype):
    x, w = (t.detach() for t in odd_views(dtype)[view])
    shape = x.shape[:-1]
    r = rand(*shape[:-1], 1, 40, seed=4, dtype=dtype).expand(*shape, 40)
    wide = rand(*shape, 90, seed=5, dtype=dtype)
    check_linear(x, w, None, r, act='tanh', dy=wide[..., 7:47])
    check_gated(x.detach(), w.detach(), rand(80, seed=3, dtype=dtype)[::2], dy=wide[..., 1:41:2])
    check_norm(x.detach(), rand(96, seed=3, dtype=dtype)[::2], x.detach(), dy=wide[..., 3:51], ds=wide[..., :1].expand(*shape, 48))


@pytest.mark.gpu
def test_single_rows_and_8bit_layouts_gpu():
    """A vector is one row; 8-bit operands take any strides."""
    x, w, b = rand(70, seed=1, dtype=BF16), rand(40, 70, seed=2, dtype=BF16), rand(40, seed=3, dtype=BF16)
    check_linear(x, w, b, rand(40, seed=4, dtype=BF16), act='swish', dy=rand(40, seed=5, dtype=BF16))
    check_norm(x.detach(), rand(70, seed=6, dtype=BF16), rand(70, seed=7, dtype=BF16), dy=rand(70, seed=8, dtype=BF16), ds=rand(70, seed=9, dtype=BF16))
    q, s = rn.quantize_rows(x.detach())
    assert q.shape == (70,) and s.shape == ()
    (q, s), (qw, sw) = rn.quantize_rows(rand(70, 111, seed=1)), rn.quantize_rows(rand(90, 111, seed=2))
    s2, sw2 = torch.stack([s, s], dim=1)[:, 0], torch.stack([sw, sw], dim=1)[:, 1]
    for rows in (5, 20, 70):
        for qx, qv in ((q[:rows, 3:83], qw[:, 7:87]), (q[:rows, :80].t().contiguous().t(), qw[:, :80].t().contiguous().t())):
            v, off = tr.sums64(qx.float(), qv.float(), None, s[:rows], sw)
            tr.assert_within(la.linear_act(qx, qv, x_scale=s2[:rows], weight_scale=sw2), v, tr.rounded(v, off, BF16), 'y')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [F16, BF16])
def test_results_larger_than_the_caches_gpu(dtype):
    """64 MB and more of results are stored past the caches: whole tiles and those at the edges, rows of the norm, forward and backward."""
    x, w = rand(2600, 64, seed=1, dtype=dtype), rand(2 * 4360, 64, seed=2, dtype=dtype, scale=0.125)
    check_gated(x, w, rand(2 * 4360, seed=3, dtype=dtype), dy=rand(2600, 4360, seed=5, dtype=dtype))
    (q, s), (qw, sw) = rn.quantize_rows(rand(4200, 64, seed=6)), rn.quantize_rows(rand(2 * 8192, 64, seed=7, scale=0.125))
    v, off = tr.sums64(q.float(), qw.float(), None, s, sw)
    a, _, a_off, _ = tr.slopes64(v[:, :8192], off[:, :8192], 'swish', 0.0, 1.0, None)
    up, up_off = v[:, 8192:], off[:, 8192:]
    want = a * up
    bound = a.abs() * up_off + up.abs() * a_off + a_off * up_off + tr.F32_ULP * want.abs()
    tr.assert_within(gf.gated_ff(q, qw, x_scale=s, weight_scale=sw, out_dtype=dtype), want, tr.rounded(want, bound, dtype), 'h')
    for shape in ((8300, 4096), (70000, 520)):
        x, w, r, dy, ds = (rand(*sh, seed=i, dtype=dtype) for i, sh in enumerate([shape, shape[-1:], shape, shape, shape]))
        check_norm(x, w, r, dy=dy, ds=ds)
        q, scale = rn.quantize_rows(x.detach())
        check_8bit_rows(q, scale, x.detach().double(), 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize('act', ['linear', 'lrelu', 'swish'])
def test_gradients_of_some_inputs_alone_gpu(act):
    """Each subset of inputs that asks for a gradient gets the bits it gets when all of them ask."""
    base = [rand(70, 96, seed=1, dtype=BF16), rand(80, 96, seed=2, dtype=BF16, scale=0.1), rand(80, seed=3, dtype=BF16)]
    extra, dy, dh = rand(70, 80, seed=4, dtype=BF16), rand(70, 80, seed=5, dtype=BF16), rand(70, 40, seed=6, dtype=BF16)
    norm = [rand(70, 80, seed=7, dtype=BF16), rand(80, seed=8, dtype=BF16), extra]

    def run(wanted, kind):
        ts = [t.clone().requires_grad_(i in wanted) for i, t in enumerate(norm if kind == 'norm' else base + ([extra] if kind == 'linear' else []))]
        if kind == 'linear':
            out = la.linear_act(ts[0], ts[1], ts[2], residual=ts[3], act=act)
        elif kind == 'gated':
            out = gf.gated_ff(ts[0], ts[1], ts[2], act=act)
        else:
            out = rn.rms_norm(ts[0], ts[1], residual=ts[2])[0]
        return dict(zip(wanted, torch.autograd.grad(out, [ts[i] for i in wanted], dh if kind == 'gated' else dy)))

    for kind, n in (('linear', 4), ('gated', 3), ('norm', 3)):
        every = run(range(n), kind)
        for mask in range(1, 2 ** n):
            wanted = [i for i in range(n) if mask >> i & 1]
            for i, g in run(wanted, kind).items():
                assert torch.equal(g, every[i]), (kind, wanted, i)


@pytest.mark.gpu
def test_a_graph_can_be_walked_twice_gpu():
    x, w = rand(33, 70, seed=1, dtype=F16).requires_grad_(True), rand(60, 70, seed=2, dtype=F16, scale=0.1).requires_grad_(True)
    y, dy = gf.gated_ff(x, w), rand(33, 30, seed=3, dtype=F16)
    first = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, (x, w), dy)))
    with torch.inference_mode():
        assert torch.equal(gf.gated_ff(x, w), y)


@pytest.mark.gpu
def test_two_streams_at_once_gpu():
    """Calls on two streams side by side, split over the summed index so that both use workspaces, give what they give alone."""
    xs = [rand(40, 9000, seed=i, dtype=BF16) for i in (1, 2)]
    w = rand(96, 9000, seed=3, dtype=BF16, scale=0.01)
    want = [la.linear_act(x, w, act='swish') for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(la.linear_act(xs[i], w, act='swish'))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.gpu
def test_offsets_past_32_bits_gpu():
    """Operands and results of more than 2^32 bytes: the last rows are what a call on them alone gives."""
    rows, width = 36000, 65536
    big = torch.zeros(rows, width, dtype=BF16, device='cuda')
    big[-70:] = rand(70, width, seed=1, dtype=BF16)
    w = rand(48, width, seed=2, dtype=BF16, scale=width ** -0.5)
    tail = big[-64:].clone()
    assert big.numel() * 2 > 2 ** 32
    y, alone = la.linear_act(big, w)[-64:].double(), la.linear_act(tail, w).double()
    v, off = tr.sums64(tail, w, None)
    tr.assert_within(y, v, tr.rounded(v, off, BF16), 'rows past 2^32')
    tr.assert_within(alone, v, tr.rounded(v, off, BF16), 'rows')
    n = rn.rms_norm(big, residual=big)[0]
    assert torch.equal(n[-64:], rn.rms_norm(tail, residual=tail)[0])
    del n
    q, s = rn.quantize_rows(big)
    q2, s2 = rn.quantize_rows(tail)
    assert torch.equal(q[-64:].float(), q2.float()) and torch.equal(s[-64:], s2)
    del q
    # as the weight of a product (its rows' gradient read down them), and as a result
    x = rand(40, 64, seed=3, dtype=BF16)
    wide = rand(rows, 64, seed=4, dtype=BF16)
    out = la.linear_act(rand(65536, 64, seed=5, dtype=BF16), wide)
    assert out.numel() * 2 > 2 ** 32
    tail_rows = rand(65536, 64, seed=5, dtype=BF16)[-50:]
    v, off = tr.sums64(tail_rows, wide, None)
    tr.assert_within(out[-50:], v, tr.rounded(v, off, BF16), 'result past 2^32')
    del out
    wl = rand(36000, 64, seed=6, dtype=BF16).requires_grad_(True)
    xl = x.requires_grad_(True)
    dy = torch.zeros(40, 36000, dtype=BF16, device='cuda')
    dy[:, -3:] = 1
    dx, dw = torch.autograd.grad(la.linear_act(xl, wl), (xl, wl), dy)
    want = wl.detach().double()[-3:].sum(dim=0).expand(40, 64)
    tr.assert_within(dx, want, tr.rounded(want, 5 * tr.F32_ULP * want.abs() + 1e-5, BF16), 'dx')
    want = x.detach().double().sum(dim=0).expand(3, 64)
    tr.assert_within(dw[-3:], want, tr.rounded(want, 50 * tr.F32_ULP * x.detach().double().abs().sum(dim=0).expand(3, 64), BF16), 'dw')
    # the summed index runs down operands of more than 2^32 bytes
    g = torch.zeros(rows, 40, dtype=BF16, device='cuda')
    g[-2:] = 1
    wb = rand(40, width, seed=7, dtype=BF16, scale=0.01).requires_grad_(True)
    dw, = torch.autograd.grad(la.linear_act(big, wb), wb, g)
    want = big[-2:].double().sum(dim=0).expand(40, width)
    tr.assert_within(dw, want, tr.rounded(want, 4 * tr.F32_ULP * big[-2:].double().abs().sum(dim=0).expand(40, width), BF16), 'dw down')


@pytest.mark.gpu
def test_results_are_reproducible_gpu():
    x, w, dy = rand(700, 1100, seed=1, dtype=BF16), rand(1000, 1100, seed=2, dtype=BF16, scale=0.03), rand(700, 500, seed=3, dtype=BF16)
    x.requires_grad_(True), w.requires_grad_(True)
    runs = []
    for _ in range(2):
        h = gf.gated_ff(x, w)
        runs.append([h, *torch.autograd.grad(h, (x, w), dy)])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.gpu
def test_empty_sizes_gpu():
    dev = 'cuda'
    for m, k, n in ((0, 8, 4), (3, 0, 4), (3, 8, 0)):
        x, w = torch.randn(m, k, device=dev, requires_grad=True), torch.randn(2 * n, k, device=dev, requires_grad=True)
        b = torch.randn(2 * n, device=dev, requires_grad=True)
        for y, want in ((la.linear_act(x, w, b, act='tanh'), torch.tanh(x @ w.t() + b)),
                        (gf.gated_ff(x, w, b), torch.nn.functional.silu((x @ w.t() + b)[:, :n]) * (x @ w.t() + b)[:, n:])):
            torch.testing.assert_close(y, want, rtol=1e-6, atol=1e-6)
            dy = torch.randn_like(y)
            for got, g in zip(torch.autograd.grad(y, (x, w, b), dy), torch.autograd.grad(want, (x, w, b), dy)):
                torch.testing.assert_close(got, g, rtol=1e-5, atol=1e-5)
    x = torch.randn(0, 8, device=dev, requires_grad=True)
    w = torch.randn(8, device=dev, requires_grad=True)
    y = rn.rms_norm(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert gx.shape == (0, 8) and not gw.any()
    q, scale = rn.quantize_rows(x.detach())
    assert q.shape == (0, 8) and scale.shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize('bad', [math.nan, math.inf, -math.inf])
def test_non_finite_values_stay_in_their_rows_and_columns_gpu(bad):
    """A NaN or infinity in one row of x (or w) shows in that row (column) of the result and nowhere else, in tiles that end behind it too."""
    for dtype in (F32, BF16):
        x, w = rand(130, 70, seed=1, dtype=dtype), rand(67, 70, seed=2, dtype=dtype)
        clean = la.linear_act(x, w, act='swish', clamp=3.0)
        x2, w2 = x.clone(), w.clone()
        x2[129, 69] = bad
        w2[66, 3] = bad
        y = la.linear_act(x2, w2, act='swish', clamp=3.0)
        assert torch.equal(y[:129, :66], clean[:129, :66])
        if math.isnan(bad):
            assert bool(y[129].isnan().all()) and bool(y[:, 66].isnan().all())
        n = rn.rms_norm(x2)
        assert torch.equal(n[:129], rn.rms_norm(x)[:129]) and bool(n[129].isnan().any())


@pytest.mark.gpu
def test_rows_behind_the_result_stay_as_they_are_gpu():
    """The kernels write rows x outer values and nothing around them."""
    lib = _hip.lib()
    for m, k, n in ((1, 64, 40), (5, 72, 33), (70, 100, 130)):
        x, w = rand(m, k, seed=1, dtype=BF16), rand(n, k, seed=2, dtype=BF16)
        y = torch.full((m + 2, n + 5), 7.0, dtype=BF16, device='cuda')
        size = lib.lvg_linear_act_work(m, n, k, 2, 0)
        work = torch.empty(max(1, size), dtype=torch.uint8, device='cuda')
        assert lib.lvg_linear_act(x.data_ptr(), w.data_ptr(), None, None, None, None, y[1:, 2:].data_ptr(), None, work.data_ptr(), size, m, n, k, k, k, 0, n + 5,
                                  2, 2, 0, 1, 0, 0.0, 1.0, -1.0, _hip.stream(x.device)) == 0
        got = y[1:m + 1, 2:n + 2].clone()
        y[1:m + 1, 2:n + 2] = 7
        assert bool((y == 7).all())
        assert torch.equal(got, la.linear_act(x, w))


# --------------------------------------------------------------------------------------------------------------------
# GPU: 8 bits.

@pytest.mark.gpu
@pytest.mark.parametrize('out', [BF16, F16])
@pytest.mark.parametrize('size', [(1, 1, 1), (1, 64, 64), (2, 7, 3), (3, 515, 5), (16, 1024, 96), (17, 130, 67), (65, 63, 129), (64, 4096, 16), (300, 128, 1000), (1030, 320, 2304), (1030, 2051, 1501)])
def test_8bit_products_gpu(size, out):
    m, k, n = size
    (q, s), (qw, sw) = rn.quantize_rows(rand(m, k, seed=1)), rn.quantize_rows(rand(2 * n, k, seed=2, scale=k ** -0.5))
    b, r = rand(2 * n, seed=3, dtype=out), rand(m, 2 * n, seed=4, dtype=out)
    v, off = tr.sums64(q.float(), qw.float(), b, s, sw)
    a, _, a_off, _ = tr.slopes64(v, off, 'lrelu', 0.2, 2 ** 0.5, None)
    want = a + r.double()
    y = la.linear_act(q, qw, b, residual=r, act='lrelu', x_scale=s, weight_scale=sw, out_dtype=out)
    tr.assert_within(y, want, tr.rounded(want, a_off + tr.F32_ULP * want.abs(), out), 'y')
    a, _, a_off, _ = tr.slopes64(v[:, :n], off[:, :n], 'swish', 0.0, 1.0, None)
    up, up_off = v[:, n:], off[:, n:]
    want = a * up
    h = gf.gated_ff(q, qw, b, x_scale=s, weight_scale=sw, out_dtype=out)
    tr.assert_within(h, want, tr.rounded(want, a.abs() * up_off + up.abs() * a_off + a_off * up_off + tr.F32_ULP * want.abs(), out), 'h')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', [(1, 1), (3, 7), (5, 64), (2, 3, 129), (7, 515), (130, 1024), (3, 4100), (2, 9001), (2, 40000)])
def test_8bit_rows_gpu(shape, dtype):
    x, w, r = rand(*shape, seed=1, dtype=dtype), rand(shape[-1], seed=2, dtype=dtype), rand(*shape, seed=3, dtype=dtype)
    q, scale = rn.quantize_rows(x)
    check_8bit_rows(q, scale, x.double(), 0.0)
    rel = (shape[-1] / 2 + 8) * tr.F32_ULP
    q, scale, total = rn.rms_norm(x, w, residual=r, eps=1e-6, quantize=True)
    s, _, want = norm64(x, w, r, 1e-6)
    check_8bit_rows(q, scale, want, rel)
    tr.assert_within(total, s, tr.rounded(s, tr.F32_ULP * s.abs(), dtype), 'sum')
    q, scale = rn.rms_norm(x, eps=0.0, quantize=True)
    check_8bit_rows(q, scale, norm64(x, None, None, 0.0)[2], rel)


@pytest.mark.gpu
def test_8bit_rows_at_the_edges_gpu():
    for width in (5, 64, 3000, 9000, 40000):
        x = torch.zeros(6, width, device='cuda')
        x[1] = 1e-30                        # below the smallest scale: zeros
        x[2, 1] = 448.0
        x[3, 2] = math.inf
        x[4, 3] = math.nan
        x[5] = 3e38
        q, scale = rn.quantize_rows(x)
        want_q, want_scale = rn.quantize_rows(x.cpu())
        assert torch.equal(scale.cpu(), want_scale) or bool(((scale.cpu() == want_scale) | (scale.cpu().isnan() & want_scale.isnan())).all())
        got, want = q.float().cpu(), want_q.float()
        assert bool(((got == want) | (got.isnan() & want.isnan())).all())


# --------------------------------------------------------------------------------------------------------------------
# GPU: norm.

@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', [(1, 1), (3, 7), (5, 64), (2, 3, 129), (7, 515), (1030, 1024), (3000, 65), (3, 2500), (5, 4096), (9, 9001), (600, 8200), (3, 40000), (70, 33000)])
def test_norm_forward_and_gradients_gpu(shape, dtype):
    x, w, r, dy, ds = (rand(*s, seed=i, dtype=dtype) for i, s in enumerate([shape, shape[-1:], shape, shape, shape]))
    check_norm(x.clone(), w.clone(), r.clone(), dy=dy, ds=ds)
    check_norm(x.clone(), w.clone(), r.clone(), dy=dy)
    check_norm(x.clone(), None, None, dy=dy)


@pytest.mark.gpu
def test_norm_through_the_sum_alone_gpu():
    x, w, r = (rand(*s, seed=i, dtype=BF16).requires_grad_(True) for i, s in enumerate([(9, 70), (70,), (9, 70)]))
    _, total = rn.rms_norm(x, w, residual=r)
    ds = rand(9, 70, seed=5, dtype=BF16)
    gx, gw, gr = torch.autograd.grad(total, (x, w, r), ds)
    assert torch.equal(gx, ds) and torch.equal(gr, ds) and not gw.any()


# --------------------------------------------------------------------------------------------------------------------
# GPU: the operators together, streams, graphs.

def block(x, r, nw, w1, w2, b2):
    y, s = rn.rms_norm(x, nw, residual=r, eps=1e-6)
    return la.linear_act(gf.gated_ff(y, w1), w2, b2, residual=s)


def block64(x, r, nw, w1, w2, b2):
    s = x + r
    y = s * (s.square().mean(dim=-1, keepdim=True) + 1e-6).rsqrt() * nw
    g, up = (y @ w1.t()).chunk(2, dim=-1)
    return (g * torch.sigmoid(g) * up) @ w2.t() + b2 + s


def block_inputs(dtype, m=77, d=136, f=200):
    return [rand(*s, seed=i, dtype=dtype, scale=c) for i, (s, c) in enumerate([((m, d), 1), ((m, d), 1), ((d,), 1), ((2 * f, d), d ** -0.5), ((d, f), f ** -0.5), ((d,), 1)])]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_block_of_all_operators_trains_gpu(dtype):
    args = [t.requires_grad_(True) for t in block_inputs(dtype)]
    dy = rand(77, 136, seed=9, dtype=dtype)
    y = block(*args)
    exact = [t.detach().double().requires_grad_(True) for t in args]
    want = block64(*exact)
    # seven roundings on the way there (sum, norm, unit, result) and back (two operands, two gradients, the norm's): their relative errors add
    # up to at most 10 u in the 2-norm, since every step's linear map has been scaled to about one
    for got, ref in zip([y, *torch.autograd.grad(y, args, dy)], [want, *torch.autograd.grad(want, exact, dy.double())]):
        assert float((got.double() - ref).norm() / ref.norm()) <= 10 * tr.u(dtype) + 300 * tr.F32_ULP


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [1, 5, 200])
def test_block_of_all_operators_serves_in_8_bits_gpu(rows):
    x, r, nw, w1, w2, b2 = block_inputs(BF16, m=rows)
    (q1, s1), (q2, s2) = rn.quantize_rows(w1), rn.quantize_rows(w2)
    q, sq, s = rn.rms_norm(x, nw, residual=r, eps=1e-6, quantize=True)
    h = gf.gated_ff(q, q1, x_scale=sq, weight_scale=s1)
    qh, sh = rn.quantize_rows(h)
    y = la.linear_act(qh, q2, b2, residual=s, x_scale=sh, weight_scale=s2)
    # the same chain in 64 bits from the same 8-bit values, step by step
    val = lambda q, s: q.double() * s.double().unsqueeze(-1)  # noqa: E731
    g, up = (val(q, sq) @ val(q1, s1).t()).chunk(2, dim=-1)
    want = g * torch.sigmoid(g) * up
    assert float((h.double() - want).norm() / want.norm()) <= tr.u(BF16) + 300 * tr.F32_ULP
    want = val(qh, sh) @ val(q2, s2).t() + b2.double() + s.double()
    assert float((y.double() - want).norm() / want.norm()) <= tr.u(BF16) + 300 * tr.F32_ULP


@pytest.mark.gpu
def test_other_streams_and_captured_graphs_gpu():
    """Eager on a side stream, and two captured graphs (forward and backward) replayed in turn with eager work between, give the eager bits.
    No eager graph of the leaves is alive when a backward pass is captured: torch ties a leaf's accumulation node to the stream of the graph that
    made it, and a captured gradient that has to wait for that stream draws it into the capture."""
    args, other = ([t.requires_grad_(True) for t in block_inputs(BF16, m=m)] for m in (9, 130))
    dys = [rand(9, 136, seed=9, dtype=BF16), rand(130, 136, seed=10, dtype=BF16)]

    def step(a, dy):
        y = block(*a)
        return [y.detach(), *torch.autograd.grad(y, a, dy)]

    want = [[t.clone() for t in step(a, dy)] for a, dy in zip((args, other), dys)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(args, dys[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    del got
    graphs = []
    for a, dy in zip((args, other), dys):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(a, dy)
        graphs.append((g, out))
    for turn in range(3):
        for (g, out), ref in zip(graphs, want):
            for t in out:
                t.zero_()
            g.replay()
            eager = step(args, dys[0])
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, ref)), turn
            assert all(torch.equal(x, y) for x, y in zip(eager, want[0])), turn


@pytest.mark.gpu
def test_second_derivatives_are_refused_gpu():
    x, w = rand(3, 8, seed=1).requires_grad_(True), rand(4, 8, seed=2).requires_grad_(True)
    g, = torch.autograd.grad(la.linear_act(x, w, act='tanh').sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [5, 70, 300])
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('act,clamp', [('relu', None), ('relu', 2.0), ('lrelu', 0.25), ('swish', 0.25), ('tanh', 0.25)])
def test_infinite_gradients_where_none_passes_gpu(act, clamp, dtype, rows):
    # relu's lower side and what the clamp cut take no gradient at all, infinite or NaN ones neither. Sums are +-1 exactly: sum(x w) = s, |s| = 1.
    outer, inner = 72, 40
    x = torch.zeros(rows, inner)
    x[:, 0] = 1
    w = torch.zeros(outer, inner)
    w[:, 0] = torch.tensor([1.0, -1.0]).repeat(outer // 2)
    x, w = (t.to('cuda', dtype).requires_grad_() for t in (x, w))
    y = la.linear_act(x, w, act=act, gain=1.0, clamp=clamp)
    dy = torch.ones(rows, outer, device='cuda', dtype=dtype)
    cut = torch.zeros(outer, dtype=torch.bool)
    if act == 'relu':
        cut[1::2] = True                                   # sums of -1
    else:
        cut[0::2] = True                                   # 1, 0.73 and 0.76 are cut at 0.25; the lower side:
        cut[1::2] = act != 'lrelu'                         # -0.2 is not, -0.27 and -0.76 are
    dy[0, cut.cuda()] = torch.inf
    dy[-1, cut.cuda()] = torch.nan
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    # relu's upper side: slope 1 (1 is below the clamp of 2); lrelu's lower side: 0.2; nothing else passes
    slope = torch.zeros(outer, dtype=torch.float64)
    if act == 'relu':
        slope[0::2] = 1
    elif act == 'lrelu':
        slope[1::2] = 0.2
    want_x = torch.zeros(rows, inner, dtype=torch.float64)
    want_x[:, 0] = (slope * w.detach().double().cpu()[:, 0]).sum()
    want_w = torch.zeros(outer, inner, dtype=torch.float64)
    want_w[:, 0] = slope * rows
    # dz is rounded once (lrelu: 0.2), the sum of equal signs once more: two half steps; the float32 sums of up to 300 terms: 300 of theirs
    bound = 2 * torch.finfo(dtype).eps / 2 + 300 * 2.0 ** -24
    for got, want in ((dx, want_x), (dw, want_w)):
        assert ((got.double().cpu() - want).abs() <= bound * want.abs()).all()
