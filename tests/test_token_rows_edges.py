"""Operators on token rows at the edges of what their documentation allows: values far from one, infinite gradients, derivative and trace modes that
pass an autograd function by, sizes near the limits of a launch, what a backward pass keeps and allocates. Bounds as in tests/helpers/token_rows.py."""

import math
import os
import subprocess
import sys

import pytest
import torch
import torch.autograd.forward_ad as fwad

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), 'helpers'))
import token_rows as tr  # noqa: E402
from test_token_rows import check_norm, rand  # noqa: E402

from torch_utils.ops import _hip
from torch_utils.ops import gated_ff as gf
from torch_utils.ops import linear_act as la
from torch_utils.ops import rms_norm as rn

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
DTYPES = [F32, F16, BF16]
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'long-video-gan_amd', 'csrc')


# --------------------------------------------------------------------------------------------------------------------
# 8-bit rows.

def same_bits(a, b):
    return torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', [(300, 5), (300, 64), (7, 515), (64, 4100), (64, 8192), (5, 40000)])
def test_8bit_rows_are_the_quotients_gpu(shape, dtype):
    """q = x / scale, one rounding of the float32 quotient: the plain form's bits, on either device. Values of 16 bits meet e4m3's ties often."""
    size = torch.exp(0.4 * torch.randn(shape[1], generator=torch.Generator().manual_seed(2)))
    x = (rand(*shape, seed=1, device='cpu') * size).to(dtype).cuda()
    q, scale = rn.quantize_rows(x)
    for want_q, want_scale in (rn.quantize_rows(x.cpu()), rn.quantize_rows(x, impl='ref')):
        assert torch.equal(scale.cpu(), want_scale.cpu())
        assert same_bits(q, want_q)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('width', [64, 515, 4100, 8192, 40000])
def test_8bit_norm_rows_are_the_quotients_gpu(width, dtype):
    """Rows of +-1 have a mean square of exactly one, so the norm to 8 bits is the weight with their signs, to 8 bits."""
    w = rand(width, seed=1, dtype=dtype)
    x = torch.where(rand(9, width, seed=2) > 0, 1.0, -1.0).to(dtype)
    q, scale = rn.rms_norm(x, w, eps=0.0, quantize=True)
    want_q, want_scale = rn.quantize_rows((x.float() * w.float()).cpu())
    assert torch.equal(scale.cpu(), want_scale) and same_bits(q, want_q)


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [5, 70])
@pytest.mark.parametrize('sx,sw,value,count', [(1.15625 * 2.0 ** -72, 1.15625 * 2.0 ** -72, 256.0, 64), (2.0 ** 40, 2.0 ** 100, 2.0 ** -9, 1), (2.0 ** 110, 2.0 ** -60, 256.0, 64),
                                               (2.0 ** -60, 2.0 ** 110, 256.0, 64)])
def test_8bit_products_with_scales_far_from_one_gpu(rows, sx, sw, value, count):
    """Results in range come out right where the product of the two scales, or of one of them and the sum, leaves float32's range; a sum of zero stays
    zero. Sums are exact, the scales' two products rounded once each, and the result."""
    inner, outer = 64, 48
    x, w = torch.zeros(rows, inner), torch.zeros(2 * outer, inner)
    x[:, :count], w[:, :count] = value, value
    x[1] = 0
    q, qw, s = x.to(E4M3).cuda(), w.to(E4M3).cuda(), torch.full((rows,), sx, device='cuda')
    v = (x.double() @ w.double().t()).cuda()
    g = v[:, :outer] * (sx * sw)
    tr.assert_within(la.linear_act(q, qw[:outer], x_scale=s, weight_scale=torch.full((outer,), sw, device='cuda')), g, tr.rounded(g, 2 * tr.F32_ULP * g.abs(), BF16), 'y')
    su = 2.0 ** -round(math.log2(float(v.max()) * sx))           # the up half is about one
    h = gf.gated_ff(q, qw, act='linear', x_scale=s, weight_scale=torch.tensor([sw, su]).repeat_interleave(outer).cuda())
    want = g * v[:, outer:] * (sx * su)
    tr.assert_within(h, want, tr.rounded(want, 6 * tr.F32_ULP * want.abs(), BF16), 'h')


# --------------------------------------------------------------------------------------------------------------------
# Norm of rows far from one.

@pytest.mark.parametrize('size', [1e15, 1e-15])
def test_plain_norm_gradient_of_rows_far_from_one_cpu(size):
    x, w, r, dy = (rand(*s, seed=i, device='cpu') for i, s in enumerate([(4, 9), (9,), (4, 9), (4, 9)]))
    check_norm(x * size, w, r * size, eps=0.0, dy=dy)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('size', [1e15, 1e-15])
@pytest.mark.parametrize('shape', [(9, 70), (5, 515), (9, 2500), (7, 8200), (3, 40000)])
def test_norm_gradient_of_rows_far_from_one_gpu(shape, size, dtype):
    """The cube of the reciprocal root leaves float32's range long before the gradient does."""
    x, w, r, dy = (rand(*s, seed=i) for i, s in enumerate([shape, shape[-1:], shape, shape]))
    x, r = (x * size).to(dtype), (r * size).to(dtype)
    check_norm(x.clone(), w.to(dtype), r, eps=0.0, dy=dy.to(dtype))
    check_norm(x.clone(), None, None, eps=0.0, dy=dy.to(dtype))


# --------------------------------------------------------------------------------------------------------------------
# Gradients that no derivative lets through, and those that one of zero does not stop.

@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', [5, 70, 300])
def test_infinite_gradients_at_a_gates_lower_side_gpu(rows, dtype):
    """relu's lower side passes no gradient to the gate, infinite or NaN ones neither. All sums are +-1 exactly."""
    outer, inner = 72, 40
    x, w = torch.zeros(rows, inner), torch.zeros(2 * outer, inner)
    x[:, 0] = 1
    w[:outer, 0] = torch.tensor([1.0, -1.0]).repeat(outer // 2)
    w[outer:, 0] = 1
    x, w, b = (t.to('cuda', dtype).requires_grad_() for t in (x, w, torch.zeros(2 * outer)))
    dy = torch.ones(rows, outer, device='cuda', dtype=dtype)
    dy[0, 1::2] = torch.inf
    dy[-1, 1::2] = torch.nan
    dw, db = torch.autograd.grad(gf.gated_ff(x, w, b, act='relu'), (w, b), dy)
    want = torch.zeros(outer, dtype=dtype, device='cuda')
    want[0::2] = rows
    assert torch.equal(db[:outer], want) and torch.equal(dw[:outer, 0], want) and not dw[:outer, 1:].any()
    # the up projection's derivative is act = 0 there, and 0 times infinity is no number
    assert bool(db[outer + 1::2].isnan().all()) and torch.equal(db[outer::2], want[0::2])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', [5, 70])
def test_nan_gradients_pass_a_derivative_of_zero_gpu(rows, dtype):
    """Where nothing is cut a NaN gradient stays one, also where the derivative has become zero (swish of -200)."""
    outer, inner = 8, 40
    x, w = torch.zeros(rows, inner), torch.zeros(2 * outer, inner)
    x[:, 0] = 1
    w[:outer, 0] = -200
    w[outer:, 0] = 1
    x, w = (t.to('cuda', dtype).requires_grad_() for t in (x, w))
    for y in (la.linear_act(x, w[:outer], act='swish'), la.linear_act(x, w[:outer], act='swish', clamp=1.0), gf.gated_ff(x, w)):
        dy = torch.ones_like(y)
        dy[2, 3] = torch.nan
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        assert bool(dx[2, 0].isnan()) and bool(dw[3, 0].isnan())
        assert bool(torch.isfinite(dx[3:]).all()) and bool(torch.isfinite(dw[4:outer]).all())


# --------------------------------------------------------------------------------------------------------------------
# Modes that watch tensors' operations.

def every_operator(device):
    """(name, function of one float tensor [6, 64], that tensor) for each operator's form without gradients."""
    w, r, nw = rand(80, 64, seed=2, device=device, scale=0.125), rand(6, 80, seed=3, device=device), rand(64, seed=4, device=device)
    return [('linear', lambda x: la.linear_act(x, w, residual=r, act='swish')),
            ('gated', lambda x: gf.gated_ff(x, w)),
            ('norm', lambda x: rn.rms_norm(x, nw)),
            ('norm and sum', lambda x: rn.rms_norm(x, nw, residual=x)),
            ('norm to 8 bits', lambda x: rn.rms_norm(x, nw, residual=x, quantize=True)),
            ('8 bits', rn.quantize_rows)], rand(6, 64, seed=1, device=device)


def test_forward_derivatives_of_the_plain_forms_cpu():
    calls, x = every_operator('cpu')
    with fwad.dual_level():
        for name, call in calls[:4]:
            out = call(fwad.make_dual(x, torch.ones_like(x)))
            assert fwad.unpack_dual(out[0] if isinstance(out, tuple) else out).tangent is not None, name


@pytest.mark.gpu
def test_forward_derivatives_are_refused_gpu():
    """The kernels have no forward derivative: a dual tensor is refused, never taken for its value alone."""
    calls, x = every_operator('cuda')
    with fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones_like(x))
        for name, call in calls:
            for grads in (True, False):
                with torch.set_grad_enabled(grads), pytest.raises(NotImplementedError):
                    call(dual)
                    pytest.fail(name)
        w = rand(80, 64, seed=2)
        with pytest.raises(NotImplementedError):
            la.linear_act(x, fwad.make_dual(w, torch.ones_like(w)))
    q, s = rn.quantize_rows(x)
    qw, sw = rn.quantize_rows(w)
    with fwad.dual_level():
        for op in (la.linear_act, gf.gated_ff):
            with pytest.raises(NotImplementedError):
                op(q, qw, x_scale=fwad.make_dual(s, torch.ones_like(s)), weight_scale=sw)
    # calls without a dual tensor go on while one is about, with leaves under no_grad too
    b, nw = rand(80, seed=5, dtype=BF16).requires_grad_(True), rand(64, seed=4).requires_grad_(True)
    with torch.no_grad():
        plain = [lambda: la.linear_act(q, qw, b, x_scale=s, weight_scale=sw), lambda: gf.gated_ff(q, qw, b, x_scale=s, weight_scale=sw),
                 lambda: rn.rms_norm(x, nw, quantize=True)[1], lambda: rn.rms_norm(x, nw), lambda: gf.gated_ff(x, w.requires_grad_(True))]
        want = [call() for call in plain]
        with fwad.dual_level():
            assert all(torch.equal(call(), t) for call, t in zip(plain, want))


@pytest.mark.gpu
def test_traced_calls_run_the_kernels_gpu():
    calls, x = every_operator('cuda')
    other = rand(6, 64, seed=9)
    q, s = rn.quantize_rows(x)
    qw, sw = rn.quantize_rows(rand(80, 64, seed=2))
    calls.append(('8-bit linear', lambda x: la.linear_act(q, qw, x_scale=s * x[:, 0].abs(), weight_scale=sw)))
    calls.append(('8-bit gated', lambda x: gf.gated_ff(q, qw, x_scale=s * x[:, 0].abs(), weight_scale=sw)))
    for name, call in calls:
        traced = torch.jit.trace(call, (x,), check_trace=False)
        for t in (other, x):
            got, want = traced(t), call(t)
            for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                assert same_bits(a.contiguous(), b.contiguous()), name


# --------------------------------------------------------------------------------------------------------------------
# What a backward pass keeps, allocates and does.

@pytest.mark.gpu
@pytest.mark.parametrize('op', ['linear', 'gated'])
def test_operands_a_gradient_does_not_need_are_not_kept_gpu(op):
    """A frozen weight's rows may change in place before the backward pass, rows without a gradient let the weight change."""
    call = (lambda x, w: la.linear_act(x, w, act='swish')) if op == 'linear' else gf.gated_ff
    base, w = rand(9, 64, seed=1).requires_grad_(True), rand(80, 64, seed=2, scale=0.125)
    want, = torch.autograd.grad(call(base, w).sum(), base)
    hidden = base * 1
    y = call(hidden, w).sum()
    with torch.no_grad():
        hidden.mul_(2)
    assert torch.equal(torch.autograd.grad(y, base)[0], want)
    x, leaf = base.detach(), w.clone().requires_grad_(True)
    want, = torch.autograd.grad(call(x, leaf).sum(), leaf)
    y = call(x, leaf).sum()
    with torch.no_grad():
        leaf.zero_()
    assert torch.equal(torch.autograd.grad(y, leaf)[0], want)


@pytest.mark.gpu
def test_a_norm_weight_may_change_before_its_own_gradient_gpu():
    x, r, dy = (rand(9, 70, seed=i) for i in range(3))
    w = rand(70, seed=3).requires_grad_(True)
    want, = torch.autograd.grad(rn.rms_norm(x, w, residual=r)[0], w, dy)
    y, total = rn.rms_norm(x, w, residual=r)
    with torch.no_grad():
        w.zero_()
    assert torch.equal(torch.autograd.grad(y, w, dy, retain_graph=True)[0], want)
    assert not torch.autograd.grad(total, w, dy)[0].any()


def test_a_bias_gradient_alone_takes_its_column_sums_alone_cpu():
    lib = _hip.lib()
    for dtype, size in ((0, 4), (2, 2)):
        rows, outer = 5000, 512
        alone, with_dz = (lib.lvg_linear_backward_work(rows, outer, 64, 1, 1, grads, dtype) for grads in (4, 5))
        assert 0 < alone < rows * outer * size <= with_dz


@pytest.mark.gpu
@pytest.mark.parametrize('act', ['linear', 'lrelu', 'swish'])
def test_a_bias_gradient_alone_gpu(act):
    x, w, b, dy = rand(700, 64, seed=1, dtype=BF16), rand(90, 64, seed=2, dtype=BF16, scale=0.125), rand(90, seed=3, dtype=BF16), rand(700, 90, seed=4, dtype=BF16)
    b.requires_grad_(True)
    alone, = torch.autograd.grad(la.linear_act(x, w, b, act=act), b, dy)
    x.requires_grad_(True)
    assert torch.equal(alone, torch.autograd.grad(la.linear_act(x, w, b, act=act), (b, x), dy)[0])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('size', [(1100, 771, 515), (1100, 768, 515), (1100, 771, 512), (3000, 1501, 1003), (40, 129, 9001)])
def test_linear_layers_of_odd_widths_train_gpu(size, dtype):
    from test_token_rows import check_linear
    m, k, n = size
    check_linear(rand(m, k, seed=1, dtype=dtype), rand(n, k, seed=2, dtype=dtype, scale=k ** -0.5), rand(n, seed=3, dtype=dtype), None, dy=rand(m, n, seed=5, dtype=dtype))


# --------------------------------------------------------------------------------------------------------------------
# Sizes near the limits of a launch.

def test_repacking_is_not_planned_past_one_launch_cpu():
    """Operands in odd rows that are too many for one repacking launch go through registers: the workspace holds no copy of them."""
    assert _hip.lib().lvg_linear_act_work(1 << 22, 4096, 4097, 2, 0) < 1 << 32


@pytest.mark.gpu
def test_more_tiles_than_two_to_the_22nd_gpu():
    rows = (1 << 28) + 64
    x = torch.zeros(rows, 8, dtype=BF16, device='cuda')
    x[-300:] = rand(300, 8, seed=1, dtype=BF16)
    w = rand(1, 8, seed=2, dtype=BF16)
    y = la.linear_act(x, w)
    assert torch.equal(y[-300:], la.linear_act(x[-300:].clone(), w)) and not y[:-300].any()


@pytest.mark.gpu
def test_more_columns_than_two_to_the_26th_gpu():
    outer = (1 << 26) + 24
    x = rand(1, 8, seed=1, dtype=BF16)
    w = torch.zeros(outer, 8, dtype=BF16, device='cuda')
    w[-300:] = rand(300, 8, seed=2, dtype=BF16)
    y = la.linear_act(x, w)
    v, off = tr.sums64(x, w[-300:], None)
    tr.assert_within(y[:, -300:], v, tr.rounded(v, off, BF16), 'y')
    assert not y[:, :-300].any()


# --------------------------------------------------------------------------------------------------------------------
# Build.

def test_objects_depend_on_the_makefile_cpu():
    """Compiler flags stand in the Makefile: a change to it rebuilds every object."""
    plan = subprocess.run(['make', '-n', '-W', 'Makefile', '-C', CSRC], capture_output=True, text=True, check=True).stdout
    for name in os.listdir(CSRC):
        if name.endswith('.hip'):
            assert f'-c {name} ' in plan, name
