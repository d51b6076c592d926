"""Dense layer on token rows with everything behind the product in its epilogue (csrc/token_gemm.h):

    y = clamp(act(x w^T + b) * gain) + residual

the dense counterpart of the convolutions' fused epilogues, with the activations of `bias_act` (the networks' own dense layers are
torch.addmm, or a product and `bias_act`). GPU tensors run the HIP kernels, forward and backward (float32, float16,
bfloat16), and the 8-bit product (e4m3 rows and weights with one scale a row, forward only); CPU tensors and impl='ref' run the
plain-PyTorch definition."""

import torch

from . import _rows
from .bias_act import _resolve, activation_funcs

SLOPE_NONE, SLOPE_SMOOTH, SLOPE_CODE = 0, 1, 2


def linear_act(x, weight, b=None, residual=None, act='linear', alpha=None, gain=None, clamp=None, x_scale=None, weight_scale=None,
               out_dtype=None, impl='cuda'):
    r"""y = clamp(act(x w^T + b) * gain) + residual.

    Args:
        x:            rows [..., inner] in float32, float16, bfloat16 or float8_e4m3fn. Any strides; rows with unit element stride that start
                      at multiples of 16 bytes are fastest.
        weight:       [outer, inner] in x's dtype.
        b:            [outer] in the result's dtype, or None.
        residual:     [..., outer] in the result's dtype, added last, or None.
        act:          key of `bias_act.activation_funcs`; alpha, gain, clamp as in `bias_act` (None = the activation's default / no clamp). As in its
                      kernel, a value that lies on the clamp exactly passes no gradient (the plain form, torch.clamp, passes it).
        x_scale:      8-bit x only: float32 [...], the value of an element is itself times its row's scale.
        weight_scale: 8-bit x only: float32 [outer], likewise for the rows of the weight.
        out_dtype:    dtype of the result: x's, or for 8-bit x float16 or bfloat16 (default bfloat16).
        impl:         'cuda' (HIP kernels when x is on the GPU) or 'ref' (plain PyTorch).

    Differentiable once in x, weight, b and residual (not with 8-bit operands), backward; a dual tensor of a forward derivative is refused. Sums are
    float32 (8-bit operands: the matrix unit adds the products of eight neighbours with 13 bits below the largest of them, these sums are float32);
    the result is rounded once. A backward pass that is captured into a graph needs leaves that no eager autograd graph still holds (torch ties a
    leaf's accumulation node to the stream of the graph that made it): drop eager results, or detach them, before the capture."""
    assert impl in ['ref', 'cuda']
    out_dtype = _check(x, weight, b, x_scale, weight_scale, out_dtype, halves=1)
    if residual is not None:
        assert residual.shape == (*x.shape[:-1], weight.shape[0]) and residual.dtype == out_dtype and residual.device == x.device
        _no_grad_with_8bit(x, residual)
    assert act in activation_funcs
    _, alpha, gain, clamp = _resolve(act, alpha, gain, clamp)
    if impl == 'ref' or not x.is_cuda:
        return _linear_act_ref(x, weight, b, residual, act, alpha, gain, clamp, x_scale, weight_scale, out_dtype)
    if _rows.watched(x, weight, b, residual):
        return _LinearAct.apply(x, weight, b, residual, x_scale, weight_scale, act, alpha, gain, clamp, out_dtype)
    return _forward(x, weight, b, residual, act, alpha, gain, clamp, x_scale, weight_scale, out_dtype, False, SLOPE_NONE)[0]


def _no_grad_with_8bit(x, *others):
    assert x.dtype != torch.float8_e4m3fn or not _rows.wants_grad(*others), 'the product of 8-bit rows has no gradient'


def _check(x, weight, b, x_scale, weight_scale, out_dtype, halves):
    """Checks what the dense products share; returns the result's dtype. halves: 2 = the weight holds two projections."""
    assert isinstance(x, torch.Tensor) and isinstance(weight, torch.Tensor)
    assert x.ndim >= 1 and weight.ndim == 2, 'x holds rows, weight is a matrix'
    dtype, device, (total, inner) = x.dtype, x.device, weight.shape
    assert x.shape[-1] == inner and total % halves == 0, f'rows of {tuple(x.shape)} do not fit a weight of {tuple(weight.shape)}'
    assert weight.dtype == dtype and weight.device == device
    if dtype == torch.float8_e4m3fn:
        out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
        assert out_dtype in (torch.float16, torch.bfloat16), '8-bit operands give a float16 or bfloat16 result'
        assert x_scale is not None and weight_scale is not None, '8-bit operands come with their scales'
        assert x_scale.dtype == weight_scale.dtype == torch.float32 and x_scale.device == weight_scale.device == device
        assert x_scale.shape == x.shape[:-1] and weight_scale.shape == (total,)
        _no_grad_with_8bit(x, x, weight, b, x_scale, weight_scale)
    else:
        assert dtype in _rows.ROW_DTYPES, f'dtype {dtype} is not supported'
        assert out_dtype is None or out_dtype == dtype, 'the result has the operands\' dtype'
        assert x_scale is None and weight_scale is None, 'scales belong to 8-bit operands'
        out_dtype = dtype
    if b is not None:
        assert b.shape == (total,) and b.dtype == out_dtype and b.device == device
    return out_dtype


def _sums_ref(x, weight, b, x_scale, weight_scale):
    """x w^T + b, 16-bit and 8-bit operands in float32."""
    x, weight = x.float(), weight.float()
    if x_scale is not None:
        x, weight = x * x_scale.unsqueeze(-1), weight * weight_scale.unsqueeze(-1)
    return torch.nn.functional.linear(x, weight, None if b is None else b.float())


def _linear_act_ref(x, weight, b, residual, act, alpha, gain, clamp, x_scale, weight_scale, out_dtype):
    """Definition of the op in stock PyTorch ops (CPU path and impl='ref')."""
    y = activation_funcs[act].func(_sums_ref(x, weight, b, x_scale, weight_scale), alpha=alpha) * gain
    if clamp >= 0:
        y = y.clamp(-clamp, clamp)
    if residual is not None:
        y = y + residual.float()
    return y.to(out_dtype)


#----------------------------------------------------------------------------
# HIP path.

def slope_kind(act, gated):
    """How the forward pass keeps the derivative: piecewise linear activations as one byte an element, smooth ones as values."""
    return SLOPE_CODE if not gated and act in ('linear', 'relu', 'lrelu') else SLOPE_SMOOTH


def _forward(x, weight, b, residual, act, alpha, gain, clamp, x_scale, weight_scale, out_dtype, gated, kind):
    """One product on x's device and the current stream: (y, slopes or None)."""
    total, inner = weight.shape
    outer = total // 2 if gated else total
    device = x.device
    x2, w2 = _rows.rows_of(x, inner), _rows.rows_of(weight, inner)
    rows = x2.shape[0]
    y = x.new_empty((rows, outer) if x.ndim == 2 else (*x.shape[:-1], outer), dtype=out_dtype)
    slopes = None
    if kind != SLOPE_NONE:
        slopes = _rows.work_of(_rows.query('lvg_linear_slope_bytes', rows, outer, total // outer if outer else 1, kind, _rows.type_code(x.dtype)), device)
    if rows == 0 or outer == 0:
        return y, slopes
    r2 = None if residual is None else _rows.rows_of(residual, outer)
    if b is not None:
        b = b.contiguous()
    if x_scale is not None:
        x_scale, weight_scale = x_scale.contiguous(), weight_scale.contiguous()
    code = _rows.type_code(x.dtype)
    size = _rows.query('lvg_linear_act_work', rows, outer, inner, code, int(gated))
    work = _rows.work_of(size, device)
    _rows.launch(device, 'lvg_linear_act',
                 x2.data_ptr(), w2.data_ptr(), None if b is None else b.data_ptr(), None if r2 is None else r2.data_ptr(),
                 None if x_scale is None else x_scale.data_ptr(), None if x_scale is None else weight_scale.data_ptr(), y.data_ptr(),
                 None if slopes is None else slopes.data_ptr(), None if work is None else work.data_ptr(), size,
                 rows, outer, inner, _rows.row_stride(x2), _rows.row_stride(w2), 0 if r2 is None else _rows.row_stride(r2), outer,
                 code, _rows.type_code(out_dtype), int(gated), activation_funcs[act].cuda_idx, kind, alpha, gain, clamp)
    return y, slopes


def keep_operands(ctx, x, weight, slopes):
    """Saves what the gradients asked for read: the rows for the weight's, the weight for the rows'."""
    need_x, need_w = ctx.needs_input_grad[:2]
    ctx.save_for_backward(x if need_w else None, weight if need_x else None, slopes)
    ctx.inner = weight.shape[1]


def _backward(dy, x, weight, slopes, inner, kind, halves, alpha, gain, need_x, need_w, need_b):
    """Gradients of x, weight and b from dy [..., outer]; kind SLOPE_NONE: dy itself times the gain is the gradient of the sums. x and weight as
    keep_operands saves them."""
    outer = dy.shape[-1]
    total = outer * halves
    dy2 = _rows.rows_of(dy, outer)
    x2, w2 = (None if t is None else _rows.rows_of(t, inner) for t in (x, weight))
    rows, device = dy2.shape[0], dy.device
    dx = dy2.new_empty((*dy.shape[:-1], inner)) if need_x else None
    dw = dy2.new_empty((total, inner)) if need_w else None
    db = dy2.new_empty(total) if need_b else None
    code = _rows.type_code(dy.dtype)
    size = _rows.query('lvg_linear_backward_work', rows, outer, inner, halves, kind, need_x + 2 * need_w + 4 * need_b, code)
    work = _rows.work_of(size, device)
    _rows.launch(device, 'lvg_linear_backward', dy2.data_ptr(), None if slopes is None else slopes.data_ptr(),
                 None if x2 is None else x2.data_ptr(), None if w2 is None else w2.data_ptr(),
                 None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(),
                 None if work is None else work.data_ptr(), size, rows, outer, inner, _rows.row_stride(dy2),
                 0 if x2 is None else _rows.row_stride(x2), 0 if w2 is None else _rows.row_stride(w2), halves, kind, alpha, gain, code)
    return dx, dw, db


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, b, residual, x_scale, weight_scale, act, alpha, gain, clamp, out_dtype):
        needed = any(ctx.needs_input_grad[:3]) and x_scale is None         # (set for leaves under no_grad too)
        kind = slope_kind(act, False) if needed and (act != 'linear' or clamp >= 0) else SLOPE_NONE
        y, slopes = _forward(x, weight, b, residual, act, alpha, gain, clamp, x_scale, weight_scale, out_dtype, False, kind)
        keep_operands(ctx, x, weight, slopes)
        ctx.args = kind, 1, alpha, gain
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, slopes = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            dx, dw, db = _backward(dy, x, weight, slopes, ctx.inner, *ctx.args, *need[:3])
        return (dx, dw, db, dy if need[3] else None) + (None,) * 7
