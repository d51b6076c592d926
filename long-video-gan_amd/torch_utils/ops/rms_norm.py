"""Root-mean-square norm of token rows with the residual's addition, and 8-bit rows with one scale each (csrc/rms_norm.hip):

    s = x + residual,   y = weight * s / sqrt(mean(s^2) + eps)
    q = y / scale in e4m3,   scale = max |y| of the row / 448

Without weight and residual it is what the mapping networks do to their input in tensor expressions (reference
model/generator_lres.py:444, LatentMappingNetwork). GPU tensors run the HIP kernels, CPU tensors and impl='ref' the plain-PyTorch definition."""

import torch

from . import _rows


def rms_norm(x, weight=None, residual=None, eps=1e-8, quantize=False, impl='cuda'):
    r"""y = weight * s / sqrt(mean(s^2) + eps), s = x + residual, over the last dimension.

    Args:
        x:        rows [..., width] in float32, float16 or bfloat16.
        weight:   [width] in x's dtype, or None (= 1).
        residual: x's shape and dtype, or None.
        eps:      added to the mean square.
        quantize: return y as float8_e4m3fn rows and their scales.
        impl:     'cuda' (HIP kernels when x is on the GPU) or 'ref' (plain PyTorch).

    Returns y; with quantize (q, scale), scale float32 [...]; with a residual also s (rounded to x's dtype) behind them. The norm is taken of
    the sum before that rounding. Differentiable once in x, weight and residual, through y and s, backward (a dual
    tensor of a forward derivative is refused); not with quantize."""
    assert impl in ['ref', 'cuda']
    assert isinstance(x, torch.Tensor) and x.ndim >= 1 and x.shape[-1] >= 1 and x.dtype in _rows.ROW_DTYPES
    assert eps >= 0
    if weight is not None:
        assert weight.shape == x.shape[-1:] and weight.dtype == x.dtype and weight.device == x.device
    if residual is not None:
        assert residual.shape == x.shape and residual.dtype == x.dtype and residual.device == x.device
    assert not (quantize and _rows.wants_grad(x, weight, residual)), '8-bit rows have no gradient'
    if impl == 'ref' or not x.is_cuda:
        out = _rms_norm_ref(x, weight, residual, eps, quantize)
    elif _rows.watched(x, weight, residual):
        out = _RmsNorm.apply(x, weight, residual, eps, quantize)
    else:
        y, scale, total, _, _ = _forward(x, weight, residual, eps, quantize, False)
        out = tuple(t for t in (y, scale, total) if t is not None)
    return out[0] if len(out) == 1 else out


def quantize_rows(x, impl='cuda'):
    """(q, scale): x [..., width] as float8_e4m3fn rows and float32 scales [...], x = q * scale; scale = max |x| of the row / 448, at least 2^-64.
    A row with a NaN has a NaN scale. For float32, float16 and bfloat16; no gradient."""
    assert impl in ['ref', 'cuda']
    assert isinstance(x, torch.Tensor) and x.ndim >= 1 and x.shape[-1] >= 1 and x.dtype in _rows.ROW_DTYPES
    assert not _rows.wants_grad(x), '8-bit rows have no gradient'
    if impl == 'ref' or not x.is_cuda:
        return _quantize_ref(x.float())
    return _QuantizeRows.apply(x) if _rows.watched() else _quantize(x)


def _quantize_ref(v):
    top = v.abs().amax(dim=-1)
    scale = (top / top.new_full((), _rows.E4M3_MAX)).clamp(min=_rows.SCALE_MIN)         # (a tensor: torch multiplies by a number's reciprocal on the GPU)
    return (v / scale.unsqueeze(-1)).clamp(-_rows.E4M3_MAX, _rows.E4M3_MAX).to(torch.float8_e4m3fn), scale


def _rms_norm_ref(x, weight, residual, eps, quantize):
    """Definition of the op in stock PyTorch ops (CPU path and impl='ref')."""
    s = x.float()
    if residual is not None:
        s = s + residual.float()
    y = s / torch.sqrt(s.square().mean(dim=-1, keepdim=True) + eps)        # (rsqrt's gradient forms a cube that leaves float32's range)
    if weight is not None:
        y = y * weight.float()
    out = _quantize_ref(y) if quantize else (y.to(x.dtype),)
    return out if residual is None else out + (s.to(x.dtype),)


#----------------------------------------------------------------------------
# HIP path.

def _forward(x, weight, residual, eps, quantize, keep):
    """(y or q, scale or None, s or None, rstd or None, rest or None) on x's device and the current stream; keep: for a backward pass, with the
    reciprocal roots and what the 16-bit sum lost in its rounding."""
    width = x.shape[-1]
    y = torch.empty_like(x, dtype=torch.float8_e4m3fn if quantize else x.dtype, memory_format=torch.contiguous_format)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32) if quantize else None
    total = torch.empty_like(x, memory_format=torch.contiguous_format) if residual is not None else None
    x2 = _rows.rows_of(x, width)
    rows = x2.shape[0]
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if keep else None
    rest = torch.empty((rows, -(-width // 8)), dtype=torch.int16, device=x.device) if keep and total is not None and x.dtype != torch.float32 else None
    if rows:
        r2 = None if residual is None else _rows.rows_of(residual, width)
        if weight is not None:
            weight = weight.contiguous()
        _rows.launch(x.device, 'lvg_rms_norm', x2.data_ptr(), None if r2 is None else r2.data_ptr(), None if weight is None else weight.data_ptr(), y.data_ptr(),
                     None if total is None else total.data_ptr(), None if rest is None else rest.data_ptr(), None if rstd is None else rstd.data_ptr(), None if scale is None else scale.data_ptr(),
                     rows, width, _rows.row_stride(x2), 0 if r2 is None else _rows.row_stride(r2), eps, _rows.type_code(x.dtype), int(quantize))
    return y, scale, total, rstd, rest


def _quantize(x):
    width = x.shape[-1]
    q = torch.empty_like(x, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    x2 = _rows.rows_of(x, width)
    if x2.shape[0]:
        _rows.launch(x.device, 'lvg_quantize_rows', x2.data_ptr(), q.data_ptr(), scale.data_ptr(), x2.shape[0], width, _rows.row_stride(x2), _rows.type_code(x.dtype))
    return q, scale


class _QuantizeRows(torch.autograd.Function):
    """For calls that are watched (see _rows.watched); rows that ask for a gradient have been refused."""
    @staticmethod
    def forward(ctx, x):
        return _quantize(x)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, quantize):
        keep = any(ctx.needs_input_grad) and not quantize
        y, scale, total, rstd, rest = _forward(x, weight, residual, eps, quantize, keep)
        ctx.set_materialize_grads(False)
        if keep:
            need_weight = ctx.needs_input_grad[0] or ctx.needs_input_grad[2]
            ctx.save_for_backward(x if total is None else total, weight if need_weight else None, rstd, rest)
        return tuple(t for t in (y, scale, total) if t is not None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds=None):
        s, weight, rstd, rest = ctx.saved_tensors
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        dw = None
        if dy is None:
            # only the sum was used
            dx = ds
            if need_w:
                dw = s.new_zeros(s.shape[-1])
        else:
            width = s.shape[-1]
            s2, dy2 = _rows.rows_of(s, width), _rows.rows_of(dy, width)
            ds2 = None if ds is None else _rows.rows_of(ds, width)
            rows, dev = s2.shape[0], s.device
            dx = torch.empty(s.shape, dtype=s.dtype, device=dev)
            code = _rows.type_code(s.dtype)
            if need_w:
                dw = torch.empty(width, dtype=s.dtype, device=dev)
            size = _rows.query('lvg_rms_norm_backward_work', rows, width, int(need_w), code)
            work = _rows.work_of(size, dev)
            if weight is not None:
                weight = weight.contiguous()
            _rows.launch(dev, 'lvg_rms_norm_backward', dy2.data_ptr(), None if ds2 is None else ds2.data_ptr(), s2.data_ptr(), None if rest is None else rest.data_ptr(),
                         None if weight is None else weight.data_ptr(), rstd.data_ptr(), dx.data_ptr(), None if dw is None else dw.data_ptr(), None if work is None else work.data_ptr(), size, rows, width,
                         _rows.row_stride(dy2), 0 if ds2 is None else _rows.row_stride(ds2), _rows.row_stride(s2), code)
        return dx if need_x else None, dw, dx if need_r else None, None, None
