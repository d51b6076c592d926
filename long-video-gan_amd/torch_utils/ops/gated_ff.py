"""Gated feed-forward unit on token rows, both projections, the activation and the product in one kernel (csrc/token_gemm.h):

    h = gain * act(x wg^T + bg) * (x wu^T + bu),   weight = [wg; wu]

`linear_act` is the projection back behind it. GPU tensors run the HIP kernels, forward and backward (float32, float16, bfloat16), and the
8-bit product (e4m3, forward only); CPU tensors and impl='ref' run the plain-PyTorch definition."""

import torch

from . import _rows
from .bias_act import _resolve, activation_funcs
from .linear_act import SLOPE_SMOOTH, SLOPE_NONE, _backward, _check, _forward, _sums_ref, keep_operands


def gated_ff(x, weight, b=None, act='swish', alpha=None, gain=1.0, x_scale=None, weight_scale=None, out_dtype=None, impl='cuda'):
    r"""h = gain * act(x wg^T + bg) * (x wu^T + bu).

    Args:
        x:            rows [..., inner] in float32, float16, bfloat16 or float8_e4m3fn.
        weight:       [2 * outer, inner] in x's dtype: the gate's rows, then those of the up projection.
        b:            [2 * outer] in the result's dtype, in the same order, or None.
        act:          key of `bias_act.activation_funcs` for the gate; alpha its parameter (None = its default).
        gain:         scale of the result (1: unlike in `bias_act`, no activation brings its own).
        x_scale, weight_scale, out_dtype, impl: as in `linear_act`; weight_scale is [2 * outer].

    Returns [..., outer]. Differentiable once in x, weight and b (not with 8-bit operands), backward; a dual tensor of a forward derivative is
    refused. Sums are float32; the result is rounded once."""
    assert impl in ['ref', 'cuda']
    out_dtype = _check(x, weight, b, x_scale, weight_scale, out_dtype, halves=2)
    assert act in activation_funcs
    _, alpha, gain, _ = _resolve(act, alpha, gain, None)
    if impl == 'ref' or not x.is_cuda:
        return _gated_ff_ref(x, weight, b, act, alpha, gain, x_scale, weight_scale, out_dtype)
    if _rows.watched(x, weight, b):
        return _GatedFF.apply(x, weight, b, x_scale, weight_scale, act, alpha, gain, out_dtype)
    return _forward(x, weight, b, None, act, alpha, gain, -1.0, x_scale, weight_scale, out_dtype, True, SLOPE_NONE)[0]


def _gated_ff_ref(x, weight, b, act, alpha, gain, x_scale, weight_scale, out_dtype):
    """Definition of the op in stock PyTorch ops (CPU path and impl='ref')."""
    gate, up = _sums_ref(x, weight, b, x_scale, weight_scale).chunk(2, dim=-1)
    return (activation_funcs[act].func(gate, alpha=alpha) * gain * up).to(out_dtype)


class _GatedFF(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, b, x_scale, weight_scale, act, alpha, gain, out_dtype):
        kind = SLOPE_SMOOTH if any(ctx.needs_input_grad[:3]) and x_scale is None else SLOPE_NONE
        h, slopes = _forward(x, weight, b, None, act, alpha, gain, -1.0, x_scale, weight_scale, out_dtype, True, kind)
        keep_operands(ctx, x, weight, slopes)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, slopes = ctx.saved_tensors
        # (the gain is in the slopes)
        return _backward(dy, x, weight, slopes, ctx.inner, SLOPE_SMOOTH, 2, 0.0, 1.0, *ctx.needs_input_grad[:3]) + (None,) * 6
