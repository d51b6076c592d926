"""What the operators on matrices of token rows (linear_act, gated_ff, rms_norm) share: views of a tensor as rows, and types."""

import math

import torch

from . import _hip

E4M3 = 4                                                   # LVG_E4M3 of the C ABI
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -64
ROW_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def rows_of(t: torch.Tensor, width: int) -> torch.Tensor:
    """[..., width] -> [rows, width] with unit element stride: a view where the strides allow it, a copy otherwise."""
    t = t.reshape(math.prod(t.shape[:-1]), width)
    return t if t.stride(1) == 1 or width <= 1 else t.contiguous()


def row_stride(t: torch.Tensor) -> int:
    """Elements between the rows of a 2-D tensor; strides of a single row mean nothing."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def type_code(dtype: torch.dtype) -> int:
    return E4M3 if dtype == torch.float8_e4m3fn else _hip.dtype_code(dtype)


def wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def work_of(size: int, device: torch.device):
    """Workspace of a call, from the current stream's pool (a captured graph gets its own)."""
    return torch.empty(size, dtype=torch.uint8, device=device) if size > 0 else None


def column_sum(part: torch.Tensor, dtype: torch.dtype, gain: float = 1.0) -> torch.Tensor:
    """gain * part.sum(dim=0), part [slots, width] float32, on part's device and the current stream."""
    out = torch.empty(part.shape[1], dtype=dtype, device=part.device)
    _hip.check(_hip.lib().lvg_column_sum(part.data_ptr(), out.data_ptr(), part.shape[0], part.shape[1], gain, _hip.dtype_code(dtype), _hip.stream(part.device)),
               'lvg_column_sum')
    return out
