"""What the operators on matrices of token rows (linear_act, gated_ff, rms_norm) share: views of a tensor as rows, and types."""

import functools
import math

import torch
from torch.autograd import forward_ad

from . import _hip

E4M3 = 4                                                   # LVG_E4M3 of the C ABI
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -64
ROW_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def rows_of(t: torch.Tensor, width: int) -> torch.Tensor:
    """[..., width] -> [rows, width] with unit element stride: a view where the strides allow it, a copy otherwise."""
    if t.ndim != 2:
        t = t.reshape(math.prod(t.shape[:-1]), width)
    return t if t.is_contiguous() or t.stride(1) == 1 or width <= 1 else t.contiguous()


def row_stride(t: torch.Tensor) -> int:
    """Elements between the rows of a 2-D tensor; strides of a single row mean nothing."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


_CODES = {torch.float32: _hip.F32, torch.float16: _hip.F16, torch.bfloat16: _hip.BF16, torch.float8_e4m3fn: E4M3}


def type_code(dtype: torch.dtype) -> int:
    return _CODES[dtype]


def wants_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def watched(*tensors) -> bool:
    """Whether a call has to go through its autograd function: for gradients; while a trace is recorded, which would otherwise see the results'
    allocations alone; and while forward derivatives are taken, which the function refuses where an input has one (the kernels have none)."""
    return forward_ad._current_level >= 0 or torch._C._get_tracing_state() is not None or wants_grad(*tensors)         # pylint: disable=protected-access


@functools.lru_cache(maxsize=4096)
def query(name: str, *args) -> int:
    """A planning query of the library (a function of its arguments alone: workspace bytes, slot counts)."""
    return _hip.check(getattr(_hip.lib(), name)(*args), name)


def launch(device: torch.device, name: str, *args):
    """The entry point `name` on the device's current stream; the launch goes to the CURRENT HIP device, so that is made the tensors' first. One
    token's worth of work takes the GPU a few microseconds: this path avoids what costs the host as much (context managers, stream objects)."""
    fn = getattr(_hip.lib(), name)
    index = device.index
    if index == torch._C._cuda_getDevice():                      # pylint: disable=protected-access
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        _hip.check(rc, name)


def work_of(size: int, device: torch.device):
    """Workspace of a call, from the current stream's pool (a captured graph gets its own)."""
    return torch.empty(size, dtype=torch.uint8, device=device) if size > 0 else None
