"""Matrix products with bias, activation and residual in their epilogue: an
attention layer's projections and a block's MLP, for a token of each request
and for whole prompts.

Kernels: csrc/linear.hip.  Float32, float16 and bfloat16; there is no
derivative (inputs that require a gradient are refused, where gradients are
recorded, and inputs with a tangent) and no CPU path.
"""

from __future__ import annotations

from functools import lru_cache

import torch
from torch.autograd import forward_ad

from . import _native as nat
from .attention import _need_no_gradient

# the activations' codes in the C interface
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_MOST = 1 << 20          # elements of a row, and between rows


@lru_cache(maxsize=4096)
def _workspace_bytes(rows: int, inner: int, outer: int, float_type: int, aligned: bool) -> int:
    """By the sizes and the alignment alone: asked for once."""

    plan = nat.LinearPlan()
    nat.check(nat.lib().cowsdm_linear_plan(rows, inner, outer, float_type, aligned, plan),
              "cowsdm_linear_plan")
    return plan.workspace_bytes


def _matrix(tensor: torch.Tensor, columns: int) -> tuple[torch.Tensor, int]:
    """A matrix whose rows can be read, and the elements between them: itself
    or a contiguous copy.  (Rows that are contiguous but not aligned go through
    a kernel of their own, which costs less than a copy.)"""

    row, column = tensor.stride()
    if column != 1 and columns > 1 or row > _MOST:
        tensor = tensor.contiguous()
        row = columns
    return tensor, 0 if tensor.shape[0] == 1 else row


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
           activation: str | None = None, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``residual + activation(x @ weight.T + bias)``: x [..., K], weight
    [N, K] as ``nn.Linear`` holds it, bias [N], residual [..., N], all of one
    type.  The activation is None, "relu", "gelu" (by the normal
    distribution), "gelu_tanh" or "silu".  Sums and everything after them are
    in float32 and rounded once.  Operands whose rows are 16-byte aligned (K
    and the strides multiples of 8, of 4 in float32) are read fastest."""

    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError('the activation must be None, "relu", "gelu", "gelu_tanh" or "silu"')
    if weight.ndim != 2 or x.ndim < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError("linear takes x [...,K] and weight [N,K]")
    outer, inner = weight.shape
    shape = (*x.shape[:-1], outer)
    if inner > _MOST:
        raise ValueError(f"linear sums over at most {_MOST} elements")
    dtype, index = x.dtype, x.get_device()
    alike = weight.dtype is dtype
    together = weight.get_device() == index
    if bias is not None:
        if bias.shape != (outer,):
            raise ValueError("linear bias must be [N]")
        alike, together = alike and bias.dtype is dtype, together and bias.get_device() == index
    if residual is not None:
        if residual.shape != shape:
            raise ValueError("linear residual must be [...,N]")
        alike = alike and residual.dtype is dtype
        together = together and residual.get_device() == index
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        _need_no_gradient(*[t for t in (x, weight, bias, residual) if t is not None])
    float_type = nat.FLOAT_TYPES.get(dtype)
    if float_type is None:
        raise TypeError("linear takes float32, float16 or bfloat16")
    if not alike:
        raise TypeError("linear inputs share one type")
    if index < 0:
        raise RuntimeError("linear inputs must be on the GPU: the kernels have no CPU path")
    if not together:
        raise ValueError("linear inputs must be on one device")
    out = x.new_empty(shape)
    rows = out.numel() // outer if outer else 0
    if not rows:
        return out
    device = out.device
    x, x_row = _matrix(x if x.ndim == 2 else x.reshape(rows, inner), inner)
    weight, weight_row = _matrix(weight, inner)
    if bias is not None and bias.stride(0) != 1:
        bias = bias.contiguous()
    residual_row = 0
    if residual is not None:
        residual, residual_row = _matrix(
            residual if residual.ndim == 2 else residual.reshape(rows, outer), outer)
    x_at, weight_at = x.data_ptr(), weight.data_ptr()
    aligned = not ((x_at | weight_at) % 16 or (x_row | weight_row) % (8 if float_type else 4))
    need = _workspace_bytes(rows, inner, outer, float_type, aligned)
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    a = nat.Linear(x_at, weight_at, nat.ptr(bias), nat.ptr(residual),
                   out.data_ptr(), x_row, weight_row, residual_row, rows, inner, outer, float_type,
                   code)
    rc = nat.lib().cowsdm_linear(a, nat.ptr(workspace), need, nat.stream_handle(device))
    if rc:
        nat.check(rc, "cowsdm_linear")
    return out
