"""Matrix products with bias, activation and residual in their epilogue: an
attention layer's projections and a block's MLP, for a token of each request
and for whole prompts.

Kernels: csrc/linear.hip.  Float32, float16 and bfloat16; there is no backward
pass (inputs that require a gradient are refused, where gradients are
recorded) and no CPU path.
"""

from __future__ import annotations

import torch

from . import _native as nat
from .attention import _need_no_gradient

# the activations' codes in the C interface
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_MOST = 1 << 20          # elements of a row, and between rows


def _matrix(tensor: torch.Tensor) -> tuple[torch.Tensor, int]:
    """A matrix whose rows can be read, and the elements between them: itself
    or a contiguous copy.  (Rows that are contiguous but not aligned are read
    element by element by the kernel, which costs less than a copy.)"""

    if tensor.stride(1) != 1 and tensor.shape[1] > 1 or tensor.stride(0) > _MOST:
        tensor = tensor.contiguous()
    if tensor.shape[0] == 1:
        return tensor, 0
    return tensor, tensor.stride(0)


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
    if bias is not None and bias.shape != (outer,):
        raise ValueError("linear bias must be [N]")
    if residual is not None and residual.shape != shape:
        raise ValueError("linear residual must be [...,N]")
    if inner > _MOST:
        raise ValueError(f"linear sums over at most {_MOST} elements")
    others = [t for t in (weight, bias, residual) if t is not None]
    _need_no_gradient(x, *others)
    dtype = x.dtype
    float_type = nat.FLOAT_TYPES.get(dtype)
    if float_type is None:
        raise TypeError("linear takes float32, float16 or bfloat16")
    if any([t.dtype is not dtype for t in others]):
        raise TypeError("linear inputs share one type")
    if not x.is_cuda:
        raise RuntimeError("linear inputs must be on the GPU: the kernels have no CPU path")
    device, index = x.device, x.get_device()
    if any([t.get_device() != index for t in others]):
        raise ValueError("linear inputs must be on one device")
    out = x.new_empty(shape)
    if not out.numel():
        return out
    rows = out.numel() // outer
    x, x_row = _matrix(x if x.ndim == 2 else x.reshape(rows, inner))
    weight, weight_row = _matrix(weight)
    if bias is not None and bias.stride(0) != 1:
        bias = bias.contiguous()
    residual_row = 0
    if residual is not None:
        residual, residual_row = _matrix(
            residual if residual.ndim == 2 else residual.reshape(rows, outer))
    a = nat.Linear(x.data_ptr(), weight.data_ptr(), nat.ptr(bias), nat.ptr(residual),
                   out.data_ptr(), x_row, weight_row, residual_row, rows, inner, outer, float_type,
                   code)
    lib = nat.lib()
    need = lib.cowsdm_linear_workspace_bytes(rows, inner, outer, float_type)
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
    rc = lib.cowsdm_linear(a, nat.ptr(workspace), need, nat.stream_handle(device))
    if rc:
        nat.check(rc, "cowsdm_linear")
    return out
