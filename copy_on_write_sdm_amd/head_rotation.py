"""The norm of query and key heads with the rotation by position, in one pass
over a projection's output: what stands between an attention layer's
projection and its attention.

Kernel: csrc/head_rotation.hip.  Float32, float16 and bfloat16; there is no
derivative (inputs that require a gradient are refused, where gradients are
recorded, and inputs with a tangent) and no CPU path.
"""

from __future__ import annotations

import math
from fractions import Fraction
from typing import Sequence

import torch

from . import _native as nat
from .attention import _float_type, _int32, _need_device, _need_no_gradient, _rows

# 2 pi to 40 digits
_FULL_TURN = Fraction(62831853071795864769252867665590057683943, 10 ** 40)


class HeadRotation:
    """How far each pair of a head's elements turns per position: frequency j
    (in radians) is ``base ** (-2 j / width)`` for the ``width`` elements that
    are rotated, or ``frequencies[j]`` where they are given (stretched or
    interpolated rotations).  Pair j is elements j and j + width / 2, or 2 j
    and 2 j + 1 where ``interleaved``.

    The kernel counts a turn in 2^-64ths (``turns`` [width / 2], int64 whose
    bits count unsigned), so that far positions are as exact as near ones."""

    def __init__(self, width: int, *, base: float = 10000.0,
                 frequencies: Sequence[float] | torch.Tensor | None = None,
                 interleaved: bool = False, device: torch.device | str = "cuda"):
        if width <= 0 or width % 8 or width > 256:
            raise ValueError("rotated head width must be a multiple of 8, at most 256")
        if frequencies is None:
            if not 0.0 < base < math.inf:
                raise ValueError("the rotation's base must be positive")
            frequencies = [base ** (-2.0 * j / width) for j in range(width // 2)]
        else:
            if isinstance(frequencies, torch.Tensor):
                frequencies = frequencies.detach().double().cpu().tolist()
            frequencies = [float(f) for f in frequencies]
            if len(frequencies) != width // 2 or not all(map(math.isfinite, frequencies)):
                raise ValueError(f"{width} rotated elements take {width // 2} finite frequencies")
        self.width, self.interleaved = width, bool(interleaved)
        self.frequencies = tuple(frequencies)
        counts = [round(Fraction(f) / _FULL_TURN * 2 ** 64) % 2 ** 64 for f in frequencies]
        self.turns = torch.tensor([c - 2 ** 64 if c >= 2 ** 63 else c for c in counts],
                                  dtype=torch.int64, device=device)

    @property
    def device(self) -> torch.device:
        return self.turns.device


def _norm_weight(weight: torch.Tensor | None, like: torch.Tensor, what: str) -> None:
    if weight is None:
        return
    if weight.shape != (like.shape[-1],) or not weight.is_contiguous():
        raise ValueError(f"the {what} norm's weight must be [D], contiguous")
    if weight.dtype is not like.dtype:
        raise TypeError("heads and their norms' weights share one type")
    if weight.get_device() != like.get_device():
        raise ValueError("the norms' weights must be on the heads' device")


def rotate_heads(query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor,
                 rotation: HeadRotation | None, *, query_norm: torch.Tensor | None = None,
                 key_norm: torch.Tensor | None = None, eps: float = 1e-6
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """Query [T, heads, D] and key [T, kv_heads, D] (any strides between rows
    and heads, as slices of a fused projection) at ``positions`` [T] (int32,
    ``PageTableStep.positions``): every head's row is divided by the root of
    its mean square (with ``eps``) and multiplied by the norm's weight [D],
    where one is given, and then its first ``rotation.width`` elements are
    rotated (none without a rotation).  Returns both, contiguous, in their
    type; everything between is in float32."""

    if query.ndim != 3 or key.ndim != 3 or key.shape[0] != query.shape[0]:
        raise ValueError("rotated heads are query [T,heads,D] and key [T,kv_heads,D]")
    rows, heads, width = query.shape
    kv_heads = key.shape[1]
    if key.shape[2] != width:
        raise ValueError("query and key heads differ in width")
    if not heads or not kv_heads:
        raise ValueError("query and key need a head each")
    if width <= 0 or width % 8 or width > 256:
        raise ValueError("head width must be a multiple of 8, at most 256")
    if not 0.0 <= eps < math.inf:
        raise ValueError("the norm's eps cannot be negative")
    rotated = 0 if rotation is None else rotation.width
    if rotated > width:
        raise ValueError(f"heads of {width} cannot be rotated in {rotated} elements")
    weights = [w for w in (query_norm, key_norm) if w is not None]
    _need_no_gradient(query, key, *weights)
    code = _float_type(query.dtype)
    if key.dtype is not query.dtype:
        raise TypeError("query and key share one type")
    _norm_weight(query_norm, query, "query")
    _norm_weight(key_norm, key, "key")
    _need_device(query, "rotated heads")
    device, index = query.device, query.get_device()
    if key.get_device() != index or (rotation is not None
                                     and rotation.turns.get_device() != index):
        raise ValueError("heads and their rotation must be on one device")
    _int32(positions, rows, index, "positions")
    query_out = query.new_empty((rows, heads, width))
    key_out = query.new_empty((rows, kv_heads, width))
    if not rows:
        return query_out, key_out
    step = 8 if code else 4
    query, q, (q_row, q_head, _) = _rows(query, step)
    key, k, (k_row, k_head, _) = _rows(key, step)
    a = nat.RotateHeads(q, k, q_row, q_head, k_row, k_head, positions.data_ptr(),
                        None if rotation is None else rotation.turns.data_ptr(),
                        nat.ptr(query_norm), nat.ptr(key_norm), query_out.data_ptr(),
                        key_out.data_ptr(), rows, heads, kv_heads, width, rotated,
                        rotation is not None and rotation.interleaved, code, eps)
    rc = nat.lib().cowsdm_rotate_heads(a, nat.stream_handle(device))
    if rc:
        nat.check(rc, "cowsdm_rotate_heads")
    return query_out, key_out
