"""Rotary positions from an fp32 table: half and interleaved pairs, part of the
head, tables scaled for long contexts, forward and gradient.

``ops.rope`` keeps the reference's formulation (fp16 2x2 matrices, half pairs,
whole heads); :func:`rotary` is the form a model's own positions take:

* :func:`rotary_table` -- (cos, sin) of every position, made once, in fp64,
  stored in fp32;
* ``b200kv::rotary(x, table, positions, interleaved, transpose, error_flag)``
  -- the turn of rows [T, H, D] (fp16, bf16, fp32), differentiable in x.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from .ops import _maybe_check_flag, _ptr, _require_cuda, _stream_ptr

ROTARY_SCALINGS = ("none", "linear", "ntk", "yarn")


def dtype_code(dtype: torch.dtype) -> int:
    """enum b200kv_dtype of a torch dtype (ValueError if the library has none)."""
    code = _lib.DTYPES.get(str(dtype).removeprefix("torch."))
    if code is None:
        raise ValueError(f"unsupported dtype {dtype}")
    return code


def rotary_table(max_pos: int, rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original_max_pos: Optional[int] = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 attention_factor: Optional[float] = None, device=None) -> torch.Tensor:
    """(cos, sin) fp32 [max_pos, rotary_dim / 2, 2] of pos * inv_i,
    inv_i = base^(-2i / rotary_dim), scaled for contexts ``factor`` times as long:

    * ``linear`` -- inv_i / factor (positions interpolated);
    * ``ntk`` -- base * factor^(rotary_dim / (rotary_dim - 2)): the fastest pair
      unchanged, the slowest interpolated;
    * ``yarn`` -- pairs that turn more than ``beta_fast`` times over
      ``original_max_pos`` keep inv_i, those under ``beta_slow`` turns take
      inv_i / factor, a linear ramp between them; cos and sin are multiplied by
      ``attention_factor`` (default 0.1 ln(factor) + 1).

    Angles are computed in fp64 and rounded once: at position 131071 an fp32
    product would already be off by 4e-3 radians.
    """
    if max_pos <= 0 or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("max_pos must be > 0 and rotary_dim even and > 0")
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"scaling must be one of {ROTARY_SCALINGS}, got {scaling!r}")
    if not factor >= 1.0 or not base > 1.0:
        raise ValueError("factor must be >= 1 and base > 1")
    half, scale = rotary_dim // 2, 1.0
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2.0))
    i = torch.arange(half, dtype=torch.float64, device=device)
    inv = base ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "yarn":
        if not original_max_pos or original_max_pos <= 0:
            raise ValueError("yarn scaling needs original_max_pos")

        def pair_of(turns: float) -> float:  # the (real) pair index that turns this often over original_max_pos
            return rotary_dim * math.log(original_max_pos / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        lo, hi = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), half - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        inv = inv * (1.0 - ramp) + inv / factor * ramp
        scale = 0.1 * math.log(factor) + 1.0
    if attention_factor is not None:
        scale = attention_factor
    angle = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv
    return (torch.stack([torch.cos(angle), torch.sin(angle)], -1) * scale).float()


def check_table(table: torch.Tensor, positions: torch.Tensor, tokens: int, head_dim: int,
                device: torch.device) -> None:
    if table.dtype != torch.float32 or table.dim() != 3 or table.shape[2] != 2 or not table.is_contiguous() \
            or table.device != device:
        raise ValueError("table must be a contiguous fp32 [max_pos, rotary_dim / 2, 2] tensor on the rows' device, "
                         f"got {tuple(table.shape)} {table.dtype} on {table.device}")
    if not 0 < 2 * table.shape[1] <= head_dim:
        raise ValueError(f"the table turns {2 * table.shape[1]} elements of a head of {head_dim}")
    if positions.dtype != torch.int32 or positions.shape != (tokens,) or not positions.is_contiguous() \
            or positions.device != device:
        raise ValueError("positions must be a contiguous int32 [T] tensor on the rows' device")


@torch.library.custom_op("b200kv::rotary", mutates_args=(), device_types="cuda")
def _rotary_op(x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, interleaved: bool, transpose: bool,
               error_flag: Optional[torch.Tensor]) -> torch.Tensor:
    _require_cuda(x, table, positions)
    if x.dim() != 3 or x.dtype not in (torch.float16, torch.bfloat16, torch.float32) or (x.stride(2) != 1
                                                                                         and x.shape[2] != 1):
        raise ValueError("x must be fp16, bf16 or fp32 [T, H, D] with a contiguous head_dim, "
                         f"got {tuple(x.shape)} {x.dtype}")
    T, H, D = x.shape
    check_table(table, positions, T, D, x.device)
    out = torch.empty((T, H, D), dtype=x.dtype, device=x.device)
    _lib.call("b200kv_rotary", x.data_ptr(), dtype_code(x.dtype), x.stride(0), x.stride(1), out.data_ptr(),
              table.data_ptr(), table.shape[0], 2 * table.shape[1], positions.data_ptr(), T, H, D, int(interleaved),
              int(transpose), _ptr(error_flag), _stream_ptr(x.device))
    _maybe_check_flag(error_flag, "rotary")
    return out


@_rotary_op.register_fake
def _(x, table, positions, interleaved, transpose, error_flag):
    return x.new_empty(x.shape)


def _rotary_setup(ctx, inputs, output):
    _, table, positions, interleaved, transpose, error_flag = inputs
    ctx.save_for_backward(table, positions)
    ctx.turn = (interleaved, transpose, error_flag)


def _rotary_backward(ctx, grad):
    table, positions = ctx.saved_tensors
    interleaved, transpose, error_flag = ctx.turn
    if grad.stride(-1) != 1:  # e.g. the expanded gradient of a sum
        grad = grad.contiguous()
    return (torch.ops.b200kv.rotary(grad, table, positions, interleaved, not transpose, error_flag), None, None, None,
            None, None)


_rotary_op.register_autograd(_rotary_backward, setup_context=_rotary_setup)


def rotary(x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, interleaved: bool = False,
           error_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows x [T, H, D] (fp16, bf16 or fp32; any token and head strides) turned at
    positions [T] (int32) by ``table`` (:func:`rotary_table`), a new contiguous
    tensor: pair i of the first rotary_dim elements is (i, i + rotary_dim / 2), or
    (2i, 2i + 1) when ``interleaved``; the other elements are copied.  fp32
    arithmetic, rounded once.  Differentiable in x (the table is a constant).  A
    position outside the table is clamped and sets ``DEVERR_BAD_LEN``."""
    return torch.ops.b200kv.rotary(x, table, positions, bool(interleaved), False, error_flag)
