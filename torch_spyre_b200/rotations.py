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

from . import _eager, _lib
from ._eager import flag_ptr, launch
from .ops import _maybe_check_flag, _require_cuda

ROTARY_SCALINGS = ("none", "linear", "ntk", "yarn")


# enum b200kv_dtype of the torch dtypes
DTYPE_CODES = {getattr(torch, name): code for name, code in _lib.DTYPES.items()}
ROTARY_DTYPES = {d: DTYPE_CODES[d] for d in (torch.float16, torch.bfloat16, torch.float32)}


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
      inv_i / factor, a ramp linear in the pair's index (it may end past the
      last pair) between them; cos and sin are multiplied by
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

        lo, hi = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        inv = inv * (1.0 - ramp) + inv / factor * ramp
        scale = 0.1 * math.log(factor) + 1.0
    if attention_factor is not None:
        scale = attention_factor
    angle = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv
    return (torch.stack([torch.cos(angle), torch.sin(angle)], -1) * scale).float()


def check_table(table: torch.Tensor, positions: torch.Tensor, tokens: int, head_dim: int,
                device: torch.device) -> None:
    shape = table.shape
    if table.dtype != torch.float32 or len(shape) != 3 or shape[2] != 2 or not table.is_contiguous() \
            or table.device != device:
        raise ValueError("table must be a contiguous fp32 [max_pos, rotary_dim / 2, 2] tensor on the rows' device, "
                         f"got {tuple(table.shape)} {table.dtype} on {table.device}")
    if not 0 < 2 * shape[1] <= head_dim:
        raise ValueError(f"the table turns {2 * shape[1]} elements of a head of {head_dim}")
    if positions.dtype != torch.int32 or positions.dim() != 1 or len(positions) != tokens \
            or not positions.is_contiguous() or positions.device != device:
        raise ValueError("positions must be a contiguous int32 [T] tensor on the rows' device")


def _rotary_impl(x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, interleaved: bool, transpose: bool,
                 error_flag: Optional[torch.Tensor]) -> torch.Tensor:
    _require_cuda(x, table, positions)
    if x.dim() != 3 or x.dtype not in ROTARY_DTYPES or (x.stride(2) != 1 and x.shape[2] != 1):
        raise ValueError("x must be fp16, bf16 or fp32 [T, H, D] with a contiguous head_dim, "
                         f"got {tuple(x.shape)} {x.dtype}")
    T, H, D = x.shape
    device = x.device
    check_table(table, positions, T, D, device)
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    launch("b200kv_rotary", device, x.data_ptr(), ROTARY_DTYPES[x.dtype], x.stride(0), x.stride(1), out.data_ptr(),
           table.data_ptr(), table.shape[0], 2 * table.shape[1], positions.data_ptr(), T, H, D, interleaved, transpose,
           flag_ptr(error_flag, device))
    _maybe_check_flag(error_flag, "rotary")
    return out


_rotary_op = torch.library.custom_op("b200kv::rotary", _rotary_impl, mutates_args=(), device_types="cuda")


@_rotary_op.register_fake
def _(x, table, positions, interleaved, transpose, error_flag):
    return x.new_empty(x.shape)


def _turn_back(grad, table, positions, interleaved, transpose, error_flag):
    if grad.stride(-1) != 1:  # e.g. the expanded gradient of a sum
        grad = grad.contiguous()
    return _turn(grad, table, positions, interleaved, not transpose, error_flag)


def _rotary_setup(ctx, inputs, output):
    _, table, positions, interleaved, transpose, error_flag = inputs
    ctx.save_for_backward(table, positions)
    ctx.turn = (interleaved, transpose, error_flag)


def _rotary_backward(ctx, grad):
    return (_turn_back(grad, *ctx.saved_tensors, *ctx.turn), None, None, None, None, None)


_rotary_op.register_autograd(_rotary_backward, setup_context=_rotary_setup)


class _Rotary(torch.autograd.Function):
    """The operator's gradient without the dispatcher (the same map turned the other way)."""

    @staticmethod
    def forward(ctx, x, table, positions, interleaved, transpose, error_flag):
        ctx.save_for_backward(table, positions)
        ctx.turn = (interleaved, transpose, error_flag)
        y = _eager.fast.rotary(x, table, positions, interleaved, transpose, error_flag)
        return _rotary_impl(x, table, positions, interleaved, transpose, error_flag) if y is None else y

    backward = staticmethod(_rotary_backward)


def _turn(x, table, positions, interleaved, transpose, error_flag):
    args = (x, table, positions, interleaved, transpose, error_flag)
    if not _eager.compiling():
        y = _eager.fast.rotary(*args)
        if y is not None:
            return y
        if _eager.plain(x) and _eager.direct(table, positions):
            return _Rotary.apply(*args) if x.requires_grad and torch.is_grad_enabled() else _rotary_impl(*args)
    return torch.ops.b200kv.rotary(*args)


def rotary(x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, interleaved: bool = False,
           error_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows x [T, H, D] (fp16, bf16 or fp32; any token and head strides) turned at
    positions [T] (int32) by ``table`` (:func:`rotary_table`), a new contiguous
    tensor: pair i of the first rotary_dim elements is (i, i + rotary_dim / 2), or
    (2i, 2i + 1) when ``interleaved``; the other elements are copied.  fp32
    arithmetic, rounded once.  Differentiable in x (the table is a constant).  A
    position outside the table is clamped and sets ``DEVERR_BAD_LEN``."""
    return _turn(x, table, positions, bool(interleaved), False, error_flag)
