"""K/V rows written to and read from the paged cache, 8-bit pools with one scale
per row and head found as the row is written.

``fp8.kv_append_fp8`` quantises with one scale per pool that the caller chose
beforehand; here every row carries its own (fp32 [num_blocks, Hkv, 64] beside a
pool of int8 or float8_e4m3fn [num_blocks, Hkv, 1, 64, 128]).  The same calls
take 16-bit pools (fp16 or bf16 [num_blocks, Hkv, D / 64, 64, 64]).

* ``b200kv::kv_store(k_new, v_new, k_pool!, v_pool!, slots, k_scales!, v_scales!, ...)``
  -- k turned by its rotary position (and q beside it), quantised, written;
* ``b200kv::kv_load(pool, slots, scales, dtype)`` -- rows gathered by slot.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _eager
from ._eager import direct, flag_ptr, launch, written
from .layout import PAGE_TOKENS
from .ops import _maybe_check_flag, _ptr, _require_cuda
from .rotations import DTYPE_CODES, ROTARY_DTYPES, check_table

DTYPES_16 = (torch.float16, torch.bfloat16)
DTYPES_8 = (torch.int8, torch.float8_e4m3fn)


def empty_row_pool(num_blocks: int, num_kv_heads: int, head_dim: int = 128, dtype: torch.dtype = torch.int8,
                   device=None) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(pool, scales) of uninitialised pages; scales is None for 16-bit dtypes."""
    if dtype in DTYPES_8:
        if head_dim != 128:
            raise ValueError("8-bit pools hold rows of 128 elements")
        pool = torch.empty((num_blocks, num_kv_heads, 1, PAGE_TOKENS, 128), dtype=dtype, device=device)
        return pool, torch.empty((num_blocks, num_kv_heads, PAGE_TOKENS), dtype=torch.float32, device=device)
    if dtype not in DTYPES_16 or head_dim not in (64, 128):
        raise ValueError(f"no pool of {dtype} with head_dim {head_dim}")
    return torch.empty((num_blocks, num_kv_heads, head_dim // 64, PAGE_TOKENS, 64), dtype=dtype, device=device), None


def check_row_pool(pool: torch.Tensor, scales: Optional[torch.Tensor], name: str) -> tuple[int, int, int]:
    """(num_blocks, Hkv, D) of a pool, its scales checked."""
    dtype, shape = pool.dtype, pool.shape
    k8 = dtype in DTYPES_8
    stick = 128 if k8 else 64
    if not (k8 or dtype in DTYPES_16) or len(shape) != 5 or shape[3] != PAGE_TOKENS or shape[4] != stick \
            or shape[2] * stick not in (64, 128) or not pool.is_contiguous():
        raise ValueError(f"{name}_pool must be contiguous [num_blocks, Hkv, D/64, 64, 64] (fp16, bf16) or "
                         f"[num_blocks, Hkv, 1, 64, 128] (int8, float8_e4m3fn), got {tuple(shape)} {dtype}")
    if k8:
        if scales is None:
            raise ValueError(f"8-bit pools need {name}_scales")
        if scales.dtype != torch.float32 or scales.shape != (shape[0], shape[1], PAGE_TOKENS) \
                or not scales.is_contiguous() or scales.device != pool.device:
            raise ValueError(f"{name}_scales must be contiguous fp32 [num_blocks, Hkv, 64] on the pool's device")
    elif scales is not None:
        raise ValueError(f"a 16-bit pool takes no {name}_scales")
    return shape[0], shape[1], shape[2] * stick


def check_row_pools(k_pool, v_pool, k_scales, v_scales) -> tuple[int, int, int]:
    shape = check_row_pool(k_pool, k_scales, "k")
    check_row_pool(v_pool, v_scales, "v")
    if k_pool.shape != v_pool.shape or k_pool.dtype != v_pool.dtype or k_pool.device != v_pool.device:
        raise ValueError("k_pool and v_pool must have the same shape, dtype and device")
    return shape


def _check_slots(slots: torch.Tensor, tokens: int, device: torch.device) -> None:
    if slots.dtype != torch.int64 or slots.dim() != 1 or len(slots) != tokens or not slots.is_contiguous() or slots.device != device:
        raise ValueError("slots must be a contiguous int64 [N] tensor on the pool's device")


def _kv_store_impl(
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    slots: torch.Tensor,
    k_scales: Optional[torch.Tensor],
    v_scales: Optional[torch.Tensor],
    q: Optional[torch.Tensor],
    table: Optional[torch.Tensor],
    positions: Optional[torch.Tensor],
    interleaved: bool,
    error_flag: Optional[torch.Tensor],
) -> torch.Tensor:
    _require_cuda(k_new, v_new, k_pool, v_pool, slots)
    NB, Hkv, D = check_row_pools(k_pool, v_pool, k_scales, v_scales)
    device, dtype = k_pool.device, k_new.dtype
    N = k_new.shape[0] if k_new.dim() == 3 else -1
    for rows, name in ((k_new, "k_new"), (v_new, "v_new")):
        if rows.shape != (N, Hkv, D) or dtype not in DTYPES_16 or rows.dtype != dtype or rows.stride(2) != 1 \
                or rows.device != device:
            raise ValueError(f"{name} must be fp16 or bf16 [N, {Hkv}, {D}] with a contiguous head_dim on the pools' "
                             f"device, got {tuple(rows.shape)} {rows.dtype}")
    if k_scales is None and k_pool.dtype != dtype:
        raise ValueError(f"a {k_pool.dtype} pool cannot take {dtype} rows")
    _check_slots(slots, N, device)
    if q is not None:
        if table is None:
            raise ValueError("q is taken to be turned: it needs a table")
        if q.dim() != 3 or q.shape[0] != N or q.shape[2] != D or q.dtype != dtype or q.stride(2) != 1 \
                or q.device != device:
            raise ValueError(f"q must be [N, Hq, {D}] of the rows' dtype with a contiguous head_dim")
        Hq, out, q_args = q.shape[1], torch.empty_like(q, memory_format=torch.contiguous_format), (
            q.data_ptr(), q.stride(0), q.stride(1))
    else:
        Hq, out, q_args = 0, k_new.new_empty((N, 0, D)), (None, 0, 0)
    if table is not None:
        if positions is None:
            raise ValueError("a table needs positions")
        check_table(table, positions, N, D, device)
        turn = (table.data_ptr(), table.shape[0], 2 * table.shape[1], positions.data_ptr())
    else:
        turn = (None, 0, 0, None)
    launch(
        "b200kv_kv_store", device, *q_args, out.data_ptr(),
        k_new.data_ptr(), k_new.stride(0), k_new.stride(1), v_new.data_ptr(), v_new.stride(0), v_new.stride(1),
        DTYPE_CODES[dtype], k_pool.data_ptr(), v_pool.data_ptr(), DTYPE_CODES[k_pool.dtype],
        _ptr(k_scales), _ptr(v_scales), slots.data_ptr(), *turn, interleaved, N, Hq, Hkv, D, NB,
        flag_ptr(error_flag, device),
    )
    _maybe_check_flag(error_flag, "kv_store")
    return out


_kv_store_op = torch.library.custom_op("b200kv::kv_store", _kv_store_impl, device_types="cuda",
                                       mutates_args=("k_pool", "v_pool", "k_scales", "v_scales"))


@_kv_store_op.register_fake
def _(k_new, v_new, k_pool, v_pool, slots, k_scales, v_scales, q, table, positions, interleaved, error_flag):
    return k_new.new_empty((k_new.shape[0], 0 if q is None else q.shape[1], k_new.shape[2]))


def kv_store(
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    slots: torch.Tensor,
    k_scales: Optional[torch.Tensor] = None,
    v_scales: Optional[torch.Tensor] = None,
    q: Optional[torch.Tensor] = None,
    table: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    error_flag: Optional[torch.Tensor] = None,
) -> Optional[torch.Tensor]:
    """Writes row n of k_new / v_new ([N, Hkv, D], fp16 or bf16) to slot slots[n],
    in one launch.

    8-bit pools take round(x * (1 / s)) with s = max|x| / qmax of the row (127 for
    int8, 448 for float8_e4m3fn), s into ``k_scales`` / ``v_scales``; 16-bit pools
    take the rows as they are.  With ``table`` and ``positions``
    (:func:`torch_spyre_b200.rotary_table`) k is turned first (not rounded
    in between); ``q`` [N, Hq, D] is turned by the same launch and returned.
    Slots must be distinct; negative slots skip their row."""
    args = (k_new, v_new, k_pool, v_pool, slots, k_scales, v_scales, q, table, positions, bool(interleaved), error_flag)
    out = None if _eager.compiling() else _eager.fast.kv_store(*args)
    if out is None:
        if direct(k_new, v_new, k_pool, v_pool, slots, k_scales, v_scales, q, table, positions):
            out = _kv_store_impl(*args)
            written(k_pool, v_pool, k_scales, v_scales)
        else:
            out = torch.ops.b200kv.kv_store(*args)
    return None if q is None else out


def _kv_load_impl(pool: torch.Tensor, slots: torch.Tensor, scales: Optional[torch.Tensor], dtype: torch.dtype,
                  error_flag: Optional[torch.Tensor]) -> torch.Tensor:
    _require_cuda(pool, slots)
    NB, Hkv, D = check_row_pool(pool, scales, "")
    N = slots.shape[0] if slots.dim() == 1 else -1
    device = pool.device
    _check_slots(slots, N, device)
    if dtype not in ROTARY_DTYPES:
        raise ValueError(f"dtype must be fp16, bf16 or fp32, got {dtype}")
    out = torch.empty((N, Hkv, D), dtype=dtype, device=device)
    launch("b200kv_kv_load", device, pool.data_ptr(), DTYPE_CODES[pool.dtype], _ptr(scales), slots.data_ptr(),
           out.data_ptr(), DTYPE_CODES[dtype], N, Hkv, D, NB, flag_ptr(error_flag, device))
    _maybe_check_flag(error_flag, "kv_load")
    return out


_kv_load_op = torch.library.custom_op("b200kv::kv_load", _kv_load_impl, mutates_args=(), device_types="cuda")


@_kv_load_op.register_fake
def _(pool, slots, scales, dtype, error_flag):
    return pool.new_empty((slots.shape[0], pool.shape[1], pool.shape[2] * pool.shape[4]), dtype=dtype)


def kv_load(pool: torch.Tensor, slots: torch.Tensor, scales: Optional[torch.Tensor] = None,
            dtype: Optional[torch.dtype] = None, error_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows [N, Hkv, D] of a pool gathered by slot (value * scale, rounded once to
    ``dtype``: fp16, bf16 or fp32; default the pool's own, fp16 for 8-bit pools).
    Negative slots give rows of zeros."""
    if dtype is None:
        dtype = pool.dtype if pool.dtype in DTYPES_16 else torch.float16
    if not _eager.compiling():
        out = _eager.fast.kv_load(pool, slots, scales, DTYPE_CODES.get(dtype, -1), error_flag)
        if out is not None:
            return out
    op = _kv_load_impl if direct(pool, slots, scales) else torch.ops.b200kv.kv_load
    return op(pool, slots, scales, dtype, error_flag)
