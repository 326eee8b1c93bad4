"""Latent attention over a paged cache of one vector a token.

A token's row has 512 latent elements, which every head takes as key and value,
and 64 rotary key elements, also shared: 1152 bytes a token in fp16 or bf16, for
any number of heads.  A head's own key (128 elements) and value (128) are
products of the latent vector with the head's weights W_k, W_v [512, 128]:

* absorbed (few new tokens): W_k is multiplied into the query, q W_k^T . c = q . W_k^T c,
  and W_v into the output, so attention runs over the rows as they are cached
  (:func:`latent_attention`);
* expanded (prompts): the rows are multiplied out, once for all queries
  (:func:`latent_prompt_attention`).

* ``b200kv::latent_attention(q_latent, q_rope, pool, block_table, ...)`` -- the
  absorbed form: drafted trees, chains or single tokens over the paged rows;
* ``b200kv::latent_store(latent, k_rope, pool!, slots, ...)`` -- rows normalised,
  turned and written, the heads' rotary queries turned beside them;
* :func:`latent_load` -- rows gathered by slot; ``b200kv::latent_commit`` -- the
  accepted path of a drafted tree, as :func:`torch_spyre_b200.tree_commit`.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _eager, _lib
from ._eager import direct, flag_ptr, launch, written
from .kv_rows import DTYPES_16, _check_slots, kv_load
from .layout import PAGE_TOKENS
from .ops import _maybe_check_flag, _ptr, _require_cuda, workspace_for
from .rotations import DTYPE_CODES, check_table
from .tree import _check_indptr, _check_sequences

RANK, ROPE, NOPE = 512, 64, 128
STICKS = (RANK + ROPE) // 64


def empty_latent_pool(num_blocks: int, dtype: torch.dtype = torch.bfloat16, device=None) -> torch.Tensor:
    """Uninitialised pages [num_blocks, 1, 9, 64, 64] of 64 rows each."""
    if dtype not in DTYPES_16:
        raise ValueError(f"latent pools are fp16 or bf16, not {dtype}")
    return torch.empty((num_blocks, 1, STICKS, PAGE_TOKENS, 64), dtype=dtype, device=device)


def _check_pool(pool: torch.Tensor) -> int:
    if pool.dtype not in DTYPES_16 or pool.dim() != 5 or pool.shape[1:] != (1, STICKS, PAGE_TOKENS, 64) \
            or not pool.is_contiguous():
        raise ValueError(f"pool must be contiguous fp16 or bf16 [num_blocks, 1, {STICKS}, 64, 64], got "
                         f"{tuple(pool.shape)} {pool.dtype}")
    return pool.shape[0]


def _latent_store_impl(
    latent: torch.Tensor,
    k_rope: torch.Tensor,
    pool: torch.Tensor,
    slots: torch.Tensor,
    q_rope: Optional[torch.Tensor],
    norm_weight: Optional[torch.Tensor],
    eps: float,
    table: Optional[torch.Tensor],
    positions: Optional[torch.Tensor],
    interleaved: bool,
    error_flag: Optional[torch.Tensor],
) -> torch.Tensor:
    _require_cuda(latent, k_rope, pool, slots)
    NB, device, dtype = _check_pool(pool), pool.device, pool.dtype
    N = latent.shape[0] if latent.dim() == 2 else -1
    for rows, name, width in ((latent, "latent", RANK), (k_rope, "k_rope", ROPE)):
        if rows.shape != (N, width) or rows.dtype != dtype or rows.stride(1) != 1 or rows.device != device:
            raise ValueError(f"{name} must be [N, {width}] of the pool's dtype with contiguous rows on its device, got "
                             f"{tuple(rows.shape)} {rows.dtype}")
    _check_slots(slots, N, device)
    if norm_weight is not None and (norm_weight.dtype != dtype or norm_weight.shape != (RANK,)
                                    or not norm_weight.is_contiguous() or norm_weight.device != device):
        raise ValueError(f"norm_weight must be contiguous [{RANK}] of the pool's dtype on its device")
    if q_rope is not None:
        if table is None:
            raise ValueError("q_rope is taken to be turned: it needs a table")
        if q_rope.dim() != 3 or q_rope.shape[0] != N or q_rope.shape[2] != ROPE or q_rope.dtype != dtype \
                or q_rope.stride(2) != 1 or q_rope.device != device:
            raise ValueError(f"q_rope must be [N, H, {ROPE}] of the pool's dtype with contiguous rows on its device")
        H, q_args = q_rope.shape[1], (q_rope.data_ptr(), q_rope.stride(0), q_rope.stride(1))
    else:
        H, q_args = 0, (None, 0, 0)
    out = latent.new_empty((N, H, ROPE))
    if table is not None:
        if positions is None:
            raise ValueError("a table needs positions")
        check_table(table, positions, N, ROPE, device)
        if table.shape[1] != ROPE // 2:
            raise ValueError(f"the table must turn all {ROPE} elements, it turns {2 * table.shape[1]}")
    launch("b200kv_latent_store", device, latent.data_ptr(), latent.stride(0), k_rope.data_ptr(), k_rope.stride(0),
           *q_args, out.data_ptr(), DTYPE_CODES[dtype], _ptr(norm_weight), eps, pool.data_ptr(), slots.data_ptr(),
           _ptr(table), 0 if table is None else table.shape[0], _ptr(positions), interleaved, N, H, NB,
           flag_ptr(error_flag, device))
    _maybe_check_flag(error_flag, "latent_store")
    return out


_latent_store_op = torch.library.custom_op("b200kv::latent_store", _latent_store_impl, device_types="cuda",
                                           mutates_args=("pool",))


@_latent_store_op.register_fake
def _(latent, k_rope, pool, slots, q_rope, norm_weight, eps, table, positions, interleaved, error_flag):
    return latent.new_empty((latent.shape[0], 0 if q_rope is None else q_rope.shape[1], ROPE))


def latent_store(
    latent: torch.Tensor,
    k_rope: torch.Tensor,
    pool: torch.Tensor,
    slots: torch.Tensor,
    q_rope: Optional[torch.Tensor] = None,
    norm_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    table: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    error_flag: Optional[torch.Tensor] = None,
) -> Optional[torch.Tensor]:
    """Writes token n's row, latent[n] ([N, 512]) and k_rope[n] ([N, 64]), to slot
    slots[n] of the pool, in one launch (strided rows will do, so both may be parts of
    one projection's output).

    With ``norm_weight`` [512] the latent part is x / sqrt(mean(x^2) + eps) * weight.
    With ``table`` ([max_pos, 32, 2], :func:`torch_spyre_b200.rotary_table`) and
    ``positions`` the key part is turned, and so is ``q_rope`` [N, H, 64] beside it,
    which is returned.  fp32 arithmetic, rounded once.  Slots must be distinct;
    negative slots skip their row."""
    args = (latent, k_rope, pool, slots, q_rope, norm_weight, float(eps), table, positions, bool(interleaved), error_flag)
    out = None if _eager.compiling() else _eager.fast.latent_store(*args)
    if out is None:
        if direct(latent, k_rope, pool, slots, q_rope, norm_weight, table, positions):
            out = _latent_store_impl(*args)
            written(pool)
        else:
            out = torch.ops.b200kv.latent_store(*args)
    return None if q_rope is None else out


def latent_load(pool: torch.Tensor, slots: torch.Tensor, dtype: Optional[torch.dtype] = None,
                error_flag: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(latent [N, 512], k_rope [N, 64]) of the rows at ``slots``, two views of one
    contiguous [N, 576] tensor (dtype fp16, bf16 or fp32; default the pool's).
    Negative slots give rows of zeros."""
    if not _eager.compiling():
        pair = _eager.fast.latent_load(pool, slots, -1 if dtype is None else DTYPE_CODES.get(dtype, 99), error_flag)
        if pair is not None:
            return pair
    NB = _check_pool(pool)
    rows = kv_load(pool.view(NB, STICKS, 1, PAGE_TOKENS, 64), slots, dtype=dtype, error_flag=error_flag)
    rows = rows.view(-1, RANK + ROPE)
    return rows[:, :RANK], rows[:, RANK:]


# ------------------------------------------------------------------- commit --
def _latent_commit_impl(pool: torch.Tensor, block_table: torch.Tensor, context_lens: torch.Tensor, path: torch.Tensor,
                        path_lens: torch.Tensor, error_flag: Optional[torch.Tensor]) -> torch.Tensor:
    _require_cuda(pool, block_table, context_lens, path, path_lens)
    NB, device = _check_pool(pool), pool.device
    B = _check_sequences(block_table, context_lens, device)
    if path.dtype != torch.int32 or path.dim() != 2 or len(path) != B or (path.shape[1] > 1 and path.stride(1) != 1) \
            or path.device != device:
        raise ValueError("path must be int32 [B, max_path] with unit column stride on the pool's device")
    if path_lens.dtype != torch.int32 or path_lens.dim() != 1 or len(path_lens) != B \
            or not path_lens.is_contiguous() or path_lens.device != device:
        raise ValueError("path_lens must be a contiguous int32 [B] tensor on the pool's device")
    new_lens = torch.empty_like(context_lens)
    launch("b200kv_latent_commit", device, pool.data_ptr(), DTYPE_CODES[pool.dtype], block_table.data_ptr(),
           block_table.stride(0), context_lens.data_ptr(), path.data_ptr(), path.stride(0) if B > 1 else path.shape[1],
           path_lens.data_ptr(), new_lens.data_ptr(), B, NB, block_table.shape[1], path.shape[1],
           flag_ptr(error_flag, device))
    _maybe_check_flag(error_flag, "latent_commit")
    return new_lens


_latent_commit_op = torch.library.custom_op("b200kv::latent_commit", _latent_commit_impl, device_types="cuda",
                                            mutates_args=("pool",))


@_latent_commit_op.register_fake
def _(pool, block_table, context_lens, path, path_lens, error_flag):
    return torch.empty_like(context_lens)


def latent_commit(pool: torch.Tensor, block_table: torch.Tensor, context_lens: torch.Tensor, path: torch.Tensor,
                  path_lens: torch.Tensor, error_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`torch_spyre_b200.tree_commit` for a latent pool: moves the rows of the
    accepted nodes path[b, :path_lens[b]] to positions context_lens[b] on, in place,
    and returns the new lengths."""
    args = (pool, block_table, context_lens, path, path_lens, error_flag)
    new_lens = None if _eager.compiling() else _eager.fast.latent_commit(*args)
    if new_lens is None:
        if not direct(pool, block_table, context_lens, path, path_lens):
            return torch.ops.b200kv.latent_commit(*args)
        new_lens = _latent_commit_impl(*args)
        written(pool)
    return new_lens


# ---------------------------------------------------------------- attention --
def _latent_attention_impl(
    q_latent: torch.Tensor,
    q_rope: torch.Tensor,
    pool: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    q_indptr: torch.Tensor,
    tree_mask: Optional[torch.Tensor],
    scale: float,
    max_nodes: int,
    error_flag: Optional[torch.Tensor],
) -> tuple[torch.Tensor, torch.Tensor]:
    return _attend(q_latent, q_rope, pool, block_table, context_lens, q_indptr, tree_mask, scale, max_nodes, error_flag,
                   True)


def _attend(q_latent, q_rope, pool, block_table, context_lens, q_indptr, tree_mask, scale, max_nodes, error_flag,
            want_lse):
    _require_cuda(q_latent, q_rope, pool, block_table, context_lens, q_indptr)
    NB, device, dtype = _check_pool(pool), pool.device, pool.dtype
    for q, name, width in ((q_latent, "q_latent", RANK), (q_rope, "q_rope", ROPE)):
        if q.dim() != 3 or q.shape[:2] != q_latent.shape[:2] or q.shape[2] != width or q.dtype != dtype \
                or q.stride(2) != 1 or q.device != device:
            raise ValueError(f"{name} must be [N, H, {width}] of the pool's dtype with contiguous rows on its device, got "
                             f"{tuple(q.shape)} {q.dtype}")
    B = _check_sequences(block_table, context_lens, device)
    _check_indptr(q_indptr, B, device)
    N, H, _ = q_latent.shape
    words = 0
    if tree_mask is not None:
        if tree_mask.dtype != torch.int64 or tree_mask.dim() != 2 or len(tree_mask) != N \
                or not tree_mask.is_contiguous() or tree_mask.device != device:
            raise ValueError("tree_mask must be a contiguous int64 [N, words] tensor on q's device")
        words = tree_mask.shape[1]
    out = torch.empty((N, H, RANK), dtype=dtype, device=device)
    lse = torch.empty((N, H), dtype=torch.float32, device=device) if want_lse else None
    if N == 0:
        return out, lse
    wbytes = _lib.lib().b200kv_latent_workspace_bytes(N, B, H)
    # An unsupported shape has no workspace size; the call below then reports why.
    ws = workspace_for(device, wbytes) if wbytes > 0 else torch.empty(0, dtype=torch.uint8, device=device)
    if wbytes > 0:
        _eager.fast.set_workspace(ws)  # where the next call finds it
    launch("b200kv_latent_attention", device, q_latent.data_ptr(), q_latent.stride(0), q_latent.stride(1),
           q_rope.data_ptr(), q_rope.stride(0), q_rope.stride(1), DTYPE_CODES[dtype], pool.data_ptr(),
           block_table.data_ptr(), block_table.stride(0), context_lens.data_ptr(), q_indptr.data_ptr(), _ptr(tree_mask),
           words, out.data_ptr(), _ptr(lse), N, B, H, NB, block_table.shape[1], max_nodes, scale, ws.data_ptr(),
           ws.numel(), flag_ptr(error_flag, device))
    _maybe_check_flag(error_flag, "latent_attention")
    return out, lse


_latent_attention_op = torch.library.custom_op("b200kv::latent_attention", _latent_attention_impl, mutates_args=(),
                                               device_types="cuda")


@_latent_attention_op.register_fake
def _(q_latent, q_rope, pool, block_table, context_lens, q_indptr, tree_mask, scale, max_nodes, error_flag):
    return q_latent.new_empty(q_latent.shape), q_latent.new_empty(q_latent.shape[:2], dtype=torch.float32)


def latent_attention(
    q_latent: torch.Tensor,
    q_rope: torch.Tensor,
    pool: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    q_indptr: torch.Tensor,
    tree_mask: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    max_nodes: Optional[int] = None,
    return_lse: bool = False,
    error_flag: Optional[torch.Tensor] = None,
):
    """Attention of every sequence's new tokens over its cached rows, absorbed form:
    each head scores a token by scale * (q_latent . latent + q_rope . k_rope) and gets the
    weighted sum of the latent parts.

    q_latent [N, H, 512] is the head's own query times its W_k^T, q_rope [N, H, 64] the
    turned part (:func:`latent_store` returns it), both of the pool's dtype; the
    result [N, H, 512] is what W_v multiplies.  The nodes of all sequences come one
    after the other; q_indptr, context_lens, tree_mask, max_nodes, the masks' meaning
    and the returned log-sum-exps are those of :func:`torch_spyre_b200.tree_attention`.
    scale defaults to that of the expanded head, 1 / sqrt(128 + 64)."""
    if scale is None:
        scale = 1.0 / math.sqrt(NOPE + ROPE)
    if max_nodes is None:
        max_nodes = q_latent.shape[0] if tree_mask is None else min(q_latent.shape[0], 64 * tree_mask.shape[1])
    args = (q_latent, q_rope, pool, block_table, context_lens, q_indptr, tree_mask, float(scale), max(1, int(max_nodes)),
            error_flag)
    pair = None if _eager.compiling() else _eager.fast.latent_attention(*args, bool(return_lse))
    if pair is None:
        plain = direct(q_latent, q_rope, pool, block_table, context_lens, q_indptr, tree_mask)
        pair = _attend(*args, return_lse) if plain else torch.ops.b200kv.latent_attention(*args)
    out, lse = pair
    return (out, lse) if return_lse else out


def _check_heads(t: torch.Tensor, name: str, like: torch.Tensor, rows: int, width: int) -> None:
    if t.dim() != 3 or t.shape != (rows, like.shape[1], width) or t.dtype != like.dtype or t.stride(2) != 1 \
            or t.device != like.device:
        raise ValueError(f"{name} must be [{rows}, {like.shape[1]}, {width}] of q's dtype with contiguous rows on its "
                         f"device, got {tuple(t.shape)} {t.dtype}")


def _latent_prompt_attention_impl(
    q: torch.Tensor,
    k_nope: torch.Tensor,
    k_rope: torch.Tensor,
    v: torch.Tensor,
    q_indptr: torch.Tensor,
    kv_indptr: torch.Tensor,
    scale: float,
    causal: bool,
    error_flag: Optional[torch.Tensor],
) -> tuple[torch.Tensor, torch.Tensor]:
    return _attend_prompt(q, k_nope, k_rope, v, q_indptr, kv_indptr, scale, causal, error_flag, True)


def _attend_prompt(q, k_nope, k_rope, v, q_indptr, kv_indptr, scale, causal, error_flag, want_lse):
    _require_cuda(q, k_nope, k_rope, v, q_indptr, kv_indptr)
    if q.dim() != 3 or q.shape[2] != NOPE + ROPE or q.dtype not in DTYPES_16 or q.stride(2) != 1:
        raise ValueError(f"q must be fp16 or bf16 [N, H, {NOPE + ROPE}] with contiguous rows, got {tuple(q.shape)} {q.dtype}")
    N, H, _ = q.shape
    M, device, dtype = k_nope.shape[0], q.device, q.dtype
    _check_heads(k_nope, "k_nope", q, M, NOPE)
    _check_heads(v, "v", q, M, NOPE)
    if k_rope.shape != (M, ROPE) or k_rope.dtype != dtype or k_rope.stride(1) != 1 or k_rope.device != device:
        raise ValueError(f"k_rope must be [{M}, {ROPE}] of q's dtype with contiguous rows on its device, got "
                         f"{tuple(k_rope.shape)} {k_rope.dtype}")
    B = q_indptr.shape[0] - 1 if q_indptr.dim() == 1 else -1
    if B < 0:
        raise ValueError("q_indptr must be int32 [B + 1]")
    for indptr, name in ((q_indptr, "q_indptr"), (kv_indptr, "kv_indptr")):
        if indptr.dtype != torch.int32 or indptr.shape != (B + 1,) or not indptr.is_contiguous() \
                or indptr.device != device:
            raise ValueError(f"{name} must be a contiguous int32 [{B + 1}] tensor on q's device")
    out = torch.empty((N, H, NOPE), dtype=dtype, device=device)
    lse = torch.empty((N, H), dtype=torch.float32, device=device) if want_lse else None
    if N == 0:
        return out, lse
    wbytes = _lib.lib().b200kv_prompt_workspace_bytes(N, M, B, H)
    ws = workspace_for(device, wbytes) if wbytes > 0 else torch.empty(0, dtype=torch.uint8, device=device)
    if wbytes > 0:
        _eager.fast.set_workspace(ws)
    launch("b200kv_latent_prompt_attention", device, q.data_ptr(), q.stride(0), q.stride(1), k_nope.data_ptr(),
           k_nope.stride(0), k_nope.stride(1), k_rope.data_ptr(), k_rope.stride(0), v.data_ptr(), v.stride(0), v.stride(1),
           DTYPE_CODES[dtype], q_indptr.data_ptr(), kv_indptr.data_ptr(), out.data_ptr(), _ptr(lse), N, M, B, H, scale,
           causal, ws.data_ptr(), ws.numel(), flag_ptr(error_flag, device))
    _maybe_check_flag(error_flag, "latent_prompt_attention")
    return out, lse


_latent_prompt_attention_op = torch.library.custom_op("b200kv::latent_prompt_attention", _latent_prompt_attention_impl,
                                                      mutates_args=(), device_types="cuda")


@_latent_prompt_attention_op.register_fake
def _(q, k_nope, k_rope, v, q_indptr, kv_indptr, scale, causal, error_flag):
    return q.new_empty((*q.shape[:2], NOPE)), q.new_empty(q.shape[:2], dtype=torch.float32)


def latent_prompt_attention(
    q: torch.Tensor,
    k_nope: torch.Tensor,
    k_rope: torch.Tensor,
    v: torch.Tensor,
    q_indptr: torch.Tensor,
    kv_indptr: torch.Tensor,
    scale: Optional[float] = None,
    causal: bool = True,
    return_lse: bool = False,
    error_flag: Optional[torch.Tensor] = None,
):
    """Attention of prompts (or chunks of them), expanded form: each head has keys and
    values of its own, multiplied out of the latent rows, and all share k_rope.

    q [N, H, 192] (128 own, 64 rotary), k_nope and v [M, H, 128] (halves of one
    product will do: strides are free), k_rope [M, 64], all fp16 or all bf16.
    Sequence b has rows q_indptr[b] .. q_indptr[b + 1] - 1 and tokens kv_indptr[b] ..
    kv_indptr[b + 1] - 1 (int32 [B + 1] both); its rows are the last of its tokens, so
    with ``causal`` row i of n sees the first m - n + i + 1 of m.  Without, all of
    them: the past of a chunk, read back by :func:`latent_load`, whose result and
    log-sum-exps :func:`torch_spyre_b200.merge_attention_states` joins with the
    chunk's own.  Returns out [N, H, 128] (and the natural-log LSE [N, H] fp32); a
    row that sees nothing gets zeros and -inf.  scale defaults to 1 / sqrt(192)."""
    if scale is None:
        scale = 1.0 / math.sqrt(NOPE + ROPE)
    args = (q, k_nope, k_rope, v, q_indptr, kv_indptr, float(scale), bool(causal), error_flag)
    pair = None if _eager.compiling() else _eager.fast.latent_prompt_attention(*args, bool(return_lse))
    if pair is None:
        plain = direct(q, k_nope, k_rope, v, q_indptr, kv_indptr)
        pair = _attend_prompt(*args, return_lse) if plain else torch.ops.b200kv.latent_prompt_attention(*args)
    out, lse = pair
    return (out, lse) if return_lse else out
