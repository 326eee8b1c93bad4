"""Verification of drafted tokens over the paged cache.

A draft is a tree of nodes per sequence, listed with parents before children;
their K/V rows sit in the cache right after the committed tokens
(:func:`torch_spyre_b200.kv_store`).  One verify step per layer:

* ``b200kv::tree_mask(parents, q_indptr, mask_words)`` -- once per step, which
  nodes each node sees (itself and its ancestors), as bits;
* ``b200kv::tree_attention(q, k_pool, v_pool, block_table, context_lens, q_indptr, ...)``
  -- attention of all nodes over committed tokens and visible nodes; without a
  mask the nodes form a chain (several tokens of one sequence, a prompt chunk);
* ``b200kv::tree_verify(parents, tokens, q_indptr, target_probs, ...)`` -- once per
  step, the accepted path and the token that comes next, from the target's and
  the drafter's probabilities and given random numbers;
* ``b200kv::tree_commit(k_pool!, v_pool!, ...)`` -- the accepted path's rows moved
  to the end of the committed tokens.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _eager, _lib
from ._eager import direct, flag_ptr, launch, written
from .kv_rows import DTYPES_16, check_row_pools
from .ops import _maybe_check_flag, _ptr, _require_cuda, workspace_for
from .rotations import DTYPE_CODES, ROTARY_DTYPES


def _check_sequences(block_table: torch.Tensor, context_lens: torch.Tensor, device: torch.device) -> int:
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1 \
            or block_table.device != device:
        raise ValueError("block_table must be int32 [B, max_blocks] with unit column stride on the pools' device")
    if context_lens.dtype != torch.int32 or context_lens.dim() != 1 \
            or len(context_lens) != len(block_table) or not context_lens.is_contiguous() or context_lens.device != device:
        raise ValueError("context_lens must be a contiguous int32 [B] tensor on the pools' device")
    return block_table.shape[0]


def _check_indptr(q_indptr: torch.Tensor, batch: int, device: torch.device) -> None:
    if q_indptr.dtype != torch.int32 or q_indptr.dim() != 1 or len(q_indptr) != batch + 1 or not q_indptr.is_contiguous() \
            or q_indptr.device != device:
        raise ValueError("q_indptr must be a contiguous int32 [B + 1] tensor on the pools' device")


# --------------------------------------------------------------------- mask --
def _tree_mask_impl(parents: torch.Tensor, q_indptr: torch.Tensor, mask_words: int,
                    error_flag: Optional[torch.Tensor]) -> torch.Tensor:
    _require_cuda(parents, q_indptr)
    if parents.dtype != torch.int32 or parents.dim() != 1 or not parents.is_contiguous():
        raise ValueError("parents must be a contiguous int32 [N] tensor")
    if q_indptr.dim() != 1 or q_indptr.shape[0] < 1:
        raise ValueError("q_indptr must be int32 [B + 1]")
    _check_indptr(q_indptr, q_indptr.shape[0] - 1, parents.device)
    mask = torch.empty((parents.shape[0], mask_words), dtype=torch.int64, device=parents.device)
    launch("b200kv_tree_mask", parents.device, parents.data_ptr(), q_indptr.data_ptr(), q_indptr.shape[0] - 1,
           parents.shape[0], mask_words, mask.data_ptr(), flag_ptr(error_flag, parents.device))
    _maybe_check_flag(error_flag, "tree_mask")
    return mask


_tree_mask_op = torch.library.custom_op("b200kv::tree_mask", _tree_mask_impl, mutates_args=(), device_types="cuda")


@_tree_mask_op.register_fake
def _(parents, q_indptr, mask_words, error_flag):
    return parents.new_empty((parents.shape[0], mask_words), dtype=torch.int64)


def tree_mask(parents: torch.Tensor, q_indptr: torch.Tensor, max_nodes: int,
              error_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Mask bits int64 [N, ceil(max_nodes / 64)] of drafted trees: node i sees
    itself and its ancestors.  parents int32 [N] are indexes inside the node's
    own sequence (nodes q_indptr[b] .. q_indptr[b + 1] - 1), smaller than the
    node's; -1 marks a root, -2 a pruned node, which sees nothing, nor do the
    nodes that descend from it."""
    args = (parents, q_indptr, max(1, -(-int(max_nodes) // 64)), error_flag)
    mask = None if _eager.compiling() else _eager.fast.tree_mask(*args)
    if mask is None:
        mask = _tree_mask_impl(*args) if direct(parents, q_indptr) else torch.ops.b200kv.tree_mask(*args)
    return mask


# ---------------------------------------------------------------- attention --
def _tree_attention_impl(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    q_indptr: torch.Tensor,
    tree_mask: Optional[torch.Tensor],
    scale: float,
    max_nodes: int,
    k_scales: Optional[torch.Tensor],
    v_scales: Optional[torch.Tensor],
    error_flag: Optional[torch.Tensor],
) -> tuple[torch.Tensor, torch.Tensor]:
    return _attend(q, k_pool, v_pool, block_table, context_lens, q_indptr, tree_mask, scale, max_nodes, k_scales,
                   v_scales, error_flag, True)


def _attend(q, k_pool, v_pool, block_table, context_lens, q_indptr, tree_mask, scale, max_nodes, k_scales, v_scales,
            error_flag, want_lse):
    _require_cuda(q, k_pool, v_pool, block_table, context_lens, q_indptr)
    NB, Hkv, D = check_row_pools(k_pool, v_pool, k_scales, v_scales)
    device, dtype = k_pool.device, q.dtype
    if q.dim() != 3 or dtype not in DTYPES_16 or q.shape[2] != D or q.stride(2) != 1 or q.device != device:
        raise ValueError(f"q must be fp16 or bf16 [N, Hq, {D}] with a contiguous head_dim on the pools' device, "
                         f"got {tuple(q.shape)} {dtype}")
    if k_scales is None and k_pool.dtype != dtype:
        raise ValueError(f"q is {dtype}, the pools are {k_pool.dtype}")
    B = _check_sequences(block_table, context_lens, device)
    _check_indptr(q_indptr, B, device)
    N, Hq, _ = q.shape
    words = 0
    if tree_mask is not None:
        if tree_mask.dtype != torch.int64 or tree_mask.dim() != 2 or len(tree_mask) != N \
                or not tree_mask.is_contiguous() or tree_mask.device != device:
            raise ValueError("tree_mask must be a contiguous int64 [N, words] tensor on q's device")
        words = tree_mask.shape[1]
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((N, Hq), dtype=torch.float32, device=device) if want_lse else None
    if N == 0:
        return out, lse
    wbytes = _lib.lib().b200kv_tree_workspace_bytes(N, B, Hq, Hkv, D)
    # An unsupported shape has no workspace size; the call below then reports why.
    ws = workspace_for(device, wbytes) if wbytes > 0 else torch.empty(0, dtype=torch.uint8, device=device)
    if wbytes > 0:
        _eager.fast.set_workspace(ws)  # where the next call finds it
    launch(
        "b200kv_tree_attention", device, q.data_ptr(), DTYPE_CODES[dtype], q.stride(0), q.stride(1),
        k_pool.data_ptr(), v_pool.data_ptr(), DTYPE_CODES[k_pool.dtype], _ptr(k_scales), _ptr(v_scales),
        block_table.data_ptr(), block_table.stride(0), context_lens.data_ptr(), q_indptr.data_ptr(),
        _ptr(tree_mask), words, out.data_ptr(), _ptr(lse),
        N, B, Hq, Hkv, D, NB, block_table.shape[1], max_nodes, scale, ws.data_ptr(), ws.numel(),
        flag_ptr(error_flag, device),
    )
    _maybe_check_flag(error_flag, "tree_attention")
    return out, lse


_tree_attention_op = torch.library.custom_op("b200kv::tree_attention", _tree_attention_impl, mutates_args=(),
                                             device_types="cuda")


@_tree_attention_op.register_fake
def _(q, k_pool, v_pool, block_table, context_lens, q_indptr, tree_mask, scale, max_nodes, k_scales, v_scales,
      error_flag):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


def tree_attention(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    q_indptr: torch.Tensor,
    tree_mask: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    max_nodes: Optional[int] = None,
    k_scales: Optional[torch.Tensor] = None,
    v_scales: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    error_flag: Optional[torch.Tensor] = None,
):
    """Attention of the drafted nodes of every sequence over its cache.

    q [N, Hq, D] fp16 or bf16, the nodes of all sequences one after the other
    (sequence b: q_indptr[b] .. q_indptr[b + 1] - 1, int32 [B + 1]); pools of q's
    dtype, or int8 / float8_e4m3fn with ``k_scales`` / ``v_scales``; context_lens
    int32 [B] counts the committed tokens, and node i's K/V row is already in the
    cache at position context_lens[b] + i.  Every node sees all committed tokens
    and the nodes whose bit its row of ``tree_mask`` has (:func:`tree_mask`; any
    mask of this form will do); without a mask, itself and the nodes before it.
    ``max_nodes`` bounds the nodes of one sequence (default: what the mask can
    hold, or N).  Returns out [N, Hq, D] (and the natural-log LSE [N, Hq] fp32);
    a node that sees nothing gets zeros and -inf.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if max_nodes is None:
        max_nodes = q.shape[0] if tree_mask is None else min(q.shape[0], 64 * tree_mask.shape[1])
    args = (q, k_pool, v_pool, block_table, context_lens, q_indptr, tree_mask, float(scale), max(1, int(max_nodes)),
            k_scales, v_scales, error_flag)
    pair = None if _eager.compiling() else _eager.fast.tree_attention(*args, bool(return_lse))
    if pair is None:
        plain = direct(q, k_pool, v_pool, block_table, context_lens, q_indptr, tree_mask, k_scales, v_scales)
        pair = _attend(*args, return_lse) if plain else torch.ops.b200kv.tree_attention(*args)
    out, lse = pair
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------- verify --
MAX_NODES = 1024  # of a sequence


def _check_probs(probs: torch.Tensor, name: str, nodes: int, device: torch.device) -> None:
    if probs.dim() != 2 or len(probs) != nodes or probs.dtype not in ROTARY_DTYPES or probs.device != device \
            or probs.shape[1] < 1 or (probs.shape[1] > 1 and probs.stride(1) != 1):
        raise ValueError(f"{name} must be fp16, bf16 or fp32 [{nodes}, vocab] with contiguous rows on parents' device, "
                         f"got {tuple(probs.shape)} {probs.dtype}")


def _tree_verify_impl(
    parents: torch.Tensor,
    tokens: torch.Tensor,
    q_indptr: torch.Tensor,
    target_probs: torch.Tensor,
    accept_u: torch.Tensor,
    sample_u: torch.Tensor,
    draft_probs: Optional[torch.Tensor],
    max_path: int,
    error_flag: Optional[torch.Tensor],
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _require_cuda(parents, tokens, q_indptr, target_probs, accept_u, sample_u)
    if parents.dtype != torch.int32 or parents.dim() != 1 or not parents.is_contiguous():
        raise ValueError("parents must be a contiguous int32 [N] tensor")
    N, device = parents.shape[0], parents.device
    if q_indptr.dim() != 1 or q_indptr.shape[0] < 1:
        raise ValueError("q_indptr must be int32 [B + 1]")
    B = q_indptr.shape[0] - 1
    _check_indptr(q_indptr, B, device)
    for t, name, n, dtype in ((tokens, "tokens", N, torch.int64), (accept_u, "accept_u", N, torch.float32),
                              (sample_u, "sample_u", B, torch.float32)):
        if t.dtype != dtype or t.dim() != 1 or len(t) != n or not t.is_contiguous() or t.device != device:
            raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} [{n}] tensor on parents' device")
    _check_probs(target_probs, "target_probs", N, device)
    if draft_probs is not None:
        _check_probs(draft_probs, "draft_probs", N, device)
        if draft_probs.dtype != target_probs.dtype or draft_probs.shape != target_probs.shape:
            raise ValueError("draft_probs must have target_probs' dtype and shape")
    if max_path < 1:
        raise ValueError(f"max_path must be >= 1, got {max_path}")
    path = torch.empty((B, max_path), dtype=torch.int32, device=device)
    path_lens = torch.empty(B, dtype=torch.int32, device=device)
    next_tokens = torch.empty(B, dtype=torch.int64, device=device)
    launch("b200kv_tree_verify", device, parents.data_ptr(), tokens.data_ptr(), q_indptr.data_ptr(),
           target_probs.data_ptr(), target_probs.stride(0), _ptr(draft_probs),
           0 if draft_probs is None else draft_probs.stride(0), DTYPE_CODES[target_probs.dtype], accept_u.data_ptr(),
           sample_u.data_ptr(), path.data_ptr(), path_lens.data_ptr(), next_tokens.data_ptr(), N, B,
           target_probs.shape[1], max_path, flag_ptr(error_flag, device))
    _maybe_check_flag(error_flag, "tree_verify")
    return path, path_lens, next_tokens


_tree_verify_op = torch.library.custom_op("b200kv::tree_verify", _tree_verify_impl, mutates_args=(), device_types="cuda")


@_tree_verify_op.register_fake
def _(parents, tokens, q_indptr, target_probs, accept_u, sample_u, draft_probs, max_path, error_flag):
    B = q_indptr.shape[0] - 1
    return parents.new_empty((B, max_path)), parents.new_empty(B), parents.new_empty(B, dtype=torch.int64)


def tree_verify(
    parents: torch.Tensor,
    tokens: torch.Tensor,
    q_indptr: torch.Tensor,
    target_probs: torch.Tensor,
    accept_u: torch.Tensor,
    sample_u: torch.Tensor,
    draft_probs: Optional[torch.Tensor] = None,
    max_path: Optional[int] = None,
    error_flag: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted tokens stay, and what comes after them.

    Node 0 of a sequence is its last token (always taken), node i the drafted
    tokens[i] (int64 [N]) after node parents[i] (int32 [N], as for
    :func:`tree_mask`; negative: not tried).  target_probs [N, vocab] (fp16, bf16,
    fp32): the target's distribution after each node; draft_probs (same type and
    shape): the one its children were drawn from independently, None where
    they were chosen without chance (a list of likely tokens).  accept_u fp32 [N]
    and sample_u fp32 [B] are uniform random numbers in [0, 1).

    From node 0 on a node's children are tried in their order: x stays if
    u * q(x) < p(x); else p becomes max(p - q, 0) over its sum (without draft_probs:
    p without x over its sum), and the next one is tried against that.  Where none
    stays, the next token is drawn from the p of that moment.  So the
    sequence's tokens have the target's distribution, whatever the drafter's is.
    64-bit arithmetic.

    Returns path int32 [B, max_path] (the nodes that stay, 0 first, then -1; at
    most ``max_path``, default the smaller of N and 1024: the nodes of the deepest
    draft are enough), path_lens int32 [B], as :func:`tree_commit` takes them, and
    next_tokens int64 [B].  At most 1024 nodes a sequence."""
    if max_path is None:
        max_path = min(max(1, parents.shape[0]), MAX_NODES)
    args = (parents, tokens, q_indptr, target_probs, accept_u, sample_u, draft_probs, int(max_path), error_flag)
    out = None if _eager.compiling() else _eager.fast.tree_verify(*args)
    if out is None:
        op = _tree_verify_impl if direct(parents, tokens, q_indptr, target_probs, accept_u, sample_u, draft_probs) \
            else torch.ops.b200kv.tree_verify
        out = op(*args)
    return out


# ------------------------------------------------------------------- commit --
def _tree_commit_impl(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    path: torch.Tensor,
    path_lens: torch.Tensor,
    k_scales: Optional[torch.Tensor],
    v_scales: Optional[torch.Tensor],
    error_flag: Optional[torch.Tensor],
) -> torch.Tensor:
    _require_cuda(k_pool, v_pool, block_table, context_lens, path, path_lens)
    NB, Hkv, D = check_row_pools(k_pool, v_pool, k_scales, v_scales)
    device = k_pool.device
    B = _check_sequences(block_table, context_lens, device)
    if path.dtype != torch.int32 or path.dim() != 2 or len(path) != B or (path.shape[1] > 1 and path.stride(1) != 1) \
            or path.device != device:
        raise ValueError("path must be int32 [B, max_path] with unit column stride on the pools' device")
    if path_lens.dtype != torch.int32 or path_lens.dim() != 1 or len(path_lens) != B \
            or not path_lens.is_contiguous() or path_lens.device != device:
        raise ValueError("path_lens must be a contiguous int32 [B] tensor on the pools' device")
    new_lens = torch.empty_like(context_lens)
    launch(
        "b200kv_tree_commit", device,
        k_pool.data_ptr(), v_pool.data_ptr(), DTYPE_CODES[k_pool.dtype], _ptr(k_scales), _ptr(v_scales),
        block_table.data_ptr(), block_table.stride(0), context_lens.data_ptr(), path.data_ptr(),
        path.stride(0) if B > 1 else path.shape[1], path_lens.data_ptr(), new_lens.data_ptr(),
        B, Hkv, D, NB, block_table.shape[1], path.shape[1], flag_ptr(error_flag, device),
    )
    _maybe_check_flag(error_flag, "tree_commit")
    return new_lens


_tree_commit_op = torch.library.custom_op("b200kv::tree_commit", _tree_commit_impl, device_types="cuda",
                                          mutates_args=("k_pool", "v_pool", "k_scales", "v_scales"))


@_tree_commit_op.register_fake
def _(k_pool, v_pool, block_table, context_lens, path, path_lens, k_scales, v_scales, error_flag):
    return torch.empty_like(context_lens)


def tree_commit(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    path: torch.Tensor,
    path_lens: torch.Tensor,
    k_scales: Optional[torch.Tensor] = None,
    v_scales: Optional[torch.Tensor] = None,
    error_flag: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Moves the K/V rows (and scales) of the accepted nodes path[b, :path_lens[b]]
    (int32, ascending; one path expanded over the batch will do) to positions context_lens[b], context_lens[b] + 1, ... of
    their sequence, in place, and returns the new lengths
    context_lens + path_lens (int32 [B])."""
    args = (k_pool, v_pool, block_table, context_lens, path, path_lens, k_scales, v_scales, error_flag)
    new_lens = None if _eager.compiling() else _eager.fast.tree_commit(*args)
    if new_lens is None:
        if not direct(k_pool, v_pool, block_table, context_lens, path, path_lens, k_scales, v_scales):
            return torch.ops.b200kv.tree_commit(*args)
        new_lens = _tree_commit_impl(*args)
        written(k_pool, v_pool, k_scales, v_scales)
    return new_lens
