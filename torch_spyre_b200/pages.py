"""A step's block tables, slots and positions, made on the GPU from the requests'
lengths: no length, page or slot passes through the host.

Free pages are a stack of block ids, ``free_pages`` int32 [capacity], of which the
first ``free_count`` int32 [1] are free; sequence b owns the first ``page_counts[b]``
entries of its row of the block table.

* ``b200kv::extend_pages(block_table!, page_counts!, free_pages, free_count!, ...)``
  -- pages for the tokens a step adds, and the tokens' slots and positions;
* ``b200kv::release_pages(block_table!, page_counts!, free_pages!, free_count!, keep_lens)``
  -- the pages past the tokens that are kept go back to the stack.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _eager
from ._eager import direct, flag_ptr, launch, written
from .ops import _maybe_check_flag, _ptr, _require_cuda


def _check_vector(t: torch.Tensor, name: str, n: Optional[int], device: torch.device,
                  dtype: torch.dtype = torch.int32) -> None:
    if t.dtype != dtype or t.dim() != 1 or (n is not None and len(t) != n) or not t.is_contiguous() or t.device != device:
        size = "[n]" if n is None else f"[{n}]"
        raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} {size} tensor on the block table's device, "
                         f"got {tuple(t.shape)} {t.dtype} on {t.device}")


def _check_state(block_table, page_counts, free_pages, free_count) -> tuple[int, torch.device]:
    _require_cuda(block_table, page_counts, free_pages, free_count)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError("block_table must be int32 [B, max_blocks] with unit column stride")
    B, device = block_table.shape[0], block_table.device
    _check_vector(page_counts, "page_counts", B, device)
    _check_vector(free_pages, "free_pages", None, device)
    _check_vector(free_count, "free_count", 1, device)
    return B, device


def _table_args(block_table):
    # a table of one row may have any stride
    stride = block_table.stride(0) if block_table.shape[0] > 1 else block_table.shape[1]
    return block_table.data_ptr(), stride


def _extend_pages_impl(
    block_table: torch.Tensor,
    page_counts: torch.Tensor,
    free_pages: torch.Tensor,
    free_count: torch.Tensor,
    context_lens: torch.Tensor,
    q_indptr: torch.Tensor,
    num_tokens: int,
    tree_mask: Optional[torch.Tensor],
    error_flag: Optional[torch.Tensor],
) -> tuple[torch.Tensor, torch.Tensor]:
    B, device = _check_state(block_table, page_counts, free_pages, free_count)
    _check_vector(context_lens, "context_lens", B, device)
    _check_vector(q_indptr, "q_indptr", B + 1, device)
    if num_tokens < 0:
        raise ValueError(f"num_tokens must be >= 0, got {num_tokens}")
    words = 0
    if tree_mask is not None:
        if tree_mask.dtype != torch.int64 or tree_mask.dim() != 2 or len(tree_mask) != num_tokens \
                or not tree_mask.is_contiguous() or tree_mask.device != device:
            raise ValueError("tree_mask must be a contiguous int64 [num_tokens, words] tensor on the block table's device")
        words = tree_mask.shape[1]
    slots = torch.empty(num_tokens, dtype=torch.int64, device=device)
    positions = torch.empty(num_tokens, dtype=torch.int32, device=device)
    launch("b200kv_extend_pages", device, *_table_args(block_table), page_counts.data_ptr(), free_pages.data_ptr(),
           free_pages.shape[0], free_count.data_ptr(), context_lens.data_ptr(), q_indptr.data_ptr(), _ptr(tree_mask),
           words, slots.data_ptr(), positions.data_ptr(), num_tokens, B, block_table.shape[1],
           flag_ptr(error_flag, device))
    _maybe_check_flag(error_flag, "extend_pages")
    return slots, positions


_extend_pages_op = torch.library.custom_op("b200kv::extend_pages", _extend_pages_impl, device_types="cuda",
                                           mutates_args=("block_table", "page_counts", "free_count"))


@_extend_pages_op.register_fake
def _(block_table, page_counts, free_pages, free_count, context_lens, q_indptr, num_tokens, tree_mask, error_flag):
    return (block_table.new_empty(num_tokens, dtype=torch.int64), block_table.new_empty(num_tokens, dtype=torch.int32))


def extend_pages(
    block_table: torch.Tensor,
    page_counts: torch.Tensor,
    free_pages: torch.Tensor,
    free_count: torch.Tensor,
    context_lens: torch.Tensor,
    q_indptr: torch.Tensor,
    num_tokens: int,
    tree_mask: Optional[torch.Tensor] = None,
    error_flag: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """(slots int64 [num_tokens], positions int32 [num_tokens]) of the tokens that
    sequence b adds behind its context_lens[b], q_indptr[b] .. q_indptr[b + 1] - 1.

    Pages that are missing are taken from the top of the stack, in the order of
    the sequences; the table, page_counts and free_count follow in place.  A
    token's position is its sequence's length plus its index, or with
    ``tree_mask`` (:func:`torch_spyre_b200.tree_mask`) plus its depth.  Tokens that
    got no page have slot -1, which :func:`torch_spyre_b200.kv_store` skips
    (``DEVERR_NO_PAGES``); so have those of a sequence whose length is negative or
    past its row of the table, which takes no page (``DEVERR_BAD_LEN``)."""
    args = (block_table, page_counts, free_pages, free_count, context_lens, q_indptr, int(num_tokens), tree_mask,
            error_flag)
    pair = None if _eager.compiling() else _eager.fast.extend_pages(*args)
    if pair is None:
        if not direct(block_table, page_counts, free_pages, free_count, context_lens, q_indptr, tree_mask):
            return torch.ops.b200kv.extend_pages(*args)
        pair = _extend_pages_impl(*args)
        written(block_table, page_counts, free_count)
    return pair


def _release_pages_impl(block_table: torch.Tensor, page_counts: torch.Tensor, free_pages: torch.Tensor,
                        free_count: torch.Tensor, keep_lens: torch.Tensor, error_flag: Optional[torch.Tensor]) -> None:
    B, device = _check_state(block_table, page_counts, free_pages, free_count)
    _check_vector(keep_lens, "keep_lens", B, device)
    launch("b200kv_release_pages", device, *_table_args(block_table), page_counts.data_ptr(), free_pages.data_ptr(),
           free_pages.shape[0], free_count.data_ptr(), keep_lens.data_ptr(), B, block_table.shape[1],
           flag_ptr(error_flag, device))
    _maybe_check_flag(error_flag, "release_pages")


_release_pages_op = torch.library.custom_op("b200kv::release_pages", _release_pages_impl, device_types="cuda",
                                            mutates_args=("block_table", "page_counts", "free_pages", "free_count"))


@_release_pages_op.register_fake
def _(block_table, page_counts, free_pages, free_count, keep_lens, error_flag):
    return None


def release_pages(block_table: torch.Tensor, page_counts: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor, keep_lens: torch.Tensor, error_flag: Optional[torch.Tensor] = None) -> None:
    """Gives the pages past ceil(keep_lens[b] / 64) of every sequence back to the
    stack, in place (keep_lens int32 [B]; 0 for a sequence that ends): after
    :func:`torch_spyre_b200.tree_commit` those that held rejected drafts.  Their
    table entries become -1.  An :func:`extend_pages` that is released whole
    leaves the stack as it was."""
    args = (block_table, page_counts, free_pages, free_count, keep_lens, error_flag)
    if not _eager.compiling() and _eager.fast.release_pages(*args):
        return
    if direct(block_table, page_counts, free_pages, free_count, keep_lens):
        _release_pages_impl(*args)
        written(block_table, page_counts, free_pages, free_count)
    else:
        torch.ops.b200kv.release_pages(*args)
