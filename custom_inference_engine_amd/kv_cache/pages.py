"""Block tables and slot maps from request lengths, on the GPU.

``step_maps`` derives what a packed step needs from its slots and new-token counts: the
packed offsets, and each row's slot, position, page and in-page offset (the index recipe of
the reference's mixed step, scheduler/mixed_module.py:99-132, one launch).  With a free
list it first gives every sequence the pages that its new tokens need, so that block tables
are kept on the device, inside a captured step if need be; ``release_pages`` gives pages
back: a finished request's, or those past the tokens that are kept.

A free list (``new_free_list``) is one int64 tensor: the count of free pages, a word of the
kernels' own, and the pages, the next one last.  Its calls follow one another: two that
overlap on different streams would hand out the same pages.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .quant import int64_index, int64_table, launch, one_device

_I64 = torch.int64
ERR_FREE = 32  # CIE_ERRBIT_FREE
MAX_SEQUENCES = 2048  # of a call


class StepMaps(NamedTuple):
    """A packed step: ``cu_seqlens`` (B + 1), and a value for each row, zeros behind the last sequence."""

    cu_seqlens: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    pages: torch.Tensor
    offsets: torch.Tensor


def new_free_list(n_pages: int, device) -> torch.Tensor:
    """The free list of a pool whose pages are all free but page 0, the padding rows'; the lowest is handed out first."""
    if n_pages < 1:
        raise AssertionError("a pool has at least page 0")
    out = torch.zeros(n_pages + 2, dtype=_I64)
    out[0] = n_pages - 1
    out[2:n_pages + 1] = torch.arange(n_pages - 1, 0, -1)
    return out.to(device)


def _check_state(lens, block_table, free_list) -> int:
    """What a call that changes tables asks of them; the pool's pages."""
    if block_table.dtype != _I64 or block_table.dim() != 2 or block_table.stride(1) != 1:
        raise AssertionError("block_table must be int64 (n_slots, pages) with dense rows")
    if lens.dtype != _I64 or lens.dim() != 1 or not lens.is_contiguous():
        raise AssertionError("lens must be contiguous int64 (n_slots,)")
    if free_list.dtype != _I64 or free_list.dim() != 1 or not free_list.is_contiguous() or free_list.shape[0] < 3:
        raise AssertionError("free_list must come from new_free_list")
    return free_list.shape[0] - 2


def step_maps(slot_ids, new_tokens, lens, block_table, page_size: int, total_T: int,
              free_list: Optional[torch.Tensor] = None, out: Optional[StepMaps] = None, err=None) -> StepMaps:
    """The maps of a step of ``total_T`` rows: sequence b feeds ``new_tokens[b]`` tokens to slot ``slot_ids[b]``.

    ``lens`` (n_slots,) are the tokens held, not advanced here; ``block_table`` (n_slots,
    pages).  With ``free_list`` each sequence (of a slot other than the padding slot 0)
    first gets the pages that its new tokens need, in order; a slot may then come once.
    Where the list has too few for all of them, none gets any (CIE_ERRBIT_FREE in
    ``err``), and rows without a page are mapped to page 0.  ``out``: tensors to write
    to, as this function returns them.
    """
    if slot_ids.dim() != 1 or new_tokens.shape != slot_ids.shape:
        raise AssertionError("slot_ids and new_tokens must have one entry per sequence")
    if lens.dim() != 1 or block_table.dim() != 2:
        raise AssertionError("lens must be (n_slots,) and block_table (n_slots, pages)")
    if total_T < 0 or page_size < 1:
        raise AssertionError("total_T must be >= 0 and page_size positive")
    B = slot_ids.shape[0]
    if out is not None:
        for t, n in zip(out, (B + 1,) + (total_T,) * 4):
            if t.dtype != _I64 or t.shape != (n,) or not t.is_contiguous():
                raise AssertionError("out must be contiguous int64: cu_seqlens (B + 1,), the others (total_T,)")
    n_pages, pages = 0, None
    if free_list is not None:
        n_pages = _check_state(lens, block_table, free_list)
        pages = free_list.data_ptr()
        dev = one_device(slot_ids, new_tokens, lens, block_table, free_list)
    else:
        dev = one_device(slot_ids, new_tokens, lens, block_table)
        lens, block_table = int64_index(lens), int64_table(block_table)
    slot_ids, new_tokens = int64_index(slot_ids), int64_index(new_tokens)
    if out is None:
        room = torch.empty(B + 1 + 4 * total_T, dtype=_I64, device=dev)  # (one allocation: half the time of five)
        out = StepMaps(*room.split_with_sizes((B + 1, total_T, total_T, total_T, total_T)))
    else:
        one_device(slot_ids, *out)
    n_slots, width = block_table.shape
    cu, slots, positions, rows_pages, offsets = out
    launch(dev, "cie_step_maps", cu.data_ptr(), slots.data_ptr(), positions.data_ptr(), rows_pages.data_ptr(),
           offsets.data_ptr(), slot_ids.data_ptr(), new_tokens.data_ptr(), lens.data_ptr(), block_table.data_ptr(),
           pages, B, total_T, page_size, n_pages, block_table.stride(0), width, min(lens.shape[0], n_slots), err=err)
    return out


def _tokens(t: torch.Tensor, slot_ids: torch.Tensor) -> torch.Tensor:
    if t.shape != slot_ids.shape:
        raise AssertionError("keep and held must have one entry per sequence")
    one_device(slot_ids, t)
    return int64_index(t)


def release_pages(free_list, slot_ids, lens, block_table, page_size: int, keep=None, held=None, err=None) -> None:
    """Gives the pages of ``slot_ids`` back to the free list, but for the first ``keep[b]`` tokens' (none by default).

    ``lens[slot]`` becomes ``keep[b]`` and the released table entries 0.  ``held[b]``: the
    tokens whose pages the sequence has, where these are more than ``lens[slot]``: after
    a ``step_maps`` whose tokens ``lens`` does not count yet (keep = those of them that
    stay).  A slot comes once, or nothing is done (CIE_ERRBIT_FREE in ``err``).  Table
    entries that hold no page (0) are not given back (CIE_ERRBIT_PAGE).
    """
    n_pages = _check_state(lens, block_table, free_list)
    if slot_ids.dim() != 1 or page_size < 1:
        raise AssertionError("slot_ids must be (B,) and page_size positive")
    dev = one_device(free_list, slot_ids, lens, block_table)
    if keep is not None:
        keep = _tokens(keep, slot_ids)
    if held is not None:
        held = _tokens(held, slot_ids)
    slot_ids = int64_index(slot_ids)
    launch(dev, "cie_release_pages", free_list.data_ptr(), slot_ids.data_ptr(), lens.data_ptr(),
           block_table.data_ptr(), None if keep is None else keep.data_ptr(),
           None if held is None else held.data_ptr(), slot_ids.shape[0], page_size,
           n_pages, block_table.stride(0), block_table.shape[1], min(lens.shape[0], block_table.shape[0]), err=err)
