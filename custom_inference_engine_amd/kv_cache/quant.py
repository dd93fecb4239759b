"""The 8-bit paged cache: quantising rows as they are written, and reading them back.

Beside ``kv_append_decode`` / ``kv_append_tokens`` of ``storage.py``, for pools of
``torch.float8_e4m3fn`` (``KVStorage(..., dtype=torch.float8_e4m3fn)``).  Every block
of 16 tokens of one kv head has a scale for its K rows and one for its V rows:
``scales`` is (n_pages, H_kv, page_size // 16, 2) float32, ``[..., 0]`` K's, ``[..., 1]``
V's, and a held value is ``pool.float() * scale``.

A scale is a power of two, 2^e with -15 <= e <= 8: the least with amax <= 448 * 2^e
over the rows written since the block's first row was.  Writing a block's row 0
starts it anew; writing another row keeps the others, which are rounded again where
the scale grows.  Rows are rounded to nearest even from their float16 inputs (the
error is at most 2^-4 of a value, or half of 2^-9 * scale under 2^-6 * scale);
values beyond +-61440, infinities among them, are held as that, NaN as NaN.  So a
held value is always a float16 value, and ``kv_read_tokens_q8`` and the attention of
``attn/quant.py`` use it exactly.
"""
from __future__ import annotations

import contextlib

import torch

from .. import _native

BLOCK = 16  # tokens that share a scale


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise AssertionError(msg)


def check_cache_q8(k: torch.Tensor, v: torch.Tensor, scales: torch.Tensor) -> None:
    """What every operator on an 8-bit cache asks of its pools and scales."""
    _require(k.dim() == 4 and k.shape == v.shape, "K/V pools must be (n_pages, H_kv, page_size, D)")
    _require(k.dtype == torch.float8_e4m3fn and v.dtype == torch.float8_e4m3fn, "K/V pools must be float8_e4m3fn")
    n_pages, h_kv, page_size, d = k.shape
    st = k.stride()
    _require(st == v.stride() and st[3] == 1 and st[2] == d,
             "K/V pools need identical strides with dense (page_size, D) rows")
    _require(page_size % BLOCK == 0, "page_size must be a multiple of 16")
    _require(tuple(scales.shape) == (n_pages, h_kv, page_size // BLOCK, 2) and scales.dtype == torch.float32
             and scales.is_contiguous(), "scales must be contiguous float32 (n_pages, H_kv, page_size // 16, 2)")


def on_device(dev: torch.device):
    """The tensors' device made current for a launch (no cost where it already is)."""
    if dev.index is None or dev.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def int64_index(t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.int64 or not t.is_contiguous():
        t = t.to(torch.int64).contiguous()
    return t


def int64_table(bt: torch.Tensor) -> torch.Tensor:
    if bt.dtype != torch.int64 or bt.stride(1) != 1:
        bt = bt.to(torch.int64).contiguous()
    return bt


def new_rows(x: torch.Tensor, h_kv: int, d: int) -> torch.Tensor:
    """New K or V as (rows, H_kv, D) that the kernels can read in 16-byte pieces."""
    _require(x.dtype == torch.float16, "new K/V must be float16")
    try:
        rows = x.view(-1, h_kv, d)
    except RuntimeError:
        rows = x.reshape(-1, h_kv, d)
    if rows.stride(2) != 1 or rows.stride(0) % 8 or rows.stride(1) % 8 or rows.data_ptr() % 16:
        rows = rows.contiguous()
    if rows.data_ptr() % 16:  # (contiguous already, at an odd address)
        rows = rows.clone()
    return rows


def kv_append_decode_q8(k_cache, v_cache, scales, k, v, slot_ids, lens, block_table, err=None) -> None:
    """``kv_append_decode`` into an 8-bit cache: row b goes to position ``lens[slot_ids[b]]`` of its slot.

    ``lens`` is the pool's per-slot length (n_slots,).  Slots other than the
    padding slot must not share the page they append to; of a slot that comes
    several times the last row is written.
    """
    check_cache_q8(k_cache, v_cache, scales)
    n_pages, h_kv, page_size, d = k_cache.shape
    dev = _native.require_device(k_cache, v_cache, scales, k, v, slot_ids, lens, block_table)
    kr, vr = new_rows(k, h_kv, d), new_rows(v, h_kv, d)
    slot_ids, lens, block_table = int64_index(slot_ids), int64_index(lens), int64_table(block_table)
    B = slot_ids.shape[0]
    _require(kr.shape[0] == B and vr.shape[0] == B, f"expected {B} new rows, got {kr.shape[0]} / {vr.shape[0]}")
    if B == 0:
        return
    lib = _native.load()
    with on_device(dev):
        _native.check(
            lib.cie_q8_append_decode(
                k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr(), kr.data_ptr(), vr.data_ptr(),
                kr.stride(0), kr.stride(1), vr.stride(0), vr.stride(1),
                slot_ids.data_ptr(), lens.data_ptr(), block_table.data_ptr(),
                B, h_kv, page_size, d, n_pages, k_cache.stride(0), k_cache.stride(1),
                block_table.stride(0), block_table.shape[1], min(lens.shape[0], block_table.shape[0]),
                _native.ptr(err), _native.stream_handle(dev),
            ),
            "cie_q8_append_decode",
        )


def kv_append_tokens_q8(k_cache, v_cache, scales, k, v, pages, offsets, err=None) -> None:
    """``kv_append_tokens`` into an 8-bit cache: row t goes to ``(pages[t], :, offsets[t])``.

    Rows in any order; of an index that comes several times the last row is written.
    """
    check_cache_q8(k_cache, v_cache, scales)
    n_pages, h_kv, page_size, d = k_cache.shape
    dev = _native.require_device(k_cache, v_cache, scales, k, v, pages, offsets)
    kr, vr = new_rows(k, h_kv, d), new_rows(v, h_kv, d)
    pages, offsets = int64_index(pages), int64_index(offsets)
    T = pages.shape[0]
    _require(offsets.shape[0] == T and kr.shape[0] == T and vr.shape[0] == T,
             "pages, offsets and new K/V must have one row per token")
    if T == 0:
        return
    lib = _native.load()
    with on_device(dev):
        _native.check(
            lib.cie_q8_append_tokens(
                k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr(), kr.data_ptr(), vr.data_ptr(),
                kr.stride(0), kr.stride(1), vr.stride(0), vr.stride(1),
                pages.data_ptr(), offsets.data_ptr(), T, h_kv, page_size, d, n_pages,
                k_cache.stride(0), k_cache.stride(1), _native.ptr(err), _native.stream_handle(dev),
            ),
            "cie_q8_append_tokens",
        )


def kv_read_tokens_q8(k_cache, v_cache, scales, pages, offsets, err=None):
    """The cached rows ``(pages[t], :, offsets[t])`` as float16: two tensors (1, T, H_kv, D).

    The values are the cache's own, exactly.  A bad index reads as zeros and is
    reported in ``err``.
    """
    check_cache_q8(k_cache, v_cache, scales)
    n_pages, h_kv, page_size, d = k_cache.shape
    dev = _native.require_device(k_cache, v_cache, scales, pages, offsets)
    pages, offsets = int64_index(pages), int64_index(offsets)
    T = pages.shape[0]
    _require(tuple(pages.shape) == (T,) and tuple(offsets.shape) == (T,), "pages / offsets must be (T,)")
    k = torch.empty((1, T, h_kv, d), dtype=torch.float16, device=dev)
    v = torch.empty_like(k)
    if T == 0:
        return k, v
    lib = _native.load()
    with on_device(dev):
        _native.check(
            lib.cie_q8_read_tokens(
                k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr(),
                pages.data_ptr(), offsets.data_ptr(), T, h_kv, page_size, d, n_pages,
                k_cache.stride(0), k_cache.stride(1), _native.ptr(err), _native.stream_handle(dev),
            ),
            "cie_q8_read_tokens",
        )
    return k, v


@torch.library.custom_op("inference::kv_append_decode_q8", mutates_args=("k_cache", "v_cache", "scales"))
def kv_append_decode_q8_op(
    k_cache: torch.Tensor, v_cache: torch.Tensor, scales: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
    slot_ids: torch.Tensor, lens: torch.Tensor, block_table: torch.Tensor,
) -> None:
    kv_append_decode_q8(k_cache, v_cache, scales, k, v, slot_ids, lens, block_table)


@kv_append_decode_q8_op.register_fake
def _(k_cache, v_cache, scales, k, v, slot_ids, lens, block_table) -> None:
    return None


@torch.library.custom_op("inference::kv_append_tokens_q8", mutates_args=("k_cache", "v_cache", "scales"))
def kv_append_tokens_q8_op(
    k_cache: torch.Tensor, v_cache: torch.Tensor, scales: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
    pages: torch.Tensor, offsets: torch.Tensor,
) -> None:
    kv_append_tokens_q8(k_cache, v_cache, scales, k, v, pages, offsets)


@kv_append_tokens_q8_op.register_fake
def _(k_cache, v_cache, scales, k, v, pages, offsets) -> None:
    return None
