"""The 8-bit paged cache: quantising rows as they are written, and reading them back.

Beside ``kv_append_decode`` / ``kv_append_tokens`` of ``storage.py``, for pools of
``torch.float8_e4m3fn`` (``KVStorage(..., dtype=torch.float8_e4m3fn)``).  Every block
of 16 tokens of one kv head has a scale for its K rows and one for its V rows:
``scales`` is (n_pages, H_kv, page_size // 16, 2) float32, ``[..., 0]`` K's, ``[..., 1]``
V's, and a held value is ``pool.float() * scale``.

A scale is a power of two, 2^e with -15 <= e <= 8: the least with amax <= 448 * 2^e
over the rows written since the block's first row was.  Writing a block's row 0
starts it anew; writing another row keeps the others, which are rounded again where
the scale grows.  Rows are rounded to nearest even from their float16 inputs: off by
2^-4 of the value, or by half a step of 2^-9 * scale under 2^-6 * scale, at most.  Each
growth may round what lies under 2^-6 of the new scale once more, by half of its step,
and as the steps double at least these add up to less than a step of the last scale:
after any growths a value x is held to 2^-4 |x| + 2^-9 * scale, and values far under
the block's largest may be held as 0.  Values beyond +-61440, infinities among them,
are held as that, NaN as NaN.  So a held value is always a float16 value, and ``kv_read_tokens_q8`` and the attention of
``attn/quant.py`` use it exactly.
"""
from __future__ import annotations

import contextlib

import torch

from .. import _native

BLOCK = 16  # tokens that share a scale
_F16, _F8, _F32, _I64 = torch.float16, torch.float8_e4m3fn, torch.float32, torch.int64
_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise AssertionError(msg)


def check_cache_q8(k: torch.Tensor, v: torch.Tensor, scales: torch.Tensor):
    """What every operator on an 8-bit cache asks of its pools and scales; the pools' shape and strides."""
    shape, st = k.shape, k.stride()
    if len(shape) != 4 or v.shape != shape:
        raise AssertionError("K/V pools must be (n_pages, H_kv, page_size, D)")
    if k.dtype != _F8 or v.dtype != _F8:
        raise AssertionError("K/V pools must be float8_e4m3fn")
    n_pages, h_kv, page_size, d = shape
    if v.stride() != st or st[3] != 1 or st[2] != d:
        raise AssertionError("K/V pools need identical strides with dense (page_size, D) rows")
    if page_size % BLOCK:
        raise AssertionError("page_size must be a multiple of 16")
    if (scales.shape != (n_pages, h_kv, page_size // BLOCK, 2) or scales.dtype != _F32
            or not scales.is_contiguous()):
        raise AssertionError("scales must be contiguous float32 (n_pages, H_kv, page_size // 16, 2)")
    return shape, st


def one_device(*tensors: torch.Tensor) -> torch.device:
    """The one HIP device of all tensors (there is no CPU path)."""
    index = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != index or index < 0:
            return _native.require_device(*tensors)  # (it says which)
    return tensors[0].device


def launch(dev: torch.device, name: str, *args, err=None) -> None:
    """One call of the C entry ``name`` on the device's current stream, with that device current."""
    fn = getattr(_native.load(), name)
    index = dev.index
    if err is not None and (err.dtype != torch.int32 or err.get_device() != index):
        raise AssertionError("err must be an int32 tensor on the operator's device")
    err = None if err is None else err.data_ptr()
    if index == _current_device():
        status = fn(*args, err, _current_stream(index))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, err, _current_stream(index))
    if status:
        _native.check(status, name)


def int64_index(t: torch.Tensor) -> torch.Tensor:
    if t.dtype != _I64 or not t.is_contiguous():
        t = t.to(_I64).contiguous()
    return t


def int64_table(bt: torch.Tensor) -> torch.Tensor:
    if bt.dtype != _I64 or bt.stride(1) != 1:
        bt = bt.to(_I64).contiguous()
    return bt


def new_rows(x: torch.Tensor, n: int, h_kv: int, d: int):
    """New K or V as n rows (H_kv, D) that the kernels can read in 16-byte pieces: the tensor that holds them
    (the caller's, or a copy), and the strides of its rows and heads."""
    if x.dtype != _F16:
        raise AssertionError("new K/V must be float16")
    shape = x.shape
    if shape != (1, n, h_kv, d) and shape != (n, h_kv, d):
        try:
            x = x.view(-1, h_kv, d)
        except RuntimeError:
            x = x.reshape(-1, h_kv, d)
        if x.shape[0] != n:
            raise AssertionError(f"expected {n} new K/V rows, one a token, got {x.shape[0]}")
    row, head, one = x.stride()[-3:]
    if one != 1 or (row | head) & 7 or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)
        row, head, one = x.stride()[-3:]
    return x, row, head


def kv_append_decode_q8(k_cache, v_cache, scales, k, v, slot_ids, lens, block_table, err=None) -> None:
    """``kv_append_decode`` into an 8-bit cache: row b goes to position ``lens[slot_ids[b]]`` of its slot.

    ``lens`` is the pool's per-slot length (n_slots,).  Slots other than the
    padding slot must not share the page they append to; of a slot that comes
    several times the last row is written.
    """
    (n_pages, h_kv, page_size, d), (s_page, s_head, _, _) = check_cache_q8(k_cache, v_cache, scales)
    dev = one_device(k_cache, v_cache, scales, k, v, slot_ids, lens, block_table)
    B = slot_ids.shape[0]
    (k, k_row, k_head), (v, v_row, v_head) = new_rows(k, B, h_kv, d), new_rows(v, B, h_kv, d)
    slot_ids, lens, block_table = int64_index(slot_ids), int64_index(lens), int64_table(block_table)
    if B == 0:
        return
    launch(dev, "cie_q8_append_decode", k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr(), k.data_ptr(),
           v.data_ptr(), k_row, k_head, v_row, v_head, slot_ids.data_ptr(), lens.data_ptr(),
           block_table.data_ptr(), B, h_kv, page_size, d, n_pages, s_page, s_head, block_table.stride(0),
           block_table.shape[1], min(lens.shape[0], block_table.shape[0]), err=err)


def kv_append_tokens_q8(k_cache, v_cache, scales, k, v, pages, offsets, err=None) -> None:
    """``kv_append_tokens`` into an 8-bit cache: row t goes to ``(pages[t], :, offsets[t])``.

    Rows in any order; of an index that comes several times the last row is written.
    Every block's rows are looked for in the whole list, so past some 32,000 rows (63 us
    at 8 heads of 128, 1.5 times their bytes' time) that search outgrows the writing
    (262,144 rows: 1.3 ms, 4 times) and several calls, cut between sequences, take less.
    """
    (n_pages, h_kv, page_size, d), (s_page, s_head, _, _) = check_cache_q8(k_cache, v_cache, scales)
    dev = one_device(k_cache, v_cache, scales, k, v, pages, offsets)
    T = pages.shape[0]
    if pages.dim() != 1 or offsets.shape != pages.shape:
        raise AssertionError("pages and offsets must have one entry per token")
    (k, k_row, k_head), (v, v_row, v_head) = new_rows(k, T, h_kv, d), new_rows(v, T, h_kv, d)
    pages, offsets = int64_index(pages), int64_index(offsets)
    if T == 0:
        return
    launch(dev, "cie_q8_append_tokens", k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr(), k.data_ptr(),
           v.data_ptr(), k_row, k_head, v_row, v_head, pages.data_ptr(), offsets.data_ptr(), T, h_kv,
           page_size, d, n_pages, s_page, s_head, err=err)


def kv_read_tokens_q8(k_cache, v_cache, scales, pages, offsets, err=None):
    """The cached rows ``(pages[t], :, offsets[t])`` as float16: two tensors (1, T, H_kv, D).

    The values are the cache's own, exactly.  A bad index reads as zeros and is
    reported in ``err``.
    """
    (n_pages, h_kv, page_size, d), (s_page, s_head, _, _) = check_cache_q8(k_cache, v_cache, scales)
    dev = one_device(k_cache, v_cache, scales, pages, offsets)
    pages, offsets = int64_index(pages), int64_index(offsets)
    T = pages.shape[0]
    _require(pages.dim() == 1 and offsets.shape == pages.shape, "pages / offsets must be (T,)")
    k = torch.empty((1, T, h_kv, d), dtype=torch.float16, device=dev)
    v = torch.empty_like(k)
    if T == 0:
        return k, v
    launch(dev, "cie_q8_read_tokens", k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
           scales.data_ptr(), pages.data_ptr(), offsets.data_ptr(), T, h_kv, page_size, d, n_pages, s_page, s_head,
           err=err)
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
