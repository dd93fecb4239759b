"""Paged GQA attention over the 8-bit cache (``kv_cache/quant.py``).

The forms of ``core.py`` with one argument more, the cache's ``scales``: decode
(plain, with the append of the new row, and from the fused QKV projection with
RoPE; on their own or from a step's ``decode_plan``, which does not depend on the
pools' type) and varlen mixed attention.  Queries, new rows and outputs are
float16; the attended values are the cache's own (byte times scale), the sums
float32, as in ``core.py``.  ``TritonQwen2Attention`` calls these where its
``KVStorage`` holds 8 bits.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from .. import _native
from ..kv_cache.quant import check_cache_q8, int64_index, int64_table, launch, new_rows, one_device
from .core import (DECODE_MAX_SPLITS, GQA_DECODE_CONFIG, _plan_workgroups, _require, default_decode_splits,
                   split_counters)


def _rows(t: torch.Tensor, n: int, width: int, what: str):
    """(1, n, width) or (n, width) float16 rows that the kernels can read: the tensor that holds them and their stride."""
    if t.dtype != torch.float16:
        raise AssertionError(f"{what} must be float16")
    shape = t.shape
    if shape != (1, n, width) and shape != (n, width):
        raise AssertionError(f"{what} must be (1, {n}, {width}), one row per token")
    row, one = t.stride()[-2:]
    if one != 1 or row & 7 or (n > 1 and row < width) or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        row = width
    return t, row if n > 1 else width


def _counters(counters: Optional[torch.Tensor], n: int, dev: torch.device) -> torch.Tensor:
    """The caller's arrival counters, or the device's own."""
    if counters is None:
        return split_counters(dev, n)
    _require(counters.dtype == torch.int32 and counters.is_contiguous() and counters.numel() >= n, "counters too small")
    _require(counters.get_device() == dev.index, "counters must be on the operator's device")
    return counters


@functools.lru_cache(maxsize=1024)
def _decode_partials_bytes(n_wg: int, H_q: int, H_kv: int, D: int) -> int:
    return _native.load().cie_paged_decode_planned_partials_bytes(n_wg, H_q, H_kv, D)


def _decode(entry, o, q_args, cache, geometry, row_args, lens, slot_ids, block_table, H_q, append, num_programs, err,
            counters, plan, dev):
    """One decode launch of the C entry ``entry`` (cie_q8_decode*): its shared arguments and buffers."""
    k, v, scales = cache
    (N_PAGES, H_kv, PAGE_SIZE, D), (s_page, s_head, _, _) = geometry
    B = slot_ids.shape[0]
    lens, slot_ids, block_table = int64_index(lens), int64_index(slot_ids), int64_table(block_table)
    n_groups = B * H_kv
    if plan is not None:  # a step's plan (decode_plan, same append mode)
        n_wg = P = _plan_workgroups(plan)
        _require(plan.get_device() == dev.index, "plan must be on the operator's device")
    else:
        P = int(num_programs) if num_programs else default_decode_splits(B, H_kv, dev)
        _require(1 <= P <= DECODE_MAX_SPLITS, "num_programs outside [1, the kernel's split limit]")
        n_wg = P * n_groups
    partials = 0
    if n_wg > n_groups:
        buffer = torch.empty(_decode_partials_bytes(n_wg, H_q, H_kv, D), dtype=torch.uint8, device=dev)
        partials = buffer.data_ptr()
        counters = _counters(counters, 2 * n_groups, dev)
    slots, width = block_table.shape
    launch(dev, entry, o.data_ptr(), *q_args, k.data_ptr(), v.data_ptr(), scales.data_ptr(), *row_args,
           lens.data_ptr(), slot_ids.data_ptr(), block_table.data_ptr(), None if plan is None else plan.data_ptr(),
           partials or None, None if counters is None else counters.data_ptr(), B, H_q, H_kv, D, PAGE_SIZE, N_PAGES,
           s_page, s_head, block_table.stride(0), width, min(lens.shape[0], slots) if append else slots, P, err=err)
    return o


def _check_decode(H_q, cache, slot_ids, block_table, rows: int):
    geometry = check_cache_q8(*cache)
    if H_q % geometry[0][1]:
        raise AssertionError("H_q must be a multiple of H_kv")
    if geometry[0][0] != block_table.shape[1]:
        raise AssertionError("block_table width must equal n_pages")
    if rows != slot_ids.shape[0]:
        raise AssertionError("decode takes one query token per sequence")
    return geometry


def _check_q(q: torch.Tensor, d: int) -> torch.Size:
    shape = q.shape
    if len(shape) != 4 or shape[0] != 1 or shape[3] != d:
        raise AssertionError("q must be (1, T, H_q, D)")
    if q.dtype != torch.float16:
        raise AssertionError("q must be float16")
    if not q.is_contiguous():
        raise AssertionError("q must be contiguous")
    return shape


def decode_gqa_attention_q8(q, k, v, scales, lens, slot_ids, block_table, num_programs=None, err=None, counters=None,
                            plan=None):
    """``decode_gqa_attention`` over an 8-bit cache: q (1, B, H_q, D) against ``lens[b]`` tokens of each slot.

    ``plan``: the step's ``decode_plan`` (``append=False``)."""
    _, B, H_q, _ = _check_q(q, k.shape[3])
    geometry = _check_decode(H_q, (k, v, scales), slot_ids, block_table, B)
    _require(lens.shape == (B,), "lens must be (B,)")
    dev = one_device(q, k, v, scales, lens, slot_ids, block_table)
    o = torch.empty_like(q)
    if B == 0:
        return o
    return _decode("cie_q8_decode", o, (q.data_ptr(),), (k, v, scales), geometry, (), lens, slot_ids, block_table, H_q, False,
                   num_programs, err, counters, plan, dev)


def decode_append_gqa_attention_q8(q, k_cache, v_cache, scales, k, v, lens, slot_ids, block_table, num_programs=None,
                                   err=None, counters=None, plan=None):
    """``decode_append_gqa_attention`` over an 8-bit cache, one launch.

    The cache and the result are those of ``kv_append_decode_q8`` followed by
    ``decode_gqa_attention_q8`` over ``lens[slot_ids] + 1`` tokens.  Slots other
    than the padding slot must be distinct."""
    _, B, H_q, D = _check_q(q, k_cache.shape[3])
    cache = (k_cache, v_cache, scales)
    geometry = _check_decode(H_q, cache, slot_ids, block_table, B)
    H_kv = geometry[0][1]
    dev = one_device(q, k_cache, v_cache, scales, k, v, lens, slot_ids, block_table)
    (k, k_row, k_head), (v, v_row, v_head) = new_rows(k, B, H_kv, D), new_rows(v, B, H_kv, D)
    o = torch.empty_like(q)
    if B == 0:
        return o
    rows = (k.data_ptr(), v.data_ptr(), k_row, k_head, v_row, v_head)
    return _decode("cie_q8_decode_append", o, (q.data_ptr(),), cache, geometry, rows, lens, slot_ids, block_table, H_q, True,
                   num_programs, err, counters, plan, dev)


def decode_qkv_rope_gqa_attention_q8(qkv, cos, sin, k_cache, v_cache, scales, lens, slot_ids, block_table,
                                     num_heads: int, num_programs=None, err=None, counters=None, plan=None):
    """``decode_qkv_rope_gqa_attention`` over an 8-bit cache, one launch.

    The new K row is rotated in float32, rounded to float16 as the float16
    cache's is, then quantised: the cache and the result are those of the split,
    ``apply_rotary_pos_emb`` and ``decode_append_gqa_attention_q8``."""
    H_q, (_, H_kv, _, D), B = int(num_heads), k_cache.shape, slot_ids.shape[0]
    cache = (k_cache, v_cache, scales)
    qkv, qkv_row = _rows(qkv, qkv.shape[-2], (H_q + 2 * H_kv) * D, "qkv")
    geometry = _check_decode(H_q, cache, slot_ids, block_table, qkv.shape[-2])
    dev = one_device(qkv, cos, sin, k_cache, v_cache, scales, lens, slot_ids, block_table)
    (cos, cos_row), (sin, sin_row) = _rows(cos, B, D, "cos"), _rows(sin, B, D, "sin")
    _require(cos_row == sin_row, "cos and sin need the same row stride")
    o = torch.empty((1, B, H_q, D), dtype=torch.float16, device=dev)
    if B == 0:
        return o
    q_args = (qkv.data_ptr(), qkv_row, cos.data_ptr(), sin.data_ptr(), cos_row)
    return _decode("cie_q8_decode_qkv_rope", o, q_args, cache, geometry, (), lens, slot_ids, block_table, H_q, True,
                   num_programs, err, counters, plan, dev)


def append_tokens_qkv_rope_q8(qkv, cos, sin, k_cache, v_cache, scales, pages, offsets, num_heads: int, err=None):
    """``append_tokens_qkv_rope`` into an 8-bit cache, one launch: returns the rotated q (1, T, H_q, D)."""
    (N_PAGES, H_kv, PAGE_SIZE, D), (s_page, s_head, _, _) = check_cache_q8(k_cache, v_cache, scales)
    H_q = int(num_heads)
    T = qkv.shape[-2]
    qkv, qkv_row = _rows(qkv, T, (H_q + 2 * H_kv) * D, "qkv")
    _require(pages.shape == (T,) and offsets.shape == (T,), "pages / offsets must be (T,)")
    dev = one_device(qkv, cos, sin, k_cache, v_cache, scales, pages, offsets)
    (cos, cos_row), (sin, sin_row) = _rows(cos, T, D, "cos"), _rows(sin, T, D, "sin")
    _require(cos_row == sin_row, "cos and sin need the same row stride")
    pages, offsets = int64_index(pages), int64_index(offsets)
    q = torch.empty((1, T, H_q, D), dtype=torch.float16, device=dev)
    if T == 0:
        return q
    launch(dev, "cie_q8_append_tokens_qkv_rope", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
           scales.data_ptr(), qkv.data_ptr(), qkv_row, cos.data_ptr(), sin.data_ptr(), cos_row,
           pages.data_ptr(), offsets.data_ptr(), T, H_q, H_kv, PAGE_SIZE, D, N_PAGES, s_page, s_head, err=err)
    return q


def mixed_plan_q8(k_cache, cu_seqlens, kv_lens, slot_ids, block_table, max_seqlen: int, total_T: int, num_heads: int,
                  err=None):
    """One mixed step's plan for ``mixed_gqa_attention_q8``, made once and used by every layer (as ``mixed_plan``).

    Returns an int32 device tensor; pass it as ``plan=`` to calls with the same
    batch, ``total_T`` (q's packed rows), heads and block table."""
    N_PAGES, H_kv, PAGE_SIZE, D = k_cache.shape
    B = slot_ids.shape[0]
    _require(num_heads % H_kv == 0, "H_q must be a multiple of H_kv")
    _require(tuple(cu_seqlens.shape) == (B + 1,) and tuple(kv_lens.shape) == (B,),
             "cu_seqlens must be (B+1,) and kv_lens (B,)")
    _require(N_PAGES == block_table.shape[1], "block_table width must equal n_pages")
    dev = one_device(k_cache, cu_seqlens, kv_lens, slot_ids, block_table)
    n = _mixed_plan_bytes(B, int(total_T), num_heads, H_kv)
    plan = torch.empty(n // 4, dtype=torch.int32, device=dev)
    _make_plan(plan.data_ptr(), n, cu_seqlens, kv_lens, slot_ids, B, total_T, max_seqlen, num_heads, k_cache.shape,
               block_table.shape[0], dev, err)
    return plan


@functools.lru_cache(maxsize=1024)
def _mixed_plan_bytes(B: int, total_T: int, H_q: int, H_kv: int) -> int:
    n = _native.load().cie_q8_mixed_plan_bytes(B, total_T, H_q, H_kv)
    _require(n > 0, "batch too large for a mixed plan")
    return n


@functools.lru_cache(maxsize=1024)
def _mixed_buffers(total_T: int, H_q: int, D: int):
    """Bytes of a call's partials, and words of its counters."""
    lib = _native.load()
    return lib.cie_q8_mixed_partials_bytes(total_T, H_q, D), lib.cie_q8_mixed_counters()


def _make_plan(plan_ptr, n_bytes, cu_seqlens, kv_lens, slot_ids, B, total_T, max_seqlen, num_heads, pool_shape, n_slots,
               dev, err):
    N_PAGES, H_kv, PAGE_SIZE, D = pool_shape
    cu_seqlens, kv_lens, slot_ids = int64_index(cu_seqlens), int64_index(kv_lens), int64_index(slot_ids)
    launch(dev, "cie_q8_mixed_plan", plan_ptr, n_bytes, cu_seqlens.data_ptr(), kv_lens.data_ptr(),
           slot_ids.data_ptr(), B, int(total_T), int(max_seqlen), num_heads, H_kv, D, PAGE_SIZE, N_PAGES,
           n_slots, err=err)


def mixed_gqa_attention_q8(q, k, v, scales, max_seqlen: int, cu_seqlens, kv_lens, slot_ids, block_table, err=None,
                           counters=None, plan=None):
    """``mixed_gqa_attention`` over an 8-bit cache: row i of sequence b attends keys [0, kv_lens[b] + i].

    q (1, total_T, H_q, D); rows outside every sequence, and those at or past
    ``max_seqlen`` in theirs (reported in ``err``), are left as
    ``torch.empty_like`` leaves them.  ``plan``: the step's ``mixed_plan_q8``;
    without one the call makes its own (a second, small launch).
    """
    _, total_T, H_q, D = _check_q(q, k.shape[3])
    (N_PAGES, H_kv, PAGE_SIZE, _), (s_page, s_head, _, _) = check_cache_q8(k, v, scales)
    B = slot_ids.shape[0]
    _require(H_q % H_kv == 0, "H_q must be a multiple of H_kv")
    _require(kv_lens.shape == (B,), "kv_lens must be (B,)")
    _require(cu_seqlens.shape == (B + 1,), "cu_seqlens must be (B+1,)")
    slots, width = block_table.shape
    _require(N_PAGES == width, "block_table width must equal n_pages")
    dev = one_device(q, k, v, scales, cu_seqlens, kv_lens, slot_ids, block_table)
    o = torch.empty_like(q)
    if B == 0 or total_T == 0 or int(max_seqlen) == 0:
        return o
    block_table = int64_table(block_table)
    plan_bytes = _mixed_plan_bytes(B, total_T, H_q, H_kv)
    n, n_ctr = _mixed_buffers(total_T, H_q, D)
    if plan is None:  # (the plan behind the partials, whose bytes are a multiple of 256)
        partials = torch.empty(n + plan_bytes, dtype=torch.uint8, device=dev)
        plan_ptr = partials.data_ptr() + n
        _make_plan(plan_ptr, plan_bytes, cu_seqlens, kv_lens, slot_ids, B, total_T, max_seqlen, H_q, k.shape, slots,
                   dev, err)
    else:
        _require(plan.dtype == torch.int32 and plan.is_contiguous() and plan.get_device() == dev.index
                 and plan.numel() * 4 >= plan_bytes, "plan must come from mixed_plan_q8 for this batch")
        partials = torch.empty(n, dtype=torch.uint8, device=dev)
        plan_ptr = plan.data_ptr()
    counters = _counters(counters, n_ctr, dev)
    launch(dev, "cie_q8_mixed", o.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), scales.data_ptr(),
           plan_ptr, plan_bytes, block_table.data_ptr(), partials.data_ptr(), n, counters.data_ptr(), B,
           total_T, H_q, H_kv, D, PAGE_SIZE, N_PAGES, s_page, s_head, block_table.stride(0), width, slots, err=err)
    return o


def _decode_config(plan):
    return {"plan": plan} if plan is not None else GQA_DECODE_CONFIG


@torch.library.custom_op("inference::gqa_decode_attention_q8", mutates_args=())
def gqa_decode_attention_q8_op(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scales: torch.Tensor,
    lens: torch.Tensor, slot_ids: torch.Tensor, block_table: torch.Tensor,
) -> torch.Tensor:
    return decode_gqa_attention_q8(q, k, v, scales, lens, slot_ids, block_table, **GQA_DECODE_CONFIG)


@gqa_decode_attention_q8_op.register_fake
def _(q, k, v, scales, lens, slot_ids, block_table):
    return torch.empty_like(q)


@torch.library.custom_op("inference::gqa_decode_append_attention_q8", mutates_args=("k_cache", "v_cache", "scales"))
def gqa_decode_append_attention_q8_op(
    q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, scales: torch.Tensor, k: torch.Tensor,
    v: torch.Tensor, lens: torch.Tensor, slot_ids: torch.Tensor, block_table: torch.Tensor,
    plan: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    return decode_append_gqa_attention_q8(q, k_cache, v_cache, scales, k, v, lens, slot_ids, block_table,
                                          **_decode_config(plan))


@gqa_decode_append_attention_q8_op.register_fake
def _(q, k_cache, v_cache, scales, k, v, lens, slot_ids, block_table, plan=None):
    return torch.empty_like(q)


@torch.library.custom_op("inference::gqa_decode_qkv_rope_attention_q8",
                         mutates_args=("k_cache", "v_cache", "scales"))
def gqa_decode_qkv_rope_attention_q8_op(
    qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    scales: torch.Tensor, lens: torch.Tensor, slot_ids: torch.Tensor, block_table: torch.Tensor,
    num_heads: int, plan: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    return decode_qkv_rope_gqa_attention_q8(qkv, cos, sin, k_cache, v_cache, scales, lens, slot_ids, block_table,
                                            num_heads, **_decode_config(plan))


@gqa_decode_qkv_rope_attention_q8_op.register_fake
def _(qkv, cos, sin, k_cache, v_cache, scales, lens, slot_ids, block_table, num_heads, plan=None):
    return qkv.new_empty((1, qkv.shape[-2], num_heads, k_cache.shape[-1]))


@torch.library.custom_op("inference::kv_append_tokens_qkv_rope_q8", mutates_args=("k_cache", "v_cache", "scales"))
def kv_append_tokens_qkv_rope_q8_op(
    qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    scales: torch.Tensor, pages: torch.Tensor, offsets: torch.Tensor, num_heads: int,
) -> torch.Tensor:
    return append_tokens_qkv_rope_q8(qkv, cos, sin, k_cache, v_cache, scales, pages, offsets, num_heads)


@kv_append_tokens_qkv_rope_q8_op.register_fake
def _(qkv, cos, sin, k_cache, v_cache, scales, pages, offsets, num_heads):
    return qkv.new_empty((1, qkv.shape[-2], num_heads, k_cache.shape[-1]))


@torch.library.custom_op("inference::gqa_mixed_attention_q8", mutates_args=())
def gqa_mixed_attention_q8_op(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scales: torch.Tensor,
    max_seqlen: int, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor,
    slot_ids: torch.Tensor, block_table: torch.Tensor, plan: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    return mixed_gqa_attention_q8(q, k, v, scales, max_seqlen, cu_seqlens, kv_lens, slot_ids, block_table, plan=plan)


@gqa_mixed_attention_q8_op.register_fake
def _(q, k, v, scales, max_seqlen, cu_seqlens, kv_lens, slot_ids, block_table, plan=None):
    return torch.empty_like(q)


@torch.library.custom_op("inference::gqa_mixed_plan_q8", mutates_args=())
def gqa_mixed_plan_q8_op(k_cache: torch.Tensor, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor,
                         slot_ids: torch.Tensor, block_table: torch.Tensor, max_seqlen: int, total_T: int,
                         num_heads: int) -> torch.Tensor:
    """A mixed step's plan for its layers' mixed attention (mixed_plan_q8)."""
    return mixed_plan_q8(k_cache, cu_seqlens, kv_lens, slot_ids, block_table, max_seqlen, total_T, num_heads)


@gqa_mixed_plan_q8_op.register_fake
def _(k_cache, cu_seqlens, kv_lens, slot_ids, block_table, max_seqlen, total_T, num_heads):
    n = _native.load().cie_q8_mixed_plan_bytes(slot_ids.shape[0], total_T, num_heads, k_cache.shape[1])
    return k_cache.new_empty((n // 4,), dtype=torch.int32)
