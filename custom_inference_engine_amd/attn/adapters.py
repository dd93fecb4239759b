"""Low-rank adapters of many requests at once, beside a shared projection.

``y[t, s] += scales[i] * B[i, s] (A[i, s] x[t])`` in place, for the slices s of y's columns
(a fused QKV projection has three) and the adapter i of row t's request; rows without one
are left as they are.  ``adapter_plan`` works out once per step which rows share an adapter
(like ``decode_plan`` / ``mixed_plan``: every layer and projection of the step reads it),
``adapter_add_`` is one launch per projection.  ``AdapterBank`` holds the weights of one
projection's adapters, ``use_adapters`` puts banks beside the projections of a model's
attention layers.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import numpy as np
import torch

from .. import _native
from ..kv_cache.quant import int64_index, launch, one_device

RANK_UNIT = 16  # a bank's ranks come in 16s
MAX_RANK = 128
_TYPES = {torch.float16: 0, torch.bfloat16: 1}  # CIE_F16, CIE_BF16
_F32, _I32 = torch.float32, torch.int32


@functools.lru_cache(maxsize=4096)
def _plan_words(T: int, n_adapters: int) -> int:
    n = _native.load().cie_adapter_plan_bytes(T, n_adapters)
    if n <= 0:
        raise AssertionError("a plan takes 1 to 1,024 adapters and at most 2^24 rows")
    return n // 4


@functools.lru_cache(maxsize=256)
def _widths(slices: tuple):
    return (ctypes.c_int64 * len(slices))(*slices), sum(slices), len(slices)


def new_adapter_plan(n_rows: int, n_adapters: int, device) -> torch.Tensor:
    """Room for the plans of a module whose steps have ``n_rows`` rows, where they need one address (a captured piece)."""
    return torch.zeros(_plan_words(n_rows, n_adapters), dtype=torch.int32, device=device)


def adapter_plan(row_slots: Optional[torch.Tensor], slot_adapters: torch.Tensor, n_adapters: int,
                 out: Optional[torch.Tensor] = None, err=None) -> torch.Tensor:
    """One step's plan: row t has adapter ``slot_adapters[row_slots[t]]``, none where that is negative.

    ``row_slots`` (T,): a mixed step's ``StepMaps.slots``, a decode step's slot ids; None:
    ``slot_adapters`` has an entry for each row.  Pass the int32 tensor as ``plan`` to the
    step's ``adapter_add_`` calls, on banks of ``n_adapters``.  ``out``: a
    ``new_adapter_plan`` of as many rows and adapters, to write to.
    """
    if slot_adapters.dim() != 1 or (row_slots is not None and row_slots.dim() != 1):
        raise AssertionError("row_slots must be (T,) and slot_adapters (n_slots,)")
    dev = one_device(slot_adapters) if row_slots is None else one_device(slot_adapters, row_slots)
    slot_adapters = int64_index(slot_adapters)
    rows, T = None, slot_adapters.shape[0]
    if row_slots is not None:
        row_slots = int64_index(row_slots)
        rows, T = row_slots.data_ptr(), row_slots.shape[0]
    words = _plan_words(T, n_adapters)
    if out is None:
        plan = torch.empty(words, dtype=torch.int32, device=dev)
    else:
        plan = out
        one_device(slot_adapters, plan)
        if plan.dtype != torch.int32 or plan.shape != (words,) or not plan.is_contiguous():
            raise AssertionError("out must come from new_adapter_plan for these rows and adapters")
    if T:
        launch(dev, "cie_adapter_plan", plan.data_ptr(), 4 * words, rows, slot_adapters.data_ptr(), T,
               slot_adapters.shape[0], n_adapters, err=err)
    return plan


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """The rows of (1, T, width)."""
    if t.dim() != 3 or t.shape[0] != 1:
        raise AssertionError(f"{name} must be (T, width) or (1, T, width)")
    return t[0]


def _share(p: int, step: int, size: int, n: int, q: int, hop: int, span: int, m: int) -> bool:
    """Whether n rows of ``size`` bytes, ``step`` apart from p on, and m of ``span`` bytes, ``hop`` apart from q on, share a byte."""
    if n > 1 and step < size:  # (rows that lie in each other: one)
        size, n = (n - 1) * step + size, 1
    if m > 1 and hop < span:
        span, m = (m - 1) * hop + span, 1
    if n == m and step == hop and n > 1:  # views of one wider tensor: row j of the second lies behind row j + k of the first
        k, r = divmod(q - p, step)
        return (r < size and -n < k < n) or (r + span > step and -n < k + 1 < n)
    rows = p + step * np.arange(n)
    hop = max(hop, 1)
    near = np.clip((rows - q - span) // hop + 1, 0, m - 1) * hop + q  # the first to end behind a row's start
    return bool(((near < rows + size) & (rows < near + span)).any())


def adapter_add_(y, x, a, b, scales, ranks, plan, slices, err=None):
    """``y`` with its rows' adapters added, in place.

    y (T, d_out) and x (T, d_in), or with a leading 1; a (n, len(slices), R, d_in), b (n,
    d_out, R), of y's type (float16 or bfloat16), R a multiple of 16 up to 128;
    ``slices``: the widths of y's parts, d_out together; scales (n,) float32; ranks (n,)
    int32: an adapter's rows of rank, those behind them being zeros in a and b.  ``plan``:
    the step's ``adapter_plan``.  A plan of other rows or adapters is reported in ``err``
    (CIE_ERRBIT_PLAN), and y left as it is.  y's memory holds nothing of the other arguments'.
    """
    yr = y if y.dim() == 2 else _rows(y, "y")
    xr = x if x.dim() == 2 else _rows(x, "x")
    (T, d_in), (y_T, y_w) = xr.shape, yr.shape
    (y_row, y_one), (x_row, x_one) = yr.stride(), xr.stride()
    widths, d_out, n_slices = _widths(slices if type(slices) is tuple else tuple(slices))
    dtype = y.dtype
    kind = _TYPES.get(dtype)
    if kind is None or x.dtype is not dtype or a.dtype is not dtype or b.dtype is not dtype:
        raise AssertionError("y, x, a and b must share float16 or bfloat16")
    if y_T != T or y_w != d_out:
        raise AssertionError(f"y must be ({T}, {d_out}): x's rows, the slices' widths")
    if (y_one != 1 and d_out > 1) or (x_one != 1 and d_in > 1):
        raise AssertionError("the rows of y and x must be dense")
    if T > 1 and y_row < d_out:
        raise AssertionError("y's rows must not share memory")
    y_ptr, x_ptr = y.data_ptr(), x.data_ptr()
    y_end = y_ptr + 2 * ((T - 1) * y_row + d_out)
    if (x_ptr < y_end and y_ptr < x_ptr + 2 * ((T - 1) * x_row + d_in)
            and T and _share(y_ptr, 2 * y_row, 2 * d_out, T, x_ptr, 2 * x_row, 2 * d_in, T)):
        raise AssertionError("x must not lie in y's memory")
    n, S, R, w = a.shape if a.dim() == 4 else (0,) * 4
    if S != n_slices or w != d_in or R % RANK_UNIT or not 0 < R <= MAX_RANK or not a.is_contiguous():
        raise AssertionError(f"a must be contiguous (n, {n_slices}, R, {d_in}), R a multiple of 16 up to 128")
    if b.shape != (n, d_out, R) or not b.is_contiguous():
        raise AssertionError(f"b must be contiguous ({n}, {d_out}, {R})")
    if scales.dtype is not _F32 or scales.shape != (n,) or not scales.is_contiguous():
        raise AssertionError(f"scales must be contiguous float32 ({n},)")
    if ranks.dtype is not _I32 or ranks.shape != (n,) or not ranks.is_contiguous():
        raise AssertionError(f"ranks must be contiguous int32 ({n},)")
    held = plan.numel()
    if plan.dtype is not _I32 or held < _plan_words(T, n) or not plan.is_contiguous():
        raise AssertionError("plan must come from adapter_plan for these rows and adapters")
    dev = one_device(y, x, a, b, scales, ranks, plan)
    if T:
        a_ptr, b_ptr, s_ptr, r_ptr, p_ptr = a.data_ptr(), b.data_ptr(), scales.data_ptr(), ranks.data_ptr(), plan.data_ptr()
        if (y_ptr < a_ptr + 2 * n * n_slices * R * d_in and a_ptr < y_end or y_ptr < b_ptr + 2 * n * d_out * R and b_ptr < y_end
                or y_ptr < s_ptr + 4 * n and s_ptr < y_end or y_ptr < r_ptr + 4 * n and r_ptr < y_end
                or y_ptr < p_ptr + 4 * held and p_ptr < y_end):  # (between y's rows, or in them)
            for t in (a, b, scales, ranks, plan):
                size = t.numel() * t.element_size()
                if _share(y_ptr, 2 * y_row, 2 * d_out, T, t.data_ptr(), size, size, 1):
                    raise AssertionError("a, b, scales, ranks and plan must not lie in y's memory")
        if T > 1 and x_row < d_in:
            xr = xr.contiguous()
            x_ptr, x_row = xr.data_ptr(), d_in
        launch(dev, "cie_adapter_add", y_ptr, y_row, x_ptr, x_row, a_ptr, b_ptr, s_ptr, r_ptr, p_ptr, 4 * held, T, n, R,
               d_in, widths, n_slices, kind, err=err)
    return y


@torch.library.custom_op("inference::adapter_add_", mutates_args=("y",))
def adapter_add_op(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor,
                   ranks: torch.Tensor, plan: torch.Tensor, slices: list[int]) -> None:
    adapter_add_(y, x, a, b, scales, ranks, plan, slices)


@adapter_add_op.register_fake
def _(y, x, a, b, scales, ranks, plan, slices) -> None:
    return None


# (an op of its own: torch does not take an argument that is written and may be left out)
@torch.library.custom_op("inference::adapter_add_reported_", mutates_args=("y", "err"))
def adapter_add_reported_op(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor,
                            ranks: torch.Tensor, plan: torch.Tensor, slices: list[int], err: torch.Tensor) -> None:
    adapter_add_(y, x, a, b, scales, ranks, plan, slices, err=err)


@adapter_add_reported_op.register_fake
def _(y, x, a, b, scales, ranks, plan, slices, err) -> None:
    return None


class AdapterBank(torch.nn.Module):
    """The adapters of one projection: ``n_adapters`` places for A and B of up to ``rank``, empty until ``load``.

    ``out_features``: the projection's width, or the widths of a fused projection's parts.
    """

    def __init__(self, n_adapters: int, rank: int, in_features: int, out_features, dtype=torch.float16, device=None):
        super().__init__()
        self.slices = tuple(out_features) if isinstance(out_features, (tuple, list)) else (out_features,)
        if not 1 <= rank <= MAX_RANK or not 1 <= n_adapters <= 1024 or not 1 <= len(self.slices) <= 4:
            raise AssertionError("a bank has 1 to 1,024 adapters of rank 1 to 128, beside 1 to 4 slices")
        if dtype not in _TYPES:
            raise AssertionError("adapters are float16 or bfloat16")
        self.n_adapters, self.rank = n_adapters, rank
        R = -(-rank // RANK_UNIT) * RANK_UNIT
        make = functools.partial(torch.zeros, device=device)
        self.register_buffer("a", make((n_adapters, len(self.slices), R, in_features), dtype=dtype), persistent=False)
        self.register_buffer("b", make((n_adapters, sum(self.slices), R), dtype=dtype), persistent=False)
        self.register_buffer("scales", make((n_adapters,), dtype=torch.float32), persistent=False)
        self.register_buffer("ranks", make((n_adapters,), dtype=torch.int32), persistent=False)

    def _apply(self, fn, recurse=True):
        # (a model that is cast casts A and B; the scales stay fp32)
        kept = self.scales
        super()._apply(fn, recurse)
        self.scales = kept.to(self.scales.device)
        return self

    @torch.no_grad()
    def load(self, i: int, a, b, scale: float = 1.0) -> None:
        """Adapter i: for each slice A (r, in_features) and B (width, r), or None for a slice without one."""
        if not 0 <= i < self.n_adapters:
            raise IndexError(f"adapter {i} of {self.n_adapters}")
        a, b = ((x,) if isinstance(x, torch.Tensor) else tuple(x) for x in (a, b))
        if len(a) != len(self.slices) or len(b) != len(self.slices):
            raise AssertionError(f"one A and one B for each of the {len(self.slices)} slices")
        r = 0
        for x, z, width in zip(a, b, self.slices):
            if (x is None) != (z is None):
                raise AssertionError("A and B of a slice come together")
            if x is not None:
                if (x.dim() != 2 or x.shape[1] != self.a.shape[3] or not 1 <= x.shape[0] <= self.rank
                        or z.shape != (width, x.shape[0])):
                    raise AssertionError(f"A must be (r, {self.a.shape[3]}) and B ({width}, r), r <= {self.rank}")
                r = max(r, x.shape[0])
        self.clear(i)
        col = 0
        for s, (x, z, width) in enumerate(zip(a, b, self.slices)):
            if x is not None:
                self.a[i, s, :x.shape[0]] = x.to(self.a)
                self.b[i, col:col + width, :x.shape[0]] = z.to(self.b)
            col += width
        self.scales[i] = float(scale)
        self.ranks[i] = r

    @torch.no_grad()
    def clear(self, i: int) -> None:
        """Empties place i: rows with this adapter are left as they are."""
        if not 0 <= i < self.n_adapters:
            raise IndexError(f"adapter {i} of {self.n_adapters}")
        for t in (self.a, self.b, self.scales, self.ranks):
            t[i] = 0

    @torch.no_grad()
    def clear_all(self) -> None:
        """Empties every place."""
        for t in (self.a, self.b, self.scales, self.ranks):
            t.zero_()

    def add_(self, y, x, plan, err=None) -> None:
        args = (y, x, self.a, self.b, self.scales, self.ranks, plan, self.slices)
        if err is None:
            adapter_add_op(*args)
        else:
            adapter_add_reported_op(*args, err)


def use_adapters(model, kv_cache, n_adapters: int, rank: int) -> list:
    """Places for ``n_adapters`` low-rank adapters beside every attention layer's QKV and output projections.

    ``use_triton_attention`` comes first, step modules and schedulers (whose graphs record
    the adapters' launches) after; again only with as many of the same rank, which
    empties them.  Returns the layers: ``layer.qkv_adapters.load(i, (A_q,
    A_k, A_v), (B_q, B_k, B_v), scale)`` and ``layer.o_adapters.load(i, A, B, scale)``
    fill place i.  A request's adapter is its slot's, ``kv_cache.slot_adapters[slot]`` (-1:
    none), which ``Scheduler.call(prompt, adapter=i)`` sets.
    """
    from .core import TritonQwen2Attention

    layers = [m for m in model.modules() if isinstance(m, TritonQwen2Attention)]
    if not layers:
        raise AssertionError("use_triton_attention(model) first")
    banks = [b for layer in layers for b in (layer.qkv_adapters, layer.o_adapters) if b is not None]
    if any((b.n_adapters, b.rank) != (n_adapters, rank) for b in banks):
        raise AssertionError("the layers have banks of other sizes, which graphs may hold")
    new = []
    for layer in layers if not banks else ():
        w, o = layer.qkv_weight, layer.original.o_proj
        new.append((AdapterBank(n_adapters, rank, w.shape[1], layer.qkv_sizes, w.dtype, w.device),
                    AdapterBank(n_adapters, rank, o.in_features, o.out_features, w.dtype, w.device)))
    kv_cache.use_adapters(n_adapters)  # (nothing has changed until here: what is refused leaves all as it was)
    for b in banks:
        b.clear_all()
    for layer, pair in zip(layers, new):
        layer.qkv_adapters, layer.o_adapters = pair
    return layers
