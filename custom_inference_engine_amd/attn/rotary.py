"""Rotary positions: half and interleaved layouts, part of a head, scaled for long contexts.

Beside the cos / sin rows that the fused append and decode calls take
(``apply_rotary_pos_emb`` of the reference's layer, attn/core.py:193-198): these
operators turn rows by their positions themselves.  Pair i of the first ``2 *
len(frequencies)`` dims of a head, (x, y), becomes ``scale * (x cos a - y sin a,
y cos a + x sin a)`` with ``a = position * frequencies[i]``: dims (i, i + half) or, with
``interleaved``, (2i, 2i + 1); the other dims are copied.  Angles are computed in 64 bits,
so far positions keep them, and for fp32 rows and tables their cos and sin too; products and
sums in fp32, rounded once.

``rotary_frequencies`` makes the table of a base and a long-context scaling; any other is
a float64 tensor of radians a position.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _native
from ..kv_cache.quant import int64_index, launch, one_device

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # CIE_F16, CIE_BF16, CIE_F32
_F64, _DENSE = torch.float64, torch.contiguous_format


# What a scaling may hold beside its type; those that a type does not use are ignored, as the model library does.
_SCALING_KEYS = {"rope_type", "type", "rope_theta", "partial_rotary_factor", "factor", "factors", "attention_factor",
                 "original_max_position_embeddings", "beta_fast", "beta_slow", "mscale", "mscale_all_dim", "truncate"}


def rotary_frequencies(rotary_dim: int, base: Optional[float] = None, scaling: Optional[dict] = None, device=None):
    """(frequencies (rotary_dim / 2,) float64, scale) of a base and a scaling.

    ``base``: the scaling's ``rope_theta`` by default, or 10,000; not another than that
    ``rope_theta``.  ``scaling`` is a model config's ``rope_scaling``, by its
    ``rope_type`` (or ``type``); keys not named here are refused, as is a
    ``partial_rotary_factor`` (``rotary_dim`` says what turns).

    * ``default``: base ** (-2i / rotary_dim).
    * ``linear``: positions divided by ``factor``.
    * ``ntk``: the base raised by factor ** (d / (d - 2)), so that the slowest pair is
      stretched by ``factor`` and the fastest is kept.
    * ``yarn``: pairs that turn more than ``beta_fast`` (32) times within
      ``original_max_position_embeddings`` are kept, those under ``beta_slow`` (1) are
      stretched by ``factor``, with a ramp between, from a whole pair to a whole pair unless
      ``truncate`` is false; ``scale`` is ``attention_factor``; or where ``mscale`` and
      ``mscale_all_dim`` are set m(mscale) / m(mscale_all_dim), m(x) = 0.1 x ln(factor) + 1 (1
      for factors up to 1); or m(1).
    * ``factors``: each frequency divided by its own ``factors[i]``; ``scale`` is
      ``attention_factor``, or 1.
    """
    scaling = {k: v for k, v in (scaling or {}).items() if v is not None}
    unknown = set(scaling) - _SCALING_KEYS
    if unknown:
        raise AssertionError(f"rope scaling has keys that are not understood: {sorted(unknown)}")
    if scaling.get("partial_rotary_factor", 1) != 1:
        raise AssertionError("rotary_dim says how much of a head turns: leave out 'partial_rotary_factor'")
    theta = scaling.get("rope_theta")
    if base is None:
        base = 10000.0 if theta is None else theta
    elif theta is not None and theta != base:
        raise AssertionError(f"base {base} is not the scaling's rope_theta {theta}")
    base = float(base)
    if rotary_dim < 2 or rotary_dim % 2 or not base > 0:
        raise AssertionError("rotary_dim must be even and positive, base positive")
    n = rotary_dim // 2
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    scale = 1.0

    def need(name):
        if name not in scaling:
            raise AssertionError(f"rope scaling '{kind}' needs '{name}'")
        return scaling[name]

    if kind == "ntk":
        if n < 2:
            raise AssertionError("rope scaling 'ntk' needs a rotary_dim of 4 or more")
        base = base * float(need("factor")) ** (rotary_dim / (rotary_dim - 2))
    freqs = [base ** (-2 * i / rotary_dim) for i in range(n)]
    if kind == "linear":
        freqs = [f / float(need("factor")) for f in freqs]
    elif kind == "yarn":
        factor, trained = float(need("factor")), need("original_max_position_embeddings")
        fast, slow = scaling.get("beta_fast") or 32, scaling.get("beta_slow") or 1
        if base == 1.0:
            raise AssertionError("rope scaling 'yarn' needs a base other than 1")
        if not fast > slow:
            raise AssertionError("rope scaling 'yarn' needs beta_fast over beta_slow")

        def pair_that_turns(times):  # (a real number) within the trained positions
            return rotary_dim * math.log(trained / (times * 2 * math.pi)) / (2 * math.log(base))

        def m(x):
            return 0.1 * x * math.log(factor) + 1 if factor > 1 else 1.0

        low, high = pair_that_turns(fast), pair_that_turns(slow)
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rotary_dim - 1)
        stretched = [min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(n)]
        freqs = [f / factor * s + f * (1 - s) for f, s in zip(freqs, stretched)]
        if scaling.get("mscale") and scaling.get("mscale_all_dim"):
            scale = m(scaling["mscale"]) / m(scaling["mscale_all_dim"])
        else:
            scale = m(1)
        scale = scaling.get("attention_factor", scale)
    elif kind == "factors":
        factors = need("factors")
        if len(factors) != n:
            raise AssertionError(f"'factors' must have {n} entries")
        freqs = [f / float(x) for f, x in zip(freqs, factors)]
        scale = scaling.get("attention_factor", 1.0)
    elif kind not in ("default", "linear", "ntk"):
        raise AssertionError(f"unknown rope scaling '{kind}': default, linear, ntk, yarn or factors")
    return torch.tensor(freqs, dtype=torch.float64, device=device), float(scale)


def _positions(positions: torch.Tensor, T: int) -> torch.Tensor:
    shape = positions.shape
    if shape[-1:] != (T,) or (len(shape) != 1 and shape != (1, T)):
        raise AssertionError("positions must have one entry per row")
    return int64_index(positions)


def _frequencies(frequencies: torch.Tensor, d: int) -> int:
    """The dims that turn."""
    shape = frequencies.shape
    if frequencies.dtype is not _F64 or len(shape) != 1 or not frequencies.is_contiguous():
        raise AssertionError("frequencies must be contiguous float64 (pairs,)")
    rot = 2 * shape[0]
    if rot < 2 or rot > d or d % 2:
        raise AssertionError(f"2 * len(frequencies) must be in [2, head_dim = {d}], head_dim even")
    return rot


def rotary_tables(positions, frequencies, dtype=torch.float16, interleaved: bool = False, scale: float = 1.0):
    """cos and sin of the positions, (1, T, 2 * pairs) each, times ``scale``: a value for each dim of a head, as the
    fused append and decode calls take them (half layout, the whole head turned)."""
    T = positions.shape[-1] if positions.dim() else 0
    rot = _frequencies(frequencies, 2 * frequencies.numel())
    if dtype not in _TYPES:
        raise AssertionError("tables are float16, bfloat16 or float32")
    dev = one_device(positions, frequencies)
    positions = _positions(positions, T)
    cos = torch.empty((1, T, rot), dtype=dtype, device=dev)
    sin = torch.empty_like(cos)
    if T:
        _native.call(dev, "cie_rotary_tables", cos.data_ptr(), sin.data_ptr(), positions.data_ptr(),
                     frequencies.data_ptr(), scale, T, rot, interleaved, _TYPES[dtype])
    return cos, sin


def apply_rotary(q, k, positions, frequencies, interleaved: bool = False, scale: float = 1.0):
    """q and k turned by their rows' positions, into new dense tensors of their shapes.

    q (1, T, H_q, D) and k (1, T, H_kv, D), or without the leading 1, float16, bfloat16 or
    float32: views into the fused QKV projection's output need no copy.  positions (T,)
    or (1, T).  ``k`` may be None.
    """
    shape, dtype = q.shape, q.dtype
    kind = _TYPES.get(dtype)
    if kind is None:
        raise AssertionError("rows must be float16, bfloat16 or float32")
    if len(shape) not in (3, 4) or (len(shape) == 4 and shape[0] != 1):
        raise AssertionError("q and k must be (1, T, heads, D) or (T, heads, D)")
    T, h_q, d = shape[-3:]
    rot = _frequencies(frequencies, d)
    if k is None:
        dev = one_device(q, positions, frequencies)
    else:
        k_shape = k.shape
        h_kv = k_shape[-2] if len(k_shape) == len(shape) else -1
        if k.dtype != dtype or k_shape != (*shape[:-2], h_kv, d):
            raise AssertionError("q and k must have the same rows, head_dim and type")
        dev = one_device(q, k, positions, frequencies)
    positions = _positions(positions, T)
    q, q_row, q_head = _dense_heads(q, d)
    q_out = torch.empty_like(q, memory_format=_DENSE)
    if k is None:
        k_out, k_ptr, to_k, h_kv, k_row, k_head = None, None, None, 0, 0, 0
    else:
        k, k_row, k_head = _dense_heads(k, d)
        k_out = torch.empty_like(k, memory_format=_DENSE)
        k_ptr, to_k = k.data_ptr(), k_out.data_ptr()
    if T and h_q + h_kv:
        _native.call(dev, "cie_rotary", q_out.data_ptr(), to_k, q.data_ptr(), k_ptr, q_row, q_head, k_row, k_head,
                     positions.data_ptr(), frequencies.data_ptr(), scale, T, h_q, h_kv, d, rot, interleaved, kind)
    return q_out, k_out


def _dense_heads(x: torch.Tensor, d: int):
    """x with the dims of a head side by side (itself, or a copy), and its strides of rows and heads."""
    st = x.stride()
    if st[-1] != 1 and d > 1:
        x = x.contiguous()
        st = x.stride()
    return x, st[-3], st[-2]


def append_tokens_qkv_rotary(qkv, positions, frequencies, k_cache, v_cache, pages, offsets, num_heads: int,
                             interleaved: bool = False, scale: float = 1.0, err=None):
    """QKV split, rotary positions and ``KVStorage.mixed_update`` in one launch, as ``append_tokens_qkv_rope``.

    Row t of ``qkv`` (1, T, (H_q + 2 H_kv) D) is turned by ``positions[t]``; its k and v
    go to ``(pages[t], :, offsets[t])`` of the 16-bit pools (qkv's type), and the turned
    q is returned, (1, T, H_q, D).  Rows with the same page and offset (padding's) leave some of
    each: any value held there is one of theirs.
    """
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        raise AssertionError("K/V pools must both be (n_pages, H_kv, page_size, D), with identical strides")
    n_pages, h_kv, page_size, d = k_cache.shape
    s_page, s_head, s_row, one = k_cache.stride()
    if one != 1 or s_row != d:
        raise AssertionError("K/V pools need dense (page_size, D) rows")
    if qkv.dtype not in (torch.float16, torch.bfloat16) or k_cache.dtype != qkv.dtype or v_cache.dtype != qkv.dtype:
        raise AssertionError("qkv and the K/V pools must share a 16-bit type")
    width = (num_heads + 2 * h_kv) * d
    if qkv.dim() != 3 or qkv.shape[0] != 1 or qkv.shape[2] != width or num_heads < 1:
        raise AssertionError(f"qkv must be (1, T, {width})")
    T = qkv.shape[1]
    if pages.shape != (T,) or offsets.shape != (T,):
        raise AssertionError("pages / offsets must be (T,)")
    rot = _frequencies(frequencies, d)
    dev = one_device(qkv, positions, frequencies, k_cache, v_cache, pages, offsets)
    positions = _positions(positions, T)
    if qkv.stride(2) != 1 or (T > 1 and qkv.stride(1) < width):
        qkv = qkv.contiguous()
    pages, offsets = int64_index(pages), int64_index(offsets)
    q = torch.empty((1, T, num_heads, d), dtype=qkv.dtype, device=dev)
    if T:
        launch(dev, "cie_kv_append_tokens_qkv_rotary", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
               qkv.data_ptr(), max(qkv.stride(1), width), positions.data_ptr(), frequencies.data_ptr(), scale,
               pages.data_ptr(), offsets.data_ptr(), T, num_heads, h_kv, page_size, d, n_pages, s_page, s_head, rot,
               interleaved, _TYPES[qkv.dtype], err=err)
    return q


@torch.library.custom_op("inference::rotary_tables", mutates_args=())
def rotary_tables_op(positions: torch.Tensor, frequencies: torch.Tensor, dtype: torch.dtype, interleaved: bool,
                     scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    return rotary_tables(positions, frequencies, dtype, interleaved, scale)


@rotary_tables_op.register_fake
def _(positions, frequencies, dtype, interleaved, scale):
    shape = (1, positions.numel(), 2 * frequencies.shape[0])
    return frequencies.new_empty(shape, dtype=dtype), frequencies.new_empty(shape, dtype=dtype)


@torch.library.custom_op("inference::apply_rotary", mutates_args=())
def apply_rotary_op(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor,
                    interleaved: bool, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    return apply_rotary(q, k, positions, frequencies, interleaved, scale)


@apply_rotary_op.register_fake
def _(q, k, positions, frequencies, interleaved, scale):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op("inference::kv_append_tokens_qkv_rotary", mutates_args=("k_cache", "v_cache"))
def kv_append_tokens_qkv_rotary_op(
    qkv: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, k_cache: torch.Tensor,
    v_cache: torch.Tensor, pages: torch.Tensor, offsets: torch.Tensor, num_heads: int, interleaved: bool, scale: float,
) -> torch.Tensor:
    return append_tokens_qkv_rotary(qkv, positions, frequencies, k_cache, v_cache, pages, offsets, num_heads,
                                    interleaved, scale)


@kv_append_tokens_qkv_rotary_op.register_fake
def _(qkv, positions, frequencies, k_cache, v_cache, pages, offsets, num_heads, interleaved, scale):
    return qkv.new_empty((1, qkv.shape[1], num_heads, k_cache.shape[-1]))


class RotaryPositions(torch.nn.Module):
    """In a model's place for its rotary embedding: what its layers get as ``position_embeddings``.

    Half layout over the whole head: cos and sin rows, one launch a step, for the layers'
    fused calls.  Otherwise the positions and the frequencies, and the layers turn their
    rows themselves (``TritonQwen2Attention.rotary``).
    """

    def __init__(self, frequencies, scale: float, interleaved: bool, tables: bool):
        super().__init__()
        self.register_buffer("frequencies", frequencies, persistent=False)
        self.scale, self.interleaved, self.tables = scale, interleaved, tables

    def _apply(self, fn, recurse=True):
        # (the model's own type is not the frequencies': only their device follows it)
        kept = self.frequencies
        super()._apply(fn, recurse)
        self.frequencies = kept.to(self.frequencies.device)
        return self

    def forward(self, x, position_ids):
        if not self.tables:
            return position_ids, self.frequencies
        if position_ids.dim() < 2 or position_ids.shape[0] == 1:
            return rotary_tables_op(position_ids, self.frequencies, x.dtype, self.interleaved, self.scale)
        # several rows of tokens (the wrapped modules' own path): side by side, and dealt to the rows again
        cos, sin = rotary_tables_op(position_ids.flatten(), self.frequencies, x.dtype, self.interleaved, self.scale)
        return cos.view(*position_ids.shape, -1), sin.view(*position_ids.shape, -1)


def use_rotary(model, frequencies, scale: float = 1.0, interleaved: bool = False) -> None:
    """Gives a model whose attention ``use_triton_attention`` has replaced the positions of ``frequencies``.

    ``rotary_frequencies`` makes them: a longer context than the model's own, part of the
    head (fewer pairs than head_dim / 2), or the interleaved layout of its checkpoint.
    Comes before step modules and schedulers, whose graphs turn rows by what they found.
    """
    from .core import TritonQwen2Attention

    layers = [m for m in model.modules() if isinstance(m, TritonQwen2Attention)]
    if not layers:
        raise AssertionError("use_triton_attention(model) first")
    rot = _frequencies(frequencies, layers[0].head_dim)
    tables = not interleaved and rot == layers[0].head_dim
    device = layers[0].qkv_weight.device
    model.model.rotary_emb = RotaryPositions(frequencies.to(device), float(scale), bool(interleaved), tables)
    for layer in layers:
        layer.rotary = None if tables else (bool(interleaved), float(scale))
