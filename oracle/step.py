"""Oracle of what a step needs before its attention: slot maps with pages from a free list, rotary
positions, low-rank adapters.  Plain loops and 64 bits on the CPU; tests only."""
from __future__ import annotations

import math

import torch


class FreeList:
    """The words of a free list: the count, a word that stays 0, the stack."""

    def __init__(self, words: list[int]):
        self.count, self.stack, self.size = words[0], words[2:2 + words[0]], len(words) - 2
        self.rest = words[2:]

    def words(self) -> list[int]:
        """What the kernels leave: words past the count are whatever was there."""
        return [self.count, 0] + self.stack + self.rest[self.count:]


def _ceil(a: int, b: int) -> int:
    return -(-a // b)


def step_maps(slot_ids, new, lens, table, page_size, T, free=None):
    """cu, (slots, positions, pages, offsets), and whether the free list served the call; ``table`` (lists) and
    ``free`` (FreeList) are changed as the call changes them."""
    n_slots, width = len(table), len(table[0])
    cu = [0]
    for n in new:
        cu.append(min(cu[-1] + max(n, 0), T))
    fresh: list[dict[int, int]] = [{} for _ in slot_ids]  # page index -> page
    served = True
    if free is not None:
        wanted, seen = [], set()
        for b, s in enumerate(slot_ids):
            n = cu[b + 1] - cu[b]
            if not 0 < s < n_slots or n == 0 or lens[s] < 0 or lens[s] + n > width * page_size:
                continue
            served &= s not in seen
            seen.add(s)
            wanted += [(b, i) for i in range(_ceil(lens[s], page_size), _ceil(lens[s] + n, page_size))]
        served &= len(wanted) <= free.count
        if served:
            for b, i in wanted:
                fresh[b][i] = table[slot_ids[b]][i] = free.stack.pop()
            free.count -= len(wanted)
    rows = []
    for b, s in enumerate(slot_ids):
        for t in range(cu[b], cu[b + 1]):
            if not 0 <= s < n_slots:
                rows.append((0, 0, 0, 0))
                continue
            pos = lens[s] + t - cu[b]
            if not 0 <= pos < width * page_size:
                rows.append((s, pos, 0, 0))
                continue
            i = pos // page_size
            held = free is None or s == 0 or i < _ceil(max(lens[s], 0), page_size)
            rows.append((s, pos, table[s][i] if held else fresh[b].get(i, 0), pos % page_size))
    rows += [(0, 0, 0, 0)] * (T - len(rows))
    return cu, rows, served


def release_pages(free, slot_ids, lens, table, page_size, keep=None, held=None) -> bool:
    """Whether it was done; ``free``, ``lens`` and ``table`` (lists) are changed."""
    n_slots, capacity = len(table), len(table[0]) * page_size
    gone, kept, seen = [], {}, set()
    for b, s in enumerate(slot_ids):
        if not 0 < s < n_slots:
            continue
        k, h = (keep[b] if keep else 0), (held[b] if held else lens[s])
        if not (0 <= k <= h <= capacity and lens[s] <= h and h >= 0):
            continue
        if s in seen:
            return False
        seen.add(s)
        kept[s] = k
        gone += [(s, i) for i in range(_ceil(k, page_size), _ceil(h, page_size))]
    if free.count + len(gone) >= free.size:
        return False
    end = free.count + len(gone)
    for s, i in reversed(gone):
        page, table[s][i] = table[s][i], 0
        if page == 0:  # no page: nothing to give back
            continue
        page = page if 0 < page < free.size else 0
        free.rest[len(free.stack)] = page
        free.stack.append(page)
    free.count = len(free.stack)
    free.rest[free.count:end] = [0] * (end - free.count)
    for s, k in kept.items():
        lens[s] = k
    return True


def rotary(x, positions, freqs, interleaved=False, scale=1.0):
    """x (T, heads, D) in float64 turned by its rows' positions, and a bound of the terms' size (|x| + |y|) * scale."""
    x = x.double()
    n = len(freqs)
    out, size = x.clone(), x.abs().clone()
    for i, f in enumerate(freqs):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        for t, p in enumerate(positions):
            angle = math.fmod(float(p) * float(f), 2 * math.pi)
            c, s = scale * math.cos(angle), scale * math.sin(angle)
            u, v = x[t, :, a], x[t, :, b]
            out[t, :, a], out[t, :, b] = u * c - v * s, v * c + u * s
            size[t, :, a] = size[t, :, b] = (u.abs() + v.abs()) * abs(scale)
    return out, size


def adapters(y, x, a, b, scales, row_adapter, slices):
    """y (T, d_out) with its rows' adapters added, in float64, and an elementwise bound of how far the kernels'
    arithmetic may be from it before the last rounding.

    Sums of products are bounded as chains of fp32 roundings (2^-23 of the terms' sizes for each
    4 products that are added at once, and one for each partial sum); A x as two values of float16
    is off by 2^-21 of it, as three of bfloat16 not at all.
    """
    split = 0.0 if y.dtype == torch.bfloat16 else 2.0 ** -21
    out, off = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64)
    d_in, R = a.shape[3], a.shape[2]
    for t, i in enumerate(row_adapter):
        if i < 0:
            continue
        col, s = 0, abs(float(scales[i]))
        xt = x[t].double()
        for k, width in enumerate(slices):
            A, B = a[i, k].double(), b[i, col:col + width].double()
            u = A @ xt
            u_off = (d_in / 4 + 32) * 2.0 ** -23 * (A.abs() @ xt.abs()) + split * u.abs() + 2.0 ** -38 * u.abs().max()
            delta = float(scales[i]) * (B @ u)
            out[t, col:col + width] += delta
            off[t, col:col + width] = s * (B.abs() @ u_off + (R / 2 + 16) * 2.0 ** -23 * (B.abs() @ u.abs())) \
                + 2.0 ** -23 * (delta.abs() + y[t, col:col + width].double().abs())
            col += width
    return out, off


def rounding(ref: torch.Tensor, dtype) -> torch.Tensor:
    """Half a step of ``dtype`` at ref, subnormals included."""
    info = torch.finfo(dtype)
    return ref.abs().clamp(min=info.smallest_normal) * (info.eps / 2)
