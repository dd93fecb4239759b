"""Plain 64-bit implementation of the 8-bit paged cache and its attention.

TEST INFRASTRUCTURE ONLY (see paged_attention.py).  A cache is the pair of its e4m3
values before scaling and its exponents, both float64; every function follows the
definition element by element or block by block, in no order that a kernel uses.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

BLOCK, TOP, LIMIT, E_MIN, E_MAX = 16, 448.0, 61440.0, -15, 8


def exponent(amax: float) -> int:
    """Least e in [-15, 8] with amax <= 448 * 2**e (8 where none is)."""
    for e in range(E_MIN, E_MAX + 1):
        if amax <= TOP * 2.0 ** e:
            return e
    return E_MAX


def round_e4m3(y: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value of float64 y, ties to even: 3 bits after the leading one, exponents from -6."""
    top = torch.frexp(y.abs().clamp_min(2.0 ** -60))[1] - 1
    step = torch.ldexp(torch.ones_like(y), top.clamp_min(-6) - 3)
    return torch.round(y / step) * step


@dataclass
class Q8Cache:
    """One pool: vals (n_pages, H, P, D) and exps (n_pages, H, P / 16), float64."""
    vals: torch.Tensor
    exps: torch.Tensor

    @classmethod
    def of(cls, pool: torch.Tensor, scales: torch.Tensor) -> "Q8Cache":
        """From a pool's bytes and its scales (n_pages, H, P / 16)."""
        return cls(pool.cpu().float().double(), torch.log2(scales.cpu().double()))

    def clone(self) -> "Q8Cache":
        return Q8Cache(self.vals.clone(), self.exps.clone())

    def values(self) -> torch.Tensor:
        return self.vals * (2.0 ** self.exps).repeat_interleave(BLOCK, 2)[..., None]

    def append(self, x: torch.Tensor, pages, offsets) -> None:
        """Rows x (T, H, D) at (pages[t], offsets[t]); of a repeated index the last row."""
        n, h_kv, page, d = self.vals.shape
        x = x.cpu().double().clamp(-LIMIT, LIMIT)  # (NaN stays)
        blocks: dict = {}
        for t, (p, o) in enumerate(zip(list(map(int, pages)), list(map(int, offsets)))):
            if 0 <= p < n and 0 <= o < page:
                blocks.setdefault((p, o // BLOCK), {})[o % BLOCK] = t
        for (p, i), rows in blocks.items():
            for h in range(h_kv):
                new = x[list(rows.values()), h]
                e = exponent(float(torch.nan_to_num(new, 0.0).abs().max()))
                block = self.vals[p, h, i * BLOCK:(i + 1) * BLOCK]
                if 0 not in rows:
                    old = int(self.exps[p, h, i])
                    e = max(e, old)
                    keep = [r for r in range(BLOCK) if r not in rows]
                    if e > old:
                        block[keep] = round_e4m3(block[keep] * 2.0 ** (old - e))
                block[list(rows)] = round_e4m3(new * 2.0 ** -e)
                self.exps[p, h, i] = e


def attend(q, kc: Q8Cache, vc: Q8Cache, seqs, block_table):
    """q (T, H_q, D); seqs: (first row, rows, slot, keys of the first row) each; row i attends keys + i keys.

    Returns the outputs and, for tolerances, sum(p |v|) of every output and the largest |v| attended."""
    T, h_q, d = q.shape
    h_kv, page = kc.vals.shape[1], kc.vals.shape[2]
    q = q.cpu().double()
    kv, vv = kc.values(), vc.values()
    o, mass, top = torch.zeros(T, h_q, d).double(), torch.zeros(T, h_q, d).double(), torch.zeros(T, h_q, 1).double()
    for t0, n, slot, keys in seqs:
        L = keys + n - 1
        if L <= 0:
            continue
        ids = block_table[slot, :-(-L // page)].cpu()
        k, v = (x[ids].transpose(0, 1).reshape(h_kv, -1, d)[:, :L] for x in (kv, vv))
        dead = torch.arange(L)[None] >= (keys + torch.arange(n))[:, None]
        for h in range(h_q):
            g = h // (h_q // h_kv)
            s = (q[t0:t0 + n, h] @ k[g].T) * d ** -0.5
            s = s.masked_fill(dead, -math.inf)
            w = torch.softmax(s, -1).nan_to_num(0.0)  # (a row without keys)
            o[t0:t0 + n, h] = w @ v[g]
            mass[t0:t0 + n, h] = w @ v[g].abs()
            top[t0:t0 + n, h] = v[g].abs().max()
    return o, mass, top


def tolerance(o, mass, top, n_keys: int):
    """What a kernel with fp16 weights, exact fp16 values and fp32 sums may be off by.

    Each weight is off by 2^-11 of itself (in numerator and sum: mass + |o|), or by half of fp16's smallest
    step, 2^-25, against a largest weight of at least 2^-8 (the reference maximum lags by 2^8 at most
    upwards, so the largest weight is 1 or more before division): n_keys * 2^-25 * top, twice; the output's
    rounding 2^-11 |o| (2^-25 where subnormal); fp32 sums and exponentials 1e-5 of mass.
    """
    return 2.0 ** -11 * (mass + 2 * o.abs()) + n_keys * 2.0 ** -24 * top + 2e-5 * mass + 2.0 ** -25
