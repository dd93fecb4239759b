"""Shared plumbing of the 8-bit cache's tests: a cache with history, and its oracle."""
import torch

from custom_inference_engine_amd import kv_append_tokens_q8
from oracle.q8_cache import Q8Cache
from tests.gpu_helpers import DEV


def rows(gen, T, h, d, loud=True):
    """fp16 rows whose magnitude differs from token to token (so that blocks grow), with channels that stand out."""
    x = torch.randn(T, h, d, generator=gen) * 0.5
    if loud:
        x = x * torch.exp(torch.randn(T, 1, 1, generator=gen))
        x = x + 8.0 * (torch.rand(1, h, d, generator=gen) < 0.05)
    return x.half()


class Case:
    """Sequences in slots 1.. with their pages anywhere in the pool.

    prior: held tokens; new: tokens to come.  The pools' unwritten bytes are ``fill``
    and unwritten scales NaN (nothing may read them into a result)."""

    def __init__(self, prior, new, h_q=14, h_kv=2, d=64, page=16, seed=0, fill=0x7f, spare=3, device=DEV):
        g = torch.Generator().manual_seed(seed)
        self.prior, self.new, self.page = list(prior), list(new), page
        self.h_q, self.h_kv, self.d, self.B, self.T = h_q, h_kv, d, len(prior), sum(new)
        need = [-(-(p + n) // page) for p, n in zip(prior, new)]
        n_pages = 1 + sum(need) + spare
        ids = 1 + torch.randperm(n_pages - 1, generator=g)
        self.table = torch.zeros(self.B + 1, n_pages, dtype=torch.int64)
        for b, x in enumerate(ids[:sum(need)].split(need)):
            self.table[1 + b, :need[b]] = x
        self.k = torch.full((n_pages, h_kv, page, d), fill, dtype=torch.uint8)
        self.v = self.k.clone()
        self.scales = torch.full((n_pages, h_kv, page // 16, 2), float("nan"))
        for name in ("k", "v", "scales"):
            setattr(self, name, getattr(self, name).to(device))
        self.k, self.v = self.k.view(torch.float8_e4m3fn), self.v.view(torch.float8_e4m3fn)
        self.slots = torch.arange(1, self.B + 1)
        self.lens = torch.tensor([0] + self.prior)
        self.kv_lens = torch.tensor(self.prior)
        self.cu = torch.tensor([0] + self.new).cumsum(0)
        self.device = device
        self.q = (torch.randn(1, self.T, h_q, d, generator=g)).half()
        self.k_new, self.v_new = rows(g, self.T, h_kv, d)[None], rows(g, self.T, h_kv, d)[None]
        self.history = [(rows(g, p, h_kv, d), rows(g, p, h_kv, d)) for p in self.prior]

    def at(self, b, first, n):
        pos = torch.arange(first, first + n)
        return self.table[1 + b][pos // self.page], pos % self.page

    def new_at(self):
        where = [self.at(b, p, n) for b, (p, n) in enumerate(zip(self.prior, self.new))]
        return torch.cat([w[0] for w in where]), torch.cat([w[1] for w in where])

    def write_history(self):
        """The held tokens through the token append, in a few calls of odd sizes."""
        for b, p in enumerate(self.prior):
            for lo in range(0, p, 1037):
                n = min(1037, p - lo)
                pages, offs = self.at(b, lo, n)
                k, v = self.history[b]
                kv_append_tokens_q8(self.k, self.v, self.scales, k[lo:lo + n].to(self.device),
                                    v[lo:lo + n].to(self.device), pages.to(self.device), offs.to(self.device))
        return self

    def oracles(self):
        """The cache as it stands: (K, V)."""
        torch.cuda.synchronize()
        s = self.scales.cpu()
        s = torch.where(s.isnan(), torch.ones_like(s), s)
        return tuple(Q8Cache.of(p, s[..., i]) for i, p in enumerate((self.k, self.v)))

    def dev(self, *names):
        return [getattr(self, n).to(self.device) for n in names]


def same_cache(case, oracles, skip_pages=()):
    """Bytes as values (NaN equal to NaN) and scales, of every page but ``skip_pages``."""
    s = case.scales.cpu()
    keep = [p for p in range(s.shape[0]) if p not in skip_pages]
    for i, (pool, want) in enumerate(zip((case.k, case.v), oracles)):
        got = pool.cpu().float().double()[keep]
        ref = want.vals[keep]
        bad = ~((got == ref) | (got.isnan() & ref.isnan()))
        assert not bad.any(), f"{'KV'[i]}: {int(bad.sum())} values differ, first at {bad.nonzero()[0].tolist()}"
        written = ~s[keep][..., i].isnan()
        assert torch.equal(s[keep][..., i][written].double(), (2.0 ** want.exps[keep])[written])
