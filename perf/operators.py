"""Performance cases of the 8-bit paged cache: written, read back, and attended.

The cache keeps K and V rows in e4m3 with one power-of-two scale for each block
of 16 tokens, kv head and K / V (``scales`` (n_pages, H_kv, page_size / 16, 2)):

* ``append``: new rows quantised into the pools, packed tokens (``rope``: from
  the fused QKV projection, rotated first).
* ``read``: cached rows back as 16-bit values.
* ``decode``: one query token per sequence against its pages; ``entry`` "plain"
  (cache only read), "append" (the new row written too) or "rope" (from the
  fused QKV projection); ``plan``: a step's plan, then ``layers`` calls on it.
* ``mixed``: varlen causal attention of prefill chunks and decode rows.

Lengths follow from the case alone, all tensor values from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False  # True: the framework's operators; False: their plain form in torch

BLOCK = 16        # tokens that share a scale
TOP = 448.0       # largest e4m3 value
LIMIT = 61440.0   # largest value held: 240 * 2**8 (16-bit values reach 65504)
E_MIN, E_MAX = -15, 8


def listed():
    return [
        # three users' next tokens, written outside the attention call: the smallest append
        _case("append_3_rows", "append", [1000, 17, 160], [1, 1, 1]),
        # a mixed step's new rows from the QKV projection: two prompt chunks and 24 running users
        _case("append_rope_464", "append", [0, 300] + _ramp(24, 128, 1024), [220, 220] + [1] * 24, rope=True),
        # four long prompts at once, 128-wide heads: the largest append
        _case("append_4x2048_d128", "append", [0, 5, 1000, 2047], [2048] * 4, h_q=32, h_kv=8, d=128),
        # one conversation's rows back, odd length
        _case("read_777", "read", [777], [0]),
        # a user's whole books back, 128-wide heads, larger pages
        _case("read_2_long", "read", [65536, 40001], [0, 0], h_q=32, h_kv=8, d=128, page=32),
        # one user's chat, 1,000 tokens in: the smallest decode
        _case("decode_1x1000", "decode", [1000], [1], entry="append"),
        # the benchmark's headline shape: 32 users, 4,096 tokens each
        _case("decode_32x4096", "decode", [4096] * 32, [1] * 32, entry="append"),
        # an odd number of users, each elsewhere in its conversation: a planned step of four layers
        _case("decode_43_ragged", "decode", _ramp(43, 512, 4096), [1] * 43, entry="rope", plan=True, layers=4),
        # a full house of long conversations, 128-wide heads: the largest decode
        _case("decode_96_d128", "decode", _ramp(96, 2048, 16384), [1] * 96, entry="plain", h_q=32, h_kv=8, d=128),
        # chunked prefill beside running decodes: the benchmark's mixed step
        _case("mixed_4x256_28", "mixed", [0, 512, 1024, 2048] + _ramp(28, 256, 2900), [256] * 4 + [1] * 28),
        # four new prompts of 2,048 tokens: compute-heavy prefill
        _case("mixed_4x2048", "mixed", [0] * 4, [2048] * 4),
        # ragged chunks over long prefixes beside decodes, 128-wide heads
        _case("mixed_ragged_d128", "mixed", [4096, 2001, 1000] + _ramp(13, 256, 4096), [1024, 701, 450] + [1] * 13,
              h_q=32, h_kv=8, d=128),
    ]


def _ramp(n, lo, hi):
    """n odd-ish lengths from lo to hi."""
    return [lo + (hi - lo) * i // max(1, n - 1) + (i % 3 if 0 < i < n - 1 else 0) for i in range(n)]


def _case(name, kind, prior, new, *, entry="plain", rope=False, plan=False, layers=1, h_q=14, h_kv=2, d=64, page=16):
    """prior / new tokens per sequence, as texts (a case holds plain values)."""
    return dict(name=name, kind=kind, prior=" ".join(map(str, prior)), new=" ".join(map(str, new)), entry=entry,
                rope=rope, plan=plan, layers=layers, h_q=h_q, h_kv=h_kv, d=d, page=page)


def _ints(text):
    return [int(x) for x in text.split()]


# (query heads, kv heads, head dim)
_HEADS = ((14, 2, 64), (14, 2, 64), (28, 4, 64), (8, 8, 64), (14, 2, 128), (32, 8, 128), (16, 1, 128))


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return w["bytes"] / 5e12 + w["flops"] / 5e14


def draw(rng):
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0.0), _cost(c))
    while True:
        h_q, h_kv, d = rng.choice(_HEADS)
        more = dict(h_q=h_q, h_kv=h_kv, d=d, page=rng.choice((16, 16, 32, 64)))
        kind = rng.choice(("append", "read", "decode", "decode", "mixed", "mixed"))
        hi = _log_int(rng, 16, 65536)
        lo = _log_int(rng, 1, hi)
        if kind == "decode":
            n = _log_int(rng, 1, 200)
            entry = rng.choice(("plain", "append", "rope"))
            plan = rng.random() < 0.4
            c = _case("", kind, [_log_int(rng, lo, hi) for _ in range(n)], [1] * n, entry=entry, plan=plan,
                      layers=rng.randint(2, 4) if plan else 1, **more)
        elif kind == "read":
            n = _log_int(rng, 1, 32)
            c = _case("", kind, [_log_int(rng, lo, hi) for _ in range(n)], [0] * n, **more)
        else:
            hi = min(hi, 8192)
            lo = min(lo, hi)
            n_pre, n_dec = rng.randint(0, 4), rng.randint(0, 48)
            if n_pre + n_dec == 0:
                continue
            top = _log_int(rng, 2, 2048)
            prior = [rng.choice((0, _log_int(rng, lo, hi))) for _ in range(n_pre)]
            prior += [_log_int(rng, lo, hi) for _ in range(n_dec)]
            new = [_log_int(rng, 2, top) for _ in range(n_pre)] + [1] * n_dec
            # (the plain form pads: its scores are at most what the largest listed case's take)
            if kind == "mixed" and len(new) * max(new) * (max(prior) + max(new)) * h_q > 4e9:
                continue
            c = _case("", kind, prior, new, rope=kind == "append" and rng.random() < 0.5, **more)
        if _cost(c) <= most[kind]:
            c.pop("name")
            return c


def work(case):
    prior, new = _ints(case["prior"]), _ints(case["new"])
    h_q, h_kv, d = case["h_q"], case["h_kv"], case["d"]
    row = h_kv * d
    if case["kind"] == "append":
        # the new rows read (rope: the queries too, and their rotary rows) and written in 8 bits
        T = sum(new)
        blocks = sum((p + n - 1) // BLOCK - p // BLOCK + 1 for p, n in zip(prior, new))
        b = T * row * 6 + blocks * h_kv * 8
        if case["rope"]:
            b += T * (4 * h_q * d + 4 * d)
        return {"bytes": b, "flops": 4 * T * row}
    if case["kind"] == "read":
        T = sum(prior)
        return {"bytes": T * row * 6 + -(-T // BLOCK) * h_kv * 8, "flops": 2 * T * row}
    # attention: every cached row and scale once, queries and outputs
    seen = [p + n for p, n in zip(prior, new)]
    T = sum(new)
    if case["kind"] == "decode" and case["entry"] == "plain":
        seen = prior
    b = sum(seen) * row * 2 + sum(-(-s // BLOCK) for s in seen) * h_kv * 8 + T * h_q * d * 4
    if case["kind"] == "decode" and case["entry"] != "plain":
        b += T * row * 6
    pairs = sum(s * n - n * (n - 1) // 2 for s, n in zip(seen, new))
    return {"bytes": case["layers"] * b, "flops": case["layers"] * 4 * pairs * h_q * d}


# ---- inputs ----

def _exponent(amax):
    """Least e with amax <= 448 * 2**e, in [-15, 8] (frexp: 448 = 0.875 * 2**9)."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(E_MIN, E_MAX)
    return torch.where(amax > 0, e, E_MIN)


def _to8(x, e):
    """x (fp32) in e4m3 at exponents e (broadcast): round to nearest even."""
    return torch.ldexp(x.clamp(-LIMIT, LIMIT), -e).to(torch.float8_e4m3fn)


def _history(T, case, gen, dev):
    """K and V rows as projections leave them: K with channels that stand out by head, both with louder tokens."""
    h, d = case["h_kv"], case["d"]
    loud = torch.exp(0.4 * torch.randn(T, 1, 1, device=dev, generator=gen))
    bias = torch.randn(1, h, d, device=dev, generator=gen) * (torch.rand(1, h, d, device=dev, generator=gen) < 0.05)
    k = torch.randn(T, h, d, device=dev, generator=gen) * 0.6 * loud + 6.0 * bias
    v = torch.randn(T, h, d, device=dev, generator=gen) * 0.5 * loud
    return k.half(), v.half()


def _spans(first, count):
    """(sequence, position) of tokens first[b] .. first[b] + count[b] of every sequence b."""
    n = torch.tensor(count)
    seq = torch.repeat_interleave(torch.arange(len(count)), n)
    return seq, torch.arange(seq.shape[0]) - (n.cumsum(0) - n)[seq] + torch.tensor(first)[seq]


def prepare(case, seed):
    with torch.inference_mode():
        dev = torch.device("cuda")
        gen = torch.Generator(dev).manual_seed(seed)
        prior, new, page = _ints(case["prior"]), _ints(case["new"]), case["page"]
        h_q, h_kv, d, B = case["h_q"], case["h_kv"], case["d"], len(prior)
        # "decode" writes its new row itself; "mixed" attends rows already written
        held = [p + n for p, n in zip(prior, new)] if case["kind"] == "mixed" else prior
        need = [-(-(p + n) // page) for p, n in zip(prior, new)]
        n_pages = 1 + sum(need)
        ids = 1 + torch.randperm(n_pages - 1, generator=torch.Generator().manual_seed(seed))  # pages anywhere in the pool
        table = torch.zeros(B + 1, n_pages, dtype=torch.int64)
        for b, x in enumerate(ids.split(need)):
            table[1 + b, :need[b]] = x
        lens = torch.tensor([0] + prior, dtype=torch.int64)
        cu = torch.zeros(B + 1, dtype=torch.int64)
        cu[1:] = torch.cumsum(torch.tensor(new), 0)
        s = {"case": case, "slots": torch.arange(1, B + 1), "table": table, "lens": lens,
             "kv_lens": torch.tensor(prior), "cu": cu}
        # each new (or, to read, each held) row's page and offset in it
        if case["kind"] == "read":
            seq, pos = _spans([0] * B, prior)
        else:
            seq, pos = _spans(prior, new)
        s["pages"], s["offsets"] = table[1 + seq, pos // page], pos % page
        s["seq"], s["pos"] = seq, pos
        s = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in s.items()}

        # the cache of one or more layers, its held rows quantised block by block
        hseq, hpos = (x.to(dev) for x in _spans([0] * B, held))
        hpage, hoff = s["table"][1 + hseq, hpos // page], hpos % page
        s["layers"] = []
        for _ in range(case["layers"]):
            pools, scales = [], []
            for x in _history(sum(held), case, gen, dev):
                rows = torch.zeros(n_pages, page, h_kv, d, dtype=torch.float16, device=dev)
                rows[hpage, hoff] = x
                rows = rows.transpose(1, 2).contiguous().view(n_pages, h_kv, page // BLOCK, BLOCK, d)
                e = _exponent(rows.abs().amax((3, 4)).float())
                pool = torch.empty(rows.shape, dtype=torch.float8_e4m3fn, device=dev)
                for i in range(0, n_pages, 4096):  # (a part at a time: it passes through fp32)
                    pool[i:i + 4096] = _to8(rows[i:i + 4096].float(), e[i:i + 4096, ..., None, None])
                pools.append(pool.view(n_pages, h_kv, page, d))
                scales.append(torch.ldexp(torch.ones_like(e, dtype=torch.float32), e))
            layer = {"k": pools[0], "v": pools[1], "scales": torch.stack(scales, -1).contiguous()}
            T = sum(new)
            if case["kind"] != "read" and T:
                k, v = _history(T, case, gen, dev)
                q = torch.randn(T, h_q, d, device=dev, generator=gen).half()
                if case["rope"] or case["entry"] == "rope":
                    layer["qkv"] = torch.cat([x.reshape(T, -1) for x in (q, k, v)], 1)[None].contiguous()
                else:
                    layer.update(q=q[None], k_new=k[None], v_new=v[None])
            s["layers"].append(layer)
        ang = s["pos"].double()[:, None] * 1e6 ** (-torch.arange(0, d, 2, device=dev).double() / d)
        s["cos"], s["sin"] = (torch.cat([f(ang)] * 2, 1).half()[None] for f in (torch.cos, torch.sin))
        s["row_in_seq"] = s["pos"] - s["kv_lens"][s["seq"]] if case["kind"] != "read" else None
        s["max_len"], s["max_new"] = max(p + n for p, n in zip(prior, new)), max(new)
        return s


# ---- one pass ----

def run(state):
    with torch.inference_mode():
        return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import custom_inference_engine_amd as cie

    case, first = s["case"], s["layers"][0]
    cache = (first["k"], first["v"], first["scales"])
    if case["kind"] == "read":
        return cie.kv_read_tokens_q8(*cache, s["pages"], s["offsets"])
    if case["kind"] == "append":
        out = list(cache)
        if case["rope"]:
            out.append(cie.append_tokens_qkv_rope_q8(first["qkv"], s["cos"], s["sin"], *cache, s["pages"], s["offsets"],
                                                     case["h_q"]))
        else:
            cie.kv_append_tokens_q8(*cache, first["k_new"], first["v_new"], s["pages"], s["offsets"])
        return out
    if case["kind"] == "mixed":
        return cie.mixed_gqa_attention_q8(first["q"], *cache, s["max_new"], s["cu"], s["kv_lens"], s["slots"], s["table"])
    append = case["entry"] != "plain"
    lens = s["lens"] if append else s["kv_lens"]
    plan = cie.decode_plan(first["k"], lens, s["slots"], s["table"], append=append) if case["plan"] else None
    out = []
    for l in s["layers"]:
        cache = (l["k"], l["v"], l["scales"])
        if case["entry"] == "rope":
            o = cie.decode_qkv_rope_gqa_attention_q8(l["qkv"], s["cos"], s["sin"], *cache, lens, s["slots"], s["table"],
                                                     case["h_q"], plan=plan)
        elif append:
            o = cie.decode_append_gqa_attention_q8(l["q"], *cache, l["k_new"], l["v_new"], lens, s["slots"], s["table"],
                                                   plan=plan)
        else:
            o = cie.decode_gqa_attention_q8(l["q"], *cache, lens, s["slots"], s["table"], plan=plan)
        out += [o, *cache] if append else [o]
    return out


def _rotate(x, cos, sin):
    """apply_rotary_pos_emb in fp32, rounded once (x (T, heads, d))."""
    x, half = x.float(), x.shape[-1] // 2
    return (x * cos[0, :, None].float() + torch.cat((-x[..., half:], x[..., :half]), -1) * sin[0, :, None].float()).half()


def _split(s, l):
    """A layer's q, k, v (T, heads, d): given, or split from its QKV rows and rotated."""
    case = s["case"]
    if "q" in l:
        return l["q"][0], l["k_new"][0], l["v_new"][0]
    q, k, v = l["qkv"][0].view(-1, case["h_q"] + 2 * case["h_kv"], case["d"]).split((case["h_q"],) + (case["h_kv"],) * 2, 1)
    return _rotate(q, s["cos"], s["sin"]), _rotate(k, s["cos"], s["sin"]), v


def _append_plain(pool, scales, x, pages, offsets):
    """Rows x (T, H, d) into (pages, offsets) of one pool; scales (n_pages, H, blocks) is a view."""
    n, h, page, d = pool.shape
    per = page // BLOCK
    block = pages * per + offsets // BLOCK
    amax = torch.zeros(n * per, h, device=x.device)
    amax.scatter_reduce_(0, block[:, None].expand(-1, h), x.abs().amax(2).float(), "amax")
    opens = torch.zeros(n * per, dtype=torch.int64, device=x.device)  # 1: written, 2: from its first row on
    opens.scatter_reduce_(0, block, 1 + (offsets % BLOCK == 0).long(), "amax")
    amax = amax.view(n, per, h).transpose(1, 2)
    opens = opens.view(n, per)[:, None].expand(n, h, per)
    old = torch.frexp(scales)[1] - 1
    e = torch.where(opens == 2, _exponent(amax), torch.where(opens == 1, torch.maximum(old, _exponent(amax)), old))
    kept = torch.where(opens == 2, e, old)  # the rows of a block that starts anew are left as they are
    rows = pool.view(n, h, per, BLOCK, d)
    pool.copy_(_to8(torch.ldexp(rows.float(), kept[..., None, None]), e[..., None, None]).view(n, h, page, d))
    at = e[pages, :, offsets // BLOCK]
    pool.view(torch.uint8)[pages, :, offsets] = _to8(x.float(), at[..., None]).view(torch.uint8)
    scales.copy_(torch.ldexp(torch.ones_like(scales), e))


def _rows_plain(l, name, pages, offsets):
    """Rows (pages, offsets) of a cache as fp32."""
    i = "kv".index(name)
    return l[name].view(torch.uint8)[pages, :, offsets].view(torch.float8_e4m3fn).float() * \
        l["scales"][pages, :, offsets // BLOCK, i][..., None]


def _attend_plain(s, l, q, seen, n_rows):
    """q (B, n_rows, h_q, d) padded; row i of sequence b attends keys [0, seen[b, i])."""
    case = s["case"]
    B, h_q, d = q.shape[0], case["h_q"], case["d"]
    h_kv = case["h_kv"]
    pos = torch.arange(s["max_len"], device=q.device)
    pages = s["table"][s["slots"]][:, pos // case["page"]]
    offs = (pos % case["page"])[None].expand(B, -1)
    k, v = (_rows_plain(l, n, pages, offs).transpose(1, 2).contiguous() for n in "kv")  # (B, h_kv, keys, d)
    q = q.float().view(B, n_rows, h_kv, h_q // h_kv, d).permute(0, 2, 3, 1, 4).reshape(B, h_kv, -1, d)
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5
    live = pos < seen.repeat(1, h_q // h_kv)[:, None, :, None]
    sc = sc.masked_fill_(~live, -math.inf)
    p = torch.exp(sc - sc.amax(3, keepdim=True).clamp_min(-1e30))
    v = v.masked_fill_((pos >= seen.amax(1)[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(p, v) / p.sum(3, keepdim=True).clamp_min(1e-30)
    return o.view(B, h_kv, h_q // h_kv, n_rows, d).permute(0, 3, 1, 2, 4).reshape(B, n_rows, h_q, d).half()


def _run_plain(s):
    case, first = s["case"], s["layers"][0]
    if case["kind"] == "read":
        return tuple(_rows_plain(first, n, s["pages"], s["offsets"]).half()[None] for n in "kv")
    if case["kind"] == "append":
        q, k, v = _split(s, first)
        _append_plain(first["k"], first["scales"][..., 0], k, s["pages"], s["offsets"])
        _append_plain(first["v"], first["scales"][..., 1], v, s["pages"], s["offsets"])
        return [first["k"], first["v"], first["scales"]] + ([q[None]] if case["rope"] else [])
    if case["kind"] == "mixed":
        B, n = s["slots"].shape[0], s["max_new"]
        q = torch.zeros(B, n, case["h_q"], case["d"], dtype=torch.float16, device=s["table"].device)
        q[s["seq"], s["row_in_seq"]] = first["q"][0]
        seen = s["kv_lens"][:, None] + 1 + torch.arange(n, device=q.device)
        seen = torch.minimum(seen, (s["kv_lens"] + s["cu"].diff())[:, None])
        return _attend_plain(s, first, q, seen, n)[s["seq"], s["row_in_seq"]][None]
    out = []
    for l in s["layers"]:
        q, k, v = _split(s, l)
        seen = s["kv_lens"][:, None]
        if case["entry"] != "plain":
            _append_plain(l["k"], l["scales"][..., 0], k, s["pages"], s["offsets"])
            _append_plain(l["v"], l["scales"][..., 1], v, s["pages"], s["offsets"])
            seen = seen + 1
        out.append(_attend_plain(s, l, q[:, None], seen, 1).transpose(0, 1))
        if case["entry"] != "plain":
            out += [l["k"], l["v"], l["scales"]]
    return out


# ---- the same in 64 bits ----

def _e4m3_64(y):
    """Nearest e4m3 value (ties to even) of y: 3 bits after the leading one, exponents from -6."""
    top = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -40)))
    step = 2.0 ** (top.clamp_min(-6) - 3)
    return (torch.round(y / step) * step).clamp(-TOP, TOP)


def _cache64(l, name):
    """(values, exponents) of a cache: e4m3 values before scaling (n, H, page, d), log2 scales (n, H, blocks)."""
    return l[name].float().double(), torch.log2(l["scales"][..., "kv".index(name)].double())


def _append64(cache, x, s):
    """The rows x (T, H, d) into a cache of _cache64, block after block in the order of their first rows."""
    vals, exps = cache
    page = s["case"]["page"]
    x = x.clamp(-LIMIT, LIMIT)
    need = torch.ceil(torch.log2(x.abs().amax(2) / TOP)).clamp(E_MIN, E_MAX)  # (T, H), exact: log2 of 1 is 0
    blocks = {}
    for t, (p, o) in enumerate(zip(s["pages"].tolist(), s["offsets"].tolist())):
        blocks.setdefault((p, o // BLOCK), []).append((o, t))
    for (p, i), rows in blocks.items():
        offs, ts = [o for o, _ in rows], [t for _, t in rows]
        e = need[ts].amax(0)
        at = slice(i * BLOCK, (i + 1) * BLOCK)
        if min(offs) % BLOCK:  # rows before these stay: their exponent can only grow
            old = exps[p, :, i]
            e = torch.maximum(e, old)
            vals[p, :, at] = _e4m3_64(vals[p, :, at] * 2.0 ** (old - e)[:, None, None])
        vals[p, :, offs] = _e4m3_64(x[ts] * 2.0 ** -e[None, :, None]).transpose(0, 1)
        exps[p, :, i] = e


def _attend64(s, caches, q, seen):
    """q (T, h_q, d) of sequences s["seq"]; row t attends seen[t] keys."""
    case, out = s["case"], torch.zeros_like(q)
    G, d, page = case["h_q"] // case["h_kv"], case["d"], case["page"]
    (kv, ke), (vv, ve) = caches
    for b in range(s["slots"].shape[0]):
        lo, hi = (int(x) for x in s["cu"][b:b + 2])
        n = int(seen[lo:hi].max())
        if n == 0:
            continue
        ids = s["table"][1 + b, :-(-n // page)]
        k, v = ((x[ids].double() * 2.0 ** e[ids].repeat_interleave(BLOCK, 2)[..., None]).transpose(0, 1)
                .reshape(case["h_kv"], -1, d)[:, :n] for x, e in ((kv, ke), (vv, ve)))
        mask = torch.arange(n, device=q.device)[None] >= seen[lo:hi, None]
        for h in range(case["h_q"]):
            sc = (q[lo:hi, h] @ k[h // G].t().contiguous()) * d ** -0.5
            out[lo:hi, h] = torch.softmax(sc.masked_fill_(mask, -math.inf), -1) @ v[h // G]
    return out


def exact(case, seed):
    if case["kind"] == "append" and sum(_ints(case["new"])) > 20000:
        return None
    with torch.inference_mode():
        s = prepare(case, seed)
        cos, sin = s["cos"][0].double()[:, None], s["sin"][0].double()[:, None]
        out = []
        for l in s["layers"]:
            if case["kind"] == "read":
                return tuple((v * 2.0 ** e.repeat_interleave(BLOCK, 2)[..., None])[s["pages"], :, s["offsets"]][None]
                             for v, e in (_cache64(l, n) for n in "kv"))
            if "q" in l:
                q, k, v = (l[n][0].double() for n in ("q", "k_new", "v_new"))
            else:
                x = l["qkv"][0].double().view(-1, case["h_q"] + 2 * case["h_kv"], case["d"])
                half = case["d"] // 2
                turned = x * cos + torch.cat((-x[..., half:], x[..., :half]), -1) * sin
                a = case["h_q"] + case["h_kv"]
                # (the cache and the attention take 16-bit rows: a rotated row is rounded to them)
                q, k, v = turned[:, :case["h_q"]], turned[:, case["h_q"]:a].half().double(), x[:, a:]
            caches = [_cache64(l, n) for n in "kv"]
            appends = case["kind"] == "append" or (case["kind"] == "decode" and case["entry"] != "plain")
            if appends:
                _append64(caches[0], k, s)
                _append64(caches[1], v, s)
            if case["kind"] != "append":
                seen = s["pos"] + (0 if case["kind"] == "decode" and not appends else 1)
                o = _attend64(s, caches, q.half().double(), seen)
                if case["kind"] == "mixed":
                    return o[None]
                out.append(o[None])
            if appends:
                out += [caches[0][0], caches[1][0], 2.0 ** torch.stack([caches[0][1], caches[1][1]], -1)]
            if case["kind"] == "append" and case["rope"]:
                out.append(q[None])
        return out
