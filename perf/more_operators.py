"""Performance cases of what a step needs before its attention: slot maps, adapters, rotary positions.

* ``step``: block tables and slot maps from request lengths, on the GPU.  ``entry`` "maps": the
  packed rows' positions, pages and offsets from tables that hold the step's pages already;
  "turn": the new tokens' pages are taken from a free list too, and given back afterwards (a
  step whose drafted tokens are dropped again), so that a pass leaves the tables as they were.
* ``rotary``: rows turned by their positions.  ``entry`` "apply": q and k split from the fused
  QKV projection; "append": q returned, k and v written into the paged pools; "tables": the
  cos / sin rows that the fused attention calls take.  ``layout`` "half" pairs dim i with
  i + rot / 2, "interleaved" 2i with 2i + 1; dims from ``rot`` on are copied.
* ``adapters``: y += scale * B (A x) with each row's own low-rank A and B, in place beside the
  shared projection's y: a step's plan of which rows share an adapter, then ``layers`` calls.

Lengths follow from the case alone, all tensor values from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False  # True: the framework's operators; False: their plain form in torch

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one user's next token: the smallest maps
        _step("maps_1", [1000], [1], 0, "maps"),
        # the benchmark's mixed step, 4 prompt chunks beside 28 decode rows, in its token bucket
        _step("maps_4x256_28", [0, 512, 1024, 2048] + _ramp(28, 256, 2900), [256] * 4 + [1] * 28, 4, "maps"),
        # 32 users with four drafted tokens each
        _step("turn_32x4", _ramp(32, 512, 4096), [4] * 32, 0, "turn"),
        # a large engine's step: 480 running users and 16 new prompts of 1,000 tokens
        _step("turn_496", [0] * 16 + _ramp(480, 64, 1500), [1000] * 16 + [1] * 480, 0, "turn"),
        # the queries and keys of 32 users' next tokens
        _rotary("rotary_32_rows", 32, 4096, "apply"),
        # a long conversation on a model whose positions are stretched fourfold: the step's tables
        _rotary("rotary_tables_1052", 1052, 120000, "tables", d=128, rot=128, scaling="yarn"),
        # an odd number of rows far out, half of each head turned in neighbouring pairs
        _rotary("rotary_part_777", 777, 1000000, "apply", h_q=32, h_kv=8, d=128, rot=64, layout="interleaved", dtype="bf16"),
        # a long prompt's rows into the cache, 128-wide heads: the largest rotary call
        _rotary("rotary_append_8192", 8192, 32768, "append", h_q=32, h_kv=8, d=128, rot=128),
        # one user's next token through one adapter, the fused QKV projection
        _adapters("adapters_1_row", [1], 1, 16, 896, (896, 128, 128)),
        # 32 users' next tokens, most on adapters of their own: a step's plan and four layers
        _adapters("adapters_32_rows", [1] * 32, 40, 16, 896, (896, 128, 128), layers=4),
        # a mixed step of requests with and without adapters of different ranks, odd width
        _adapters("adapters_mixed_1052", [256] * 4 + [1] * 28, 12, 64, 1000, (1000,), none=0.25, ragged=True, layers=2),
        # four new prompts of 2,048 tokens, 4,096 wide: the largest adapter call
        _adapters("adapters_4x2048", [2048] * 4, 8, 64, 4096, (4096,), dtype="bf16"),
    ]


def _ramp(n, lo, hi):
    """n odd-ish lengths from lo to hi."""
    return [lo + (hi - lo) * i // max(1, n - 1) + (i % 3 if 0 < i < n - 1 else 0) for i in range(n)]


def _step(name, prior, new, pad, entry, page=16):
    return dict(name=name, kind="step", prior=" ".join(map(str, prior)), new=" ".join(map(str, new)), pad=pad,
                entry=entry, page=page)


def _rotary(name, rows, far, entry, h_q=14, h_kv=2, d=64, rot=64, layout="half", scaling="none", dtype="fp16", page=16):
    return dict(name=name, kind="rotary", rows=rows, far=far, entry=entry, h_q=h_q, h_kv=h_kv, d=d, rot=rot,
                layout=layout, scaling=scaling, dtype=dtype, page=page)


def _adapters(name, new, n, rank, d_in, slices, none=0.0, ragged=False, layers=1, dtype="fp16"):
    """n adapters in the bank, of ``rank`` (ragged: of 1 to rank); a part ``none`` of the requests has none."""
    return dict(name=name, kind="adapters", new=" ".join(map(str, new)), n=n, rank=rank, d_in=d_in,
                slices=" ".join(map(str, slices)), none=none, ragged=ragged, layers=layers, dtype=dtype)


def _ints(text):
    return [int(x) for x in text.split()]


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
        kind = rng.choice(("step", "rotary", "adapters"))
        if kind == "step":
            n_pre, n_dec = rng.choice((0, 1, _log_int(rng, 1, 16))), rng.choice((0, _log_int(rng, 1, 480)))
            if n_pre + n_dec == 0:
                continue
            hi, top, page = _log_int(rng, 16, 32768), _log_int(rng, 2, 2048), rng.choice((16, 16, 32, 64))
            prior = [rng.choice((0, _log_int(rng, 1, hi))) for _ in range(n_pre)] + [_log_int(rng, 1, hi) for _ in range(n_dec)]
            new = [_log_int(rng, 2, top) for _ in range(n_pre)] + [rng.choice((1, 1, 4))] * n_dec
            c = _step("", prior, new, rng.choice((0, rng.randint(0, 40))), rng.choice(("maps", "turn")), page)
            need = sum(-(-(p + n) // page) for p, n in zip(prior, new))
            if need * len(prior) > 2e7:  # (the table has a column for each page)
                continue
        elif kind == "rotary":
            h_q, h_kv, d = rng.choice(((14, 2, 64), (14, 2, 64), (28, 4, 64), (8, 8, 64), (14, 2, 128), (32, 8, 128), (16, 1, 128)))
            entry = rng.choice(("apply", "apply", "append", "tables"))
            rot = d if entry == "tables" else rng.choice((d, d, d // 2, d // 4, 2 * rng.randint(1, d // 2)))
            c = _rotary("", _log_int(rng, 1, 8192), _log_int(rng, 256, 2000000), entry, h_q, h_kv, d, rot,
                        rng.choice(("half", "half", "interleaved")), rng.choice(("none", "linear", "yarn")),
                        rng.choice(("fp16", "fp16", "bf16")), rng.choice((16, 32, 64)))
        else:
            n_pre, n_dec, top = rng.choice((0, 0, rng.randint(1, 6))), rng.choice((0, _log_int(rng, 1, 256))), _log_int(rng, 2, 2048)
            if n_pre + n_dec == 0:
                continue
            new = [_log_int(rng, 2, top) for _ in range(n_pre)] + [1] * n_dec
            d_in = rng.choice((896, 1792, 4096, 8 * rng.randint(8, 512), rng.randint(64, 4096)))
            slices = rng.choice(((d_in,), (896, 128, 128), (4096,), (2048, 256, 256), (rng.randint(8, 4096), rng.randint(8, 1024))))
            c = _adapters("", new, _log_int(rng, 1, 128), rng.choice((8, 16, 16, 32, 64)), d_in, slices,
                          rng.choice((0.0, 0.25)), rng.random() < 0.5, rng.randint(1, 4), rng.choice(("fp16", "bf16")))
            # (the plain form takes each request's own weights, in 32 bits)
            if len(new) * len(slices) * c["rank"] * (d_in + max(slices)) > 4e8 or len(new) * max(new) * (d_in + sum(slices)) > 4e8:
                continue
        if _cost(c) <= most[kind]:
            c.pop("name")
            return c


def _ids(case):
    """Each request's adapter (-1: none) and each adapter's rank."""
    r = random.Random(case["n"] * 1000003 + len(case["new"]))
    ids = [-1 if r.random() < case["none"] else r.randrange(case["n"]) for _ in _ints(case["new"])]
    return ids, [r.randint(1, case["rank"]) if case["ragged"] else case["rank"] for _ in range(case["n"])]


def work(case):
    if case["kind"] == "step":
        prior, new, P = _ints(case["prior"]), _ints(case["new"]), case["page"]
        B, T = len(prior), sum(new) + case["pad"]
        # slots, new and held lengths in; a table word for each page that gets rows; four words a row out
        b = 8 * (3 * B + B + 1 + 4 * T + sum((p + n - 1) // P - p // P + 1 for p, n in zip(prior, new)))
        if case["entry"] == "turn":  # new pages: from the list into the table, and back
            b += 8 * 4 * sum(-(-(p + n) // P) - -(-p // P) for p, n in zip(prior, new)) + 8 * 3 * B
        return {"bytes": b, "flops": 0}
    if case["kind"] == "rotary":
        T, d, h = case["rows"], case["d"], case["h_q"] + case["h_kv"]
        b = 8 * T + 4 * case["rot"]
        if case["entry"] == "tables":
            return {"bytes": b + 4 * T * d, "flops": 2 * T * d}
        if case["entry"] == "append":
            b += 16 * T + 4 * T * case["h_kv"] * d
        return {"bytes": b + 4 * T * h * d, "flops": 3 * T * h * case["rot"]}
    new, slices = _ints(case["new"]), _ints(case["slices"])
    ids, ranks = _ids(case)
    S, out = len(slices), sum(slices)
    T = sum(n for n, i in zip(new, ids) if i >= 0)
    b = T * 2 * (case["d_in"] + 2 * out) + sum(2 * ranks[i] * (S * case["d_in"] + out) for i in set(ids) if i >= 0)
    f = sum(2 * n * ranks[i] * (S * case["d_in"] + out) for n, i in zip(new, ids) if i >= 0)
    return {"bytes": case["layers"] * b + 8 * sum(new), "flops": case["layers"] * f}


# ---- inputs ----

def frequencies(case):
    """Radians a position for each pair, and the factor of cos and sin."""
    r, base = case["rot"], 1e6
    f = [base ** (-2 * i / r) for i in range(r // 2)]
    if case["scaling"] == "linear":
        return [x / 4.0 for x in f], 1.0
    if case["scaling"] == "yarn":
        # pairs that turn over 32 times in the trained 32,768 positions stay, under once are stretched, a ramp between
        s, trained = 4.0, 32768
        at = [r * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (32, 1)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), r - 1)
        keep = [1 - min(max((i - lo) / max(hi - lo, 1e-3), 0), 1) for i in range(r // 2)]
        return [x / s * (1 - k) + x * k for x, k in zip(f, keep)], 0.1 * math.log(s) + 1
    return f, 1.0


def _spans(first, count):
    """(sequence, position) of tokens first[b] .. first[b] + count[b] of every sequence b."""
    n = torch.tensor(count)
    seq = torch.repeat_interleave(torch.arange(len(count)), n)
    return seq, torch.arange(seq.shape[0]) - (n.cumsum(0) - n)[seq] + torch.tensor(first)[seq]


def prepare(case, seed):
    with torch.inference_mode():
        dev = torch.device("cuda")
        gen = torch.Generator(dev).manual_seed(seed)
        host = torch.Generator().manual_seed(seed)
        s = {"case": case}
        if case["kind"] == "step":
            prior, new, P = _ints(case["prior"]), _ints(case["new"]), case["page"]
            B = len(prior)
            need = [-(-(p + n) // P) for p, n in zip(prior, new)]
            held = need if case["entry"] == "maps" else [-(-p // P) for p in prior]
            n_pages = 1 + sum(need)
            ids = 1 + torch.randperm(n_pages - 1, generator=host)  # pages anywhere in the pool
            slot = 1 + torch.randperm(B, generator=host)           # slots in any order
            table = torch.zeros(B + 1, n_pages, dtype=torch.int64)
            free = ids[sum(held):]
            for b, x in enumerate(ids[:sum(held)].split(held)):
                table[slot[b], :held[b]] = x
            lens = torch.zeros(B + 1, dtype=torch.int64)
            lens[slot] = torch.tensor(prior)
            # the free list: its count, a word of its own, and the pages, the next one last
            flist = torch.zeros(2 + n_pages, dtype=torch.int64)
            flist[0] = len(free)
            flist[2:2 + len(free)] = free
            s.update(slots=slot, new=torch.tensor(new), lens=lens, table=table, free=flist, T=sum(new) + case["pad"],
                     prior=torch.tensor(prior), held=torch.tensor(prior) + torch.tensor(new), most=max(need))
        elif case["kind"] == "rotary":
            T, d, h_q, h_kv, P = case["rows"], case["d"], case["h_q"], case["h_kv"], case["page"]
            f, s["scale"] = frequencies(case)
            s["freqs"] = torch.tensor(f, dtype=torch.float64)
            # a few requests' packed rows, each a run of positions
            n_req = max(1, min(T, 1 + T // 300))
            first = torch.randint(0, case["far"], (n_req,), generator=host)
            row = torch.arange(T)
            s["pos"] = first[row * n_req // T] + row
            if case["entry"] != "tables":
                s["qkv"] = torch.randn(1, T, (h_q + 2 * h_kv) * d, device=dev, generator=gen).to(_TYPES[case["dtype"]])
            if case["entry"] == "append":
                n_pages = 1 + -(-T // P)
                page = 1 + torch.randperm(n_pages - 1, generator=host)
                s["pages"], s["offsets"] = page[row // P], row % P
                s["k"], s["v"] = (torch.randn(n_pages, h_kv, P, d, device=dev, generator=gen).to(_TYPES[case["dtype"]])
                                  for _ in range(2))
        else:
            new, slices = _ints(case["new"]), _ints(case["slices"])
            ids, ranks = _ids(case)
            T, B, S, n, t = sum(new), len(new), len(slices), case["n"], _TYPES[case["dtype"]]
            R = -(-case["rank"] // 16) * 16  # the bank's rows of rank: whole 16s, zeros behind an adapter's own
            seq, at = _spans([0] * B, new)
            slot = 1 + torch.randperm(B, generator=host)
            by_slot = torch.full((B + 1,), -1)
            by_slot[slot] = torch.tensor(ids)
            s.update(row_slots=slot[seq], by_slot=by_slot, seq=seq, at=at, ids=torch.tensor(ids), slices=tuple(slices),
                     ranks=torch.tensor(ranks, dtype=torch.int32), scales=0.5 + torch.rand(n, generator=host), most=max(new))
            live = (torch.arange(R) < torch.tensor(ranks)[:, None]).to(dev)
            s["layers"] = []
            for _ in range(case["layers"]):
                a = torch.randn(n, S, R, case["d_in"], device=dev, generator=gen) * case["d_in"] ** -0.5
                b = torch.randn(n, sum(slices), R, device=dev, generator=gen) * 0.3
                s["layers"].append({
                    "a": (a * live[:, None, :, None]).to(t), "b": (b * live[:, None]).to(t),
                    "x": torch.randn(T, case["d_in"], device=dev, generator=gen).to(t),
                    "y": torch.randn(T, sum(slices), device=dev, generator=gen).to(t)})
        return {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in s.items()}


# ---- one pass ----

def run(state):
    with torch.inference_mode():
        return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import custom_inference_engine_amd as cie

    case = s["case"]
    if case["kind"] == "step":
        turn = case["entry"] == "turn"
        m = cie.step_maps(s["slots"], s["new"], s["lens"], s["table"], case["page"], s["T"],
                          free_list=s["free"] if turn else None)
        if turn:
            cie.release_pages(s["free"], s["slots"], s["lens"], s["table"], case["page"], keep=s["prior"], held=s["held"])
        return [m.cu_seqlens, m.slots, m.positions, m.pages, m.offsets, s["lens"], s["table"], s["free"]]
    if case["kind"] == "rotary":
        how = dict(interleaved=case["layout"] == "interleaved", scale=s["scale"])
        if case["entry"] == "tables":
            return cie.rotary_tables(s["pos"], s["freqs"], dtype=_TYPES[case["dtype"]], **how)
        if case["entry"] == "append":
            q = cie.append_tokens_qkv_rotary(s["qkv"], s["pos"], s["freqs"], s["k"], s["v"], s["pages"], s["offsets"],
                                             case["h_q"], **how)
            return [q, s["k"], s["v"]]
        q, k, _ = s["qkv"].view(1, case["rows"], -1, case["d"]).split((case["h_q"],) + (case["h_kv"],) * 2, 2)
        return cie.apply_rotary(q, k, s["pos"], s["freqs"], **how)
    plan = cie.adapter_plan(s["row_slots"], s["by_slot"], case["n"])
    return [cie.adapter_add_(l["y"], l["x"], l["a"], l["b"], s["scales"], s["ranks"], plan, s["slices"])
            for l in s["layers"]]


def _step_plain(s):
    case, P, lens, table, free = s["case"], s["case"]["page"], s["lens"], s["table"], s["free"]
    slots, new = s["slots"], s["new"]
    prior = lens[slots]
    end = new.cumsum(0)
    cu = torch.cat((torch.zeros_like(end[:1]), end))
    col = torch.arange(s["most"], device=slots.device)
    if case["entry"] == "turn":  # the pages past those held, from the list's end on
        have, want = (prior + P - 1) // P, (prior + new + P - 1) // P
        rank = (want - have).cumsum(0) - want
        fresh = (col >= have[:, None]) & (col < want[:, None])
        taken = free[(free[0] + 1 - rank[:, None] - col).clamp(2, free.shape[0] - 1)]
        rows = table[:, :s["most"]]
        rows[slots] = torch.where(fresh, taken, rows[slots])
        free[0] -= (want - have).sum()
    row = torch.arange(s["T"], device=slots.device)
    seq = torch.searchsorted(end, row, right=True)
    live = seq < slots.shape[0]
    seq = seq.clamp(max=slots.shape[0] - 1)
    slot = torch.where(live, slots[seq], 0)
    pos = torch.where(live, lens[slot] + row - cu[seq], 0)
    out = [cu, slot, pos, torch.where(live, table[slot, pos // P], 0), pos % P]
    if case["entry"] == "turn":  # all of it back: the list's words are still there
        held, keep = (s["held"] + P - 1) // P, (s["prior"] + P - 1) // P
        back = (col >= keep[:, None]) & (col < held[:, None])
        rank = (held - keep).cumsum(0) - held
        n = (held - keep).sum()
        ids = rows[slots]
        at = torch.where(back, free[0] + n + 1 - rank[:, None] - col, 1)
        free.scatter_(0, at.flatten(), torch.where(back, ids, 0).flatten())
        rows[slots] = torch.where(back, 0, ids)
        lens[slots] = s["prior"]
        free[0] += n
    return out + [lens, table, free]


def _cos_sin(s):
    """cos and sin (rows, pairs) in 32 bits, of angles taken in 64."""
    ang = torch.remainder(s["pos"].double()[:, None] * s["freqs"], 2 * math.pi)
    return (torch.cos(ang) * s["scale"]).float(), (torch.sin(ang) * s["scale"]).float()


def _turn(x, cos, sin, layout):
    """x (rows, heads, d) with its first 2 * pairs dims turned; in the type of cos and sin."""
    x, n = x.to(cos.dtype), cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    if layout == "half":
        a, b = x[..., :n], x[..., n:2 * n]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * n:]), -1)
    a, b = x[..., :2 * n:2], x[..., 1:2 * n:2]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), x[..., 2 * n:]), -1)


def _rotary_rows(s, cos, sin):
    """The turned queries, the turned keys and the values, (rows, heads, d)."""
    case = s["case"]
    q, k, v = s["qkv"][0].view(case["rows"], -1, case["d"]).split((case["h_q"],) + (case["h_kv"],) * 2, 1)
    return _turn(q, cos, sin, case["layout"]), _turn(k, cos, sin, case["layout"]), v


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "step":
        return _step_plain(s)
    if case["kind"] == "rotary":
        t = _TYPES[case["dtype"]]
        cos, sin = _cos_sin(s)
        if case["entry"] == "tables":
            return tuple(_both(x, case["layout"]).to(t)[None] for x in (cos, sin))
        q, k, v = _rotary_rows(s, cos, sin)
        if case["entry"] == "apply":
            return q.to(t)[None], k.to(t)[None]
        s["k"][s["pages"], :, s["offsets"]] = k.to(t)
        s["v"][s["pages"], :, s["offsets"]] = v
        return [q.to(t)[None], s["k"], s["v"]]
    # each request's rows side by side, padded, with its adapter's weights
    at = s["ids"].clamp(min=0)
    scale = torch.where(s["ids"] >= 0, s["scales"][at], 0)[:, None, None]
    B, S, n = at.shape[0], len(s["slices"]), s["most"]
    return [_adapters_plain(s, l, at, scale, B, S, n) for l in s["layers"]]


def _both(x, layout):
    """A factor for each dim from one for each pair."""
    return torch.cat((x, x), -1) if layout == "half" else x.repeat_interleave(2, -1)


def _adapters_plain(s, l, at, scale, B, S, n):
    x = torch.zeros(B, n, l["x"].shape[1], device=l["x"].device)
    x[s["seq"], s["at"]] = l["x"].float()
    a = l["a"][at].float()  # (B, S, R, d_in)
    R = a.shape[2]
    u = torch.matmul(x, a.view(B, S * R, -1).transpose(1, 2).contiguous()).view(B, n, S, R)
    b = l["b"][at].float()  # (B, d_out, R)
    which = torch.repeat_interleave(torch.arange(S, device=x.device), torch.tensor(s["slices"], device=x.device))
    # a column's slice picks its own ranks: B's columns spread over all of them, zeros elsewhere
    wide = (which[:, None] == torch.arange(S, device=x.device))[None, :, :, None] * b[:, :, None]
    d = torch.matmul(u.flatten(2), wide.flatten(2).transpose(1, 2).contiguous()) * scale
    l["y"].copy_(l["y"].float() + d[s["seq"], s["at"]])
    return l["y"]


# ---- the same in 64 bits ----

def exact(case, seed):
    if case["kind"] == "step":
        return None  # (whole numbers)
    with torch.inference_mode():
        s = prepare(case, seed)
        if case["kind"] == "rotary":
            f, scale = frequencies(case)
            n, x = len(f), None
            turns = s["pos"].double()[:, None] * (torch.tensor(f, dtype=torch.float64, device="cuda") / (2 * math.pi))
            z = torch.polar(torch.full_like(turns, scale), 2 * math.pi * (turns - turns.round()))  # a turn as a complex factor
            if case["entry"] == "tables":
                whole = torch.cat((z, z), 1) if case["layout"] == "half" else torch.stack((z, z), 2).flatten(1)
                return whole.real[None], whole.imag[None]
            x = s["qkv"][0].double().view(case["rows"], -1, case["d"])
            heads = x[:, :case["h_q"] + case["h_kv"]]
            if case["layout"] == "half":
                w = torch.complex(heads[..., :n].contiguous(), heads[..., n:2 * n].contiguous()) * z[:, None]
                turned = torch.cat((w.real, w.imag, heads[..., 2 * n:]), -1)
            else:
                w = torch.view_as_complex(heads[..., :2 * n].reshape(*heads.shape[:2], n, 2)) * z[:, None]
                turned = torch.cat((torch.view_as_real(w).flatten(-2), heads[..., 2 * n:]), -1)
            q, k = turned[:, :case["h_q"]], turned[:, case["h_q"]:]
            if case["entry"] == "apply":
                return q[None], k[None]
            pools = [s["k"].double(), s["v"].double()]
            for pool, rows in zip(pools, (k, x[:, case["h_q"] + case["h_kv"]:])):
                pool[s["pages"], :, s["offsets"]] = rows
            return [q[None], *pools]
        new, slices = _ints(case["new"]), _ints(case["slices"])
        ids, _ = _ids(case)
        out = []
        for l in s["layers"]:
            y, lo = l["y"].double(), 0
            for n, i in zip(new, ids):
                if i >= 0:
                    x, c = l["x"][lo:lo + n].double(), 0
                    for k, width in enumerate(slices):
                        u = x @ l["a"][i, k].double().t().contiguous()
                        y[lo:lo + n, c:c + width] += float(s["scales"][i]) * (u @ l["b"][i, c:c + width].double().t().contiguous())
                        c += width
                lo += n
            out.append(y)
        return out
