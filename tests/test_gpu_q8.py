"""The 8-bit paged cache on the GPU: written, read back and attended, against plain 64-bit implementations."""
import pytest
import torch

import custom_inference_engine_amd as cie
from custom_inference_engine_amd import _native
from custom_inference_engine_amd.graphs import StepGraph
from oracle import paged_attention as paged
from oracle import q8_cache as ref
from tests.gpu_helpers import DEV, err_word, note
from tests.q8_helpers import Case, rows, same_cache

pytestmark = pytest.mark.gpu

PAGE, LEN, OFFSET, SPLIT, PLAN = 1, 2, 4, 8, 16


def append_tokens(c, err=None, order=None):
    pages, offs = c.new_at()
    order = torch.arange(c.T) if order is None else order
    cie.kv_append_tokens_q8(c.k, c.v, c.scales, c.k_new[:, order].to(DEV), c.v_new[:, order].to(DEV),
                            pages[order].to(DEV), offs[order].to(DEV), err=err)


def oracle_append(c, oracles, order=None):
    pages, offs = c.new_at()
    order = torch.arange(c.T) if order is None else order
    for o, x in zip(oracles, (c.k_new, c.v_new)):
        o.append(x[0, order], pages[order], offs[order])


# ---- append ----

SHAPES = [
    dict(prior=[0], new=[1]),
    dict(prior=[0, 15, 16, 17, 31], new=[1, 1, 1, 1, 1]),
    dict(prior=[0, 5, 20, 37, 0], new=[17, 1, 3, 1, 0]),
    dict(prior=[3, 100], new=[64, 33], page=32, d=128),
    dict(prior=[7, 0, 90], new=[45, 2, 1], page=48, h_kv=1, h_q=7),
    dict(prior=[60, 130], new=[70, 1], page=64, h_kv=8, h_q=8),
    dict(prior=[1, 2030, 0], new=[1500, 700, 333]),  # more than 2,048 tokens: four a workgroup
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s['prior']}+{s['new']}")
def test_token_append(native_lib, shape):
    note(f"q8 token append {shape}")
    c = Case(**shape, seed=1).write_history()
    want = c.oracles()
    err = err_word()
    append_tokens(c, err)
    oracle_append(c, want)
    same_cache(c, want)
    assert int(err) == 0


def test_history_in_pieces_is_the_definition(native_lib):
    """Write_history's own calls, against the oracle on the same pieces (blocks cut by call borders)."""
    note("q8 history")
    c = Case(prior=[40], new=[0])
    k, v = c.history[0]
    oracles = c.oracles()
    for lo, n in ((0, 3), (3, 1), (4, 15), (19, 13), (32, 8)):
        pages, offs = c.at(0, lo, n)
        cie.kv_append_tokens_q8(c.k, c.v, c.scales, k[lo:lo + n].to(DEV), v[lo:lo + n].to(DEV), pages.to(DEV),
                                offs.to(DEV))
        for o, x in zip(oracles, (k, v)):
            o.append(x[lo:lo + n], pages, offs)
    same_cache(c, oracles)


def test_token_append_in_any_order_and_twice(native_lib):
    """A shuffled list, and one with every index twice: the last row of an index, with no race on its block."""
    note("q8 append order")
    for seed in range(3):
        c = Case(prior=[5, 33], new=[50, 40], seed=seed).write_history()
        want = c.oracles()
        g = torch.Generator().manual_seed(seed)
        order = torch.cat([torch.randperm(c.T, generator=g), torch.randperm(c.T, generator=g)])
        pages, offs = c.new_at()
        k = rows(g, 2 * c.T, c.h_kv, c.d)
        v = rows(g, 2 * c.T, c.h_kv, c.d)
        cie.kv_append_tokens_q8(c.k, c.v, c.scales, k.to(DEV), v.to(DEV), pages[order].to(DEV), offs[order].to(DEV))
        for o, x in zip(want, (k, v)):
            o.append(x, pages[order], offs[order])
        same_cache(c, want)


def test_append_values_at_the_edges(native_lib):
    """Zeros, subnormals, infinities, the largest fp16, NaN, negative zero; a tiny block that grows to the largest."""
    note("q8 append edges")
    c = Case(prior=[0], new=[8], h_kv=2, h_q=2)
    x = c.k_new
    x[:, 0] = 0
    x[:, 1] = 2.0 ** -24
    x[:, 2] = -0.0
    x[:, 3] = 2.0 ** -15
    x[0, 4, 0, ::2] = float("inf")
    x[0, 4, 1, 5] = float("-inf")
    x[0, 5, 0, 7] = float("nan")
    x[:, 6] = 65504.0
    x[:, 7] = -61440.0
    c.v_new = x.flip(1).contiguous()
    want = c.oracles()
    for t in range(8):  # token by token: every growth
        pages, offs = c.at(0, t, 1)
        cie.kv_append_tokens_q8(c.k, c.v, c.scales, c.k_new[:, t:t + 1].to(DEV), c.v_new[:, t:t + 1].to(DEV),
                                pages.to(DEV), offs.to(DEV))
        for o, y in zip(want, (c.k_new, c.v_new)):
            o.append(y[0, t:t + 1], pages, offs)
        same_cache(c, want)


@pytest.mark.parametrize("shape", [
    dict(prior=[0, 1, 14, 15, 16, 31, 47, 100]),
    dict(prior=[5, 70, 64], page=32, d=128, h_kv=8, h_q=32),
    dict(prior=[5, 70, 64, 128] * 70, page=64, h_kv=1, h_q=4),
], ids=["edges", "page32", "batch280"])
def test_decode_append(native_lib, shape):
    note(f"q8 decode append {len(shape['prior'])}")
    c = Case(new=[1] * len(shape["prior"]), **shape, seed=2).write_history()
    want = c.oracles()
    err = err_word()
    cie.kv_append_decode_q8(c.k, c.v, c.scales, *c.dev("k_new", "v_new", "slots", "lens", "table"), err=err)
    oracle_append(c, want)
    same_cache(c, want)
    assert int(err) == 0


def test_decode_append_padding_and_a_slot_twice(native_lib):
    """Padding rows (slot 0) touch page 0 only; of a slot that comes twice the last row is written."""
    note("q8 decode append padding")
    c = Case(prior=[9, 33], new=[1, 1], seed=3).write_history()
    want = c.oracles()
    g = torch.Generator().manual_seed(5)
    k, v = rows(g, 6, 2, 64), rows(g, 6, 2, 64)
    slots = torch.tensor([0, 2, 1, 0, 2, 0])
    cie.kv_append_decode_q8(c.k, c.v, c.scales, k[None].to(DEV), v[None].to(DEV), slots.to(DEV), c.lens.to(DEV),
                            c.table.to(DEV))
    pages, offs = c.new_at()
    for o, x in zip(want, (k, v)):
        o.append(x[[2, 4, 5]], [int(pages[0]), int(pages[1]), 0], [int(offs[0]), int(offs[1]), 0])
    same_cache(c, want)


def test_append_bad_indices(native_lib):
    note("q8 append errors")
    c = Case(prior=[4, 20, 8], new=[1, 1, 1], seed=4).write_history()
    want = c.oracles()
    n = c.k.shape[0]
    err = err_word()
    pages, offs = c.new_at()
    pages[0], offs[2] = n + 5, 16
    cie.kv_append_tokens_q8(c.k, c.v, c.scales, *c.dev("k_new", "v_new"), pages.to(DEV), offs.to(DEV), err=err)
    assert int(err) == PAGE | OFFSET
    for o, x in zip(want, (c.k_new, c.v_new)):
        o.append(x[0, 1:2], pages[1:2], offs[1:2])
    same_cache(c, want)
    err.zero_()
    slots, lens = torch.tensor([-1, 99, 3]), c.lens.clone()
    lens[3] = n * 16
    cie.kv_append_decode_q8(c.k, c.v, c.scales, *c.dev("k_new", "v_new"), slots.to(DEV), lens.to(DEV),
                            c.table.to(DEV), err=err)
    assert int(err) == PAGE | LEN
    same_cache(c, want)


def test_append_strided(native_lib):
    """K and V out of a fused projection's rows, and pools that are every other page of larger ones."""
    note("q8 append strided")
    c = Case(prior=[6, 40], new=[20, 3], seed=6).write_history()
    want = c.oracles()
    fused = torch.zeros(1, c.T, 18 * 64, dtype=torch.float16, device=DEV)
    fused[..., 896:1024] = c.k_new.to(DEV).view(1, c.T, 128)
    fused[..., 1024:] = c.v_new.to(DEV).view(1, c.T, 128)
    wide = [torch.zeros(2 * c.k.shape[0], *c.k.shape[1:], dtype=torch.uint8, device=DEV) for _ in "kv"]
    for w, p in zip(wide, (c.k, c.v)):
        w[::2] = p.view(torch.uint8)
    c.k, c.v = (w.view(torch.float8_e4m3fn)[::2] for w in wide)
    pages, offs = c.new_at()
    cie.kv_append_tokens_q8(c.k, c.v, c.scales, fused[..., 896:1024].view(1, c.T, 2, 64),
                            fused[..., 1024:].view(1, c.T, 2, 64), pages.to(DEV), offs.to(DEV))
    oracle_append(c, want)
    same_cache(c, want)
    assert all(not w[1::2].any() for w in wide)
    k, _ = cie.kv_read_tokens_q8(c.k, c.v, c.scales, pages.to(DEV), offs.to(DEV))
    assert torch.equal(k[0].cpu().double(), want[0].values()[pages, :, offs])


def rope_tables(pos, d):
    ang = pos.double()[:, None] * 1e6 ** (-torch.arange(0, d, 2).double() / d)
    return [torch.cat([f(ang)] * 2, 1).half()[None] for f in (torch.cos, torch.sin)]


def rotate(x, cos, sin):
    return paged.rope(x[0], cos[0], sin[0])[None]


def fused_rows(c):
    return torch.cat([x[0].reshape(c.T, -1) for x in (c.q, c.k_new, c.v_new)], 1)[None].contiguous()


@pytest.mark.parametrize("shape", [
    dict(prior=[0, 5, 100], new=[40, 1, 17]),
    dict(prior=[30, 0], new=[1, 70], d=128, h_q=32, h_kv=8, page=32),
    dict(prior=[0], new=[2100], h_q=4, h_kv=1),
], ids=["d64", "d128", "long"])
def test_rope_append_is_rotate_then_append(native_lib, shape):
    note(f"q8 rope append {shape}")
    c = Case(**shape, seed=7).write_history()
    want = c.oracles()
    pages, offs = c.new_at()
    pos = torch.cat([torch.arange(p, p + n) for p, n in zip(c.prior, c.new)])
    cos, sin = rope_tables(pos, c.d)
    err = err_word()
    q = cie.append_tokens_qkv_rope_q8(fused_rows(c).to(DEV), cos.to(DEV), sin.to(DEV), c.k, c.v, c.scales,
                                      pages.to(DEV), offs.to(DEV), c.h_q, err=err)
    assert torch.equal(q.cpu(), rotate(c.q, cos, sin))
    c.k_new = rotate(c.k_new, cos, sin)
    oracle_append(c, want)
    same_cache(c, want)
    assert int(err) == 0


# ---- read ----

@pytest.mark.parametrize("shape", [dict(prior=[1]), dict(prior=[77, 16, 3], page=32),
                                   dict(prior=[130, 64], d=128, h_kv=8, h_q=8, page=64)], ids=str)
def test_read_back(native_lib, shape):
    note(f"q8 read {shape}")
    c = Case(new=[0] * len(shape["prior"]), **shape, seed=8).write_history()
    where = [c.at(b, 0, p) for b, p in enumerate(c.prior)]
    pages, offs = torch.cat([w[0] for w in where]), torch.cat([w[1] for w in where])
    order = torch.randperm(len(pages), generator=torch.Generator().manual_seed(0))
    pages, offs = pages[order], offs[order]
    got = cie.kv_read_tokens_q8(c.k, c.v, c.scales, pages.to(DEV), offs.to(DEV))
    for g, o in zip(got, c.oracles()):
        assert g.shape == (1, len(pages), c.h_kv, c.d)
        assert torch.equal(g[0].cpu().double(), o.values()[pages, :, offs])
    # what was written, to half a step of e4m3 (2^-4 of a value; under the smallest normal 2^-10 of the scale, once
    # for its own rounding and at most once for each of a block's growths: the scale at least doubles each time, so
    # in all less than 2 * 2^-10 of the last)
    k = torch.cat([h[0] for h in c.history])[order].double()
    s = c.scales[..., 0].cpu()[pages, :, offs // 16].double()[..., None]
    assert ((got[0][0].cpu().double() - k).abs() <= k.abs() * 2.0 ** -4 + s * 2.0 ** -9).all()


def test_read_bad_indices_are_zeros(native_lib):
    note("q8 read errors")
    c = Case(prior=[20], new=[0]).write_history()
    err = err_word()
    k, v = cie.kv_read_tokens_q8(c.k, c.v, c.scales, torch.tensor([10 ** 9, -1, 1, 1], device=DEV),
                                 torch.tensor([0, 0, 16, -1], device=DEV), err=err)
    assert not k.any() and not v.any() and int(err) == PAGE | OFFSET
    k, v = cie.kv_read_tokens_q8(c.k, c.v, c.scales, *[torch.zeros(0, dtype=torch.int64, device=DEV)] * 2)
    assert k.shape == (1, 0, 2, 64)


# ---- decode ----

def check_attention(got, want, n_keys, what=""):
    o, mass, top = want
    err = (got.cpu().double() - o).abs()
    tol = ref.tolerance(o, mass, top, n_keys)
    assert torch.isfinite(got).all(), what
    assert (err <= tol).all(), f"{what}: {int((err > tol).sum())} of {err.numel()} off, worst {float((err / tol).max()):.2f} of tolerance"


def decode_seqs(c, lens):
    return [(b, 1, b + 1, int(n)) for b, n in enumerate(lens)]


DECODE = [
    (dict(prior=[0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129]), [None, 1, 2, 5, 64]),
    (dict(prior=[1000]), [None, 1, 16, 64]),
    (dict(prior=[300, 4097, 77], d=128, h_q=32, h_kv=8), [None, 1, 3]),
    (dict(prior=[50, 260], page=48, h_q=16, h_kv=1), [None, 7]),
    (dict(prior=[50, 260], page=64, h_q=8, h_kv=8, d=128), [None, 2]),
    (dict(prior=[9000], h_q=16, h_kv=1, d=128), [1, 9]),  # a wave of more than 64 tiles
]


@pytest.mark.parametrize("shape,splits", DECODE, ids=[str(d[0]["prior"])[:30] + f"d{d[0].get('d', 64)}" for d in DECODE])
def test_decode(native_lib, shape, splits):
    c = Case(new=[1] * len(shape["prior"]), **shape, seed=9).write_history()
    want = ref.attend(c.q[0], *c.oracles(), decode_seqs(c, c.prior), c.table)
    for P in splits:
        note(f"q8 decode {shape} splits {P}")
        err = err_word()
        o = cie.decode_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales, *c.dev("kv_lens", "slots", "table"),
                                        num_programs=P, err=err)
        check_attention(o[0], want, max(c.prior), f"splits {P}")
        assert int(err) == 0
    plan = cie.decode_plan(c.k, *c.dev("kv_lens", "slots", "table"), append=False)
    o = cie.decode_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales, *c.dev("kv_lens", "slots", "table"), plan=plan)
    check_attention(o[0], want, max(c.prior), "planned")


def decode_append(c, plan=None, P=None, err=None):
    return cie.decode_append_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales,
                                              *c.dev("k_new", "v_new", "lens", "slots", "table"), plan=plan,
                                              num_programs=P, err=err)


@pytest.mark.parametrize("shape", [
    dict(prior=[0, 1, 14, 15, 16, 17, 31, 47, 100, 1000]),
    dict(prior=[5, 70, 64, 700], page=32, d=128, h_q=32, h_kv=8),
    dict(prior=[13, 200], page=64, h_q=16, h_kv=1, d=128),
    dict(prior=[4200, 3], h_q=4, h_kv=1),  # the new row's tile past a wave's first 64
], ids=["edges", "d128", "page64", "long"])
@pytest.mark.parametrize("form", ["1", "3", "default", "planned"])
def test_decode_append_is_append_then_decode(native_lib, shape, form):
    """Bytes, scales and outputs of the fused launch, for rows that grow their block and rows that do not."""
    for seed in (10, 11):
        c = Case(new=[1] * len(shape["prior"]), **shape, seed=seed).write_history()
        if seed == 11:
            c.k_new *= 30  # every block grows
        want = c.oracles()
        P = int(form) if form.isdigit() else None
        plan = cie.decode_plan(c.k, *c.dev("lens", "slots", "table")) if form == "planned" else None
        note(f"q8 decode append {shape} {form}")
        err = err_word()
        o = decode_append(c, plan, P, err)
        oracle_append(c, want)
        same_cache(c, want)
        seqs = decode_seqs(c, [p + 1 for p in c.prior])
        check_attention(o[0], ref.attend(c.q[0], *want, seqs, c.table), max(c.prior) + 1, form)
        assert int(err) == 0


@pytest.mark.parametrize("shape", [dict(prior=[0, 15, 33, 500]), dict(prior=[64, 77], d=128, h_q=32, h_kv=8, page=32),
                                   dict(prior=[2, 4300], d=128, h_q=7, h_kv=1)], ids=["d64", "d128", "g7"])
def test_decode_rope_is_rotate_then_decode(native_lib, shape):
    c = Case(new=[1] * len(shape["prior"]), **shape, seed=12).write_history()
    cos, sin = rope_tables(c.kv_lens, c.d)
    qkv = fused_rows(c)
    before = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.scales)]
    c.q, c.k_new = rotate(c.q, cos, sin), rotate(c.k_new, cos, sin)
    o = {P: decode_append(c, P=P) for P in (1, 4)}
    after = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.scales)]
    for P in (1, 4):
        note(f"q8 decode rope {shape} splits {P}")
        k, v, s = (t.clone() for t in before)
        got = cie.decode_qkv_rope_gqa_attention_q8(qkv.to(DEV), cos.to(DEV), sin.to(DEV), k.view(torch.float8_e4m3fn),
                                                   v.view(torch.float8_e4m3fn), s, *c.dev("lens", "slots", "table"),
                                                   c.h_q, num_programs=P)
        assert torch.equal(got, o[P])
        assert torch.equal(k, after[0]) and torch.equal(v, after[1])
        assert torch.equal(s.view(torch.int32), after[2].view(torch.int32))


def test_decode_padding_rows_and_bad_indices(native_lib):
    note("q8 decode padding")
    c = Case(prior=[40, 90], new=[1, 1], seed=13).write_history()
    want = ref.attend(c.q[0], *c.oracles(), decode_seqs(c, c.prior), c.table)
    q = torch.cat([c.q, c.q, c.q[:, :1]], 1).to(DEV)
    slots = torch.tensor([1, 2, 0, -3, 77], device=DEV)
    lens = torch.tensor([40, 90, 0, 5, 5], device=DEV)
    err = err_word()
    o = cie.decode_gqa_attention_q8(q, c.k, c.v, c.scales, lens, slots, c.table.to(DEV), err=err)
    check_attention(o[0, :2], want, 90)
    assert not o[0, 2:].any() and int(err) == PAGE  # no keys: zeros
    # an appending batch with padding rows: the real rows as without them
    c2 = Case(prior=[40, 90], new=[1, 1], seed=13).write_history()
    o2 = decode_append(c2)
    k = torch.cat([c.k_new, c.k_new], 1).to(DEV)
    o = cie.decode_append_gqa_attention_q8(q[:, :4], c.k, c.v, c.scales, k, torch.cat([c.v_new] * 2, 1).to(DEV),
                                           c.lens.to(DEV), torch.tensor([1, 2, 0, 0], device=DEV), c.table.to(DEV),
                                           num_programs=int(256 // 4))
    want2 = ref.attend(c2.q[0], *c2.oracles(), decode_seqs(c2, [41, 91]), c2.table)
    check_attention(o[0, :2], want2, 91)
    check_attention(o2[0], want2, 91)
    same_cache(c, c2.oracles(), skip_pages=(0,))
    err.zero_()
    bad = c.table.clone()
    bad[1, 0] = 10 ** 6
    cie.decode_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales, *c.dev("kv_lens", "slots"), bad.to(DEV), err=err)
    assert int(err) == PAGE
    err.zero_()
    cie.decode_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales, torch.tensor([-1, 10 ** 7], device=DEV),
                                c.slots.to(DEV), c.table.to(DEV), err=err)
    assert int(err) & LEN


def test_decode_far_pages(native_lib):
    """Page offsets past 2^32 bytes: append, decode, read and mixed on the last pages of a pool of 4.6 GB."""
    note("q8 far pages")
    n = 280_000
    c = Case(prior=[70], new=[1], d=128, h_q=8, h_kv=8, seed=14)
    k = torch.empty(n, 8, 16, 128, dtype=torch.uint8, device=DEV)
    v = torch.empty_like(k)
    scales = torch.empty(n, 8, 1, 2, device=DEV)
    small = c.k.shape[0]
    table = torch.where(c.table > 0, c.table + n - small, 0)
    c.k, c.v, c.scales = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), scales
    c.table = torch.zeros(2, n, dtype=torch.int64)
    c.table[:, :small] = table
    assert int(table.max()) * 8 * 16 * 128 > 2 ** 32
    c.write_history()
    o = decode_append(c)
    last = slice(n - small, n)
    near = [ref.Q8Cache.of(p[last], scales[last][..., i]) for i, p in enumerate((c.k, c.v))]
    seen = (table - (n - small)).clamp(min=0)
    want = ref.attend(c.q[0], *near, [(0, 1, 1, 71)], seen)
    check_attention(o[0], want, 71)
    pages, offs = c.at(0, 0, 71)
    got, _ = cie.kv_read_tokens_q8(c.k, c.v, c.scales, pages.to(DEV), offs.to(DEV))
    assert torch.equal(got[0].cpu().double(), near[0].values()[pages - (n - small), :, offs])
    m = cie.mixed_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales, 1, *c.dev("cu", "kv_lens", "slots", "table"))
    check_attention(m[0], want, 71)


# ---- mixed ----

def mixed_seqs(c):
    return [(int(c.cu[b]), n, b + 1, p + 1) for b, (p, n) in enumerate(zip(c.prior, c.new)) if n]


MIXED = [
    dict(prior=[0], new=[1]),
    dict(prior=[0], new=[2]),
    dict(prior=[0, 5, 20, 37, 0, 1000], new=[17, 1, 3, 1, 0, 1]),
    dict(prior=[0, 100, 512], new=[256, 37, 129]),
    dict(prior=[0, 3000], new=[300, 40]),
    dict(prior=[9000, 4000, 30], new=[1, 2, 1]),                    # split narrow items
    dict(prior=[6000], new=[64]),                                   # split wide items
    dict(prior=[20000], new=[1], h_q=4, h_kv=1),                    # 64 chunks at most
    dict(prior=[0, 700, 64], new=[65, 33, 1], d=128, h_q=32, h_kv=8, page=32),
    dict(prior=[2500], new=[90], d=128, h_q=16, h_kv=1),
    dict(prior=[10, 0], new=[50, 140], page=48, h_q=8, h_kv=8),     # one head a group: 128-row tiles
    dict(prior=[i * 7 % 90 for i in range(90)], new=[i % 4 for i in range(90)]),
]


@pytest.mark.parametrize("shape", MIXED, ids=lambda s: f"{str(s['prior'])[:24]}+{str(s['new'])[:20]}d{s.get('d', 64)}")
def test_mixed(native_lib, shape):
    note(f"q8 mixed {shape}")
    c = Case(**shape, seed=15).write_history()
    append_tokens(c)
    want = ref.attend(c.q[0], *c.oracles(), mixed_seqs(c), c.table)
    n = max(p + m for p, m in zip(c.prior, c.new))
    args = (c.q.to(DEV), c.k, c.v, c.scales, max(c.new), *c.dev("cu", "kv_lens", "slots", "table"))
    err = err_word()
    o = cie.mixed_gqa_attention_q8(*args, err=err)
    check_attention(o[0], want, n)
    plan = cie.mixed_plan_q8(c.k, *c.dev("cu", "kv_lens", "slots", "table"), max(c.new), c.T, c.h_q, err=err)
    assert torch.equal(cie.mixed_gqa_attention_q8(*args, plan=plan, err=err), o)
    assert int(err) == 0
    counters = cie.attn.core.split_counters(torch.device(DEV), 1)
    assert not counters.any()


def test_mixed_leaves_other_rows_and_caps_rows(native_lib):
    """Rows before and after the sequences are not written; rows at or past max_seqlen neither."""
    note("q8 mixed other rows")
    c = Case(prior=[20, 0, 5], new=[9, 40, 1], seed=16).write_history()
    append_tokens(c)
    want = ref.attend(c.q[0], *c.oracles(), mixed_seqs(c), c.table)
    T = c.T + 20
    at = torch.arange(3, 3 + c.T)
    q = torch.zeros(1, T, 14, 64, dtype=torch.float16)
    q[0, at] = c.q[0]
    cu = torch.tensor([3, 12, 52, 53, 53, 53])  # and two sequences without rows
    slots, kv = torch.tensor([1, 2, 3, 0, 0]), torch.tensor([20, 0, 5, 0, 0])
    lib = _native.load()
    o = torch.full((1, T, 14, 64), 7.0, dtype=torch.float16, device=DEV)
    err = err_word()

    def call(max_seqlen, cu):
        qd, sl, kvd, cud, tb = (x.to(DEV) for x in (q, slots, kv, cu, c.table))
        plan = cie.mixed_plan_q8(c.k, cud, kvd, sl, tb, max_seqlen, T, 14, err=err)
        n = lib.cie_q8_mixed_partials_bytes(T, 14, 64)
        parts = torch.empty(n, dtype=torch.uint8, device=DEV)
        ctr = torch.zeros(lib.cie_q8_mixed_counters(), dtype=torch.int32, device=DEV)
        rc = lib.cie_q8_mixed(o.data_ptr(), qd.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), c.scales.data_ptr(),
                              plan.data_ptr(), plan.numel() * 4, tb.data_ptr(), parts.data_ptr(), n, ctr.data_ptr(),
                              5, T, 14, 2, 64, 16, c.k.shape[0], c.k.stride(0), c.k.stride(1), tb.stride(0),
                              tb.shape[1], tb.shape[0], err.data_ptr(), _native.stream_handle(torch.device(DEV)))
        assert rc == 0
        torch.cuda.synchronize()

    call(40, cu)
    check_attention(o[0, at], want, 40)
    rest = torch.ones(T, dtype=torch.bool)
    rest[at] = False
    assert (o[0, rest] == 7.0).all() and int(err) == 0
    o.fill_(7.0)
    call(8, cu)
    assert int(err) == LEN
    kept = torch.cat([torch.arange(3, 11), torch.arange(12, 20), torch.tensor([52])])
    check_attention(o[0, kept], tuple(x[kept - 3] for x in want), 40)
    gone = torch.ones(T, dtype=torch.bool)
    gone[kept] = False
    assert (o[0, gone] == 7.0).all()


def test_mixed_bad_sequences_and_plans(native_lib):
    note("q8 mixed errors")
    c = Case(prior=[20, 30], new=[9, 4], seed=17).write_history()
    append_tokens(c)
    want = ref.attend(c.q[0], *c.oracles(), mixed_seqs(c), c.table)
    err = err_word()
    q, tb, cu = c.q.to(DEV), c.table.to(DEV), c.cu.to(DEV)
    o = cie.mixed_gqa_attention_q8(q, c.k, c.v, c.scales, 9, cu, c.kv_lens.to(DEV), torch.tensor([55, 2], device=DEV),
                                   tb, err=err)
    assert int(err) == PAGE
    check_attention(o[0, 9:], tuple(x[9:] for x in want), 40)
    err.zero_()
    o = cie.mixed_gqa_attention_q8(q, c.k, c.v, c.scales, 9, cu, torch.tensor([20, 10 ** 9], device=DEV),
                                   c.slots.to(DEV), tb, err=err)
    assert int(err) == LEN
    check_attention(o[0, :9], tuple(x[:9] for x in want), 40)
    err.zero_()
    plan = cie.mixed_plan_q8(c.k, cu, *c.dev("kv_lens", "slots", "table"), 9, c.T + 1, 14, err=err)
    cie.mixed_gqa_attention_q8(q, c.k, c.v, c.scales, 9, cu, *c.dev("kv_lens", "slots", "table"), plan=plan, err=err)
    assert int(err) == PLAN
    # overlapping sequences: more items than the plan holds
    err.zero_()
    many = torch.tensor([0, c.T] * 200 + [0], device=DEV)
    B = many.shape[0] - 1
    cie.mixed_gqa_attention_q8(q, c.k, c.v, c.scales, c.T, many, torch.zeros(B, dtype=torch.int64, device=DEV),
                               torch.ones(B, dtype=torch.int64, device=DEV), tb, err=err)
    assert int(err) & PAGE  # (the ranges that run backwards)


# ---- streams, graphs ----

def test_two_streams_and_graph_replays(native_lib):
    """A step (append from the projection, mixed attention, then planned decodes) captured and replayed, with eager
    calls of the same operators between the replays and on another stream with its own counters."""
    note("q8 graph")
    c = Case(prior=[33, 700, 5], new=[1, 1, 1], seed=18).write_history()
    c2 = Case(prior=[33, 700, 5], new=[1, 1, 1], seed=18).write_history()
    cos, sin = (x.to(DEV) for x in rope_tables(c.kv_lens, 64))
    qkv = fused_rows(c).to(DEV)
    lens, slots, table, cu, kvl = c.dev("lens", "slots", "table", "cu", "kv_lens")

    def step(x):
        def fn():
            q = cie.append_tokens_qkv_rope_q8(qkv, cos, sin, x.k, x.v, x.scales, *pages, 14)
            a = cie.mixed_gqa_attention_q8(q, x.k, x.v, x.scales, 1, cu, kvl, slots, table)
            plan = cie.decode_plan(x.k, lens, slots, table)
            b = cie.decode_qkv_rope_gqa_attention_q8(qkv, cos, sin, x.k, x.v, x.scales, lens, slots, table, 14, plan=plan)
            k, v = cie.kv_read_tokens_q8(x.k, x.v, x.scales, *pages)
            return a, b, k, v
        return fn

    pages = [x.to(DEV) for x in c.new_at()]
    eager = [x.clone() for x in step(c2)()]
    g1, g2 = StepGraph(step(c)), StepGraph(step(c))  # two graphs on the same counters
    for i in range(4):
        outs = [x.clone() for x in (g1 if i % 2 else g2).replay()]
        again = step(c2)()
        torch.cuda.synchronize()
        for a, b, e in zip(outs, again, eager):
            assert torch.equal(a, e) and torch.equal(b, e)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    n = _native.load().cie_q8_mixed_counters()
    own = torch.zeros(max(n, 64), dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        o = cie.mixed_gqa_attention_q8(c2.q.to(DEV), c2.k, c2.v, c2.scales, 1, cu, kvl, slots, table, counters=own)
        d = cie.decode_gqa_attention_q8(c2.q.to(DEV), c2.k, c2.v, c2.scales, kvl + 1, slots, table, counters=own)
    main = cie.mixed_gqa_attention_q8(c2.q.to(DEV), c2.k, c2.v, c2.scales, 1, cu, kvl, slots, table)
    torch.cuda.synchronize()
    assert torch.equal(o, main) and not own.any()
    want = ref.attend(c2.q[0], *c2.oracles(), decode_seqs(c2, [34, 701, 6]), c2.table)
    check_attention(d[0], want, 701)
    check_attention(o[0], want, 701)


def test_unaligned_queries_are_refused(native_lib):
    note("q8 refusals on the device")
    c = Case(prior=[20], new=[1]).write_history()
    q = torch.zeros(14 * 64 + 1, dtype=torch.float16, device=DEV)[1:].view(1, 1, 14, 64)
    with pytest.raises(RuntimeError, match="invalid argument"):
        cie.decode_gqa_attention_q8(q, c.k, c.v, c.scales, *c.dev("kv_lens", "slots", "table"))
    with pytest.raises(AssertionError, match="counters"):
        cie.mixed_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales, 1, *c.dev("cu", "kv_lens", "slots", "table"),
                                   counters=torch.zeros(4, dtype=torch.int32, device=DEV))
    with pytest.raises(AssertionError, match="num_programs"):
        cie.decode_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales, *c.dev("kv_lens", "slots", "table"),
                                    num_programs=65)


# ---- larger calls, extremes, plans of other calls ----

@pytest.mark.parametrize("shape", [
    dict(prior=[0] * 3, new=[1500] * 3, h_q=16, h_kv=4),
    dict(prior=[9000], new=[900]),
    dict(prior=[6000], new=[700], h_q=16, h_kv=8, d=128),
], ids=["prefill", "split64", "split128"])
def test_mixed_whole_tiles(native_lib, shape):
    """Launches large enough for tiles of 128 columns, unsplit and split over the keys."""
    note(f"q8 mixed whole tiles {shape}")
    test_mixed(native_lib, shape)


def test_long_token_append_is_that_in_pieces(native_lib):
    """17,700 tokens in one call (16 a workgroup) and in calls of 1,037 leave the same cache."""
    note("q8 long append")
    one, many = (Case(prior=[3, 0], new=[17000, 700], h_kv=1, h_q=1, seed=20).write_history() for _ in range(2))
    append_tokens(one)
    pages, offs = many.new_at()
    for lo in range(0, many.T, 1037):
        s = slice(lo, lo + 1037)
        cie.kv_append_tokens_q8(many.k, many.v, many.scales, many.k_new[:, s].to(DEV), many.v_new[:, s].to(DEV),
                                pages[s].to(DEV), offs[s].to(DEV))
    for a, b in ((one.k, many.k), (one.v, many.v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(one.scales.view(torch.int32), many.scales.view(torch.int32))


@pytest.mark.parametrize("shape", [dict(h_q=14, h_kv=2), dict(h_q=8, h_kv=2, d=128)], ids=["d64", "d128"])
def test_decode_append_of_extremes(native_lib, shape):
    """A block's rows one decode at a time, from tiny to the largest fp16, infinities and a NaN: the cache of the
    definition, and results that are NaN only in the heads that hold one."""
    note(f"q8 decode extremes {shape}")
    c = Case(prior=[14], new=[1], seed=21, **shape).write_history()
    want = c.oracles()
    c.table[1, 1] = 1 + c.table[1, 0] % 4  # (another of the four pages)
    steps = [2.0 ** -24, -0.0, 2.0 ** -15, 0.3, 447.0, 65504.0, float("-inf"), float("inf"), -61441.0, float("nan")]
    d = c.d
    for i, x in enumerate(steps):
        pos = 14 + i
        k = torch.randn(1, 1, c.h_kv, d, generator=torch.Generator().manual_seed(i)).half() * 0.01
        v = -k.flip(3)
        k[0, 0, 0, i * d // len(steps)] = x
        v[0, 0, 0, d - 1 - i] = -x
        c.lens[1] = pos
        o = cie.decode_append_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales, k.to(DEV), v.to(DEV),
                                               *c.dev("lens", "slots", "table"), num_programs=1 + i % 3)
        page, off = int(c.table[1, pos // 16]), pos % 16
        for w, y in zip(want, (k, v)):
            w.append(y[0], [page], [off])
        same_cache(c, want)
        group = c.h_q // c.h_kv
        assert torch.isfinite(o[0, 0, group:]).all()
        assert bool(o[0, 0, :group].isnan().all()) == (x != x) and bool(torch.isfinite(o[0, 0, :group]).all()) == (x == x)
        first = 0 if abs(x) < 1 else group  # (scores of thousands are off by more than the tolerance counts)
        seen = ref.attend(c.q[0], *want, [(0, 1, 1, pos + 1)], c.table)
        check_attention(o[0, :, first:], tuple(y[:, first:] for y in seen), pos + 1, f"{x}")
    # the NaN through the other forms: split decodes, and the last of mixed rows in narrow and wide items
    args = (c.k, c.v, c.scales)
    lens, table = torch.tensor([24], device=DEV), c.table.to(DEV)
    outs = [cie.decode_gqa_attention_q8(c.q.to(DEV), *args, lens, c.slots.to(DEV), table, num_programs=P)
            for P in (1, 2, 5)]
    for n in (1, 2, 20):
        q = c.q.to(DEV).expand(1, n, -1, -1).contiguous()
        outs.append(cie.mixed_gqa_attention_q8(q, *args, n, torch.tensor([0, n], device=DEV), lens - n,
                                               c.slots.to(DEV), table)[:, -1:])
    for o in outs:
        assert o[0, 0, :group].isnan().all()
        check_attention(o[0, :, group:], tuple(y[:, group:] for y in seen), 24)


def test_index_types_and_row_layouts(native_lib):
    """int32 indices, and new rows as (B, H_kv, D), (B, 1, H_kv, D) or every other head of a wider tensor."""
    note("q8 index types")
    c = Case(prior=[20, 47, 5], new=[1, 1, 1], seed=22).write_history()
    base = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.scales)]
    want = decode_append(c)
    after = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.scales)]
    wide = torch.zeros(3, 4, 64, dtype=torch.float16, device=DEV)
    wide[:, ::2] = c.k_new[0].to(DEV)
    v = c.v_new.to(DEV)
    for k, vv in ((c.k_new[0].to(DEV), v[0]), (c.k_new.transpose(0, 1).to(DEV), v.transpose(0, 1)), (wide[:, ::2], v)):
        for t, b in zip((c.k.view(torch.uint8), c.v.view(torch.uint8), c.scales), base):
            t.copy_(b)
        o = cie.decode_append_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales, k, vv,
                                               *(x.int() for x in c.dev("lens", "slots", "table")))
        assert torch.equal(o, want)
        for t, a in zip((c.k.view(torch.uint8), c.v.view(torch.uint8), c.scales.view(torch.int32)), after):
            assert torch.equal(t, a.view(t.dtype))


def test_plans_of_other_calls_are_not_followed(native_lib):
    note("q8 other plans")
    c = Case(prior=[20, 700, 5], new=[1, 1, 1], seed=23).write_history()
    before = c.k.view(torch.uint8).clone()
    err = err_word()
    plain = cie.decode_plan(c.k, *c.dev("kv_lens", "slots", "table"), append=False)
    app = cie.decode_plan(c.k, *c.dev("lens", "slots", "table"))
    decode_append(c, plain, err=err)  # the other append mode, either way
    torch.cuda.synchronize()
    assert int(err) == PLAN and torch.equal(c.k.view(torch.uint8), before)
    err.zero_()
    cie.decode_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales, *c.dev("kv_lens", "slots", "table"), plan=app, err=err)
    assert int(err) == PLAN
    err.zero_()  # a plan of three sequences for two: those are right
    o = cie.decode_gqa_attention_q8(c.q[:, :2].contiguous().to(DEV), c.k, c.v, c.scales, c.kv_lens[:2].to(DEV),
                                    c.slots[:2].to(DEV), c.table.to(DEV), plan=plain, err=err)
    assert int(err) == PLAN
    want = ref.attend(c.q[0], *c.oracles(), decode_seqs(c, c.prior), c.table)
    check_attention(o[0], tuple(x[:2] for x in want), 700)
    # cu_seqlens that runs backwards: an empty plan
    err.zero_()
    plan = cie.mixed_plan_q8(c.k, torch.tensor([0, 2, 1, 3], device=DEV), *c.dev("kv_lens", "slots", "table"), 3, 3,
                             14, err=err)
    assert int(plan[0]) == 0 and int(err) == PAGE


def test_operands_elsewhere_are_refused(native_lib):
    """Counters, plans and error words that the device cannot use, before anything is launched."""
    note("q8 operands elsewhere")
    c = Case(prior=[20], new=[1]).write_history()
    decode = (c.q.to(DEV), c.k, c.v, c.scales, *c.dev("kv_lens", "slots", "table"))
    mixed = (c.q.to(DEV), c.k, c.v, c.scales, 1, *c.dev("cu", "kv_lens", "slots", "table"))
    plan = cie.decode_plan(c.k, *c.dev("kv_lens", "slots", "table"), append=False)
    host = torch.zeros(4096, dtype=torch.int32)
    for call in (lambda: cie.decode_gqa_attention_q8(*decode, num_programs=2, counters=host),
                 lambda: cie.decode_gqa_attention_q8(*decode, plan=plan.cpu()),
                 lambda: cie.decode_gqa_attention_q8(*decode, err=host[:1]),
                 lambda: cie.mixed_gqa_attention_q8(*mixed, counters=host),
                 lambda: cie.mixed_gqa_attention_q8(*mixed, plan=plan.cpu()),
                 lambda: cie.kv_read_tokens_q8(*decode[1:4], *[torch.zeros(1, 1, dtype=torch.int64, device=DEV)] * 2)):
        with pytest.raises(AssertionError):
            call()


def test_rope_append_of_many_heads_and_rows(native_lib):
    test_rope_append_is_rotate_then_append(native_lib, dict(prior=[20, 3], new=[1100, 1], h_q=4, h_kv=4, d=128))


def test_mixed_of_many_sequences(native_lib):
    """More sequences, and more query tiles, than the plan's threads; split tiles among the last ones."""
    prior = [i * 13 % 70 for i in range(600)]
    new = [i % 4 for i in range(600)]
    prior[7], prior[590], new[590], prior[595], new[595] = 3000, 5000, 1, 4000, 60
    shape = dict(prior=prior, new=new, h_q=4, h_kv=2)
    test_mixed(native_lib, shape)
    # 2,100 rows in half tiles of 4: 525 beside one decode row over a long prefix
    test_mixed(native_lib, dict(prior=[0] * 7 + [3000], new=[300] * 7 + [1], h_q=16, h_kv=1))
