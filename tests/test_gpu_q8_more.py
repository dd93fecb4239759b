"""The 8-bit cache on the GPU, further cases: plans of other calls, NaN in masked places, merges of every form."""
import pytest
import torch

import custom_inference_engine_amd as cie
from oracle import q8_cache as ref
from tests.gpu_helpers import DEV, err_word, note
from tests.q8_helpers import Case
from tests.test_gpu_q8 import PLAN, append_tokens, check_attention, decode_seqs, mixed_seqs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,h_q,h_kv", [(64, 14, 2), (128, 32, 8)])
@pytest.mark.parametrize("append", [False, True])
def test_decode_plan_of_fewer_sequences(native_lib, append, d, h_q, h_kv):
    """A plan of two sequences, split four ways each, has a workgroup for each of the (sequence, kv head) pairs of a
    call of eight, which then brings no partials: nothing of it is followed.  One with more workgroups than the
    call's pairs is right for its sequences, and the call reports the missing ones."""
    prior = [300, 90, 5, 0, 64, 200, 17, 33]
    c = Case(prior=prior, new=[1] * 8, h_q=h_q, h_kv=h_kv, d=d, seed=30).write_history()
    lens = c.dev("lens" if append else "kv_lens")[0]
    slots, table, k_new, v_new = c.dev("slots", "table", "k_new", "v_new")
    before = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.scales)]
    err = err_word()

    def plan(n, splits):
        return cie.decode_plan(c.k, lens if append else lens[:n], slots[:n], table, append=append, num_programs=splits)

    def call(n, p):
        q = c.q[:, :n].contiguous().to(DEV)
        if append:
            return cie.decode_append_gqa_attention_q8(q, c.k, c.v, c.scales, k_new[:, :n].contiguous(),
                                                      v_new[:, :n].contiguous(), lens, slots[:n], table, plan=p, err=err)
        return cie.decode_gqa_attention_q8(q, c.k, c.v, c.scales, lens[:n], slots[:n], table, plan=p, err=err)

    note(f"q8 plan of two for eight, as many workgroups, append {append} d {d}")
    call(8, plan(2, 4))
    torch.cuda.synchronize()
    assert int(err) == PLAN
    for t, b in zip((c.k.view(torch.uint8), c.v.view(torch.uint8), c.scales.view(torch.int32)), before):
        assert torch.equal(t, b.view(t.dtype))
    err.zero_()
    note(f"q8 plan of two for eight, more workgroups, append {append} d {d}")
    o = call(8, plan(2, 8))
    torch.cuda.synchronize()
    assert int(err) == PLAN
    seen = decode_seqs(c, [p + append for p in prior])
    want = ref.attend(c.q[0], *c.oracles(), seen[:2], c.table)
    check_attention(o[0, :2], tuple(x[:2] for x in want), 301)
    err.zero_()
    for splits in (1, 3):  # its own plan, unsplit and split: followed without a report
        o = call(8, plan(8, splits))
        torch.cuda.synchronize()
        assert int(err) == 0
        check_attention(o[0], ref.attend(c.q[0], *c.oracles(), seen, c.table), 301)
    with pytest.raises(RuntimeError, match="invalid argument"):  # fewer workgroups than pairs
        call(8, plan(2, 1))
    assert not cie.attn.core.split_counters(torch.device(DEV), 1).any()


NANS = [  # (shape, positions of the last sequence that hold a NaN in V, and in K)
    (dict(prior=[0], new=[128], h_q=4, h_kv=4), [100], []),             # one head a group: 128 rows a tile
    (dict(prior=[0], new=[70], h_q=4, h_kv=4, d=128), [0, 3, 69], [68]),
    (dict(prior=[37], new=[100]), [40, 41, 57, 136], [129]),            # 18 rows a tile
    (dict(prior=[0, 30], new=[60, 90], d=128, h_q=32, h_kv=8, page=32), [33, 118, 119], []),
    (dict(prior=[5], new=[14], h_q=2, h_kv=2), [12, 18], [9]),          # narrow items of several rows
    (dict(prior=[21], new=[2]), [22], []),
    (dict(prior=[300], new=[4], d=128, h_q=32, h_kv=8), [301, 303], [302]),
    (dict(prior=[6000], new=[64]), [5, 6031], [6050]),                  # split over the keys
    (dict(prior=[9000], new=[2], h_q=4, h_kv=1), [9001], []),
    (dict(prior=[0] * 3, new=[1500] * 3, h_q=16, h_kv=4), [700, 1499], []),  # whole tiles
    (dict(prior=[6000], new=[700], h_q=16, h_kv=8, d=128), [6350, 6351], []),
]


@pytest.mark.parametrize("shape,in_v,in_k", NANS, ids=lambda x: f"{x['prior']}+{x['new']}d{x.get('d', 64)}" if isinstance(x, dict) else str(x))
def test_mixed_nan_reaches_the_rows_that_attend_it(native_lib, shape, in_v, in_k):
    """A NaN in V is NaN in that dim of its head's rows from its own on, one in K in every dim; earlier rows, which mask
    the key, are as if it were any number."""
    note(f"q8 mixed nan {shape} {in_v} {in_k}")
    c = Case(**shape, seed=31).write_history()
    last, g = c.B - 1, torch.Generator().manual_seed(32)
    t0, prior = int(c.cu[last]), c.prior[last]
    held = {p: (int(torch.randint(c.h_kv, (1,), generator=g)), int(torch.randint(c.d, (1,), generator=g)))
            for p in in_v + in_k}
    nan = torch.tensor([float("nan"), -float("nan")]).half()
    nan[1] = torch.tensor([-512], dtype=torch.int16).view(torch.float16)[0]  # 0xfe00: negative
    for x, where in ((c.v_new, in_v), (c.k_new, in_k)):
        for i, p in enumerate(where):
            h, dim = held[p]
            if p >= prior:
                x[0, t0 + p - prior, h, dim] = nan[i % 2]
            else:  # (in the rows held before)
                pages, offs = c.at(last, p, 1)
                (c.v if x is c.v_new else c.k).view(torch.uint8)[int(pages), h, int(offs), dim] = 0x7f + 0x80 * (i % 2)
    append_tokens(c)
    want = torch.zeros(c.T, c.h_q, c.d, dtype=torch.bool)  # NaN
    group = c.h_q // c.h_kv
    for where, whole in ((in_v, False), (in_k, True)):
        for p in where:
            h, dim = held[p]
            rows = slice(max(t0, t0 + p - prior), c.T)
            want[rows, h * group:(h + 1) * group, slice(None) if whole else dim] = True
    kc, vc = c.oracles()
    for x in (kc, vc):
        x.vals.nan_to_num_(0.0)
    seen = ref.attend(c.q[0], kc, vc, mixed_seqs(c), c.table)
    args = (c.q.to(DEV), c.k, c.v, c.scales, max(c.new), *c.dev("cu", "kv_lens", "slots", "table"))
    for _ in range(2):
        o = cie.mixed_gqa_attention_q8(*args)[0].cpu()
        assert torch.equal(o.isnan(), want)
        check_attention(o.masked_fill(want, 0.0), tuple(x.masked_fill(want, 0.0) if x.shape == want.shape else x for x in seen),
                        max(p + n for p, n in zip(c.prior, c.new)))


def plan_items(c, plan):
    """A mixed plan's items: (row, rows, g, slot, pos, first and last key tile, chunk, chunks) each."""
    words = plan.cpu()
    return [tuple(words[12 + 12 * i:21 + 12 * i].tolist()) for i in range(int(words[0]))]


MERGES = [  # (shape, columns times D / 4 of the split tile, its chunks): every form of the merge, and the cap on chunks
    (dict(prior=[9000], new=[3]), (257, 512), (9, 48)),                                # two pieces a thread, D = 64
    (dict(prior=[9000], new=[2], d=128, h_q=8, h_kv=1), (257, 512), (9, 48)),          # the same at D = 128
    (dict(prior=[9000], new=[2], d=128, h_q=14, h_kv=2), (257, 512), (9, 48)),
    (dict(prior=[3000], new=[3], d=128, h_q=8, h_kv=1), (257, 1024), (2, 8)),          # four, chunks a few
    (dict(prior=[3000], new=[5], d=64), (257, 1024), (2, 8)),
    (dict(prior=[2300], new=[1], d=128, h_q=32, h_kv=8), (1, 256), (2, 16)),           # one
    (dict(prior=[12000], new=[1], d=128, h_q=16, h_kv=2), (1, 256), (17, 48)),
    (dict(prior=[9000], new=[40], d=128, h_q=4, h_kv=1), (513, 2048), (9, 48)),        # eight
    (dict(prior=[65500], new=[1], h_q=4, h_kv=1), (1, 256), (48, 48)),                 # the cap, a narrow item's
    (dict(prior=[40000], new=[20], h_q=4, h_kv=1), (513, 2048), (48, 48)),             # and a wide one's
    (dict(prior=[30001], new=[11], h_q=7, h_kv=1, d=128), (513, 2048), (48, 48)),      # (9 rows a half tile: 63 x 32)
    (dict(prior=[20000], new=[360], h_q=7, h_kv=1, d=128), (2049, 4096), (9, 48)),     # sixteen: 18 rows a whole one
    (dict(prior=[20000], new=[360], h_q=7, h_kv=1), (1025, 2048), (9, 48)),
]


@pytest.mark.parametrize("shape,units,chunks", MERGES, ids=lambda x: f"{x['prior']}+{x['new']}d{x.get('d', 64)}" if isinstance(x, dict) else str(x))
def test_mixed_merge_forms(native_lib, shape, units, chunks):
    note(f"q8 mixed merge {shape}")
    c = Case(**shape, seed=33).write_history()
    append_tokens(c)
    want = ref.attend(c.q[0], *c.oracles(), mixed_seqs(c), c.table)
    args = (c.q.to(DEV), c.k, c.v, c.scales, max(c.new), *c.dev("cu", "kv_lens", "slots", "table"))
    err = err_word()
    plan = cie.mixed_plan_q8(c.k, *c.dev("cu", "kv_lens", "slots", "table"), max(c.new), c.T, c.h_q, err=err)
    items = plan_items(c, plan)
    kt = -(-(c.prior[0] + c.new[0]) // 16)
    split = [i for i in items if i[8] > 1]
    assert split and max(abs(i[1]) for i in split) * (c.h_q // c.h_kv) * c.d // 4 in range(units[0], units[1] + 1)
    assert chunks[0] <= max(i[8] for i in items) <= chunks[1]
    for g in range(c.h_kv):  # the chunks of every tile cover its keys once
        for row in {i[0] for i in items}:
            tile = sorted(i for i in items if i[2] == g and i[0] == row)
            at = 0
            for i in sorted(tile, key=lambda i: i[7]):
                assert i[5] == at and i[6] >= at
                at = i[6]
            assert at == -(-(tile[0][4] + abs(tile[0][1])) // 16) <= kt and len(tile) == tile[0][8]
    o = cie.mixed_gqa_attention_q8(*args, plan=plan, err=err)
    check_attention(o[0], want, c.prior[0] + c.new[0])
    assert int(err) == 0 and torch.equal(cie.mixed_gqa_attention_q8(*args, plan=plan), o)
    assert not cie.attn.core.split_counters(torch.device(DEV), 1).any()


def test_mixed_ranges_that_run_backwards_leave_the_plan_empty(native_lib):
    """cu_seqlens that falls anywhere: no item, the page bit alone, and no row of the outputs computed."""
    note("q8 mixed backwards")
    c = Case(prior=[20, 30], new=[9, 4], seed=17).write_history()
    append_tokens(c)
    many = torch.tensor([0, c.T] * 200 + [0], device=DEV)
    B = many.shape[0] - 1
    lens, slots = torch.zeros(B, dtype=torch.int64, device=DEV), torch.ones(B, dtype=torch.int64, device=DEV)
    err = err_word()
    plan = cie.mixed_plan_q8(c.k, many, lens, slots, c.table.to(DEV), c.T, c.T, c.h_q, err=err)
    assert int(err) == 1 and int(plan[0]) == 0
    cie.mixed_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales, c.T, many, lens, slots, c.table.to(DEV), plan=plan, err=err)
    torch.cuda.synchronize()
    assert int(err) == 1


@pytest.mark.parametrize("shape", [dict(prior=[0], new=[8192], h_q=8, h_kv=8), dict(prior=[700], new=[6000], h_q=32, h_kv=8, d=128)],
                         ids=["d64", "d128"])
def test_mixed_items_of_many_stages(native_lib, shape):
    """Unsplit wide items of more than 64 stages: a wave gathers its page ids and scales more than once."""
    note(f"q8 mixed many stages {shape}")
    c = Case(**shape, seed=34).write_history()
    append_tokens(c)
    index = c.dev("cu", "kv_lens", "slots", "table")
    plan = cie.mixed_plan_q8(c.k, *index, c.T, c.T, c.h_q)
    assert max(i[6] - i[5] for i in plan_items(c, plan) if i[8] == 1) > 4 * 64
    o = cie.mixed_gqa_attention_q8(c.q.to(DEV), c.k, c.v, c.scales, c.T, *index, plan=plan)[0]
    oracles = c.oracles()
    for first in (0, c.T // 2 - 7, c.T - 40):  # (some rows: the rest differ by their keys only)
        want = ref.attend(c.q[0], *oracles, [(first, 40, 1, c.prior[0] + first + 1)], c.table)
        rows = slice(first, first + 40)
        check_attention(o[rows], tuple(x[rows] for x in want), c.prior[0] + c.T)
    assert torch.isfinite(o).all()
