"""The 8-bit cache on the GPU, further cases: plans of other calls, NaN in masked places, merges of every form."""
import pytest
import torch

import custom_inference_engine_amd as cie
from oracle import q8_cache as ref
from tests.gpu_helpers import DEV, err_word, note
from tests.q8_helpers import Case
from tests.test_gpu_q8 import PLAN, check_attention, decode_seqs

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
