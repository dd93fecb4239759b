"""Slot maps, rotary positions and adapters without a GPU: refusals, sizes, frequencies, and the schedulers' bookkeeping."""
import math
import os
import re

import pytest
import torch
from transformers import Qwen2Config
from transformers.models.qwen2.modeling_qwen2 import Qwen2RotaryEmbedding

import custom_inference_engine_amd as cie
from custom_inference_engine_amd import _build
from custom_inference_engine_amd.scheduler import Scheduler
from oracle import step as ref
from tests import test_asm_order as asm

I64 = torch.int64


def idx(*v):
    return torch.tensor(v, dtype=I64)


# ---- slot maps ----

def maps_args(**over):
    a = dict(slot_ids=idx(1, 2), new_tokens=idx(3, 1), lens=torch.zeros(3, dtype=I64),
             block_table=torch.zeros((3, 8), dtype=I64), page_size=16, total_T=4, free_list=None, out=None)
    a.update(over)
    return a


@pytest.mark.parametrize("over", [
    dict(slot_ids=idx(1)), dict(slot_ids=idx(1, 2)[None], new_tokens=idx(3, 1)[None]), dict(lens=torch.zeros((3, 1), dtype=I64)),
    dict(block_table=torch.zeros(3, dtype=I64)), dict(total_T=-1), dict(page_size=0),
    dict(free_list=torch.zeros(10)), dict(free_list=torch.zeros(2, dtype=I64)), dict(free_list=torch.zeros((5, 2), dtype=I64)),
    dict(free_list=cie.new_free_list(8, "cpu"), lens=torch.zeros(3, dtype=torch.int32)),
    dict(free_list=cie.new_free_list(8, "cpu"), block_table=torch.zeros((3, 8), dtype=torch.int32)),
    dict(free_list=cie.new_free_list(8, "cpu"), block_table=torch.zeros((8, 3), dtype=I64).t()),
    dict(out=cie.StepMaps(idx(0, 0, 0), *[torch.zeros(5, dtype=I64)] * 4)),
    dict(out=cie.StepMaps(idx(0, 0), *[torch.zeros(4, dtype=I64)] * 4)),
    dict(out=cie.StepMaps(idx(0, 0, 0), *[torch.zeros(4, dtype=torch.int32)] * 4)),
])
def test_step_maps_refuses(over):
    with pytest.raises(AssertionError):
        cie.step_maps(**maps_args(**over))


@pytest.mark.parametrize("over", [
    dict(slot_ids=idx(1, 2)[None]), dict(lens=torch.zeros(3)), dict(block_table=torch.zeros((3, 8))), dict(page_size=0),
    dict(free_list=torch.zeros(8)), dict(keep=idx(1)), dict(held=idx(1, 2, 3)),
])
def test_release_pages_refuses(over):
    a = dict(free_list=cie.new_free_list(8, "cpu"), slot_ids=idx(1, 2), lens=torch.zeros(3, dtype=I64),
             block_table=torch.zeros((3, 8), dtype=I64), page_size=16)
    a.update(over)
    if "keep" in over or "held" in over:  # (these are looked at on the device)
        with pytest.raises((AssertionError, RuntimeError)):
            cie.release_pages(**a)
        return
    with pytest.raises(AssertionError):
        cie.release_pages(**a)


def test_no_cpu_path():
    freqs = cie.rotary_frequencies(64)[0]
    q = torch.zeros((1, 2, 4, 64), dtype=torch.float16)
    for call in (lambda: cie.step_maps(**maps_args()),
                 lambda: cie.step_maps(**maps_args(free_list=cie.new_free_list(8, "cpu"))),
                 lambda: cie.release_pages(cie.new_free_list(8, "cpu"), idx(1), torch.zeros(3, dtype=I64),
                                           torch.zeros((3, 8), dtype=I64), 16),
                 lambda: cie.rotary_tables(idx(1, 2), freqs), lambda: cie.apply_rotary(q, q, idx(1, 2), freqs),
                 lambda: cie.adapter_plan(idx(1, 2), idx(0, 0, 1), 2)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_free_list():
    words = cie.new_free_list(5, "cpu")
    assert words.tolist() == [4, 0, 4, 3, 2, 1, 0] and words.dtype == I64
    assert cie.new_free_list(1, "cpu").tolist() == [0, 0, 0]
    with pytest.raises(AssertionError):
        cie.new_free_list(0, "cpu")


def test_oracle_takes_and_gives_back():
    """The plain loops' own pin: a hand-worked step of three sequences, undone by its release."""
    table = [[0] * 4 for _ in range(4)]
    table[1][:2], table[2][0] = [7, 3], 5
    lens, free = [0, 20, 16, 0], ref.FreeList([4, 0, 9, 8, 2, 6, 0, 0, 0, 0, 0, 0])
    before = [r[:] for r in table], free.words()
    cu, rows, ok = ref.step_maps([2, 1, 3], [2, 13, 17], lens, table, 16, 34, free)
    assert ok and cu == [0, 2, 15, 32]
    assert table[2][:2] == [5, 6] and table[1][:3] == [7, 3, 2] and table[3][:2] == [8, 9] and free.count == 0
    assert rows[:3] == [(2, 16, 6, 0), (2, 17, 6, 1), (1, 20, 3, 4)] and rows[14] == (1, 32, 2, 0)
    assert rows[31] == (3, 16, 9, 0) and rows[32:] == [(0, 0, 0, 0)] * 2
    assert ref.release_pages(free, [2, 1, 3], lens, table, 16, [16, 20, 0], [18, 33, 17])
    assert (table, free.words()) == before and lens == [0, 20, 16, 0]


def _call_maps(lib, **over):
    a = dict(cu=16, slots=32, pos=48, pages=64, offs=80, ids=96, new=112, lens=128, bt=144, free=160, B=2, T=4, page=16,
             n_pages=8, stride=8, width=8, n_slots=3)
    a.update(over)
    return lib.cie_step_maps(*list(a.values()), None, None)


@pytest.mark.parametrize("over,code", [
    (dict(B=-1), -1), (dict(T=-1), -1), (dict(page=0), -1), (dict(width=0), -1), (dict(stride=7), -1), (dict(n_slots=0), -1),
    (dict(n_pages=0), -1), (dict(cu=0), -1), (dict(slots=0), -1), (dict(offs=0), -1), (dict(ids=0), -1), (dict(lens=0), -1),
    (dict(B=2049), -2), (dict(T=(1 << 24) + 1), -2), (dict(n_pages=(1 << 24) + 1), -2), (dict(width=1 << 25, stride=1 << 25), -2),
    (dict(page=1 << 31), -2),
])
def test_step_maps_entry_rejects(native_lib, over, code):
    assert _call_maps(native_lib, **over) == code


@pytest.mark.parametrize("over,code", [
    (dict(B=-1), -1), (dict(page=0), -1), (dict(n_pages=0), -1), (dict(stride=7), -1), (dict(free=0), -1), (dict(ids=0), -1),
    (dict(B=2049), -2), (dict(n_pages=1 << 25), -2), (dict(B=0, free=0), 0),
])
def test_release_pages_entry_rejects(native_lib, over, code):
    a = dict(free=16, ids=32, lens=48, bt=64, keep=0, held=0, B=2, page=16, n_pages=8, stride=8, width=8, n_slots=3)
    a.update(over)
    assert native_lib.cie_release_pages(*list(a.values()), None, None) == code


# ---- rotary ----

@pytest.mark.parametrize("scaling", [
    None,
    {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
    {"type": "yarn", "factor": 10.0, "original_max_position_embeddings": 4096, "beta_fast": 16, "beta_slow": 2,
     "attention_factor": 0.9},
], ids=["default", "linear", "yarn", "yarn_10"])
@pytest.mark.parametrize("d,base", [(64, 1e6), (128, 1e4)])
def test_frequencies_are_the_models_own(scaling, d, base):
    """Against the rotary embedding of the models this framework runs, whose frequencies are fp32 (three roundings)."""
    cfg = Qwen2Config(hidden_size=14 * d, num_attention_heads=14, num_key_value_heads=2, rope_theta=base,
                      max_position_embeddings=32768,
                      rope_scaling=dict(scaling, rope_type=scaling.get("rope_type", scaling.get("type"))) if scaling else None)
    emb = Qwen2RotaryEmbedding(cfg)
    freqs, scale = cie.rotary_frequencies(d, base, scaling)
    assert freqs.dtype == torch.float64 and freqs.shape == (d // 2,)
    want = emb.inv_freq.double()
    # (base ** x in fp32: the exponent's rounding counts ln(base) < 14 times)
    assert ((freqs - want).abs() <= want * (14 + 6) * 2.0 ** -23).all()
    assert abs(scale - emb.attention_scaling) <= 1e-6


def test_other_frequencies():
    plain = cie.rotary_frequencies(16, 100.0)[0]
    assert torch.allclose(plain, 100.0 ** (-torch.arange(0, 16, 2).double() / 16), rtol=1e-14)
    ntk = cie.rotary_frequencies(16, 100.0, {"rope_type": "ntk", "factor": 8.0})[0]
    assert ntk[0] == 1 and math.isclose(ntk[-1], plain[-1] / 8, rel_tol=1e-12)  # the slowest pair is stretched by the factor
    own, scale = cie.rotary_frequencies(4, 100.0, {"rope_type": "factors", "factors": [1, 5.0], "attention_factor": 1.2})
    assert torch.allclose(own, torch.tensor([1.0, 0.02], dtype=torch.float64)) and scale == 1.2


@pytest.mark.parametrize("args", [
    (7,), (0,), (8, 0.0), (8, 1e4, {"rope_type": "linear"}), (8, 1e4, {"rope_type": "yarn", "factor": 2.0}),
    (8, 1e4, {"rope_type": "other"}), (8, 1e4, {"rope_type": "factors", "factors": [1, 2]}), (2, 1e4, {"type": "ntk", "factor": 2.0}),
])
def test_frequencies_refuse(args):
    with pytest.raises(AssertionError):
        cie.rotary_frequencies(*args)


def test_rotary_refuses():
    f16 = torch.float16
    q, k = torch.zeros((1, 5, 4, 64), dtype=f16), torch.zeros((1, 5, 2, 64), dtype=f16)
    pos, freqs = torch.arange(5), cie.rotary_frequencies(64)[0]
    for bad in ((q[0, 0], k, pos, freqs), (q, k[:, :4], pos, freqs), (q, k.float(), pos, freqs), (q, k[..., :32], pos, freqs),
                (q.int(), k.int(), pos, freqs), (q, k, pos, freqs.float()), (q, k, pos, cie.rotary_frequencies(66)[0]),
                (q, k, pos, freqs[:0]), (q, k, pos, freqs[None]), (q, k, pos, freqs[::2]), (q[..., :63], k[..., :63], pos, freqs)):
        with pytest.raises(AssertionError):
            cie.apply_rotary(*bad)
    with pytest.raises((AssertionError, RuntimeError)):
        cie.apply_rotary(q, k, pos[:4], freqs)
    for dtype in (torch.int32, torch.float64):
        with pytest.raises(AssertionError):
            cie.rotary_tables(pos, freqs, dtype)
    pool = torch.zeros((3, 2, 16, 64), dtype=f16)
    qkv = torch.zeros((1, 5, 8 * 64), dtype=f16)
    at = torch.zeros(5, dtype=I64)
    for bad in ((qkv, pos, freqs, pool, pool[:2], at, at, 4), (qkv, pos, freqs, pool.float(), pool.float(), at, at, 4),
                (qkv.bfloat16(), pos, freqs, pool, pool, at, at, 4), (qkv, pos, freqs, pool, pool, at[:3], at, 4),
                (qkv, pos, freqs, pool, pool, at, at, 5), (qkv[0], pos, freqs, pool, pool, at, at, 4),
                (qkv, pos, freqs, pool.transpose(2, 3), pool.transpose(2, 3), at, at, 4),
                (qkv, pos, cie.rotary_frequencies(80)[0], pool, pool, at, at, 4)):
        with pytest.raises(AssertionError):
            cie.append_tokens_qkv_rotary(*bad)


@pytest.mark.parametrize("over,code", [
    (dict(T=-1), -1), (dict(rot=7), -1), (dict(rot=66), -1), (dict(rot=0), -1), (dict(D=63), -1), (dict(H_q=0, H_kv=0), -1),
    (dict(pos=0), -1), (dict(freqs=0), -1), (dict(q=0), -1), (dict(k_out=0), -1), (dict(dtype=3), -2), (dict(H_q=65536), -2),
    (dict(T=0, q=0), 0),
])
def test_rotary_entry_rejects(native_lib, over, code):
    a = dict(q_out=16, k_out=32, q=48, k=64, qt=256, qh=64, kt=128, kh=64, pos=80, freqs=96, scale=1.0, T=5, H_q=4, H_kv=2, D=64,
             rot=64, interleaved=0, dtype=0)
    a.update(over)
    assert native_lib.cie_rotary(*list(a.values()), None) == code


@pytest.mark.parametrize("over,code", [
    (dict(T=-1), -1), (dict(stride=511), -1), (dict(page=0), -1), (dict(n_pages=0), -1), (dict(H_kv=0), -1), (dict(rot=65), -1),
    (dict(pages=0), -1), (dict(v=0), -1), (dict(dtype=2), -2),
])
def test_rotary_append_entry_rejects(native_lib, over, code):
    a = dict(q=16, k=32, v=48, qkv=64, stride=512, pos=80, freqs=96, scale=1.0, pages=112, offs=128, T=5, H_q=4, H_kv=2, page=16,
             D=64, n_pages=3, ps=2048, hs=1024, rot=64, interleaved=0, dtype=0)
    a.update(over)
    assert native_lib.cie_kv_append_tokens_qkv_rotary(*list(a.values()), None, None) == code


# ---- adapters ----

def test_adapters_refuse():
    f16 = torch.float16
    y, x = torch.zeros((5, 96), dtype=f16), torch.zeros((5, 64), dtype=f16)
    a, b = torch.zeros((3, 2, 16, 64), dtype=f16), torch.zeros((3, 96, 16), dtype=f16)
    scales, ranks = torch.ones(3), torch.full((3,), 16, dtype=torch.int32)
    plan = torch.zeros(8 + 3 * 20, dtype=torch.int32)
    good = dict(y=y, x=x, a=a, b=b, scales=scales, ranks=ranks, plan=plan, slices=(64, 32))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cie.adapter_add_(**good)
    for over in (dict(y=y[:4]), dict(y=y[:, :95]), dict(y=y.float()), dict(x=x.bfloat16()), dict(x=x[:, :63]), dict(a=a[:, :1]),
                 dict(a=a[..., :8, :]), dict(a=a[0]), dict(b=b[:2]), dict(b=b.transpose(1, 2)), dict(scales=scales.half()),
                 dict(scales=scales[:2]), dict(ranks=ranks.long()), dict(plan=plan[:20]), dict(plan=plan.long()),
                 dict(slices=(96,)), dict(slices=(64, 31)), dict(y=y[:1].expand(5, 96)), dict(y=y.t()),
                 dict(a=torch.zeros((3, 2, 144, 64), dtype=f16), b=torch.zeros((3, 96, 144), dtype=f16)),
                 dict(y=y.float(), x=x.float(), a=a.float(), b=b.float()), dict(y=y[None, None]), dict(x=x[None].expand(2, 5, 64)),
                 dict(x=y[:, :64])):
        with pytest.raises(AssertionError):
            cie.adapter_add_(**{**good, **over})
    with pytest.raises(AssertionError):
        cie.adapter_plan(idx(1, 2)[None], idx(0, 1), 2)
    with pytest.raises(AssertionError):
        cie.adapter_plan(idx(1, 2), idx(0, 1)[None], 2)


def test_plan_sizes(native_lib):
    words = lambda T, n: native_lib.cie_adapter_plan_bytes(T, n) // 4  # noqa: E731
    assert words(1, 1) == 8 + 20 and words(5, 3) == 8 + 3 * 20
    # every dealing of T rows to at most n adapters fits: the worst is one row for all adapters but one
    for T, n in ((1, 5), (40, 40), (100, 7), (1536, 1000), (1537, 1000), (5000, 3)):
        m = 16 if T <= 1536 else 32
        g = min(T, n)
        worst = (g - 1) + -(-(T - g + 1) // m)
        assert words(T, n) >= 8 + worst * (4 + m)
    for T, n in ((-1, 3), (5, 0), (5, 1025), ((1 << 24) + 1, 3)):
        assert native_lib.cie_adapter_plan_bytes(T, n) == -1


@pytest.mark.parametrize("over,code", [
    (dict(T=-1), -1), (dict(R=0), -1), (dict(R=24), -2), (dict(R=144), -2), (dict(N=0), -1), (dict(N=1025), -2), (dict(d_in=0), -1),
    (dict(n_slices=0), -1), (dict(n_slices=5), -2), (dict(dtype=2), -2), (dict(y=0), -1), (dict(plan=0), -1), (dict(plan=72), -1),
    (dict(b=24), -1), (dict(plan_bytes=200), -1), (dict(ys=95), -1), (dict(xs=63), -1), (dict(widths=(64, 0)), -1), (dict(T=0, y=0), 0),
])
def test_adapter_entry_rejects(native_lib, over, code):
    import ctypes

    a = dict(y=16, ys=96, x=32, xs=64, a=48, b=64, scales=80, ranks=96, plan=112, plan_bytes=4 * (8 + 3 * 20), T=5, N=3, R=16, d_in=64,
             widths=(64, 32), n_slices=2, dtype=0)
    a.update(over)
    a["widths"] = (ctypes.c_int64 * 5)(*a["widths"])
    assert native_lib.cie_adapter_add(*list(a.values()), None, None) == code


def test_adapter_plan_entry_rejects(native_lib):
    plan = native_lib.cie_adapter_plan
    n = 4 * (8 + 3 * 20)
    assert plan(16, n, 32, 48, -1, 4, 3, None, None) == -1
    assert plan(16, n, 32, 48, 5, 0, 3, None, None) == -1
    assert plan(16, n - 4, 32, 48, 5, 4, 3, None, None) == -1
    assert plan(16, n, 0, 48, 5, 4, 3, None, None) == -1  # an entry for each row
    assert plan(0, n, 32, 48, 5, 4, 3, None, None) == -1
    assert plan(16, 1 << 30, 32, 48, 5, 4, 1025, None, None) == -2


def test_bank_on_the_host():
    bank = cie.AdapterBank(2, 20, 24, (16, 8), dtype=torch.float16)
    g = torch.Generator().manual_seed(0)
    a, b = torch.randn(3, 24, generator=g), torch.randn(8, 3, generator=g)
    bank.load(1, (None, a), (None, b), scale=2.0)
    assert bank.ranks.tolist() == [0, 3] and bank.scales.tolist() == [0.0, 2.0]
    assert torch.equal(bank.a[1, 1, :3], a.half()) and not bank.a[1, 0].any() and not bank.a[1, 1, 3:].any()
    assert torch.equal(bank.b[1, 16:, :3], b.half()) and not bank.b[1, :16].any() and not bank.b[1, :, 3:].any()
    for bad in (lambda: bank.load(2, (None, a), (None, b)), lambda: bank.load(0, a, b), lambda: bank.load(0, (a, a), (None, b)),
                lambda: bank.load(0, (None, a[:, :3]), (None, b)), lambda: bank.load(0, (None, a), (None, b[:, :2])),
                lambda: bank.clear(-1), lambda: bank.load(0, (None, torch.zeros(21, 24)), (None, torch.zeros(8, 21)))):
        with pytest.raises((AssertionError, IndexError)):
            bad()
    assert bank.ranks.tolist() == [0, 3]  # (a refused load leaves the bank as it is)
    for bad in (dict(rank=0), dict(rank=129), dict(n_adapters=0), dict(n_adapters=1025), dict(out_features=(1,) * 5),
                dict(dtype=torch.float32)):
        with pytest.raises(AssertionError):
            cie.AdapterBank(**{**dict(n_adapters=2, rank=8, in_features=8, out_features=8), **bad})


# ---- what uses them ----

def _cfg():
    return Qwen2Config(hidden_size=896, num_attention_heads=14, num_key_value_heads=2, intermediate_size=256,
                       num_hidden_layers=1, vocab_size=128, max_position_embeddings=512)


def test_storage_state():
    kv = cie.KVStorage(_cfg(), max_cache_len=64, page_size=16, n_slots=3, device="cpu", dtype=torch.float16)
    assert kv.free_list is None and kv.slot_adapters is None
    kv.use_adapters(5)
    kv.slot_adapters[1] = 3
    kv.reset([1])
    assert kv.slot_adapters.tolist() == [-1, -1, -1]
    kv.manage_pages()
    assert kv.free_list.tolist() == [3, 0, 3, 2, 1, 0]
    kv.lens[1] = 2
    with pytest.raises(AssertionError):
        kv.manage_pages()


class CountingExecutor:
    """A step executor that keeps a pool's lengths as the step modules would, and its pages as ``step_maps`` would."""

    def __init__(self, kv):
        self.kv, self.adapters = kv, []

    def _step(self, slots, counts):
        kv = self.kv
        self.adapters.append({s: int(kv.slot_adapters[s]) for s in slots})
        lens, table, free = kv.lens.tolist(), kv.block_table.tolist(), ref.FreeList(kv.free_list.tolist())
        assert ref.step_maps(slots, counts, lens, table, kv.page_size, sum(counts), free)[2], "pages run short on the device"
        kv.block_table.copy_(torch.tensor(table))
        kv.free_list.copy_(torch.tensor(free.words()))
        for s, n in zip(slots, counts):
            kv.lens[s] += n
        return [1] * len(slots)

    def decode(self, slot_ids):
        return self._step(slot_ids, [1] * len(slot_ids))

    def mixed(self, chunks, slot_ids):
        return self._step(slot_ids, [len(c) for c in chunks])


def _release(free_list, slots, lens, table, page_size, err=None):
    li, ta, fr = lens.tolist(), table.tolist(), ref.FreeList(free_list.tolist())
    assert ref.release_pages(fr, slots.tolist(), li, ta, page_size)
    lens.copy_(torch.tensor(li))
    table.copy_(torch.tensor(ta))
    free_list.copy_(torch.tensor(fr.words()))


def test_scheduler_with_pages_on_the_device(monkeypatch):
    """Pages are only counted on the host: the device's list never runs short, through admissions, chunked prefills and
    preemptions, each request keeps its adapter, and everything is given back."""
    kv = cie.KVStorage(_cfg(), max_cache_len=192, page_size=16, n_slots=4, device="cpu", dtype=torch.float16)
    kv.manage_pages()
    kv.use_adapters(4)
    before = kv.free_list[0].item()

    monkeypatch.setattr("custom_inference_engine_amd.kv_cache.pages.release_pages", _release)
    executor = CountingExecutor(kv)
    sched = Scheduler(None, kv, eos_token_ids={128}, max_new_tokens=16, token_budget=160, executor=executor)
    lengths, adapters = (60, 70, 50, 9, 64), [2, -1, 0, 3, -1]
    results = sched.generate([[5] * n for n in lengths], adapters)
    assert all(len(r.new_tokens) == 16 for r in results) and sched.stats.preemptions == 2
    assert kv.free_list[0] == before and not kv.lens.any() and not kv.block_table.any()
    assert (kv.slot_adapters == -1).all()
    seen = {i for step in executor.adapters for i in step.values()}
    assert seen == set(adapters)
    with pytest.raises(ValueError):
        sched.generate([[1]], [1, 2])


def test_a_failed_step_leaks_no_pages(monkeypatch):
    """A step that took pages and failed: the loop's end leaves the pool empty and its list whole."""
    monkeypatch.setattr("custom_inference_engine_amd.kv_cache.pages.release_pages", _release)
    kv = cie.KVStorage(_cfg(), max_cache_len=192, page_size=16, n_slots=4, device="cpu", dtype=torch.float16)
    kv.manage_pages()
    kv.use_adapters(1)
    executor = CountingExecutor(kv)

    def fails(chunks, slot_ids):
        lens = kv.lens.clone()
        executor._step(slot_ids, [len(c) for c in chunks])
        kv.lens.copy_(lens)  # (its tokens were never counted)
        raise ZeroDivisionError

    executor.mixed = fails
    sched = Scheduler(None, kv, eos_token_ids={128}, max_new_tokens=16, token_budget=160, executor=executor)
    future = sched.call([1] * 40, adapter=0)
    with pytest.raises(ZeroDivisionError):
        sched.loop()
    assert isinstance(future.exception(), ZeroDivisionError)
    assert torch.equal(kv.free_list, cie.new_free_list(kv.n_pages, "cpu")) and not kv.lens.any() and not kv.block_table.any()
    assert (kv.slot_adapters == -1).all()


def test_a_slot_named_twice_is_reset_once(monkeypatch):
    monkeypatch.setattr("custom_inference_engine_amd.kv_cache.pages.release_pages", _release)
    kv = cie.KVStorage(_cfg(), max_cache_len=192, page_size=16, n_slots=4, device="cpu", dtype=torch.float16)
    kv.manage_pages()
    kv.use_adapters(1)
    CountingExecutor(kv)._step([1, 2], [20, 3])
    kv.reset([2, 1, 2, 0, 0])
    assert sorted(kv.free_list[2:13].tolist()) == list(range(1, 12)) and kv.free_list[0] == 11
    assert not kv.lens.any() and not kv.block_table.any()


def test_pages_that_are_managed_report_errors():
    kv = cie.KVStorage(_cfg(), max_cache_len=192, page_size=16, n_slots=4, device="cpu", dtype=torch.float16)
    kv.manage_pages()
    kv.check_pages()
    for bits, text in ((32, "free pages"), (2, "bad slots"), (33, "free pages")):
        kv.page_err.fill_(bits)
        with pytest.raises(RuntimeError, match=text):
            kv.check_pages()
        kv.check_pages()


def test_scheduler_refuses_adapters_it_has_not():
    kv = cie.KVStorage(_cfg(), max_cache_len=192, page_size=16, n_slots=4, device="cpu", dtype=torch.float16)
    sched = Scheduler(None, kv, eos_token_ids={128}, max_new_tokens=16, token_budget=160, executor=object())
    assert isinstance(sched.call([1, 2], adapter=0).exception(), ValueError)
    kv.use_adapters(2)
    assert isinstance(sched.call([1, 2], adapter=2).exception(), ValueError)
    assert isinstance(sched.call([1, 2], adapter=-2).exception(), ValueError)
    assert not sched.call([1, 2], adapter=1).done()


@pytest.mark.parametrize("src,honoured", [("rotary.hip", True), ("adapters.hip", True), ("step_maps.hip", False)])
def test_which_kernels_honour_nans(src, honoured):
    """A NaN in a row comes out of it: the last flag of the two counts."""
    flags = [f for f in _build.source_flags(src) if f in ("-fhonor-nans", "-fno-honor-nans")]
    assert (flags[-1] == "-fhonor-nans") == honoured


@pytest.mark.skipif(not os.path.exists(asm.HIPCC), reason="hipcc not available")
@pytest.mark.parametrize("src,kernels", [("step_maps.hip", 6), ("rotary.hip", 2), ("adapters.hip", 2)])
def test_assembly_of_the_step_kernels(src, kernels, tmp_path, monkeypatch):
    """Sums round to fp32 before they become 16-bit values, nothing takes the packed fp32 forms, spills registers or
    needs the caches written back."""
    monkeypatch.setattr(_build, "HIPCC_FLAGS", _build.source_flags(src))
    text = asm._assembly(src, tmp_path)
    assert "buffer_wbl2" not in text and "buffer_inv" not in text
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
    assert set(re.findall(r"\.vgpr_spill_count:\s*(\d+)", text)) == {"0"}
    bodies = asm._kernels(text)
    assert len(bodies) >= kernels
    for name, body in bodies.items():
        assert not any(asm.FMA_MIX_F16.match(l) for l in body), name
