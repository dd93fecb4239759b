"""Slot maps, rotary positions and adapters without a GPU: what calls refuse, configs that change the frequencies, and
what a pool's state goes through."""
import random

import pytest
import torch
from transformers import Qwen2Config, Qwen2ForCausalLM
from transformers.models.qwen2.modeling_qwen2 import Qwen2RotaryEmbedding

import custom_inference_engine_amd as cie
from custom_inference_engine_amd.attn import adapters as ad
from custom_inference_engine_amd.scheduler import Scheduler

I64 = torch.int64


# ---- adapters ----

def test_rows_that_share_memory():
    """Against the sets of their bytes."""
    r = random.Random(0)
    seen = [0, 0]
    for _ in range(4000):
        n, m = r.choice((1, 2, 3, 5)), r.choice((1, 2, 3, 5))
        size, span = r.randint(1, 6), r.randint(1, 6)
        step = r.randint(size, 14) if n > 1 else r.randint(0, 14)
        hop = r.choice((step, r.randint(0, 14)))
        p, q = 100, 100 + r.randint(-40, 40)
        first = {p + step * i + j for i in range(n) for j in range(size)}
        second = {q + hop * i + j for i in range(m) for j in range(span)}
        assert ad._share(p, step, size, n, q, hop, span, m) == bool(first & second), (p, step, size, n, q, hop, span, m)
        seen[bool(first & second)] += 1
    assert min(seen) > 500


def adapter_args(buf, y, x):
    a, b = torch.zeros((3, 2, 16, 64), dtype=torch.float16), torch.zeros((3, 96, 16), dtype=torch.float16)
    return dict(y=y, x=x, a=a, b=b, scales=torch.ones(3), ranks=torch.full((3,), 16, dtype=torch.int32),
                plan=torch.zeros(8 + 3 * 20, dtype=torch.int32), slices=(64, 32))


def test_adapters_refuse_shared_memory():
    """x anywhere in y's rows is refused; columns of one wider tensor beside each other, or rows behind each other, are not."""
    f16 = torch.float16
    wide, flat = torch.zeros((5, 300), dtype=f16), torch.zeros(4000, dtype=f16)
    y = wide[:, 100:196]
    for left in (37, 40, 95, 99, 100, 150, 195):
        with pytest.raises(AssertionError, match="y's memory"):
            cie.adapter_add_(**adapter_args(wide, y, wide[:, left:left + 64]))
    for x in (wide[:, 100:164].contiguous(), wide[:, 36:100], wide[:, 196:260], wide[:, 0:64]):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            cie.adapter_add_(**adapter_args(wide, y, x))
    y = flat[:480].view(5, 96)
    for x, shared in ((flat[480:800].view(5, 64), False), (flat[479:799].view(5, 64), True), (flat[90:154].expand(5, 64), True),
                      (flat[480:544].expand(5, 64), False), (flat[100:900].view(5, 160)[:, :64], True)):
        with pytest.raises(AssertionError if shared else RuntimeError):
            cie.adapter_add_(**adapter_args(flat, y, x))
    with pytest.raises(AssertionError):  # one row too
        cie.adapter_add_(**adapter_args(flat, flat[None, :96], flat[None, 95:159]))


def _model():
    cfg = Qwen2Config(hidden_size=896, num_attention_heads=14, num_key_value_heads=2, intermediate_size=256,
                      num_hidden_layers=1, vocab_size=128, max_position_embeddings=512)
    model = Qwen2ForCausalLM(cfg).half().eval()
    cie.use_triton_attention(model)
    return cfg, model


def _pool(cfg, n_slots=4):
    return cie.KVStorage(cfg, max_cache_len=192, page_size=16, n_slots=n_slots, device="cpu", dtype=torch.float16)


def test_a_layer_with_adapters_wants_a_plan():
    """A step that would leave its rows without their adapters says so: no plan in the metadata, or no cache at all."""
    cfg, model = _model()
    kv = _pool(cfg)
    layer, = cie.use_adapters(model, kv, 2, 8)
    hidden, emb = torch.zeros(1, 3, 896, dtype=torch.float16), (torch.ones(1, 3, 64).half(), torch.zeros(1, 3, 64).half())
    meta = cie.AttentionMetadata(token_count=3, full_decode=False, device="cpu")
    with pytest.raises(AssertionError, match="adapter_plan"):
        layer(hidden, emb, kv_manager=kv, metadata=meta)
    with pytest.raises(AssertionError, match="adapters"):
        layer(hidden, emb)


def test_state_that_graphs_hold_stays_where_it_is():
    """manage_pages and use_adapters again: the same tensors, as after the first call, or a refusal."""
    cfg, model = _model()
    kv = _pool(cfg)
    kv.manage_pages()
    held = [kv.free_list, kv.page_err]
    kv.free_list[0] = 2
    kv.manage_pages()
    assert kv.free_list is held[0] and kv.page_err is held[1]
    assert torch.equal(kv.free_list, cie.new_free_list(kv.n_pages, "cpu"))
    layer, = cie.use_adapters(model, kv, 2, 8)
    slots, banks = kv.slot_adapters, (layer.qkv_adapters, layer.o_adapters)
    tensors = [t for b in banks for t in (b.a, b.b, b.scales, b.ranks)]
    banks[1].load(1, torch.ones(3, 896), torch.ones(896, 3))
    kv.slot_adapters[1] = 1
    assert cie.use_adapters(model, kv, 2, 8) == [layer]
    assert kv.slot_adapters is slots and (slots == -1).all()
    assert (layer.qkv_adapters, layer.o_adapters) == banks
    assert all(x is y and not y.any() for x, y in zip(tensors, [t for b in banks for t in (b.a, b.b, b.scales, b.ranks)]))
    for n, rank in ((3, 8), (2, 16), (2, 7)):
        with pytest.raises(AssertionError):
            cie.use_adapters(model, kv, n, rank)
    with pytest.raises(AssertionError):
        kv.use_adapters(5)
    assert kv.slot_adapters is slots and kv.n_adapters == 2
    other = _pool(cfg)  # another pool of the same model
    assert cie.use_adapters(model, other, 2, 8) == [layer] and other.n_adapters == 2


def test_a_scheduler_before_manage_pages_stops():
    """A scheduler that keeps the tables itself does not go on with a pool that keeps its own."""
    cfg, _ = _model()
    kv = _pool(cfg)
    sched = Scheduler(None, kv, eos_token_ids={128}, max_new_tokens=16, token_budget=160, executor=object())
    kv.manage_pages()
    future = sched.call([1, 2])
    with pytest.raises(RuntimeError, match="manage_pages"):
        sched.loop()
    assert future.exception() is not None
    kv.use_adapters(2)
    executor = type("Executor", (), {"n_adapters": 0})()  # whose graphs have none
    sched = Scheduler(None, kv, eos_token_ids={128}, max_new_tokens=16, token_budget=160, executor=executor)
    future = sched.call([1, 2], adapter=1)
    assert future.done() and isinstance(future.exception(), ValueError)


def test_any_number_of_slots_is_reset(monkeypatch):
    """A call gives back the pages of 2,048 sequences at most."""
    cfg, _ = _model()
    kv = _pool(cfg, n_slots=5000)
    kv.manage_pages()
    parts = []
    monkeypatch.setattr("custom_inference_engine_amd.kv_cache.pages.release_pages",
                        lambda free_list, slots, *rest, err=None: parts.append(slots.tolist()))
    kv.reset(list(range(4999, -1, -1)))
    assert max(map(len, parts)) <= 2048 and sum(parts, []) == list(range(4999, -1, -1))
    parts.clear()
    kv.reset([])
    assert not any(parts)


# ---- rotary ----

YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}


@pytest.mark.parametrize("scaling", [
    dict(YARN, mscale=1.0, mscale_all_dim=1.0), dict(YARN, mscale=0.707, mscale_all_dim=1.0), dict(YARN, mscale=0.7),
    dict(YARN, mscale_all_dim=0.7), dict(YARN, mscale=0.7, mscale_all_dim=0.0),
    dict(YARN, mscale=0.7, mscale_all_dim=0.5, attention_factor=1.1), dict(YARN, attention_factor=0.0),
    dict(YARN, truncate=False), dict(YARN, truncate=True), dict(YARN, truncate=False, beta_fast=4, beta_slow=2), dict(YARN, beta_fast=None),
    dict(YARN, factor=1.0, mscale=2.0, mscale_all_dim=1.0), dict(YARN, factor=0.5),
    dict(YARN, rope_theta=1e4), {"rope_type": "linear", "factor": 2.0, "rope_theta": 5e5}, {"rope_type": "default", "rope_theta": 1e6},
    {"rope_type": "linear", "factor": 2.0, "partial_rotary_factor": 1.0}, {"rope_type": "linear", "factor": 2.0, "attention_factor": 3.0},
], ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_every_key_of_a_scaling_counts(scaling, d):
    """The config's own rope_scaling, as the model library keeps it, against its rotary embedding's fp32 frequencies:
    three roundings and a power (ln(base) < 14 times the exponent's), and a ramp of four more of the unscaled frequency."""
    cfg = Qwen2Config(hidden_size=14 * d, num_attention_heads=14, num_key_value_heads=2, rope_theta=1e6,
                      max_position_embeddings=32768, rope_scaling=dict(scaling))
    emb = Qwen2RotaryEmbedding(cfg)
    held = dict(cfg.rope_scaling)
    assert held["rope_theta"] == scaling.get("rope_theta", 1e6)
    freqs, scale = cie.rotary_frequencies(d, scaling=held)
    plain = held["rope_theta"] ** (-torch.arange(0, d, 2).double() / d)
    want = emb.inv_freq.double()
    assert ((freqs - want).abs() <= (20 * want + 4 * plain) * 2.0 ** -23).all()
    assert abs(scale - emb.attention_scaling) <= 1e-6
    again, _ = cie.rotary_frequencies(d, held["rope_theta"], held)
    assert torch.equal(again, freqs)


@pytest.mark.parametrize("base,scaling", [
    (None, dict(YARN, short_factor=[1.0])), (None, dict(YARN, llama_4_scaling_beta=0.1)), (1e4, dict(YARN, rope_theta=1e6)),
    (None, {"rope_type": "linear", "factor": 2.0, "partial_rotary_factor": 0.5}), (None, {"partial_rotary_factor": 0.5}),
    (None, {"rope_type": "default", "mrope_section": [8, 12, 12]}), (None, dict(YARN, beta_fast=1, beta_slow=32)),
    (None, {"rope_type": "linear", "factor": None}), (-1.0, None), (None, {"rope_theta": 0.0}),
])
def test_keys_that_are_not_understood_are_refused(base, scaling):
    with pytest.raises(AssertionError):
        cie.rotary_frequencies(64, base, scaling)


def test_adapters_that_are_refused_leave_the_pool_alone():
    cfg, model = _model()
    kv = _pool(cfg)
    for n, rank in ((2, 500), (2, 0), (5000, 8)):
        with pytest.raises(AssertionError):
            cie.use_adapters(model, kv, n, rank)
        assert kv.slot_adapters is None and kv.n_adapters == 0
    kv.use_adapters(2)
    with pytest.raises(AssertionError):
        cie.use_adapters(model, kv, 3, 8)
    layer, = cie.use_adapters(model, kv, 2, 8)
    assert layer.qkv_adapters.n_adapters == 2
