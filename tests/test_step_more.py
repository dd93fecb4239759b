"""Slot maps, rotary positions and adapters without a GPU: what calls refuse, configs that change the frequencies, and
what a pool's state goes through."""
import random

import pytest
import torch
from transformers import Qwen2Config, Qwen2ForCausalLM

import custom_inference_engine_amd as cie
from custom_inference_engine_amd.attn import adapters as ad

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
