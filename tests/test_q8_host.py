"""The 8-bit cache without a GPU: its oracle's pins, refusals, storage, fake impls."""
import ctypes

import pytest
import torch
from transformers import Qwen2Config

import custom_inference_engine_amd as cie
from oracle import q8_cache as ref


def test_oracle_rounding_is_e4m3():
    """The oracle's rounding is torch's cast on every fp16 value in range, and idempotent."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[x.abs() <= 448].double()
    got = ref.round_e4m3(x)
    assert torch.equal(got, x.float().to(torch.float8_e4m3fn).double())
    assert torch.equal(ref.round_e4m3(got), got)


def test_every_held_value_is_an_fp16_value():
    byte = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().double()
    for e in range(ref.E_MIN, ref.E_MAX + 1):
        v = byte[byte.abs() <= (240 if e == 8 else 448)] * 2.0 ** e
        assert torch.equal(v.half().double(), v)


def test_oracle_exponent_borders():
    for e in range(-15, 8):
        edge = torch.tensor(448.0 * 2.0 ** e).half()
        assert ref.exponent(float(edge)) == e
        above = (edge.view(torch.int16) + 1).view(torch.float16)
        assert ref.exponent(float(above)) == e + 1
    assert ref.exponent(0.0) == -15 and ref.exponent(61440.0) == 8


def test_oracle_block_grows_and_starts_anew():
    c = ref.Q8Cache(torch.zeros(2, 1, 16, 1).double(), torch.zeros(2, 1, 1).double())
    c.append(torch.tensor([1.0, 0.3]).view(2, 1, 1), [1, 1], [0, 1])
    assert c.exps[1, 0, 0] == -8 and c.values()[1, 0, 0, 0] == 1.0
    c.append(torch.full((1, 1, 1), 1000.0), [1], [2])  # grows: the others are rounded again
    assert c.exps[1, 0, 0] == 2
    assert c.values()[1, 0, :3, 0].tolist() == [1.0, 0.3125, 1024.0]
    c.append(torch.full((1, 1, 1), 0.5), [1], [0])  # row 0: anew
    assert c.exps[1, 0, 0] == -9
    # a mistake planted in the oracle's own rule must show: without starting anew the exponent stays
    assert max(2, ref.exponent(0.5)) != c.exps[1, 0, 0]


def _cfg(**more):
    return Qwen2Config(hidden_size=896, num_attention_heads=14, num_key_value_heads=2, intermediate_size=256,
                       num_hidden_layers=2, vocab_size=128, max_position_embeddings=512, **more)


def test_storage_in_8_bits():
    kv = cie.KVStorage(_cfg(), max_cache_len=100, page_size=32, n_slots=5, device="cpu", dtype=torch.float8_e4m3fn)
    assert kv.keys[0].shape == (4, 2, 32, 64) and kv.keys[0].element_size() == 1
    assert kv.scales[1].shape == (4, 2, 2, 2) and kv.scales[1].is_contiguous()
    assert cie.KVStorage(_cfg(), 100, 16, 5, "cpu", torch.float16).scales is None
    with pytest.raises(AssertionError, match="multiple of 16"):
        cie.KVStorage(_cfg(), max_cache_len=100, page_size=8, n_slots=5, device="cpu", dtype=torch.float8_e4m3fn)
    x = torch.zeros(1, 1, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="HIP device"):
        kv.decode_update(0, torch.tensor([1]), x, x)
    with pytest.raises(RuntimeError, match="HIP device"):
        kv.mixed_update(0, torch.tensor([1]), torch.tensor([0]), x, x)
    with pytest.raises(RuntimeError, match="HIP device"):
        kv.read_tokens(0, torch.tensor([1]), torch.tensor([0]))


def _args():
    return dict(q=torch.zeros(1, 2, 14, 64, dtype=torch.float16),
                k=torch.zeros(6, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn),
                v=torch.zeros(6, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn),
                scales=torch.ones(6, 2, 1, 2), lens=torch.tensor([3, 4]), slot_ids=torch.tensor([1, 2]),
                block_table=torch.zeros(3, 6, dtype=torch.int64))


@pytest.mark.parametrize("change,match", [
    (lambda a: a.update(q=a["q"][:, :, :13].contiguous()), "multiple"),
    (lambda a: a.update(q=a["q"].float()), "float16"),
    (lambda a: a.update(q=a["q"].transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
    (lambda a: a.update(q=a["q"][..., :32].contiguous()), "q must be"),
    (lambda a: a.update(k=a["k"].view(torch.uint8)), "float8_e4m3fn"),
    (lambda a: a.update(v=a["v"][:5]), "pools must be"),
    (lambda a: a.update(scales=a["scales"].double()), "scales"),
    (lambda a: a.update(scales=torch.ones(6, 2, 2, 2)), "scales"),
    (lambda a: a.update(scales=torch.ones(6, 2, 1, 4)[..., ::2]), "scales"),
    (lambda a: a.update(block_table=a["block_table"][:, :5]), "n_pages"),
    (lambda a: a.update(lens=a["lens"][:1]), "lens"),
    (lambda a: a.update(slot_ids=a["slot_ids"][:1], lens=a["lens"][:1]), "one query token"),
])
def test_decode_refusals(change, match):
    a = _args()
    change(a)
    with pytest.raises(AssertionError, match=match):
        cie.decode_gqa_attention_q8(**a)


def test_other_refusals():
    a = _args()
    cache = (a["k"], a["v"], a["scales"])
    x = torch.zeros(1, 2, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="HIP device"):
        cie.decode_gqa_attention_q8(**a)
    with pytest.raises(RuntimeError, match="HIP device"):
        cie.decode_append_gqa_attention_q8(a["q"], *cache, x, x, a["lens"], a["slot_ids"], a["block_table"])
    with pytest.raises(AssertionError, match="cu_seqlens"):
        cie.mixed_gqa_attention_q8(a["q"], *cache, 1, torch.tensor([0, 1]), a["lens"], a["slot_ids"], a["block_table"])
    with pytest.raises(AssertionError, match="kv_lens"):
        cie.mixed_gqa_attention_q8(a["q"], *cache, 1, torch.tensor([0, 1, 2]), a["lens"][:1], a["slot_ids"],
                                   a["block_table"])
    with pytest.raises(AssertionError, match="page_size"):
        k8 = torch.zeros(6, 2, 8, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
        cie.kv_read_tokens_q8(k8, k8, torch.ones(6, 2, 0, 2), a["lens"], a["lens"])
    with pytest.raises(AssertionError, match="qkv must be"):
        cie.decode_qkv_rope_gqa_attention_q8(x.view(1, 2, 128), x, x, *cache, a["lens"], a["slot_ids"],
                                             a["block_table"], 14)


def test_abi_refuses_before_launching(native_lib):
    """Host-side checks of the C entry points: nothing is launched (there is no GPU here)."""
    p = ctypes.c_void_p(4096)
    EINVAL, EUNSUP = -1, -2

    def append(D=64, page=16, H=2, stride=2048, T=1, kp=p, ks=128):
        return native_lib.cie_q8_append_tokens(kp, p, p, p, p, ks, 64, 128, 64, p, p, T, H, page, D, 4, stride, 1024,
                                               None, None)

    assert append(D=96) == EUNSUP and append(D=63) == EUNSUP and append(page=24) == EUNSUP
    assert append(H=0) == EINVAL and append(T=-1) == EINVAL and append(stride=2040) == EINVAL
    assert append(kp=None) == EINVAL and append(kp=ctypes.c_void_p(4100)) == EINVAL and append(ks=100) == EINVAL
    assert append(T=0) == 0

    def decode(D=64, hq=14, page=16, splits=1, plan=None, parts=p, B=2):
        return native_lib.cie_q8_decode(p, p, p, p, p, p, p, p, plan, parts, p, B, hq, 2, D, page, 4, 2048, 1024, 4,
                                        4, 3, splits, None, None)

    assert decode(D=32) == EUNSUP and decode(hq=34) == EUNSUP and decode(page=8) == EUNSUP
    assert decode(hq=13) == EINVAL and decode(splits=0) == EINVAL and decode(splits=65) == EUNSUP
    assert decode(splits=2, parts=None) == EINVAL and decode(plan=p, splits=3) == EINVAL and decode(B=0) == 0

    def mixed(B=2, T=8, D=64, hq=14, parts=None, n=None):
        n = native_lib.cie_q8_mixed_partials_bytes(T, hq, D) if n is None else n
        return native_lib.cie_q8_mixed(p, p, p, p, p, p, 1 << 20, p, parts, n, p, B, T, hq, 2, D, 16, 4, 2048, 1024,
                                       4, 4, 3, None, None)

    assert mixed() == EINVAL and mixed(parts=p, n=16) == EINVAL and mixed(D=32) == EUNSUP
    assert mixed(hq=34) == EUNSUP and mixed(B=4096) == EUNSUP and mixed(T=0) == 0
    assert native_lib.cie_q8_mixed_plan_bytes(-1, 8, 14, 2) == -1
    assert native_lib.cie_q8_mixed_plan_bytes(4096, 8, 14, 2) == -1
    assert native_lib.cie_q8_mixed_plan(p, 16, p, p, p, 2, 8, 8, 14, 2, 64, 16, 4, 3, None, None) == EINVAL


def test_fake_impls(native_lib):
    a = {k: v.to("meta") for k, v in _args().items()}
    ops = torch.ops.inference
    assert ops.gqa_decode_attention_q8(a["q"], a["k"], a["v"], a["scales"], a["lens"], a["slot_ids"],
                                       a["block_table"]).shape == a["q"].shape
    qkv = torch.empty(1, 2, 18 * 64, dtype=torch.float16, device="meta")
    cs = torch.empty(1, 2, 64, dtype=torch.float16, device="meta")
    assert ops.kv_append_tokens_qkv_rope_q8(qkv, cs, cs, a["k"], a["v"], a["scales"], a["lens"], a["lens"],
                                            14).shape == (1, 2, 14, 64)
    n = native_lib.cie_q8_mixed_plan_bytes(2, 2, 14, 2) // 4
    cu = torch.zeros(3, dtype=torch.int64, device="meta")
    assert ops.gqa_mixed_plan_q8(a["k"], cu, a["lens"], a["slot_ids"], a["block_table"], 2, 2, 14).shape == (n,)


def test_piecewise_cuts_at_the_8_bit_attention():
    from custom_inference_engine_amd.piecewise import utils

    g = torch.fx.Graph()
    x = g.placeholder("x")
    kv_lens = g.call_function(torch.add, (x, 1))
    y = g.call_function(utils.MIXED_ATTENTION_Q8, (x, x, x, x), {"kv_lens": kv_lens})
    z = g.call_function(torch.mul, (y, 2))
    g.output(z)
    ids = utils.create_partition(torch.fx.GraphModule({}, g))
    assert utils.is_attention(y) and ids[y] % 2 == 1 and ids[kv_lens] == ids[y] and ids[z] == ids[y] + 1
