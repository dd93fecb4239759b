"""Rotary positions on the GPU against 64 bits.

Tolerance: an output is rounded once (half a step of its type); cos and sin are off by 2^-21 at most (the
reduced angle's rounding to fp32, pi 2^-24, and 2 steps of each), two products and a sum by 2^-23 of the
terms: 2^-20 (|x| + |y|) scale together.
"""
import math

import pytest
import torch
from transformers import Qwen2Config
from transformers.models.qwen2.modeling_qwen2 import Qwen2RotaryEmbedding

import custom_inference_engine_amd as cie
from oracle import step as ref
from tests.gpu_helpers import DEV, err_word, note

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def near(got, want, size, what):
    got = got.double().cpu()
    bad = (got - want).abs() > ref.rounding(want, what[0]) + 2.0 ** -20 * size
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, first at {bad.nonzero()[0].tolist()}"



def case(T, h_q, h_kv, d, rot, dtype, far=5000, seed=0, base=1e4):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(1, T, (h_q + 2 * h_kv) * d, generator=g).to(dtype)
    pos = torch.randint(0, far, (T,), generator=g)
    freqs, _ = cie.rotary_frequencies(rot, base)
    return qkv, pos, freqs


def split(qkv, h_q, h_kv, d):
    return qkv.view(1, qkv.shape[1], -1, d).split((h_q, h_kv, h_kv), 2)


SHAPES = [(1, 14, 2, 64, 64), (5, 14, 2, 64, 32), (33, 4, 4, 128, 128), (3, 8, 1, 64, 20), (7, 2, 1, 80, 48), (2, 3, 1, 6, 2),
          (129, 1, 1, 256, 256), (9, 5, 3, 96, 96), (64, 14, 2, 66, 66), (17, 32, 8, 128, 64), (6, 3, 2, 64, 52), (6, 3, 2, 64, 56), (6, 3, 2, 64, 60), (11, 2, 2, 40, 18),
          (4, 2, 1, 30, 16), (4, 2, 1, 24, 14), (3, 2, 1, 42, 34)]


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=str)
@pytest.mark.parametrize("T,h_q,h_kv,d,rot", SHAPES)
def test_apply(T, h_q, h_kv, d, rot, dtype, interleaved):
    qkv, pos, freqs = case(T, h_q, h_kv, d, rot, dtype, seed=T)
    q, k, v = split(qkv.to(DEV), h_q, h_kv, d)
    note(f"apply_rotary T={T} heads {h_q}/{h_kv} d={d} rot={rot} {dtype}")
    got = cie.apply_rotary(q, k, pos.to(DEV), freqs.to(DEV), interleaved=interleaved, scale=1.25)
    for x, y, name in zip(split(qkv, h_q, h_kv, d), got, "qk"):
        assert y.shape == x.shape and y.is_contiguous() and y.dtype == dtype
        want, size = ref.rotary(x[0], pos.tolist(), freqs.tolist(), interleaved, 1.25)
        near(y[0], want, size, (dtype, name))
        assert torch.equal(y[0, ..., rot:].cpu(), x[0, ..., rot:])  # the rest of a head is copied


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("T,h_q,h_kv,d,rot,page", [(1, 14, 2, 64, 64, 16), (77, 14, 2, 64, 32, 16), (33, 8, 8, 128, 128, 32),
                                                   (40, 4, 2, 96, 20, 16), (5, 3, 1, 66, 66, 8), (21, 3, 2, 64, 52, 16),
                                                   (21, 3, 2, 64, 60, 16)])
def test_append(T, h_q, h_kv, d, rot, page, dtype, interleaved):
    qkv, pos, freqs = case(T, h_q, h_kv, d, rot, dtype, seed=T)
    n_pages = 3 + -(-T // page)
    pools = [torch.full((n_pages, h_kv, page, d), float("nan"), dtype=dtype, device=DEV) for _ in range(2)]
    where = torch.randperm(n_pages * page)[:T]
    pages, offsets = where // page, where % page
    err = err_word()
    note(f"append_tokens_qkv_rotary T={T} heads {h_q}/{h_kv} d={d} rot={rot} {dtype}")
    q = cie.append_tokens_qkv_rotary(qkv.to(DEV), pos.to(DEV), freqs.to(DEV), *pools, pages.to(DEV), offsets.to(DEV), h_q,
                                     interleaved=interleaved, scale=0.75, err=err)
    assert int(err) == 0
    x = split(qkv, h_q, h_kv, d)
    held = [p.cpu() for p in pools]
    for y, x_, name in ((q[0].cpu(), x[0], "q"), (held[0][pages, :, offsets], x[1], "k")):
        want, size = ref.rotary(x_[0], pos.tolist(), freqs.tolist(), interleaved, 0.75)
        near(y, want, size, (dtype, name))
    assert torch.equal(held[1][pages, :, offsets], x[2][0])
    for p in held:  # nothing else is written
        p[pages, :, offsets] = float("nan")
        assert p.isnan().all()
    same = cie.apply_rotary(x[0].to(DEV), x[1].to(DEV), pos.to(DEV), freqs.to(DEV), interleaved=interleaved, scale=0.75)
    assert torch.equal(same[0], q) and torch.equal(same[1][0].cpu(), pools[0].cpu()[pages, :, offsets])


def test_append_of_bad_pages_and_offsets():
    qkv, pos, freqs = case(4, 4, 2, 64, 64, F16)
    pools = [torch.zeros((3, 2, 16, 64), dtype=F16, device=DEV) for _ in range(2)]
    for pages, offsets, bit in (([1, 3, 2, -1], [0, 0, 0, 0], 1), ([1, 1, 1, 1], [0, 16, -1, 3], 4)):
        err = err_word()
        q = cie.append_tokens_qkv_rotary(qkv.to(DEV), pos.to(DEV), freqs.to(DEV), *pools, torch.tensor(pages, device=DEV),
                                         torch.tensor(offsets, device=DEV), 4, err=err)
        assert int(err) == bit
        want, size = ref.rotary(split(qkv, 4, 2, 64)[0][0], pos.tolist(), freqs.tolist())
        near(q[0], want, size, (F16, "q"))  # the queries of such rows are turned all the same
    rows = pools[1].cpu()
    assert (rows[1, :, [0, 3]] != 0).any() and (rows[2, :, 0] != 0).any() and (rows[0] == 0).all() and (rows[1, :, 15] == 0).all()


@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
def test_far_positions(dtype):
    """Angles past what fp32 products hold: positions to 2^40, where the fp64 product is still good to 2^-13 of a turn;
    the oracle takes the same product (Python's floats), reduced exactly."""
    pos = torch.tensor([0, 1, 2 ** 20 + 1, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 31, -1, -70001])
    qkv, _, freqs = case(len(pos), 4, 2, 64, 64, dtype)
    q, k, _ = split(qkv.to(DEV), 4, 2, 64)
    got, _ = cie.apply_rotary(q, k, pos.to(DEV), freqs.to(DEV))
    want, size = ref.rotary(split(qkv, 4, 2, 64)[0][0], pos.tolist(), freqs.tolist())
    # (the product's own rounding, 2^-53 of up to 2^31 radians each side, is 2^-22 each: within the bound doubled)
    near(got[0], want, 4 * size, (dtype, "q"))


def test_angle_zero_and_quarter_turns():
    """Position 0 leaves rows as they are; a frequency of pi / 2 takes (x, y) to (-y, x), (-x, -y), (y, -x)."""
    x = torch.randn(1, 4, 2, 8, dtype=F32)
    got, none = cie.apply_rotary(x.to(DEV), None, torch.arange(4, device=DEV),
                                 torch.full((4,), math.pi / 2, dtype=torch.float64, device=DEV))
    a, b = x[0, ..., :4], x[0, ..., 4:]
    want = torch.stack([torch.cat(p, -1) for p in ((a[0], b[0]), (-b[1], a[1]), (-a[2], -b[2]), (b[3], -a[3]))])
    assert none is None and torch.equal(got[0, 0].cpu(), x[0, 0])
    assert (got[0].cpu() - want).abs().max() <= 2.0 ** -20 * x.abs().max() * 2


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=str)
@pytest.mark.parametrize("T,rot", [(1, 64), (77, 128), (5, 20), (300, 2), (40, 48)])
def test_tables(T, rot, dtype, interleaved):
    _, pos, freqs = case(T, 1, 1, rot, rot, dtype, far=200000)
    note(f"rotary_tables T={T} rot={rot} {dtype}")
    cos, sin = cie.rotary_tables(pos[None].to(DEV), freqs.to(DEV), dtype, interleaved, 1.5)
    angle = pos.double()[:, None] * freqs
    for got, want in ((cos, 1.5 * angle.cos()), (sin, 1.5 * angle.sin())):
        want = want.repeat_interleave(2, 1) if interleaved else torch.cat((want, want), 1)
        assert got.shape == (1, T, rot) and got.dtype == dtype
        near(got[0], want, torch.full_like(want, 1.5), (dtype, "table"))


@pytest.mark.parametrize("scaling", [None, {"rope_type": "linear", "factor": 4.0},
                                     {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}],
                         ids=["default", "linear", "yarn"])
def test_tables_are_the_models_own(scaling):
    """Within fp16 of the model's own rotary embedding, which takes its angles in fp32: positions up to 512 only."""
    cfg = Qwen2Config(hidden_size=896, num_attention_heads=14, num_key_value_heads=2, rope_theta=1e6,
                      max_position_embeddings=32768, rope_scaling=scaling)
    pos = torch.arange(0, 512, 3)[None]
    cos, sin = Qwen2RotaryEmbedding(cfg)(torch.zeros(1, dtype=F32), pos)
    freqs, scale = cie.rotary_frequencies(64, 1e6, scaling)
    got = cie.rotary_tables(pos.to(DEV), freqs.to(DEV), scale=scale)
    for a, b in zip(got, (cos, sin)):
        # (fp32 frequencies and angles: 3 roundings of up to 512 radians, 2^-14 in all; fp16: 2^-11 of values up to 1.14)
        assert (a.cpu().double() - b.double()).abs().max() <= 2.0 ** -14 + 1.14 * 2.0 ** -11


def test_non_finite_values_stay_in_their_pairs():
    x = torch.randn(1, 6, 2, 64, dtype=F16)
    x[0, 2, 1, 5], x[0, 3, 0, 40] = float("nan"), float("inf")
    freqs = cie.rotary_frequencies(64)[0].to(DEV)
    pos = torch.arange(7, 13, device=DEV)
    got = cie.apply_rotary(x.to(DEV), None, pos, freqs)[0].cpu()
    bad = ~got.isfinite()
    assert bad.sum() == 4 and bad[0, 2, 1, 5] and bad[0, 2, 1, 37] and bad[0, 3, 0, 40] and bad[0, 3, 0, 8]
    assert got[0, 2, 1, 5].isnan() and got[0, 2, 1, 37].isnan()


def test_strides_and_alignments():
    """Rows, heads and pools at any stride and 2-byte alignment, and packed int32 positions."""
    qkv, pos, freqs = case(11, 3, 2, 64, 32, F16)
    want = cie.apply_rotary(*(t.contiguous().to(DEV) for t in split(qkv, 3, 2, 64)[:2]), pos.to(DEV), freqs.to(DEV))
    base = torch.zeros(11 * 501 + 7, dtype=F16, device=DEV)
    odd = base[7:].view(11, 501)[:, :7 * 64]
    odd.copy_(qkv[0])
    views = [odd[:, 64 * a:64 * b].view(11, b - a, 64) if odd.is_contiguous() else odd.unflatten(1, (7, 64))[:, a:b]
             for a, b in ((0, 3), (3, 5))]
    got = cie.apply_rotary(*views, pos.int().to(DEV), freqs.to(DEV))
    assert all(torch.equal(a, b[0]) for a, b in zip(got, want))
    swapped = qkv.view(11, 7, 64).transpose(0, 1).contiguous().to(DEV).transpose(0, 1)  # heads outermost
    got = cie.apply_rotary(swapped[:, :3], swapped[:, 3:5], pos.to(DEV), freqs.to(DEV))
    assert all(torch.equal(a, b[0]) for a, b in zip(got, want))
    pool = torch.zeros((9, 2, 16, 64), dtype=F16, device=DEV)[::2]
    pools = (pool, torch.zeros((9, 2, 16, 64), dtype=F16, device=DEV)[::2])
    at = torch.arange(11, device=DEV)
    q = cie.append_tokens_qkv_rotary(odd[None], pos.to(DEV), freqs.to(DEV), *pools, at % 5, at, 3)
    assert torch.equal(q, want[0]) and torch.equal(pools[0][at % 5, :, at], want[1][0])


def test_no_rows():
    freqs = cie.rotary_frequencies(64)[0].to(DEV)
    q, k = cie.apply_rotary(torch.empty((1, 0, 4, 64), dtype=F16, device=DEV), torch.empty((1, 0, 2, 64), dtype=F16, device=DEV),
                            torch.empty(0, dtype=torch.int64, device=DEV), freqs)
    assert q.shape == (1, 0, 4, 64) and k.shape == (1, 0, 2, 64)
    assert cie.rotary_tables(torch.empty(0, dtype=torch.int64, device=DEV), freqs)[0].shape == (1, 0, 64)


def test_captured():
    qkv, pos, freqs = case(37, 14, 2, 64, 64, F16)
    qkv, pos, freqs = qkv.to(DEV), pos.to(DEV), freqs.to(DEV)
    q, k, _ = split(qkv, 14, 2, 64)
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        out = cie.apply_rotary(q, k, pos, freqs)
    for i in range(3):
        pos += 1000 * i
        graph.replay()
        want = cie.apply_rotary(q, k, pos, freqs)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
