"""The 8-bit cache without a GPU, further cases: how it is built, and what its paths refuse and accept."""
import types

import pytest
import torch
from transformers import Qwen2Config

import custom_inference_engine_amd as cie
from custom_inference_engine_amd import _build
from custom_inference_engine_amd.scheduler import decode_module, mixed_module
from custom_inference_engine_amd.scheduler.scheduler import ModuleExecutor
from oracle import q8_cache as ref


@pytest.mark.parametrize("src", _build.SOURCES)
def test_kernels_that_keep_nans_are_built_to(src, tmp_path, monkeypatch):
    """A NaN held in an 8-bit cache has to come out of its attention: no such file may be compiled as if none existed."""
    seen = []

    def run(cmd, **_):
        seen.append(cmd)
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(_build.subprocess, "run", run)
    _build._compile(src, False, str(tmp_path))
    assert ("-fno-honor-nans" in seen[0]) != src.startswith("q8_")
    assert "-ffast-math" not in seen[0] and "-packed-fp32-ops" in seen[0]


def config():
    return Qwen2Config(hidden_size=896, num_attention_heads=14, num_key_value_heads=2, intermediate_size=256,
                       num_hidden_layers=2, vocab_size=128, max_position_embeddings=512)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float8_e4m3fn], ids=str)
def test_piecewise_buffer_needs_no_dtype_of_the_model(dtype, monkeypatch):
    """The attention outputs' buffer has the cache's type, float16 beside an 8-bit one; the model's object, which need
    not have one, is not asked."""
    for module, name in ((decode_module, "DecodeModule"), (mixed_module, "FullMixedModule"),
                         (mixed_module, "PiecewiseMixedModule")):
        monkeypatch.setattr(module, name, lambda *args, **kw: types.SimpleNamespace(**kw))
    kv = cie.KVStorage(config(), max_cache_len=64, page_size=16, n_slots=3, device="cpu", dtype=dtype)
    model = object()
    executor = ModuleExecutor(model, kv, [1, 2], [16, 128, 160], pool=object(), piecewise_above=128)
    assert executor.buffer.dtype == (torch.float16 if dtype == torch.float8_e4m3fn else dtype)
    assert executor.buffer.shape == (1, 160, 14, 64) and executor.mixed_modules[160].buffer is executor.buffer
    assert not hasattr(executor.mixed_modules[128], "buffer")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("index", [torch.int64, torch.int32], ids=str)
def test_read_tokens_of_a_16_bit_cache(dtype, index):
    """Rows in any order, as mixed_update takes them; what lies outside the pool reads as zeros, as from an 8-bit cache."""
    kv = cie.KVStorage(config(), max_cache_len=64, page_size=16, n_slots=3, device="cpu", dtype=dtype)
    g = torch.Generator().manual_seed(0)
    for pool in (kv.keys[1], kv.values[1]):
        pool.copy_(torch.randn(pool.shape, generator=g))
    kv.keys[1][0, :, 0] = float("nan")  # (what a clamped index would read)
    n = kv.n_pages
    pages = torch.tensor([3, 0, n, -1, 2, 1, 1, 10 ** 6], dtype=index)
    offs = torch.tensor([15, 7, 0, 0, 0, 16, -1, 3], dtype=index)
    held = [True, True, False, False, True, False, False, False]
    for got, pool in zip(kv.read_tokens(1, pages, offs), (kv.keys[1], kv.values[1])):
        assert got.shape == (1, 8, 2, 64) and got.dtype == dtype
        for t, ok in enumerate(held):
            want = pool[int(pages[t]), :, int(offs[t])] if ok else torch.zeros(2, 64, dtype=dtype)
            assert torch.equal(got[0, t], want)
    none = kv.read_tokens(0, pages[:0], offs[:0])
    assert [x.shape for x in none] == [(1, 0, 2, 64)] * 2


def test_held_values_stay_within_the_stated_error():
    """Rows that come one at a time, each of which may make the block grow: 2^-4 |x| + 2^-9 * scale, and half of the
    second where a row has seen no growth.  Half of it alone does not hold after growths."""
    g = torch.Generator().manual_seed(4)
    past_half = 0
    for case in range(200):
        c = ref.Q8Cache(torch.zeros(1, 1, 16, 64).double(), torch.zeros(1, 1, 1).double())
        grow = torch.cumsum(torch.randint(0, 3, (16,), generator=g), 0)
        x = (torch.randn(16, 1, 64, generator=g) * 2.0 ** (grow - 12.0 - 2 * torch.rand(16, generator=g))[:, None, None])
        x = (x * 2.0 ** (-9.0 * torch.rand(16, 1, 64, generator=g))).half()
        for t in range(16):
            before = float(c.exps[0, 0, 0])
            c.append(x[t:t + 1], [0], [t])
            scale = 2.0 ** float(c.exps[0, 0, 0])
            want = x[:t + 1, 0].double()
            off = (c.values()[0, 0, :t + 1] - want).abs()
            assert (off <= want.abs() * 2.0 ** -4 + scale * 2.0 ** -9).all()
            assert (off[t] <= torch.maximum(want[t].abs() * 2.0 ** -4, torch.tensor(scale * 2.0 ** -10))).all()
            assert t == 0 or c.exps[0, 0, 0] >= before
            past_half += int((off > torch.maximum(want.abs() * 2.0 ** -4, torch.tensor(scale * 2.0 ** -10))).sum())
    assert past_half > 0
    # 2.51 steps are held as 3; in steps twice as large, 1.5, as 2: off by 0.745 of such a step
    c = ref.Q8Cache(torch.zeros(1, 1, 16, 1).double(), torch.zeros(1, 1, 1).double())
    x = 2.51 * 2.0 ** -9
    c.append(torch.tensor([448.0, x]).view(2, 1, 1), [0, 0], [0, 1])
    assert c.values()[0, 0, 1, 0] == 3 * 2.0 ** -9
    c.append(torch.tensor([800.0]).view(1, 1, 1), [0], [2])
    assert c.exps[0, 0, 0] == 1 and c.values()[0, 0, 1, 0] == 2 * 2.0 ** -8
    assert abs(2 * 2.0 ** -8 - x) > 0.74 * 2.0 ** -8
