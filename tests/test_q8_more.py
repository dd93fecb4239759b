"""The 8-bit cache without a GPU, further cases: how it is built, and what its paths refuse and accept."""
import os
import re
import types
from collections import Counter

import pytest
import torch
from transformers import Qwen2Config

import custom_inference_engine_amd as cie
from custom_inference_engine_amd import _build
from custom_inference_engine_amd.scheduler import decode_module, mixed_module
from custom_inference_engine_amd.scheduler.scheduler import ModuleExecutor
from oracle import q8_cache as ref
from tests import test_asm_order as asm


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


@pytest.mark.parametrize("lead", [(1,), ()], ids=["3d", "2d"])
def test_fake_impls_of_the_projection_forms_take_both_layouts(lead):
    """(1, n, width) and (n, width) rows, which the calls accept, have outputs of n rows in a traced graph too."""
    n, width = 5, 18 * 64
    qkv, cs = (torch.empty(*lead, n, w, dtype=torch.float16, device="meta") for w in (width, 64))
    k = torch.empty(6, 2, 16, 64, dtype=torch.float8_e4m3fn, device="meta")
    scales = torch.empty(6, 2, 1, 2, device="meta")
    i, table = torch.empty(n, dtype=torch.int64, device="meta"), torch.empty(9, 6, dtype=torch.int64, device="meta")
    ops = torch.ops.inference
    assert ops.kv_append_tokens_qkv_rope_q8(qkv, cs, cs, k, k.clone(), scales, i, i, 14).shape == (1, n, 14, 64)
    assert ops.gqa_decode_qkv_rope_attention_q8(qkv, cs, cs, k, k.clone(), scales, i, i, table, 14).shape == (1, n, 14, 64)


def test_default_splits_are_the_current_devices(monkeypatch):
    """A device without an index is the current one, each time it is asked."""
    from custom_inference_engine_amd.attn import core

    cus, current = {0: 256, 1: 64}, [0]
    monkeypatch.setattr(core.torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(core.torch.cuda, "get_device_properties", lambda d: types.SimpleNamespace(
        multi_processor_count=cus[getattr(d, "index", d) if getattr(d, "index", d) is not None else current[0]]))
    for cached in (core._cu_count, getattr(core, "_device_cus", core._cu_count)):
        getattr(cached, "cache_clear", lambda: None)()
    try:
        any_device = torch.device("cuda")
        assert core.default_decode_splits(4, 2, any_device) == 32
        current[0] = 1
        assert core.default_decode_splits(4, 2, any_device) == 8
        assert core.default_decode_splits(4, 2, torch.device("cuda", 0)) == 32
        assert core.default_decode_splits(4, 2) == 32  # (no device: 256 CUs)
    finally:
        core._device_cus.cache_clear()


# ---- a mixed plan's capacity: the plan kernel's arithmetic, over every group size ----

SLOTS, COLS, MIN_SHARE, MAX_CHUNKS, SMALL = 256, 128, 32, 48, 80


def plan_of(lens, kv_lens, G, h_kv):
    """(items, partial rows, arrival words, columns of a wide tile) of the plan kernel for these sequences."""
    def cut(L, cols):
        narrow = L * G <= 16
        R = L if narrow else cols // G
        return narrow, R, -(-L // R)

    seqs = [(L, c, times) for (L, c), times in Counter(zip(lens, kv_lens)).items() if L]
    total = []
    for cols in (COLS, COLS // 2):
        w = 0.0
        for L, c, times in seqs:
            narrow, R, n = cut(L, cols)
            w += times * (((c + L) >> 6) + 1.0 if narrow else n * ((c >> 4) + 2) + R * n * (n + 1) / 32 + 1)
        total.append(w)
    per = 1.001 * h_kv / SLOTS
    small = total[0] * per <= SMALL
    cols, want = (COLS // 2, total[1]) if small else (COLS, total[0])
    want = int(min(2.0 ** 26, want * per + 1))
    items = rows_out = words = 0
    for L, c, times in seqs:
        narrow, R, n_rt = cut(L, cols)
        share = (max(MIN_SHARE, 4 * want if narrow else want) + 3) & ~3
        for r in range(n_rt):
            rows = min(R, L - r * R)
            n = min(MAX_CHUNKS, -(-((c + r * R + rows + 15) >> 4) // share))
            items += times * n * h_kv
            if n > 1:
                rows_out += times * n * rows * G * h_kv
                words += times * h_kv
    return items, rows_out, words, cols


def test_mixed_plans_fit_what_the_sizes_promise(native_lib):
    """Items, partial rows and arrival words of batches chosen to need many: one row more than a whole or a half tile
    holds (5 heads a group: 25 rows, one whole tile and three half ones), many short sequences, long prefixes."""
    g = torch.Generator().manual_seed(9)

    def rand(lo, hi):
        return int(torch.randint(lo, hi + 1, (1,), generator=g))

    seen = set()
    for G in range(1, 17):
        half, whole = COLS // 2 // G, COLS // G
        edges = [1, half, half + 1, 2 * half + 1, whole, whole + 1, 2 * whole, 2 * whole + 1, 3 * half + 1]
        batches = []
        for h_kv in (1, 2, 3, 8, 32):
            for L in edges:
                for B in (1, 7, 64, 500, 2048):
                    batches += [([L] * B, [0] * B, h_kv), ([L] * B, [rand(0, 3000)] * B, h_kv)]
            for L in (1, 2, 16 // G + 1, whole, 700, 9000):
                batches += [([L], [c], h_kv) for c in (0, 511, 512, 4000, 65536, 2 ** 20)]
            for _ in range(40):
                B = rand(1, 60)
                batches.append(([rand(0, 1) * rand(0, 2 ** rand(0, 9)) for _ in range(B)],
                                [rand(0, 2 ** rand(0, 16)) for _ in range(B)], h_kv))
            # the largest launches of half tiles: batches of edge lengths up to the limit of W
            for L in edges:
                for B in range(1, 2048, 97):
                    batches.append(([L] * B, [0] * B, h_kv))
        for lens, kv_lens, h_kv in batches:
            T, B, h_q = sum(lens), len(lens), G * h_kv
            if T == 0:
                continue
            items, rows, words, cols = plan_of(lens, kv_lens, G, h_kv)
            assert 48 + 48 * items <= native_lib.cie_q8_mixed_plan_bytes(B, T, h_q, h_kv), (G, h_kv, lens[0], B)
            assert rows * (64 + 2) * 4 <= native_lib.cie_q8_mixed_partials_bytes(T, h_q, 64), (G, h_kv, lens[0], B)
            assert 2 * words <= native_lib.cie_q8_mixed_counters(), (G, h_kv, lens[0], B)
            seen.add((cols, rows > 0))
    assert seen == {(COLS, True), (COLS, False), (COLS // 2, True), (COLS // 2, False)}
    assert plan_of([25], [0], 5, 1)[0] == 3  # one whole tile would have held them


# ---- the kernels' assembly ----

@pytest.mark.skipif(not os.path.exists(asm.HIPCC), reason="hipcc not available")
@pytest.mark.parametrize("src,kernel", [("q8_decode.hip", "q8_decode_kernel"), ("q8_mixed.hip", "q8_mixed_kernel"),
                                        ("q8_append.hip", "q8_append_kernel")])
def test_assembly_of_the_8_bit_kernels(src, kernel, tmp_path, monkeypatch):
    """Partial states are stored before their arrival is counted, rotations round to fp32 first, and nothing takes
    the packed fp32 forms; as the 16-bit kernels, with the files' own flags."""
    monkeypatch.setattr(_build, "HIPCC_FLAGS", _build.source_flags(src))
    text = asm._assembly(src, tmp_path)
    assert "buffer_wbl2" not in text and "buffer_inv" not in text
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
    kernels = {n: b for n, b in asm._kernels(text).items() if kernel in n}
    assert kernels
    for name, body in kernels.items():
        assert not any(asm.FMA_MIX_F16.match(l) for l in body), name
        if src != "q8_append.hip":
            asm._check_arrival(name, body)
            parts = [l for l in body if asm.STORE.match(l) and "dwordx4" in l and "buffer_store" in l]
            assert parts and all("sc1" in l for l in parts), name
