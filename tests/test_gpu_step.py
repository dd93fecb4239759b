"""Slot maps, adapters and rotary positions together, as a step uses them: by hand on one layer's operators, and
through the step modules and the scheduler on a small Qwen2."""
import copy

import pytest
import torch
from transformers import Qwen2Config, Qwen2ForCausalLM

import custom_inference_engine_amd as cie
from custom_inference_engine_amd import KVStorage, use_adapters, use_rotary, use_triton_attention
from custom_inference_engine_amd.scheduler import DecodeModule, FullMixedModule, MixedModule, Scheduler
from oracle import paged_attention as attn
from oracle import step as ref
from tests.gpu_helpers import DEV, err_word, note

pytestmark = pytest.mark.gpu
H_Q, H_KV, D = 14, 2, 64


def test_a_layer_by_hand():
    """Two steps of one layer: maps with pages from the list, the projection's adapters, turned rows into the pools, mixed
    attention; against the oracles in 64 bits (attention within the suite's bar)."""
    g = torch.Generator().manual_seed(0)
    hidden, widths = 96, (H_Q * D, H_KV * D, H_KV * D)
    page, n_pages, n_slots = 16, 40, 5
    k_pool, v_pool = (torch.full((n_pages, H_KV, page, D), 3.0, dtype=torch.float16, device=DEV) for _ in range(2))
    free = cie.new_free_list(n_pages, DEV)
    lens = torch.zeros(n_slots, dtype=torch.int64, device=DEV)
    table = torch.zeros((n_slots, n_pages), dtype=torch.int64, device=DEV)
    by_slot = torch.tensor([-1, 1, -1, 0, 1], device=DEV)
    bank = cie.AdapterBank(2, 24, hidden, widths, device=DEV)
    for i, r in enumerate((24, 5)):
        bank.load(i, [torch.randn(r, hidden, generator=g) * 0.1 for _ in widths],
                  [torch.randn(w, r, generator=g) * 0.3 for w in widths], scale=0.5 + i)
    weight = (torch.randn(sum(widths), hidden, generator=g) * 0.1).half()
    freqs, scale = cie.rotary_frequencies(48, 1e6, {"rope_type": "linear", "factor": 2.0})  # part of the head
    rows_of = {s: [[], []] for s in range(n_slots)}  # each slot's turned k and its v, as the pools should hold them

    for slots, new in (([3, 1, 4], [21, 33, 1]), ([1, 2, 3, 4], [1, 40, 1, 1])):
        T = sum(new) + 3
        x = torch.randn(1, T, hidden, generator=g).half()
        ids, n_new = torch.tensor(slots, device=DEV), torch.tensor(new, device=DEV)
        note(f"layer by hand T={T}")
        err = err_word()
        m = cie.step_maps(ids, n_new, lens, table, page, T, free_list=free, err=err)
        qkv = torch.nn.functional.linear(x.to(DEV), weight.to(DEV))
        plain = qkv.cpu()
        plan = cie.adapter_plan(m.slots, by_slot, 2, err=err)
        cie.adapter_add_(qkv, x.to(DEV), bank.a, bank.b, bank.scales, bank.ranks, plan, bank.slices, err=err)
        q = cie.append_tokens_qkv_rotary(qkv, m.positions, freqs.to(DEV), k_pool, v_pool, m.pages, m.offsets, H_Q,
                                         interleaved=True, scale=scale, err=err)
        o = cie.mixed_gqa_attention(q, k_pool, v_pool, T, m.cu_seqlens, lens[ids], ids, table, err=err)
        torch.cuda.synchronize()
        assert int(err) == 0

        row_slot = m.slots.tolist()
        row_adapter = [int(by_slot[s]) for s in row_slot]
        want, off = ref.adapters(plain[0], x[0], bank.a.cpu(), bank.b.cpu(), bank.scales.cpu(), row_adapter, widths)
        got = qkv[0].cpu()
        assert ((got.double() - want).abs() <= off + ref.rounding(want.abs() + off, torch.float16)).all()
        heads = got.view(T, -1, D)
        turned, size = ref.rotary(heads[:, :H_Q + H_KV], m.positions.tolist(), freqs.tolist(), True, scale)
        near = ref.rounding(turned, torch.float16) + 2.0 ** -20 * size
        assert ((q[0].cpu().double() - turned[:, :H_Q]).abs() <= near[:, :H_Q]).all()
        pages, offs = m.pages.cpu(), m.offsets.cpu()
        n = sum(new)
        held = k_pool.cpu()[pages, :, offs][:n]
        assert ((held.double() - turned[:n, H_Q:]).abs() <= near[:n, H_Q:]).all()
        assert torch.equal(v_pool.cpu()[pages, :, offs][:n], heads[:n, H_Q + H_KV:])
        wm, written = attn.mixed_attention(q.cpu(), k_pool.cpu(), v_pool.cpu(), m.cu_seqlens.cpu(), lens[ids].cpu(), ids.cpu(),
                                           table.cpu())
        assert written.sum() == n
        assert ((o[0].float().cpu() - wm)[written].abs() <= 2e-3 + 1e-2 * wm[written].abs()).all()
        for t in range(n):  # the pools hold every earlier row too
            rows_of[row_slot[t]][0].append(held[t])
            rows_of[row_slot[t]][1].append(heads[t, H_Q + H_KV:])
        lens[ids] += n_new
        for s in range(1, n_slots):
            pos = torch.arange(int(lens[s]))
            at = table[s].cpu()[pos // page], pos % page
            for pool, rows in zip((k_pool, v_pool), rows_of[s]):
                assert len(rows) == len(pos)
                if rows:
                    assert torch.equal(pool.cpu()[at[0], :, at[1]], torch.stack(rows))
    cie.release_pages(free, torch.tensor([1, 2, 3, 4], device=DEV), lens, table, page)
    assert int(free[0]) == n_pages - 1 and sorted(free[2:n_pages + 1].tolist()) == list(range(1, n_pages))


def _config(**more):
    cfg = Qwen2Config(hidden_size=896, num_attention_heads=H_Q, num_key_value_heads=H_KV, intermediate_size=1024,
                      num_hidden_layers=2, vocab_size=512, max_position_embeddings=4096, rope_theta=1e6, rms_norm_eps=1e-6,
                      tie_word_embeddings=True, **more)
    cfg._attn_implementation = "sdpa"
    return cfg


def _models(cfg):
    torch.manual_seed(0)
    theirs = Qwen2ForCausalLM(cfg).float().eval()
    with torch.no_grad():  # (weights of the size of a trained model's, so that attention is not uniform)
        for layer in theirs.model.layers:
            for p in (layer.self_attn.q_proj, layer.self_attn.k_proj):
                p.weight.mul_(4)
    ours = copy.deepcopy(theirs).half().to(DEV)
    use_triton_attention(ours)
    return theirs, ours


def _logits(model, tokens):
    with torch.no_grad():
        return model(input_ids=torch.tensor([tokens]), use_cache=False).logits[0, -1]


def _rel(a, b):
    return ((a.float().cpu() - b).norm() / b.norm()).item()


def _prompts(*lengths, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 512, (n,), generator=g).tolist() for n in lengths]


def _adapters(layers, n, rank, seed):
    """Random adapters in every place, and how to merge one into a plain model's weights."""
    g = torch.Generator().manual_seed(seed)
    kept = []
    for i in range(n):
        r, scale, per_layer = rank - 3 * i, 1.0 + i, []
        for layer in layers:
            a = [torch.randn(r, 896, generator=g) * 0.05 for _ in range(4)]
            b = [torch.randn(w, r, generator=g) * 0.1 for w in (*layer.qkv_sizes, 896)]
            layer.qkv_adapters.load(i, a[:3], b[:3], scale)
            layer.o_adapters.load(i, a[3], b[3], scale)
            per_layer.append([scale * (y.half().float() @ x.half().float()) for x, y in zip(a, b)])
        kept.append(per_layer)

    def merged(model, i):
        model = copy.deepcopy(model)
        with torch.no_grad():
            for layer, deltas in zip(model.model.layers, kept[i] if i >= 0 else ()):
                at = layer.self_attn
                for p, d in zip((at.q_proj, at.k_proj, at.v_proj, at.o_proj), deltas):
                    p.weight.add_(d)
        return model
    return merged


def test_requests_with_their_own_adapters(native_lib):
    """A packed prefill and captured decode steps of four requests with three adapters among them and none: each one's
    logits are those of the plain model with its adapter merged into the weights."""
    cfg = _config()
    theirs, ours = _models(cfg)
    kv = KVStorage(cfg, max_cache_len=2048, page_size=16, n_slots=6, device=DEV, dtype=torch.float16)
    kv.manage_pages()
    merged = _adapters(use_adapters(ours, kv, 3, 20), 3, 20, seed=1)
    note("adapters: capturing")
    dec, mix = DecodeModule(ours, kv, batch_size=4), FullMixedModule(ours, kv, batch_size=5, token_count=128)
    eager = MixedModule(ours, kv, token_count=128)
    slots, which, prompts = [1, 2, 3, 5], [2, -1, 0, 2], _prompts(37, 5, 20, 11)
    for s, i in zip(slots, which):
        kv.slot_adapters[s] = i
    models = [merged(theirs, i) for i in which]
    assert _rel(_logits(models[0], prompts[0]), _logits(theirs, prompts[0])) > 0.2  # an adapter is felt
    bar = 2e-2  # (the suite's for fp16 logits of this model)

    note("adapters: prefill")
    nxt = mix.forward(prompts, slots)
    seqs = [p + [t] for p, t in zip(prompts, nxt)]
    for i in range(4):
        assert _rel(mix.last_logits[i], _logits(models[i], prompts[i])) < bar, i
    for step in range(2):
        note(f"adapters: decode {step}")
        nxt = dec.forward(slots)
        for i in range(4):
            assert _rel(dec.logits[i], _logits(models[i], seqs[i])) < bar, (step, i)
            seqs[i].append(nxt[i])
    note("adapters: mixed step of decode rows, and a slot with another request's adapter")
    kv.reset([2])
    kv.slot_adapters[2] = 1
    more = _prompts(30, seed=8)[0]
    nxt = eager.forward([[s[-1]] for s in (seqs[0], seqs[2])] + [more], [1, 3, 2])
    for got, model, seq in zip(eager.last_logits, (models[0], models[2], merged(theirs, 1)), (seqs[0], seqs[2], more)):
        assert _rel(got, _logits(model, seq)) < bar
    kv.reset([1, 2, 3, 5])
    assert int(kv.free_list[0]) == kv.n_pages - 1 and kv.lens.eq(0).all() and kv.block_table.eq(0).all()


@pytest.mark.parametrize("managed", [False, True])
@pytest.mark.parametrize("piecewise", [False, True])
def test_scheduler_with_adapters_and_pages_on_the_device(native_lib, piecewise, managed):
    """Requests with adapters of their own served with preemption: every token is the merged model's greedy choice, up to
    the fp16 path's error; where the pool manages its pages, the list is whole again afterwards."""
    torch._dynamo.reset()
    cfg = _config()
    theirs, ours = _models(cfg)
    kv = KVStorage(cfg, max_cache_len=192, page_size=16, n_slots=4, device=DEV, dtype=torch.float16)
    if managed:
        kv.manage_pages()
    merged = _adapters(use_adapters(ours, kv, 2, 16), 2, 16, seed=2)
    note("scheduler with adapters: capturing")
    sched = Scheduler(ours, kv, eos_token_ids={512}, max_new_tokens=16, token_budget=160, piecewise_mixed=piecewise)
    prompts, which = _prompts(60, 70, 50, 9, 64, seed=11), [0, -1, 1, 1, 0]
    note("scheduler with adapters: generate")
    with torch.inference_mode():
        results = sched.generate(prompts, which)
    torch.cuda.synchronize()
    assert sched.stats.preemptions == 2
    for p, i, r in zip(prompts, which, results):
        seq = p + r.new_tokens
        with torch.no_grad():
            logits = merged(theirs, i)(input_ids=torch.tensor([seq[:-1]]), use_cache=False).logits[0]
        for j, tok in enumerate(r.new_tokens):
            row = logits[len(p) - 1 + j]
            assert float(row.max() - row[tok]) <= 2e-2 * float(row.max() - row.min()), (i, j)
    assert kv.lens.eq(0).all() and kv.block_table.eq(0).all() and kv.slot_adapters.eq(-1).all()
    if managed:
        assert int(kv.free_list[0]) == kv.n_pages - 1 and kv.free_list[1] == 0
        assert sorted(kv.free_list[2:kv.n_pages + 1].tolist()) == list(range(1, kv.n_pages))


def test_maps_of_the_step_modules(native_lib):
    """The mixed step's maps are those that the CPU form of the module derives."""
    cfg = _config()
    _, ours = _models(cfg)
    kv = KVStorage(cfg, max_cache_len=1024, page_size=16, n_slots=6, device=DEV, dtype=torch.float16)
    mod = MixedModule(ours, kv, token_count=64)
    kv.block_table[1:] = torch.randperm(5 * kv.n_pages, device=DEV).view(5, -1) % kv.n_pages
    kv.lens[1:] = torch.tensor([0, 31, 200, 16, 5], device=DEV)
    with torch.inference_mode():
        mod.upload([[1] * 17, [2], [3] * 30], [4, 2, 5])
        mod._prepare()
        got = [t.clone() for t in (mod.cu_seqlens, mod.positions, mod.metadata.pages, mod.metadata.offsets)]
        mod._prepare_host(kv, mod.batch_size)
        for a, b in zip(got, (mod.cu_seqlens, mod.positions, mod.metadata.pages, mod.metadata.offsets)):
            assert torch.equal(a, b)
    assert mod.row_slots.tolist() == [4] * 17 + [2] + [5] * 30 + [0] * 16


def test_out_of_pages(native_lib):
    """A pool that manages its pages says when a step finds too few, keeps every token it held, and goes on when some are
    free again; eagerly and in graphs."""
    cfg = _config()
    _, ours = _models(cfg)
    kv = KVStorage(cfg, max_cache_len=6 * 16, page_size=16, n_slots=4, device=DEV, dtype=torch.float16)
    kv.manage_pages()
    mix, dec = MixedModule(ours, kv, token_count=64), DecodeModule(ours, kv, batch_size=2)
    full = FullMixedModule(ours, kv, batch_size=3, token_count=64)
    note("out of pages")
    mix.forward([[1] * 32, [2] * 32], [1, 2])  # four of five pages
    held = kv.keys[0][kv.block_table[1, :2]].clone()
    for module in (mix, full):
        with pytest.raises(RuntimeError, match="free pages"):
            module.forward([[3] * 20], [3])
        kv.lens[3] = 0  # (the caller drops the step)
        assert int(kv.free_list[0]) == 1 and not kv.block_table[3].any()
    with pytest.raises(RuntimeError, match="free pages"):
        dec.forward([1, 2])  # a page each
    kv.lens[1:3] = 32
    assert torch.equal(kv.keys[0][kv.block_table[1, :2]], held)
    kv.reset([2])
    assert int(kv.free_list[0]) == 3
    dec.forward([1])
    assert kv.lens.tolist() == [0, 33, 0, 0] and int(kv.block_table[1, 2]) > 0
    kv.reset_pages()
    assert int(kv.free_list[0]) == 5 and not kv.lens.any() and not kv.block_table.any()


def test_a_model_that_is_cast_keeps_its_adapters(native_lib):
    cfg = _config()
    _, ours = _models(cfg)
    kv = KVStorage(cfg, max_cache_len=256, page_size=16, n_slots=3, device=DEV, dtype=torch.float16)
    layers = use_adapters(ours, kv, 2, 8)
    layers[0].o_adapters.load(1, torch.ones(3, 896), torch.ones(896, 3), scale=0.3)
    ours.half()
    bank = layers[0].o_adapters
    assert bank.scales.dtype == torch.float32 and bank.ranks.dtype == torch.int32 and bank.a.dtype == torch.float16
    assert bank.scales[1] == torch.tensor(0.3)


def _run(ours, kv, prompts, theirs, bar=2e-2):
    """A prefill and two decode steps of every prompt against another model's logits (the suite's bar for fp16)."""
    dec, mix = DecodeModule(ours, kv, batch_size=2), MixedModule(ours, kv, token_count=128)
    slots = [1, 2]
    nxt = mix.forward(prompts, slots)
    seqs = [p + [t] for p, t in zip(prompts, nxt)]
    for i in range(2):
        assert _rel(mix.last_logits[i], _logits(theirs, prompts[i])) < bar, i
    for step in range(2):
        nxt = dec.forward(slots)
        for i in range(2):
            assert _rel(dec.logits[i], _logits(theirs, seqs[i])) < bar, (step, i)
            seqs[i].append(nxt[i])


def test_stretched_positions(native_lib):
    """A model whose config stretches its positions: rows turned by ``rotary_frequencies`` of the same config."""
    scaling = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}
    theirs, ours = _models(_config(rope_scaling=scaling))
    kv = KVStorage(ours.config, max_cache_len=512, page_size=16, n_slots=4, device=DEV, dtype=torch.float16)
    kv.manage_pages()
    prompts = _prompts(100, 9)
    ours.model.rotary_emb = None
    use_rotary(ours, *cie.rotary_frequencies(D, 1e6, scaling))
    note("stretched positions")
    _run(ours, kv, prompts, theirs)
    plain, _ = _models(_config())
    assert _rel(_logits(plain, prompts[0]), _logits(theirs, prompts[0])) > 4e-2  # the stretch is felt


def test_interleaved_positions(native_lib):
    """A checkpoint of interleaved layout: the plain model's q and k rows dealt to neighbouring dims attend as before."""
    theirs, ours = _models(_config())
    deal = torch.arange(D).view(2, D // 2).t().flatten()  # new dim 2i, 2i + 1 <- old i, i + D / 2
    with torch.no_grad():
        for layer in ours.model.layers:
            at = layer.self_attn
            rows = torch.arange(sum(at.qkv_sizes)).view(-1, D)
            rows[:H_Q + H_KV] = rows[:H_Q + H_KV][:, deal]
            at.qkv_weight.copy_(at.qkv_weight[rows.flatten()])
            at.qkv_bias.copy_(at.qkv_bias[rows.flatten()])
    kv = KVStorage(ours.config, max_cache_len=512, page_size=16, n_slots=4, device=DEV, dtype=torch.float16)
    kv.manage_pages()
    use_rotary(ours, *cie.rotary_frequencies(D, 1e6), interleaved=True)
    note("interleaved positions")
    _run(ours, kv, _prompts(50, 9), theirs)
    with pytest.raises(AssertionError):  # the wrapped module has no such positions
        ours(input_ids=torch.tensor([[1, 2]], device=DEV), use_cache=False)


@pytest.mark.parametrize("decode", [False, True], ids=["mixed", "decode"])
@pytest.mark.parametrize("rot", [0, 64, 40], ids=["tables", "interleaved", "part"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float8_e4m3fn], ids=["fp16_cache", "8_bit_cache"])
def test_a_replaced_layer_is_its_operators(native_lib, dtype, rot, decode):
    """One layer of the model, with adapters and each kind of positions, on both caches: its output and the cache, bit for
    bit, from the operators called one by one."""
    cfg = _config()
    _, ours = _models(cfg)
    kvs = [KVStorage(cfg, max_cache_len=512, page_size=16, n_slots=5, device=DEV, dtype=dtype) for _ in range(2)]
    layers = use_adapters(ours, kvs[0], 2, 16)
    _adapters(layers, 2, 16, seed=3)
    layer = layers[1]
    freqs, scale = cie.rotary_frequencies(rot or D, 1e6)
    freqs = freqs.to(DEV)
    how = dict(interleaved=rot == 64, scale=scale)
    use_rotary(ours, freqs, scale, interleaved=rot == 64)
    slots, new = ([1, 2, 4], [1, 1, 1]) if decode else ([4, 1, 2], [20, 1, 13])
    T = sum(new)
    slot_ids, n_new = torch.tensor(slots, device=DEV), torch.tensor(new, device=DEV)
    g = torch.Generator().manual_seed(2)
    past = [torch.randn(1, 50, H_KV, D, generator=g).half().to(DEV) for _ in range(2)]
    at = torch.arange(50, device=DEV)
    for kv in kvs:  # what the sequences hold
        kv.block_table[1:] = 1 + torch.arange(4 * 7, device=DEV).view(4, 7).repeat(1, 5)[:, :kv.n_pages]
        kv.lens[1:] = torch.tensor([50, 17, 0, 30], device=DEV)
        for s in range(1, 5):
            kv.mixed_update(1, kv.block_table[s][at // 16], at % 16, *past)
    hidden = torch.randn(1, T, 896, generator=g).half().to(DEV)
    by_slot = torch.tensor([-1, 1, -1, 0, 0], device=DEV)
    a, b = kvs
    note(f"a layer and its operators: {dtype} rot={rot} decode={decode}")
    with torch.inference_mode():
        m = cie.step_maps(slot_ids, n_new, a.lens, a.block_table, 16, T)
        meta = cie.AttentionMetadata(token_count=T, full_decode=decode, device=DEV)
        meta.slot_ids, meta.cu_seqlens, meta.pages, meta.offsets = slot_ids, m.cu_seqlens, m.pages, m.offsets
        meta.adapter_plan = cie.adapter_plan(m.slots, by_slot, 2)
        emb = ours.model.rotary_emb(hidden, m.positions[None])
        got, _ = layer(hidden, emb, kv_manager=a, metadata=meta)

        def adapted(y, x, bank):
            return cie.adapter_add_(y, x, bank.a, bank.b, bank.scales, bank.ranks, meta.adapter_plan, bank.slices)

        qkv = adapted(torch.nn.functional.linear(hidden, layer.qkv_weight, layer.qkv_bias), hidden, layer.qkv_adapters)
        q, k, v = qkv.view(1, T, -1, D).split((H_Q, H_KV, H_KV), 2)
        if rot:
            q, k = cie.apply_rotary(q, k, m.positions, freqs, **how)
        else:
            cos, sin = cie.rotary_tables(m.positions, freqs, **how)
        cache = (b.keys[1], b.values[1]) + ((b.scales[1],) if b.scales else ())
        f8 = "_q8" if b.scales else ""
        call = lambda name, *args, **kw: getattr(cie, name + f8)(*args, **kw)  # noqa: E731
        prior = b.lens[slot_ids]
        if decode and rot:
            o = call("decode_append_gqa_attention", q, *cache, k, v, b.lens, slot_ids, b.block_table)
        elif decode:
            o = call("decode_qkv_rope_gqa_attention", qkv, cos, sin, *cache, b.lens, slot_ids, b.block_table, H_Q)
        else:
            if rot:
                b.mixed_update(1, m.pages, m.offsets, k, v)
            else:
                q = call("append_tokens_qkv_rope", qkv, cos, sin, *cache, m.pages, m.offsets, H_Q)
            o = call("mixed_gqa_attention", q, *cache, T, m.cu_seqlens, prior, slot_ids, b.block_table)
        o = o.reshape(1, T, H_Q * D)
        want = adapted(layer.original.o_proj(o), o, layer.o_adapters)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    for x, y in zip((a.keys[1], a.values[1]), (b.keys[1], b.values[1])):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert a.scales is None or torch.equal(a.scales[1], b.scales[1])


def test_frequencies_keep_their_type():
    """A model that is cast after use_rotary keeps 64-bit frequencies."""
    _, ours = _models(_config())
    freqs, scale = cie.rotary_frequencies(D, 1e6)
    use_rotary(ours, freqs, scale)
    ours.half()
    assert ours.model.rotary_emb.frequencies.dtype == torch.float64
    assert torch.equal(ours.model.rotary_emb.frequencies.cpu(), freqs)
