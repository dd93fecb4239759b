"""The framework's own paths on an 8-bit cache: the drop-in layer, the step modules, the Scheduler."""
import copy

import pytest
import torch
from transformers import Qwen2Config, Qwen2ForCausalLM

import custom_inference_engine_amd as cie
from custom_inference_engine_amd.scheduler import DecodeModule, FullMixedModule, MixedModule, Scheduler
from custom_inference_engine_amd.scheduler.scheduler import ModuleExecutor, batch_buckets, token_buckets
from oracle import paged_attention as paged
from oracle import q8_cache as ref
from tests.gpu_helpers import DEV, note

pytestmark = pytest.mark.gpu


def config(layers=2, h_q=14, h_kv=2, hidden=896):
    cfg = Qwen2Config(hidden_size=hidden, num_attention_heads=h_q, num_key_value_heads=h_kv, intermediate_size=512,
                      num_hidden_layers=layers, vocab_size=512, max_position_embeddings=4096, rope_theta=1e6,
                      tie_word_embeddings=True)
    cfg._attn_implementation = "sdpa"
    return cfg


def model_of(cfg, seed=0):
    torch.manual_seed(seed)
    model = Qwen2ForCausalLM(cfg).half().to(DEV).eval()
    cie.use_triton_attention(model)
    return model


def storage(cfg, page=16, tokens=512, slots=4, dtype=torch.float8_e4m3fn):
    kv = cie.KVStorage(cfg, max_cache_len=tokens, page_size=page, n_slots=slots, device=DEV, dtype=dtype)
    per = (kv.n_pages - 1) // (slots - 1)
    ids = 1 + torch.randperm(kv.n_pages - 1, generator=torch.Generator().manual_seed(3))
    for s in range(1, slots):
        kv.block_table[s, :per] = ids[(s - 1) * per:s * per]
    return kv


@pytest.mark.parametrize("fuse_append,fuse_rope", [(True, True), (True, False), (False, False)])
@pytest.mark.parametrize("h_q,h_kv,hidden", [(14, 2, 896), (8, 4, 1024)], ids=["d64", "d128"])
def test_layer_prefill_then_decode(native_lib, fuse_append, fuse_rope, h_q, h_kv, hidden):
    """A layer's two steps against projections, rotation, quantised cache and attention in 64 bits."""
    note(f"q8 layer {fuse_append} {fuse_rope} {h_q}")
    cfg = config(1, h_q, h_kv, hidden)
    model = model_of(cfg)
    layer = model.model.layers[0].self_attn
    with torch.no_grad():
        layer.qkv_bias.copy_(torch.randn(layer.qkv_bias.shape, generator=torch.Generator().manual_seed(1)))
    layer.fuse_append, layer.fuse_rope = fuse_append, fuse_rope
    kv = storage(cfg)
    d = kv.head_dim
    caches = [ref.Q8Cache(p[0].cpu().float().double(), torch.zeros(kv.scales[0].shape[:3]).double())
              for p in (kv.keys, kv.values)]
    g = torch.Generator().manual_seed(2)
    prior = [0, 0]
    for new, decode in (([37, 20], False), ([1, 1], True), ([1, 1], True)):
        T = sum(new)
        hidden_states = torch.randn(1, T, hidden, generator=g).half()
        pos = torch.cat([torch.arange(p, p + n) for p, n in zip(prior, new)])
        seq = torch.cat([torch.full((n,), b) for b, n in enumerate(new)])
        meta = cie.AttentionMetadata(token_count=T, full_decode=decode, device=DEV)
        meta.prepare_full_graph(2)
        meta.write_slot_ids([1, 2])
        meta.write_cu_seqlens([0, new[0], T])
        pages = kv.block_table.cpu()[1 + seq, pos // 16]
        meta.write_pages(pages)
        meta.write_offsets(pos % 16)
        cos, sin = model.model.rotary_emb(hidden_states.to(DEV), pos[None].to(DEV))
        with torch.inference_mode():
            out, _ = layer(hidden_states.to(DEV), (cos, sin), kv_manager=kv, metadata=meta)
            qkv = torch.nn.functional.linear(hidden_states.to(DEV), layer.qkv_weight, layer.qkv_bias).cpu()
            kv.mixed_advance(torch.tensor([1, 2], device=DEV), torch.tensor(new, device=DEV))
        q, k, v = qkv[0].split(layer.qkv_sizes, -1)
        q, k, v = (x.reshape(T, -1, d) for x in (q, k, v))
        if fuse_rope:
            q, k = paged.rope(q, cos[0].cpu(), sin[0].cpu()), paged.rope(k, cos[0].cpu(), sin[0].cpu())
        else:  # HF's rotation, in fp16 steps
            from transformers.models.qwen2.modeling_qwen2 import apply_rotary_pos_emb
            q, k = (x[0].cpu() for x in apply_rotary_pos_emb(q[None].to(DEV), k[None].to(DEV), cos, sin,
                                                             unsqueeze_dim=2))
        for c, x in zip(caches, (k, v)):
            c.append(x, pages, pos % 16)
        seqs = [(0, new[0], 1, prior[0] + 1), (new[0], new[1], 2, prior[1] + 1)]
        o, mass, top = ref.attend(q, *caches, seqs, kv.block_table)
        w = layer.original.o_proj.weight.cpu().double()
        want = o.reshape(T, -1) @ w.T
        # the attention's tolerance through |w|, the product's fp16 rounding and fp32 sums
        tol = ref.tolerance(o, mass, top, 64).reshape(T, -1) @ w.abs().T
        tol += 2.0 ** -11 * want.abs() + 1e-5 * (o.reshape(T, -1).abs() @ w.abs().T) + 2.0 ** -25
        assert ((out[0].cpu().double() - want).abs() <= tol).all()
        got_k, got_v = kv.read_tokens(0, pages.to(DEV), (pos % 16).to(DEV))
        for x, c in zip((got_k, got_v), caches):
            assert torch.equal(x[0].cpu().double(), c.values()[pages, :, pos % 16])
        prior = [p + n for p, n in zip(prior, new)]


def test_step_modules_replay_is_eager(native_lib):
    """FullMixedModule's graph against MixedModule's eager step, then DecodeModule's graph against an eager step:
    logits, pools and scales, bit for bit, over several steps."""
    note("q8 step modules")
    cfg = config()
    model = model_of(cfg)
    a, b = storage(cfg), storage(cfg)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (50, 9, 77)]
    graph, eager = FullMixedModule(model, a, batch_size=3, token_count=96), MixedModule(model, b, token_count=96)

    def same():
        torch.cuda.synchronize()
        for x, y in zip(a.keys + a.values, b.keys + b.values):  # (page 0 holds padding rows)
            assert torch.equal(x.view(torch.uint8)[1:], y.view(torch.uint8)[1:])
        for x, y in zip(a.scales, b.scales):
            assert torch.equal(x[1:], y[1:])
        assert torch.equal(a.lens, b.lens)

    for chunk in ([p[:30] for p in prompts], [prompts[0][30:], None, prompts[2][30:]]):
        feed = [(c, s) for c, s in zip(chunk, (1, 2, 3)) if c]
        t1 = graph.forward([c for c, _ in feed], [s for _, s in feed])
        t2 = eager.forward([c for c, _ in feed], [s for _, s in feed])
        assert t1 == t2 and torch.equal(graph.last_logits, eager.last_logits)
        same()
    module = DecodeModule(model, a, batch_size=4)
    other = DecodeModule(model, b, batch_size=4)
    for step in range(20):  # past a block's border in every slot
        t1 = module.forward([1, 2, 3])
        with torch.inference_mode():
            other.upload([1, 2, 3])
            logits = other._step()[:3]
            t2 = torch.argmax(logits, -1)
            b.last_generated[other.slots[:3]] = t2
        assert t1 == t2.tolist() and torch.equal(module.logits[:3], logits)
        same()


def test_scheduler_on_an_8_bit_cache(native_lib):
    """Requests served with preemption and page reuse: the graphs' tokens are the eager modules', every slot and
    page is released."""
    note("q8 scheduler")
    cfg = config()
    g = torch.Generator().manual_seed(11)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (60, 70, 50, 9, 64)]
    got = []
    for graphs in (True, False):
        model = model_of(cfg)
        kv = cie.KVStorage(cfg, max_cache_len=192, page_size=16, n_slots=4, device=DEV, dtype=torch.float8_e4m3fn)
        executor = None if graphs else ModuleExecutor(model, kv, batch_buckets(4), token_buckets(160), graph_mixed=False)
        sched = Scheduler(model, kv, eos_token_ids={512}, max_new_tokens=16, token_budget=160, executor=executor)
        with torch.inference_mode():
            res = sched.generate(prompts)
        assert sched.stats.preemptions == 2
        assert kv.lens.eq(0).all() and kv.block_table.eq(0).all()
        assert all(len(r.new_tokens) == 16 for r in res)
        got.append([r.new_tokens for r in res])
    assert got[0] == got[1]


def test_scheduler_piecewise_on_an_8_bit_cache(native_lib):
    """The piecewise backend cuts at the 8-bit attention: its tokens are the full graphs'."""
    note("q8 piecewise")
    torch._dynamo.reset()
    cfg = config()
    g = torch.Generator().manual_seed(12)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (150, 20, 10)]
    got = []
    for piecewise in (True, False):
        model = model_of(cfg)
        kv = cie.KVStorage(cfg, max_cache_len=1024, page_size=16, n_slots=4, device=DEV, dtype=torch.float8_e4m3fn)
        sched = Scheduler(model, kv, eos_token_ids={512}, max_new_tokens=4, token_budget=192, piecewise_mixed=piecewise)
        with torch.inference_mode():
            got.append([r.new_tokens for r in sched.generate(prompts)])
        if piecewise:
            used = [sched.executor.mixed_modules[t] for t in sched.stats.mixed_steps if t > 128]
            assert used and all(m.backend.compiles == 1 and m.backend.piece_replays > 0 for m in used)
    assert got[0] == got[1]


def test_compiled_layer_is_eager(native_lib):
    """torch.compile(fullgraph=True) of a decode and a mixed step on an 8-bit cache."""
    note("q8 compiled layer")
    torch._dynamo.reset()
    cfg = config(1)
    model = model_of(cfg)
    layer = model.model.layers[0].self_attn
    for decode in (False, True):
        T = 2 if decode else 6
        outs = []
        for compiled in (False, True):
            kv = storage(cfg)
            kv.lens[1], kv.lens[2] = 5, 9
            meta = cie.AttentionMetadata(token_count=T, full_decode=decode, device=DEV)
            meta.prepare_full_graph(2)
            meta.write_slot_ids([1, 2])
            meta.write_cu_seqlens([0, 1, 2] if decode else [0, 4, 6])
            pos = torch.tensor([5, 9] if decode else [5, 6, 7, 8, 9, 10])
            seq = torch.tensor([1, 2] if decode else [1] * 4 + [2] * 2)
            meta.write_pages(kv.block_table.cpu()[seq, pos // 16])
            meta.write_offsets(pos % 16)
            x = torch.randn(1, T, 896, generator=torch.Generator().manual_seed(1)).half().to(DEV)
            pe = model.model.rotary_emb(x, pos[None].to(DEV))

            def fn(x, cos, sin):
                return layer(x, (cos, sin), kv_manager=kv, metadata=meta)[0]

            if compiled:
                fn = torch.compile(fn, backend="aot_eager", fullgraph=True)
            with torch.inference_mode():
                outs.append([fn(x, *pe), kv.keys[0].view(torch.uint8), kv.values[0].view(torch.uint8), kv.scales[0]])
        for a, b in zip(*outs):
            assert torch.equal(a, b)
