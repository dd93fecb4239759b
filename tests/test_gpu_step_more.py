"""Steps that are refused, and state that is turned on twice or late, through the step modules and the scheduler on a
small Qwen2."""
import pytest
import torch

import custom_inference_engine_amd as cie
from custom_inference_engine_amd import KVStorage, use_adapters, use_rotary
from custom_inference_engine_amd.scheduler import DecodeModule, FullMixedModule, MixedModule, PiecewiseMixedModule, Scheduler
from tests.gpu_helpers import DEV, note
from tests.test_gpu_step import D, H_KV, H_Q, _adapters, _config, _logits, _models, _prompts, _rel

pytestmark = pytest.mark.gpu


def _pool(cfg, pages=6, managed=True, slots=5):
    kv = KVStorage(cfg, max_cache_len=pages * 16, page_size=16, n_slots=slots, device=DEV, dtype=torch.float16)
    if managed:
        kv.manage_pages()
    return kv


def _state(kv):
    words = kv.free_list.tolist()
    return kv.lens.tolist(), kv.block_table.tolist(), words[:2 + words[0]], kv.last_generated.tolist()


def _whole(kv):
    """Each page of the pool is held by one slot, or free, once."""
    held = [p for s, n in enumerate(kv.lens.tolist()) for p in kv.block_table[s, :-(-n // 16)].tolist()]
    words = kv.free_list.tolist()
    assert words[1] == 0 and sorted(words[2:2 + words[0]] + held) == list(range(1, kv.n_pages))


@pytest.mark.parametrize("kind", ["eager", "graph", "piecewise"])
def test_a_refused_step_changes_nothing(native_lib, kind):
    """A mixed step and a decode step that find too few pages leave lengths, tables, list and last tokens as they were;
    their slots are reset like any other, and what then runs is what runs in a pool that never refused a step."""
    torch._dynamo.reset()
    cfg = _config()
    _, ours = _models(cfg)

    def modules(kv):
        if kind == "graph":
            mix = FullMixedModule(ours, kv, batch_size=4, token_count=64)
        elif kind == "piecewise":
            mix = PiecewiseMixedModule(ours, kv, token_count=64,
                                       buffer=torch.zeros(1, 64, H_Q, D, dtype=torch.float16, device=DEV))
        else:
            mix = MixedModule(ours, kv, token_count=64)
        return mix, DecodeModule(ours, kv, batch_size=2)

    kv, other = _pool(cfg), _pool(cfg)
    (mix, dec), (mix2, dec2) = modules(kv), modules(other)
    prompts = _prompts(32, 31, 20, 17)
    note(f"refused steps: {kind}")
    for m in (mix, mix2):
        m.forward(prompts[:2], [1, 2])  # four of five pages
    for _ in range(2):
        before = _state(kv)
        for chunks, slots in ((prompts[2:3], [3]), ([[5], prompts[3], [6]], [2, 3, 1])):
            with pytest.raises(RuntimeError, match="free pages"):
                mix.forward(chunks, slots)
            assert _state(kv) == before
        kv.reset([3])
        assert _state(kv) == before
        kv.check_pages()
    for d in (dec, dec2):  # slot 1 takes the last page, slot 2 needs none yet
        d.forward([1, 2])
    assert _state(kv) == _state(other)
    before = _state(kv)
    with pytest.raises(RuntimeError, match="free pages"):
        dec.forward([2])  # its 33rd token
    assert _state(kv) == before
    for pool in (kv, other):
        pool.reset([1])
        _whole(pool)
    assert int(kv.free_list[0]) == 3
    for _ in range(3):
        got, want = dec.forward([2]), dec2.forward([2])
        assert got == want and torch.equal(dec.logits[0], dec2.logits[0])
    assert mix.forward([prompts[2]], [3]) == mix2.forward([prompts[2]], [3])
    assert torch.equal(mix.last_logits, mix2.last_logits) and _state(kv) == _state(other)
    _whole(kv)


def test_a_step_that_some_sequences_cannot_take(native_lib):
    """One sequence would run past its table's row while another gets a page: nothing is kept, and the page is free again."""
    cfg = _config()
    _, ours = _models(cfg)
    kv = _pool(cfg, pages=5)
    mix, dec = MixedModule(ours, kv, token_count=96), DecodeModule(ours, kv, batch_size=2)
    note("a sequence past its table's row")
    mix.forward([[3] * 16], [1])
    kv.lens[2] = 80  # (a slot that a caller has set beyond its pages)
    before = _state(kv)
    with pytest.raises(RuntimeError, match="lengths"):
        mix.forward([[1], [2] * 20, [4]], [2, 3, 1])
    assert _state(kv) == before
    with pytest.raises(RuntimeError, match="lengths"):
        dec.forward([1, 2])
    assert _state(kv) == before
    kv.lens[2] = 0
    dec.forward([1])
    assert kv.lens.tolist() == [0, 17, 0, 0, 0] and int(kv.free_list[0]) == 2
    _whole(kv)


@pytest.mark.parametrize("kind", ["eager", "graph"])
def test_a_pool_whose_tables_the_caller_keeps_reports_too(native_lib, kind):
    """A sequence past its table's row stops a mixed step with an error, and leaves the pool as it was."""
    cfg = _config()
    _, ours = _models(cfg)
    kv = _pool(cfg, pages=4, managed=False)
    mix = FullMixedModule(ours, kv, batch_size=3, token_count=32) if kind == "graph" else MixedModule(ours, kv, token_count=32)
    kv.block_table[1, :2], kv.block_table[2, 0] = torch.tensor([1, 3], device=DEV), 2
    note(f"past the table's row: {kind}")
    first = mix.forward([[5] * 7, [6] * 9], [1, 2])
    kv.lens[1] = 60
    before = kv.lens.clone(), kv.last_generated.clone()
    with pytest.raises(RuntimeError, match="lengths"):
        mix.forward([[1] * 5, [2]], [1, 2])
    assert torch.equal(kv.lens, before[0]) and torch.equal(kv.last_generated, before[1])
    kv.lens[1], kv.lens[2] = 0, 0
    assert mix.forward([[5] * 7, [6] * 9], [1, 2]) == first and kv.lens.tolist() == [0, 7, 9, 0, 0]


def test_adapters_that_do_not_fit_are_reported(native_lib):
    """A bank of other adapters than the step's plan, by the op and through a layer; a slot's adapter past the last one,
    in mixed and decode steps: an error, and no step is counted."""
    cfg = _config()
    _, ours = _models(cfg)
    kv = _pool(cfg, pages=8, managed=False)
    layers = use_adapters(ours, kv, 3, 16)
    kv.block_table[1, :2] = torch.tensor([1, 2], device=DEV)
    mix, dec = MixedModule(ours, kv, token_count=32), DecodeModule(ours, kv, batch_size=2)
    kv.slot_adapters[1] = 1
    note("adapters that do not fit")
    mix.forward([[1] * 9], [1])
    kv.slot_adapters[1] = 3
    for step in (lambda: mix.forward([[1] * 9], [1]), lambda: dec.forward([1])):
        last = kv.last_generated.clone()
        with pytest.raises(RuntimeError, match="adapters"):
            step()
        assert kv.lens.tolist() == [0, 9, 0, 0, 0] and torch.equal(kv.last_generated, last)
    kv.slot_adapters[1] = 1
    dec.forward([1])
    assert kv.lens.tolist() == [0, 10, 0, 0, 0]
    other = cie.AdapterBank(2, 16, 896, 896, dtype=torch.float16, device=DEV)
    x, y, err = torch.ones(1, 5, 896).half().to(DEV), torch.ones(1, 5, 896).half().to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    plan = cie.adapter_plan(None, torch.zeros(5, dtype=torch.int64, device=DEV), 300)
    other.add_(y, x, plan, err)
    assert int(err) == 16 and (y == 1).all()
    layers[0].o_adapters = other
    with pytest.raises(RuntimeError, match="adapters"):
        mix.forward([[1] * 9], [1])
    assert kv.lens.tolist() == [0, 10, 0, 0, 0]


def test_pages_and_adapters_turned_on_late(native_lib):
    """Modules and schedulers made before: their steps are refused, and a scheduler takes no request whose adapter its
    graphs would leave out."""
    cfg = _config()
    _, ours = _models(cfg)
    kv = _pool(cfg, pages=16, managed=False)
    sched = Scheduler(ours, kv, eos_token_ids={512}, max_new_tokens=4, token_budget=160)
    mix, dec = MixedModule(ours, kv, token_count=32), DecodeModule(ours, kv, batch_size=2)
    kv.use_adapters(2)
    future = sched.call([1, 2, 3], adapter=1)
    assert future.done() and isinstance(future.exception(), ValueError)
    for step in (lambda: mix.forward([[1, 2]], [1]), lambda: dec.forward([1])):
        with pytest.raises(RuntimeError, match="before the step modules"):
            step()
    assert not kv.lens.any()
    kv = _pool(cfg, pages=16, managed=False)
    mix, dec = FullMixedModule(ours, kv, batch_size=2, token_count=32), DecodeModule(ours, kv, batch_size=2)
    kv.manage_pages()
    for step in (lambda: mix.forward([[1, 2]], [1]), lambda: dec.forward([1])):
        with pytest.raises(RuntimeError, match="before the step modules"):
            step()
    assert not kv.lens.any()


def test_turned_on_twice_under_graphs(native_lib):
    """Graphs recorded between two calls of manage_pages and use_adapters go on with the pool's own words."""
    cfg = _config()
    theirs, ours = _models(cfg)
    kv = _pool(cfg, pages=16)
    layers = use_adapters(ours, kv, 2, 16)
    mix, dec = FullMixedModule(ours, kv, batch_size=2, token_count=32), DecodeModule(ours, kv, batch_size=2)
    note("turned on twice")
    kv.manage_pages()
    assert use_adapters(ours, kv, 2, 16) == layers
    merged = _adapters(layers, 2, 16, seed=6)
    prompt = _prompts(20)[0]
    kv.slot_adapters[2] = 1
    nxt = mix.forward([prompt], [2])
    assert _rel(mix.last_logits[0], _logits(merged(theirs, 1), prompt)) < 2e-2
    dec.forward([2])
    assert _rel(dec.logits[0], _logits(merged(theirs, 1), prompt + nxt)) < 2e-2
    assert int(kv.free_list[0]) == 13
    _whole(kv)
    kv.reset([2])
    assert int(kv.free_list[0]) == 15


def test_the_wrapped_modules_path_after_use_rotary(native_lib):
    """A model that is called without a cache, on one row of tokens and on several (padded or not): as before use_rotary,
    up to the tables' rounding."""
    cfg = _config()
    _, ours = _models(cfg)
    g = torch.Generator().manual_seed(1)
    calls = [dict(input_ids=torch.randint(0, 512, (b, n), generator=g).to(DEV)) for b, n in ((1, 7), (3, 7), (2, 1))]
    mask = torch.ones(3, 7, dtype=torch.int64, device=DEV)
    mask[1, :4] = 0
    calls.append(dict(calls[1], attention_mask=mask, position_ids=(mask.cumsum(1) - 1).clamp(min=0)))
    with torch.inference_mode():
        want = [ours(**c, use_cache=False).logits for c in calls]
        use_rotary(ours, *cie.rotary_frequencies(D, 1e6))
        note("the wrapped modules' path")
        for c, w in zip(calls, want):
            got = ours(**c, use_cache=False).logits
            assert got.shape == w.shape and _rel(got, w.float().cpu()) < 2e-2
        rows = torch.tensor([[0, 1, 2], [70000, 5, 9]], device=DEV)
        cos, sin = ours.model.rotary_emb(want[0], rows)
        for t, one in ((cos, 0), (sin, 1)):
            assert t.shape == (2, 3, D)
            assert torch.equal(t, torch.cat([cie.rotary_tables(r, ours.model.rotary_emb.frequencies)[one] for r in rows]))


@pytest.mark.parametrize("kind", ["decode", "graph", "piecewise", "eager"])
def test_other_positions_after_a_module_was_made(native_lib, kind):
    """Recorded steps keep the frequencies that they read and are refused; an eager module turns by the new ones."""
    torch._dynamo.reset()
    cfg = _config()
    theirs, ours = _models(cfg)
    kv = _pool(cfg, pages=16)
    use_rotary(ours, *cie.rotary_frequencies(D, 1e4))
    mix = MixedModule(ours, kv, token_count=32)
    if kind == "decode":
        made = DecodeModule(ours, kv, batch_size=1)
    elif kind == "graph":
        made = FullMixedModule(ours, kv, batch_size=2, token_count=32)
    elif kind == "piecewise":
        made = PiecewiseMixedModule(ours, kv, token_count=32, buffer=torch.zeros(1, 32, H_Q, D, dtype=torch.float16, device=DEV))
    first = ours.model.rotary_emb.frequencies.data_ptr()
    use_rotary(ours, *cie.rotary_frequencies(D, 1e6))
    note(f"other positions: {kind}")
    prompt = _prompts(20)[0]
    nxt = mix.forward([prompt], [1])
    assert _rel(mix.last_logits[0], _logits(theirs, prompt)) < 2e-2
    if kind == "eager":
        return
    assert made.rotary_emb.frequencies.data_ptr() == first
    lens = kv.lens.clone()
    with pytest.raises(RuntimeError, match="use_rotary"):
        made.forward([1]) if kind == "decode" else made.forward([nxt], [1])
    assert torch.equal(kv.lens, lens)
