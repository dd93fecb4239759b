"""Free lists after calls whose pages they did not have: what holds no page is not given back."""
import random

import pytest
import torch

import custom_inference_engine_amd as cie
from oracle import step as ref
from tests.gpu_helpers import DEV, err_word
from tests.test_gpu_step_maps import FREE, PAGE, Pool

pytestmark = pytest.mark.gpu


def whole(pool):
    """The list's pages and the tables', each page of the pool once."""
    held = [p for s, n in enumerate(pool.lens) for p in pool.table[s][:-(-n // pool.page)]]
    words = pool.d_free.tolist()
    assert sorted(words[2:2 + words[0]] + held) == list(range(1, pool.n_pages))


@pytest.mark.parametrize("held,new,free", [([16, 16, 5], [1, 1, 1], 1), ([60, 30], [70, 1], 3), ([0], [40], 2), ([3] * 40, [30] * 40, 79)])
def test_a_turn_that_was_refused(held, new, free):
    """Maps whose pages run short, then the release of what they were to give: the list, the tables and the lengths are as
    before, and the next turn is served from pages that no other holds."""
    need = sum(-(-h // 16) for h in held)
    pool = Pool(held, 16, 1 + need + free)
    slots = list(range(len(held), 0, -1))
    h, n = held[::-1], new[::-1]
    before = pool.d_free.clone(), pool.d_table.clone(), pool.d_lens.clone()
    for _ in range(2):
        assert not pool.step(slots, n, sum(n), True)
        err = err_word()
        pool.release(slots, keep=h, held=[a + b for a, b in zip(h, n)], err=err)
        # (pages that were never given: reported, or refused where they are more than the list has room for)
        assert int(err) in (PAGE, FREE)
        for a, b in zip(before, (pool.d_free, pool.d_table, pool.d_lens)):
            assert torch.equal(a[:2 + int(before[0][0])] if a.dim() == 1 and a.numel() == pool.n_pages + 2 else a,
                               b[:2 + int(before[0][0])] if b.dim() == 1 and b.numel() == pool.n_pages + 2 else b)
    assert pool.step(slots[-1:], [1], 1, True)
    pool.lens[slots[-1]] += 1
    pool.up()
    whole(pool)


@pytest.mark.parametrize("n_pages", [60, 9000, 70000])
def test_gaps_are_closed(n_pages):
    """Tables with entries that hold no page at their ends, between others and everywhere: what is left keeps its order,
    in pools of one, some and many workgroups' releases."""
    r = random.Random(n_pages)
    each = (n_pages - 10) // 3
    pool = Pool([each * 16 - 3, each * 16, 16 * (each // 2), 0], 16, n_pages, slots=6)
    for i in range(each):
        if i >= each - 5 or i % 7 == 3:
            pool.table[1][i] = 0
        if r.random() < 0.5:
            pool.table[2][i] = 0
    for i in range(each // 2):
        pool.table[3][i] = 0
    pool.up()
    err = err_word()
    assert pool.release([3, 1, 4, 2], keep=[0, 20, 0, 0], err=err)
    assert int(err) == PAGE
    words = pool.d_free.tolist()
    assert words[1] == 0 and len(set(words[2:2 + words[0]])) == words[0] and min(words[2:2 + words[0]]) > 0
    assert pool.step([3], [64], 64, True)
    err = err_word()
    assert pool.release([3, 1], held=[64, 20], err=err) and int(err) == 0


def test_gaps_in_a_graph():
    """A turn that is refused in one replay and served in the next."""
    pool = Pool([16, 16], 16, 8, free=1)
    slots, new, keep = torch.tensor([1, 2], device=DEV), torch.tensor([5, 1], device=DEV), torch.tensor([16, 16], device=DEV)
    held = keep + new

    def turn():
        maps = cie.step_maps(slots, new, pool.d_lens, pool.d_table, 16, 6, free_list=pool.d_free)
        cie.release_pages(pool.d_free, slots, pool.d_lens, pool.d_table, 16, keep=keep, held=held)
        return maps

    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        maps = turn()
    for n in ([5, 1], [5, 0], [5, 1], [0, 3]):
        new.copy_(torch.tensor(n))
        held.copy_(keep + new)
        graph.replay()
        torch.cuda.synchronize()
        _, rows, _ = ref.step_maps([1, 2], n, pool.lens, pool.table, 16, 6, pool.free)
        ref.release_pages(pool.free, [1, 2], pool.lens, pool.table, 16, [16, 16], held.tolist())
        assert torch.stack(maps[1:], 1).tolist() == [list(x) for x in rows]
        pool.same()
        assert pool.free.count == 1
