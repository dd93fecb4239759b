"""Block tables and slot maps on the GPU against plain loops: every word, and what the free list holds after."""
import random

import pytest
import torch

import custom_inference_engine_amd as cie
from oracle import step as ref
from tests.gpu_helpers import DEV, err_word, note

pytestmark = pytest.mark.gpu
PAGE, LEN, FREE = 1, 2, 32


class Pool:
    """Slots with their pages anywhere in the pool, and the free pages in any order."""

    def __init__(self, held, page, n_pages, seed=0, slots=None, free=None):
        r = random.Random(seed)
        need = [-(-h // page) for h in held]
        ids = r.sample(range(1, n_pages), n_pages - 1)
        n_slots = slots or len(held) + 1
        self.page, self.n_pages = page, n_pages
        self.lens = [0] * n_slots
        self.table = [[0] * n_pages for _ in range(n_slots)]
        at = 0
        for s, (h, n) in enumerate(zip(held, need), 1):
            self.lens[s] = h
            self.table[s][:n] = ids[at:at + n]
            at += n
        stack = ids[at:] if free is None else ids[at:at + free]
        self.free = ref.FreeList([len(stack), 0] + stack + [0] * (n_pages - len(stack)))
        self.up()

    def up(self):
        self.d_lens, self.d_table, self.d_free = (torch.tensor(x, dtype=torch.int64, device=DEV)
                                                  for x in (self.lens, self.table, self.free.words()))

    def step(self, slots, new, T, managed, err=None):
        note(f"step_maps B={len(slots)} T={T} managed={managed}")
        got = cie.step_maps(torch.tensor(slots, dtype=torch.int64, device=DEV),
                            torch.tensor(new, dtype=torch.int64, device=DEV), self.d_lens, self.d_table, self.page, T,
                            free_list=self.d_free if managed else None, err=err)
        cu, rows, served = ref.step_maps(slots, new, self.lens, self.table, self.page, T, self.free if managed else None)
        assert got.cu_seqlens.tolist() == cu
        assert torch.stack(got[1:], 1).tolist() == [list(x) for x in rows]
        self.same()
        return served

    def release(self, slots, keep=None, held=None, err=None):
        note(f"release_pages B={len(slots)}")
        up = lambda x: None if x is None else torch.tensor(x, dtype=torch.int64, device=DEV)  # noqa: E731
        cie.release_pages(self.d_free, up(slots), self.d_lens, self.d_table, self.page, keep=up(keep), held=up(held), err=err)
        done = ref.release_pages(self.free, slots, self.lens, self.table, self.page, keep, held)
        self.same()
        return done

    def same(self):
        assert self.d_lens.tolist() == self.lens
        assert self.d_free.tolist() == self.free.words()
        assert self.d_table.tolist() == self.table


@pytest.mark.parametrize("managed", [False, True])
@pytest.mark.parametrize("held,new,page,pad", [
    ([1000], [1], 16, 0), ([0], [1], 16, 0), ([15, 16, 17], [1, 1, 1], 16, 1), ([0, 31, 32, 33], [33, 1, 1, 0], 32, 7),
    ([5, 0, 100, 64], [300, 1, 17, 1], 16, 100), ([0], [1], 1, 0), ([3] * 40, [4] * 40, 7, 0), ([0, 0, 0], [0, 0, 0], 16, 5),
    ([100] * 300, [1] * 300, 64, 3), (list(range(257)), [1 + i % 5 for i in range(257)], 16, 0),
])
def test_maps(managed, held, new, page, pad):
    pages = 2 + sum(-(-(h + n) // page) for h, n in zip(held, new))
    pool = Pool(held, page, pages)
    slots = list(range(1, len(held) + 1))
    random.Random(1).shuffle(slots)
    new = [new[s - 1] for s in slots]
    if not managed:  # the tables hold the new tokens' pages already
        ref.step_maps(slots, new, pool.lens, pool.table, page, sum(new), pool.free)
        pool.up()
    err = err_word()
    assert pool.step(slots, new, sum(new) + pad, managed, err)
    assert int(err) == 0


def test_many_rows_and_sequences():
    """More rows than the grid's threads, and the most sequences of a call."""
    r = random.Random(3)
    held = [r.randrange(40) for _ in range(2047)]
    new = [r.choice((0, 1, 1, 90)) for _ in held]
    pool = Pool(held, 16, 1 + sum(-(-(h + n) // 16) for h, n in zip(held, new)))
    err = err_word()
    assert pool.step(list(range(1, 2048)) + [0], new + [3], sum(new) + 70000, True, err)
    assert int(err) == 0 and pool.free.count == 0
    assert pool.release(list(range(1, 2048)) + [0], keep=held + [0], held=[h + n for h, n in zip(held, new)] + [0], err=err)
    assert int(err) == 0
    assert pool.release(list(range(2047, 0, -1)), err=err) and pool.free.count == pool.n_pages - 1
    assert int(err) == 0 and not any(pool.lens)


def test_padding_entries():
    """Padded sequences (slot 0, no tokens), and decode buckets (slot 0, a token each): page 0, and no page taken."""
    pool = Pool([16, 3], 16, 8)
    err = err_word()
    assert pool.step([1, 2, 0, 0], [1, 1, 0, 0], 4, True, err)
    assert pool.step([0, 2, 0, 0], [1, 1, 1, 1], 4, True, err)
    assert int(err) == 0 and pool.free.count == 4


@pytest.mark.parametrize("B", [1, 3, 40, 500])
def test_giving_back_undoes_taking(B):
    held = [(7 * b) % 50 for b in range(B)]
    new = [1 + (11 * b) % 60 for b in range(B)]
    pool = Pool(held, 16, 3 + sum(-(-(h + n) // 16) for h, n in zip(held, new)))
    before = pool.d_free.clone(), pool.d_table.clone(), pool.d_lens.clone()
    slots = list(range(B, 0, -1))
    h, n = held[::-1], new[::-1]
    for _ in range(3):
        assert pool.step(slots, n, sum(new), True)
        assert pool.release(slots, keep=h, held=[a + b for a, b in zip(h, n)])
        for a, b in zip(before, (pool.d_free, pool.d_table, pool.d_lens)):
            assert torch.equal(a, b)
    assert pool.step(slots, n, sum(new), True)
    assert pool.release(slots, keep=[a + 1 for a in h], held=[a + b for a, b in zip(h, n)])  # a token of each stays


def test_too_few_pages_gives_none():
    pool = Pool([16, 16, 5], 16, 20, free=1)
    err = err_word()
    assert not pool.step([1, 2, 3], [1, 1, 1], 3, True, err)
    assert int(err) == FREE
    assert pool.step([3, 2], [1, 1], 2, True)  # one page is enough for these
    assert pool.free.count == 0


def test_a_slot_twice():
    pool = Pool([16, 5], 16, 20)
    err = err_word()
    assert not pool.step([1, 2, 1], [1, 1, 1], 3, True, err)
    assert int(err) == FREE
    err = err_word()
    assert not pool.release([1, 2, 1], err=err)
    assert int(err) == FREE
    assert pool.step([1, 2, 1], [1, 1, 0], 3, True)  # without tokens it may
    pool = Pool([16, 5], 16, 20)
    assert pool.step([1, 2, 1], [1, 1, 0], 2, False)  # and where nothing is taken


def test_giving_back_twice_is_refused_or_empty():
    pool = Pool([40, 20], 16, 6)  # a full pool but for none
    err = err_word()
    assert pool.release([1, 2], err=err) and pool.free.count == 5
    assert pool.release([1, 2], err=err) and int(err) == 0  # the slots are empty
    assert not pool.release([1], held=[16], err=err)  # the list holds every page
    assert int(err) == FREE


@pytest.mark.parametrize("managed", [False, True])
def test_bad_slots_counts_and_lengths(managed):
    pool = Pool([20, 5], 16, 4, slots=5)
    err = err_word()
    pool.step([1, 9, 2, -1], [1, 2, 1, 2], 8, managed, err)
    assert int(err) == PAGE
    err = err_word()
    pool.step([1, 2], [-3, 2], 4, managed, err)
    assert int(err) == LEN
    err = err_word()
    pool.step([1, 2], [2, 5], 4, managed, err)  # past the rows
    assert int(err) == LEN
    pool.lens[3], pool.lens[4] = 63, -2
    pool.up()
    err = err_word()
    pool.step([3, 4, 2], [3, 4, 1], 8, managed, err)  # past the table's row, and before it
    assert int(err) == LEN


@pytest.mark.parametrize("page", [1, 16, 1 << 30])
@pytest.mark.parametrize("new", [1, 3])
def test_any_word_as_a_length(page, new):
    """A length whose sum with the new tokens passes 63 bits takes no page and writes no table entry."""
    lens = torch.tensor([0, (1 << 63) - 1, 2], device=DEV)
    table = torch.full((3, 8), 5, device=DEV)
    free, err = cie.new_free_list(8, DEV), err_word()
    got = cie.step_maps(torch.tensor([1, 2], device=DEV), torch.tensor([new, 1], device=DEV), lens, table, page, new + 1,
                        free_list=free, err=err)
    assert int(err) == LEN and got.pages.tolist()[:new] == [0] * new and got.offsets.tolist()[:new] == [0] * new
    assert int(free[0]) == (6 if page == 1 else 7)  # (the other sequence's, where it needs one)
    table[2, 2 // page] = 5
    assert bool((table == 5).all())


def test_release_of_bad_sequences_leaves_them():
    pool = Pool([20, 5, 33], 16, 8, slots=6)
    err = err_word()
    assert pool.release([9, 1, -1, 0], err=err)
    assert int(err) == PAGE
    err = err_word()
    assert pool.release([2, 3], keep=[6, 33], err=err)  # more than it holds
    assert int(err) == LEN
    err = err_word()
    assert pool.release([2, 3], keep=[0, 0], held=[4, 500], err=err)  # fewer than lens, more than the table's row
    assert int(err) == LEN


def test_bad_page_ids_come_out_as_page_0():
    pool = Pool([20], 16, 6)
    pool.table[1][1] = 77
    pool.up()
    err = err_word()
    assert pool.release([1], err=err)
    assert int(err) == PAGE and pool.free.count == 5
    pool.d_free[pool.free.count - 1 + 2] = 99  # the stack's top
    pool.free.stack[-1] = pool.free.rest[pool.free.count - 1] = 99
    err = err_word()
    got = cie.step_maps(torch.tensor([1], device=DEV), torch.tensor([2], device=DEV), pool.d_lens, pool.d_table, 16, 2,
                        free_list=pool.d_free, err=err)
    assert int(err) == PAGE and got.pages.tolist() == [0, 0] and got.offsets.tolist() == [0, 1]
    assert pool.d_table[1, 0] == 0 and pool.d_free[0] == 4


def test_positions_past_32_bits():
    """A page of 2^30 tokens: positions and offsets are 64-bit words."""
    held = [5 * (1 << 30) + 7, 3]
    lens = torch.tensor([0] + held, device=DEV)
    table = torch.arange(3 * 8, device=DEV).view(3, 8)
    got = cie.step_maps(torch.tensor([2, 1], device=DEV), torch.tensor([2, 3], device=DEV), lens, table, 1 << 30, 5)
    assert got.positions.tolist() == [3, 4] + [held[0] + i for i in range(3)]
    assert got.pages.tolist() == [16, 16, 13, 13, 13] and got.offsets.tolist() == [3, 4, 7, 8, 9]


def test_strided_table_and_other_index_types():
    pool = Pool([20, 40], 16, 9)
    wide = torch.full((3, 20), -1, dtype=torch.int64, device=DEV)
    wide[:, :9] = pool.d_table
    cu, rows, _ = ref.step_maps([2, 1], [8, 3], pool.lens, pool.table, 16, 12)
    for table, kind in ((wide[:, :9], torch.int64), (pool.d_table.int(), torch.int32)):
        got = cie.step_maps(torch.tensor([2, 1], dtype=kind, device=DEV), torch.tensor([8, 3], dtype=kind, device=DEV),
                            pool.d_lens.to(kind), table, 16, 12)
        assert got.cu_seqlens.tolist() == cu and torch.stack(got[1:], 1).tolist() == [list(x) for x in rows]
    managed = wide[:, :9]
    got = cie.step_maps(torch.tensor([1, 2], device=DEV), torch.tensor([20, 10], device=DEV), pool.d_lens, managed, 16, 30,
                        free_list=pool.d_free)
    cu, rows, _ = ref.step_maps([1, 2], [20, 10], pool.lens, pool.table, 16, 30, pool.free)
    assert torch.stack(got[1:], 1).tolist() == [list(x) for x in rows]
    assert managed.tolist() == pool.table and (wide[:, 9:] == -1).all()


def test_another_stream_and_out():
    pool = Pool([20, 40], 16, 12)
    out = cie.StepMaps(torch.full((3,), -1, device=DEV), *(torch.full((12,), -1, device=DEV) for _ in range(4)))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = cie.step_maps(torch.tensor([2, 1], device=DEV), torch.tensor([8, 3], device=DEV), pool.d_lens, pool.d_table,
                            16, 12, free_list=pool.d_free, out=out)
    side.synchronize()
    assert got is out
    cu, rows, _ = ref.step_maps([2, 1], [8, 3], pool.lens, pool.table, 16, 12, pool.free)
    assert out.cu_seqlens.tolist() == cu and torch.stack(out[1:], 1).tolist() == [list(x) for x in rows]
    pool.same()


def test_captured_turns():
    """A turn in a graph: replayed between eager turns on the same free list, each as the loops say."""
    pool = Pool([20, 40, 7], 16, 30)
    slots, new = torch.tensor([2, 1, 3], device=DEV), torch.tensor([30, 3, 9], device=DEV)
    keep = torch.tensor([41, 20, 9], device=DEV)
    held = torch.tensor([70, 23, 16], device=DEV)

    def turn():
        maps = cie.step_maps(slots, new, pool.d_lens, pool.d_table, 16, 50, free_list=pool.d_free)
        cie.release_pages(pool.d_free, slots, pool.d_lens, pool.d_table, 16, keep=keep, held=held)
        return maps

    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        maps = turn()
    pool.same()  # (capturing runs nothing)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        s, n = slots.tolist(), new.tolist()
        cu, rows, _ = ref.step_maps(s, n, pool.lens, pool.table, 16, 50, pool.free)
        ref.release_pages(pool.free, s, pool.lens, pool.table, 16, keep.tolist(), held.tolist())
        assert maps.cu_seqlens.tolist() == cu and torch.stack(maps[1:], 1).tolist() == [list(x) for x in rows]
        pool.same()
        for t, x in ((new, [5 + i, 1, 30]), (keep, [42 + i, 21, 10]), (held, [41 + i + 5 + i, 21, 39])):
            t.copy_(torch.tensor(x))
        new[1] = 1 - (i > 0)
        lens = [pool.lens[x] for x in s]
        held.copy_(torch.tensor(lens).to(DEV) + new)
        keep.copy_(torch.minimum(keep, held))
        assert pool.release([3], keep=[lens[2] // 2])
        lens[2] //= 2
        held[2] = lens[2] + new[2]
        keep[2] = lens[2]
