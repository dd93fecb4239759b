"""Low-rank adapters on the GPU against 64 bits: the bound is the oracle's own (``oracle/step.py``), and one rounding
to the element type."""
import pytest
import torch

import custom_inference_engine_amd as cie
from oracle import step as ref
from tests.gpu_helpers import DEV, err_word, note

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
PAGE, PLAN, ADAPTER = 1, 16, 64


class Case:
    def __init__(self, ids, n, rank, d_in, slices, dtype, ranks=None, seed=0):
        g = torch.Generator().manual_seed(seed)
        T, R, out = len(ids), -(-rank // 16) * 16, sum(slices)
        self.ids, self.n, self.slices, self.dtype = ids, n, slices, dtype
        self.ranks = torch.tensor(ranks or [rank] * n, dtype=torch.int32)
        live = torch.arange(R) < self.ranks[:, None]
        self.a = (torch.randn(n, len(slices), R, d_in, generator=g) * d_in ** -0.5 * live[:, None, :, None]).to(dtype)
        self.b = (torch.randn(n, out, R, generator=g) * live[:, None]).to(dtype)
        self.scales = 0.25 + torch.rand(n, generator=g)
        self.x, self.y = torch.randn(T, d_in, generator=g).to(dtype), torch.randn(T, out, generator=g).to(dtype)

    def up(self):
        return [t.to(DEV) for t in (self.y, self.x, self.a, self.b, self.scales, self.ranks)]

    def run(self, err=None):
        y, *rest = self.up()
        note(f"adapters T={len(self.ids)} n={self.n} a={tuple(self.a.shape)} slices={self.slices} {self.dtype}")
        plan = cie.adapter_plan(None, torch.tensor(self.ids, dtype=torch.int64, device=DEV), self.n, err=err)
        assert cie.adapter_add_(y, *rest, plan, self.slices, err=err) is y
        return y.cpu()

    def check(self, got):
        want, off = ref.adapters(self.y, self.x, self.a, self.b, self.scales, self.ids, self.slices)
        bad = (got.double() - want).abs() > off + ref.rounding(want.abs() + off, self.dtype)
        assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, first at {bad.nonzero()[0].tolist()}"
        none = torch.tensor([i < 0 for i in self.ids], dtype=torch.bool)
        assert torch.equal(got[none], self.y[none])


def spread(T, n, none=0.2, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, n, (T,), generator=g)
    return torch.where(torch.rand(T, generator=g) < none, -1, ids).tolist()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("ids,n,rank,d_in,slices", [
    ([0], 1, 16, 64, (64,)),
    ([0], 1, 1, 8, (8,)),
    ([3], 5, 8, 896, (896, 128, 128)),
    (spread(32, 40), 40, 16, 896, (896, 128, 128)),
    (spread(33, 3), 3, 32, 200, (72,)),
    (spread(100, 7), 7, 64, 512, (512, 64)),
    (spread(45, 4), 4, 128, 1024, (136, 72, 64, 200)),
    (spread(70, 4), 4, 48, 328, (264, 72)),
    ([1] * 50 + [0] * 31 + [-1] * 10 + [1], 2, 24, 320, (192,)),
    ([-1] * 20, 3, 16, 64, (64,)),
    ([2] * 16 + [1] * 17 + [0] * 15, 3, 80, 136, (80, 88, 96)),
])
def test_products(ids, n, rank, d_in, slices, dtype):
    case = Case(ids, n, rank, d_in, slices, dtype, seed=len(ids))
    err = err_word()
    case.check(case.run(err))
    assert int(err) == 0


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("d_in,slices", [(1, (1,)), (7, (3, 5)), (100, (100,)), (893, (67, 129)), (64, (65,)), (130, (64, 1, 63))])
def test_odd_widths(d_in, slices, dtype):
    """Widths that leave no 16-byte pieces go value by value."""
    case = Case(spread(21, 3), 3, 20, d_in, slices, dtype)
    case.check(case.run())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
def test_ranks_of_their_own(dtype):
    ranks = [1, 16, 17, 64, 0, 33]
    case = Case(spread(60, 6, none=0.1), 6, 64, 256, (128, 64), dtype, ranks=ranks)
    case.check(case.run())
    empty = torch.tensor([i == 4 for i in case.ids])
    assert empty.any() and torch.equal(case.run()[empty], case.y[empty])  # an empty place


@pytest.mark.parametrize("T,n", [(1536, 3), (1537, 3), (2500, 300), (4100, 1), (5000, 1024), (8200, 2), (70000, 5)])
def test_many_rows(T, n):
    """Both tile heights; rows dealt over one, few and many adapters."""
    case = Case(spread(T, n, none=0.1), n, 16, 64, (64,), F16)
    case.check(case.run())


def test_plan_is_the_rows_in_order():
    """Tiles of one adapter, adapters and their rows ascending: the same plan every time."""
    for T, n in ((1, 1), (50, 4), (700, 9), (1537, 5), (8192, 3), (8193, 3), (9000, 700), (17000, 40), (100000, 1024)):
        ids = spread(T, n, seed=T)
        on_device = torch.tensor(ids, dtype=torch.int64, device=DEV)
        note(f"plan T={T} n={n}")
        plan = cie.adapter_plan(None, on_device, n).tolist()
        m = 16 if T <= 1536 else 32
        want = []
        for a in range(n):
            rows = [t for t, i in enumerate(ids) if i == a]
            want += [(a, rows[k:k + m]) for k in range(0, len(rows), m)]
        assert plan[:4] == [len(want), T, n, m]
        tiles = [plan[8 + k * (4 + m):8 + (k + 1) * (4 + m)] for k in range(len(want))]
        assert [(t[0], t[4:4 + t[1]]) for t in tiles] == want


def test_plan_at_one_address():
    ids = torch.tensor(spread(40, 3), device=DEV)
    room = cie.new_adapter_plan(40, 3, DEV)
    assert cie.adapter_plan(None, ids, 3, out=room) is room
    want = cie.adapter_plan(None, ids, 3)
    n = int(want[0])
    for t in (room, want):  # (words behind a tile's rows are whatever was there)
        tiles = t[8:8 + 20 * n].view(n, 20)
        tiles[:, 2:4] = 0
        tiles[:, 4:].masked_fill_(torch.arange(16, device=DEV) >= tiles[:, 1:2], 0)
    assert torch.equal(room[:5], want[:5]) and torch.equal(room[8:8 + 20 * n], want[8:8 + 20 * n])
    for bad in (cie.new_adapter_plan(70, 3, DEV), cie.new_adapter_plan(40, 4, DEV), room.long()):
        with pytest.raises(AssertionError):
            cie.adapter_plan(None, ids, 3, out=bad)


def test_plan_of_slots():
    """Rows' adapters through their slots; bad slots and adapters have none, and are reported."""
    by_slot = torch.tensor([-1, 2, 0, -5, 1, 3], device=DEV)
    row_slots = torch.tensor([1, 1, 4, 0, 2, 3, 1, 5], device=DEV)
    plan = cie.adapter_plan(row_slots, by_slot, 4).tolist()
    tiles = [plan[8 + 20 * k:28 + 20 * k] for k in range(plan[0])]
    assert [(t[0], t[4:4 + t[1]]) for t in tiles] == [(0, [4]), (1, [2]), (2, [0, 1, 6]), (3, [7])]
    for slots, n, bit in ((row_slots, 3, ADAPTER), (torch.tensor([1, 6, 2], device=DEV), 4, PAGE),
                          (torch.tensor([-1, 1], device=DEV), 4, PAGE)):
        err = err_word()
        plan = cie.adapter_plan(slots, by_slot, n, err=err)
        assert int(err) == bit
        rows = [r for k in range(int(plan[0])) for r in plan[12 + 20 * k:12 + 20 * k + int(plan[9 + 20 * k])].tolist()]
        assert 7 not in rows if bit == ADAPTER else all(0 < int(slots[r]) < 6 for r in rows)


def test_a_plan_of_other_rows_is_refused():
    case = Case(spread(30, 3), 3, 16, 64, (64,), F16)
    y, *rest = case.up()
    plan = cie.adapter_plan(None, torch.tensor(spread(40, 3), device=DEV), 3)
    err = err_word()
    cie.adapter_add_(y, *rest, plan, case.slices, err=err)
    assert int(err) == PLAN and torch.equal(y.cpu(), case.y)
    plan = cie.adapter_plan(None, torch.tensor(spread(30, 3), device=DEV), 9)
    err = err_word()
    cie.adapter_add_(y, *rest, plan, case.slices, err=err)
    assert int(err) == PLAN and torch.equal(y.cpu(), case.y)


def test_a_row_does_not_depend_on_its_neighbours():
    """Bit for bit the same row alone, among others, at another place and in the other tile height."""
    case = Case(spread(40, 2, none=0), 2, 32, 200, (72, 40), F16)
    y = case.run()
    for t in (0, 7, 39):
        one = Case([case.ids[t]], 2, 32, 200, (72, 40), F16)
        one.a, one.b, one.scales, one.ranks = case.a, case.b, case.scales, case.ranks
        one.x, one.y = case.x[t:t + 1], case.y[t:t + 1]
        assert torch.equal(one.run()[0], y[t])
    many = Case([case.ids[t % 40] for t in range(2400)], 2, 32, 200, (72, 40), F16)
    many.a, many.b, many.scales, many.ranks = case.a, case.b, case.scales, case.ranks
    many.x, many.y = case.x.repeat(60, 1), case.y.repeat(60, 1)
    assert torch.equal(many.run(), y.repeat(60, 1))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
def test_values_past_the_types_range(dtype):
    """A x beyond fp16's largest value, and far under its smallest, keeps its bits: only y has to hold the result."""
    for up, down in ((2.0 ** 12, 2.0 ** -14), (2.0 ** -14, 2.0 ** 12)):
        case = Case(spread(20, 2, none=0), 2, 16, 512, (64,), dtype)
        case.a, case.b = (case.a.float() * up).to(dtype), (case.b.float() * down).to(dtype)
        case.x = (case.x.float() * 2.0 ** (8 if up > 1 else -8)).to(dtype)
        case.scales = case.scales * 2.0 ** (-6 if up > 1 else 10)
        case.check(case.run())


def test_infinities_and_nans_stay_in_their_rows():
    case = Case([0, 1, 0, -1, 0], 2, 16, 96, (64, 8), F16)
    case.x[1, 5] = float("nan")
    case.x[2, 7] = float("inf")
    case.x[3, 9] = float("nan")  # a row without an adapter
    clean = Case([0, 1, 0, -1, 0], 2, 16, 96, (64, 8), F16)
    got, want = case.run(), clean.run()
    assert torch.equal(got[[0, 3, 4]], want[[0, 3, 4]])
    assert got[1].isnan().all() and not got[2].isfinite().any()
    # one infinite rank beside finite ones: the infinity comes out with B's sign, the others are not lost in it
    case = Case([0], 1, 16, 16, (16,), F16)
    case.a.zero_()
    case.a[0, 0, 0, 0], case.a[0, 0, 1, 1] = 60000.0, 1.0
    case.x[0] = 0
    case.x[0, 0], case.x[0, 1] = float("inf"), 2.0
    case.a[0, 0, 1, 0] = 0.0
    case.b.fill_(1.0)
    got = case.run()
    assert got[0].isnan().all()  # (0 * inf in the other ranks, as in the plain form)
    case.x[0, 0] = 60000.0
    case.b[:, :, 0] = 0.0
    got = case.run()
    assert torch.equal(got, (case.y.float() + case.scales * 2.0).half())


def test_strides_and_leading_dims():
    """y and x as views: columns of a wider tensor (aligned or not), a leading 1, rows shared in x."""
    case = Case(spread(19, 3), 3, 16, 64, (64, 16), F16)
    want = case.run()
    y, x, *rest = case.up()
    plan = cie.adapter_plan(None, torch.tensor(case.ids, device=DEV), 3)
    for left, width in ((8, 120), (3, 101)):
        wide_y = torch.full((1, 19, width), 7.0, dtype=F16, device=DEV)
        wide_x = torch.full((1, 19, width), float("nan"), dtype=F16, device=DEV)
        wide_y[0, :, left:left + 80], wide_x[0, :, left:left + 64] = y, x
        cie.adapter_add_(wide_y[..., left:left + 80], wide_x[..., left:left + 64], *rest, plan, case.slices)
        assert torch.equal(wide_y[0, :, left:left + 80].cpu(), want)
        assert (wide_y[..., :left] == 7).all() and (wide_y[..., left + 80:] == 7).all()
    same = x[:1].expand(19, 64)
    a, b = y.clone(), y.clone()
    cie.adapter_add_(a, same, *rest, plan, case.slices)
    cie.adapter_add_(b, same.contiguous(), *rest, plan, case.slices)
    assert torch.equal(a, b)


def test_no_rows():
    case = Case([0], 2, 16, 64, (64,), F16)
    y, x, *rest = case.up()
    plan = cie.adapter_plan(None, torch.empty(0, dtype=torch.int64, device=DEV), 2)
    cie.adapter_add_(y[:0], x[:0], *rest, plan, case.slices)


def test_bank():
    """What load puts in place: slices without an adapter, ranks of their own, a place that is filled anew and emptied."""
    g = torch.Generator().manual_seed(0)
    bank = cie.AdapterBank(3, 20, 96, (64, 32, 32), dtype=F16, device=DEV)
    assert bank.a.shape == (3, 3, 32, 96) and bank.b.shape == (3, 128, 32)
    make = lambda *s: torch.randn(*s, generator=g).half()  # noqa: E731
    bank.load(1, (make(20, 96), None, make(20, 96)), (make(64, 20), None, make(32, 20)), scale=3.0)
    a, b = (make(4, 96), None, make(7, 96)), (make(64, 4), None, make(32, 7))
    bank.load(1, a, b, scale=0.5)
    assert bank.ranks.tolist() == [0, 7, 0]
    x, y = make(1, 5, 96), make(1, 5, 128)
    plan = cie.adapter_plan(None, torch.tensor([1, 0, -1, 1, 2], device=DEV), 3)
    out = y.to(DEV)
    bank.add_(out, x.to(DEV), plan)
    want = y.double()
    for t in (0, 3):
        want[0, t, :64] += 0.5 * (b[0].double() @ (a[0].double() @ x[0, t].double()))
        want[0, t, 96:] += 0.5 * (b[2].double() @ (a[2].double() @ x[0, t].double()))
    # (|A x| <= 96 terms: fp32 sums are off by 2^-15 of some 40, then 7 ranks; y's rounding 2^-11)
    assert ((out.cpu().double() - want).abs() <= 0.02 + 2.0 ** -11 * want.abs()).all()
    assert torch.equal(out[0, [1, 2, 4]].cpu(), y[0, [1, 2, 4]])
    bank.clear(1)
    again = y.to(DEV)
    bank.add_(again, x.to(DEV), plan)
    assert torch.equal(again.cpu(), y) and not bank.a.any() and not bank.b.any()


def test_captured_with_other_adapters():
    """A plan and its products in a graph: the slots' adapters, rows and weights of each replay count."""
    case = Case(spread(30, 4), 4, 32, 128, (64, 32), F16)
    y, x, a, b, scales, ranks = case.up()
    by_slot = torch.tensor([-1, 0, 1, 2, 3], device=DEV)
    slots = torch.tensor([i + 1 for i in case.ids], device=DEV)
    out = torch.empty_like(y)
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        out.copy_(y)
        cie.adapter_add_(out, x, a, b, scales, ranks, cie.adapter_plan(slots, by_slot, 4), case.slices)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        case.check(out.cpu())
        want = y.clone()
        cie.adapter_add_(want, x, a, b, scales, ranks, cie.adapter_plan(slots, by_slot, 4), case.slices)
        assert torch.equal(out, want)
        by_slot.copy_(torch.tensor([-1, 3, 2, -1, i]))
        x.mul_(0.5)
        a[1] += 0.125
        case.ids = [int(by_slot[s]) for s in slots]
        case.x, case.a = x.cpu(), a.cpu()


def test_another_stream():
    case = Case(spread(64, 8), 8, 16, 512, (512,), F16)
    want = case.run()
    side = torch.cuda.Stream()
    y, *rest = case.up()
    ids = torch.tensor(case.ids, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        cie.adapter_add_(y, *rest, cie.adapter_plan(None, ids, 8), case.slices)
    side.synchronize()
    assert torch.equal(y.cpu(), want)
