"""Low-rank adapters where their arithmetic could lose bits or a call could reach past what it was given: sums that
cancel, slices of different sizes, words that are no plan, plans of more rows than a wave keeps."""
import pytest
import torch

import custom_inference_engine_amd as cie
from oracle import step as ref
from tests.gpu_helpers import DEV, err_word, note

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
PLAN = 16


def add(x, a, b, scales, slices, y=None, ids=None):
    """y (zeros) with adapter 0 added to every row, on the GPU; the error word is checked."""
    T, n = x.shape[0], a.shape[0]
    ids = torch.zeros(T, dtype=torch.int64) if ids is None else ids
    y = torch.zeros(T, sum(slices), dtype=x.dtype) if y is None else y
    ranks = torch.full((n,), a.shape[2], dtype=torch.int32)
    note(f"adapters T={T} a={tuple(a.shape)} slices={slices} {x.dtype}")
    err = err_word()
    y, x, a, b, scales, ranks, ids = (t.to(DEV) for t in (y, x, a, b, scales, ranks, ids))
    cie.adapter_add_(y, x, a, b, scales, ranks, cie.adapter_plan(None, ids, n, err=err), slices, err=err)
    assert int(err) == 0
    return y.cpu()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("T,R,d_in,slices", [(1, 16, 64, (64,)), (3, 64, 64, (64, 8)), (5, 16, 67, (9, 65)), (40, 128, 72, (136,)),
                                             (2000, 16, 64, (64, 64)), (1700, 64, 72, (72,)), (1600, 32, 67, (65,))])
def test_products_that_cancel(T, R, d_in, slices, dtype):
    """Two ranks whose A x is 1 + 2^-9 + 2^-k and -(1 + 2^-9), added by B's ones: 2^-k is left, whole.  (Every partial
    sum is a 24-bit value, so nothing rounds; 2^-k, beside 2^-9 and 1, is the third group of eight bits of A x.)"""
    for k in (17, 18, 22):
        x, a = torch.zeros(T, d_in), torch.zeros(1, len(slices), R, d_in)
        x[:, 0], x[:, 1], x[:, 2] = 1.0, 2.0 ** -9, 2.0 ** -9
        a[0, :, 3, 0], a[0, :, 3, 1], a[0, :, 3, 2] = 1.0, 1.0, 2.0 ** (9 - k)
        a[0, :, R - 1, 0], a[0, :, R - 1, 1] = -1.0, -1.0
        b = torch.zeros(1, sum(slices), R)
        b[..., 3] = b[..., R - 1] = 1.0
        got = add(x.to(dtype), a.to(dtype), b.to(dtype), torch.tensor([2.0 ** 10]), slices)
        assert (got == 2.0 ** (10 - k)).all(), (k, got.unique().tolist())


@pytest.mark.parametrize("T,R,d_in,widths", [(1, 16, 64, (64, 8)), (3, 64, 64, (64, 72)), (40, 32, 67, (9, 65)), (5, 128, 64, (8, 64)),
                                             (2000, 16, 64, (64, 64)), (1700, 32, 64, (72, 8))])
def test_a_small_slice_beside_a_large_one(T, R, d_in, widths):
    """A slice whose A x is 2^-24 of the other's keeps its own bits, wherever it stands: of 2^-10 + 2^-28 and -2^-10, added
    by B's ones, 2^-28 is left, whole."""
    for small in (0, 1):
        x, a, b = torch.zeros(T, d_in), torch.zeros(1, 2, R, d_in), torch.zeros(1, sum(widths), R)
        x[:, 0], x[:, 1] = 1.0, 2.0 ** -14
        a[0, 1 - small, 0, 0] = 2.0 ** 14
        a[0, small, 3, 0], a[0, small, 3, 1], a[0, small, R - 1, 0] = 2.0 ** -10, 2.0 ** -14, -(2.0 ** -10)
        lo = small * widths[0]
        b[0, lo:lo + widths[small], 3] = b[0, lo:lo + widths[small], R - 1] = 1.0
        got = add(x.half(), a.half(), b.half(), torch.tensor([2.0 ** 20]), widths)
        want = torch.zeros(T, sum(widths))
        want[:, lo:lo + widths[small]] = 2.0 ** -8
        assert torch.equal(got.float(), want), small


def test_slices_of_different_sizes():
    """One slice's A scaled by 2^10 and another's by 2^-12 (their B scaled back), against each slice's own bound."""
    g = torch.Generator().manual_seed(4)
    for T, R, d_in, slices in ((9, 16, 64, (64, 64, 8)), (30, 64, 200, (136, 72, 64)), (1800, 32, 67, (65, 9, 64))):
        T_ids = torch.randint(-1, 2, (T,), generator=g)
        a, b = torch.randn(2, 3, R, d_in, generator=g) * d_in ** -0.5, torch.randn(2, sum(slices), R, generator=g)
        col = 0
        for s, e in enumerate((10, 0, -12)):
            a[:, s] *= 2.0 ** e
            b[:, col:col + slices[s]] *= 2.0 ** -e
            col += slices[s]
        a, b, x, y = a.half(), b.half(), torch.randn(T, d_in, generator=g).half(), torch.randn(T, sum(slices), generator=g).half()
        scales = torch.tensor([0.5, 2.0])
        got = add(x, a, b, scales, slices, y=y, ids=T_ids)
        want, off = ref.adapters(y, x, a, b, scales, T_ids.tolist(), slices)
        assert ((got.double() - want).abs() <= off + ref.rounding(want.abs() + off, F16)).all()


@pytest.mark.parametrize("T", [20, 2000])
@pytest.mark.parametrize("word", [-5, -(1 << 31), (1 << 31) - 1, 0])
def test_words_that_are_no_plan(T, word):
    """A buffer of the right size with anything in it: reported, nothing written."""
    g = torch.Generator().manual_seed(0)
    x, y = torch.randn(T, 64, generator=g).half().to(DEV), torch.randn(T, 128, generator=g).half().to(DEV)
    a, b = torch.randn(3, 1, 16, 64, generator=g).half().to(DEV), torch.randn(3, 128, 16, generator=g).half().to(DEV)
    scales, ranks = torch.ones(3, device=DEV), torch.full((3,), 16, dtype=torch.int32, device=DEV)
    plan = cie.new_adapter_plan(T, 3, DEV).fill_(word)
    err, kept = err_word(), y.clone()
    note(f"no plan T={T} word={word}")
    cie.adapter_add_(y, x, a, b, scales, ranks, plan, (128,), err=err)
    assert int(err) == PLAN and torch.equal(y, kept)


def test_a_plan_of_more_rows_than_a_wave_keeps():
    """Past about a million rows a wave counts its rows anew when it writes them: the same order, each row once."""
    T, n = 1_200_007, 37
    g = torch.Generator().manual_seed(0)
    row_slots = torch.randint(0, 90, (T,), generator=g)
    row_slots[300_000:700_000] = 5  # (a long prompt's)
    by_slot = torch.randint(-1, n, (90,), generator=g)
    by_slot[5] = 11
    err = err_word()
    note(f"plan T={T} n={n}")
    plan = cie.adapter_plan(row_slots.to(DEV), by_slot.to(DEV), n, err=err)
    assert int(err) == 0
    ids = by_slot[row_slots]
    rows = torch.sort(ids, stable=True).indices[int((ids < 0).sum()):]
    counts = torch.bincount(ids[ids >= 0], minlength=n)
    tiles_of = (counts + 31) // 32
    tiles = int(tiles_of.sum())
    words = plan.cpu()
    assert words[:4].tolist() == [tiles, T, n, 32]
    got = words[8:8 + 36 * tiles].view(tiles, 36)
    assert torch.equal(got[:, 0].long(), torch.repeat_interleave(torch.arange(n), tiles_of))
    live = torch.arange(32) < got[:, 1:2]
    assert torch.equal(got[:, 4:][live].long(), rows)
    x, y = torch.randn(T, 8, generator=g).half(), torch.zeros(T, 8).half()
    a, b = torch.randn(n, 1, 16, 8, generator=g).half(), torch.randn(n, 8, 16, generator=g).half()
    ranks = torch.full((n,), 16, dtype=torch.int32)
    out = cie.adapter_add_(y.to(DEV), x.to(DEV), a.to(DEV), b.to(DEV), torch.ones(n, device=DEV), ranks.to(DEV), plan, (8,))
    some = torch.randint(0, T, (400,), generator=g)
    want, off = ref.adapters(y[some], x[some], a, b, torch.ones(n), ids[some].tolist(), (8,))
    assert ((out.cpu()[some].double() - want).abs() <= off + ref.rounding(want.abs() + off, F16)).all()


def test_weights_in_y_are_refused():
    """A bank whose tensors lie in y's rows, and one between them, which is taken."""
    room = torch.zeros(64 * 1024, dtype=F16, device=DEV)
    y = room[:20 * 2048].view(20, 2048)[:, 100:164]
    x, plan = torch.ones(20, 8).half().to(DEV), cie.adapter_plan(None, torch.zeros(20, dtype=torch.int64, device=DEV), 1)
    scales, ranks = torch.ones(1, device=DEV), torch.full((1,), 16, dtype=torch.int32, device=DEV)
    a, b = torch.ones(1, 1, 16, 8).half().to(DEV), torch.ones(1, 64, 16).half().to(DEV)
    for lo in (0, 60, 163, 2048, 19 * 2048 + 40):
        for bad in (dict(a=room[lo:lo + 128].view(1, 1, 16, 8)), dict(b=room[lo:lo + 1024].view(1, 64, 16))):
            args = {**dict(a=a, b=b), **bad}
            with pytest.raises(AssertionError, match="y's memory"):
                cie.adapter_add_(y, x, args["a"], args["b"], scales, ranks, plan, (64,))
    room[2048 + 200:2048 + 328] = 1.0  # (an A of ones between two rows)
    between = room[2048 + 200:2048 + 328].view(1, 1, 16, 8)
    cie.adapter_add_(y, x, between, b, scales, ranks, plan, (64,))
    assert (y == 16 * 8).all() and (between == 1).all()
