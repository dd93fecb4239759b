"""Rotary positions of fp32 rows and tables: cos and sin keep all 24 bits."""
import math

import pytest
import torch

import custom_inference_engine_amd as cie
from oracle import step as ref
from tests.gpu_helpers import DEV, note

pytestmark = pytest.mark.gpu
F32 = torch.float32


def exact(pos, freqs, scale):
    """cos and sin (T, pairs) in 64 bits, times scale."""
    angle = torch.tensor([[math.fmod(p * f, 2 * math.pi) for f in freqs.tolist()] for p in pos.tolist()], dtype=torch.float64)
    return scale * angle.cos(), scale * angle.sin()


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("T,rot", [(1, 64), (40, 128), (33, 20), (5, 2), (200, 66)])
def test_fp32_tables_are_rounded_once(T, rot, interleaved):
    """Half a step of the value, and what the angle is off: positions under 2^13, whose products with a frequency and 1 / 2 pi
    are off by three roundings of 2^-53 (2^-38 radians), on either side."""
    g = torch.Generator().manual_seed(T)
    pos = torch.randint(0, 8192, (T,), generator=g)
    for scale in (1.0, 0.1 * math.log(4) + 1):
        freqs, _ = cie.rotary_frequencies(rot, 1e4)
        note(f"fp32 tables T={T} rot={rot}")
        got = cie.rotary_tables(pos.to(DEV), freqs.to(DEV), dtype=F32, interleaved=interleaved, scale=scale)
        for t, want in zip(got, exact(pos, freqs, scale)):
            want = torch.cat((want, want), 1) if not interleaved else want.repeat_interleave(2, 1)
            assert ((t[0].cpu().double() - want).abs() <= ref.rounding(want, F32) + 2.0 ** -37).all()


@pytest.mark.parametrize("T,d,rot", [(300, 64, 64), (70, 128, 32), (33, 64, 20)])
def test_fp32_rows(T, d, rot):
    """cos and sin rounded once, a product, a sum: four halves of a step of the terms."""
    g = torch.Generator().manual_seed(d)
    x, pos = torch.randn(1, T, 6, d, generator=g), torch.randint(0, 8192, (T,), generator=g)
    freqs, _ = cie.rotary_frequencies(rot, 1e4)
    for interleaved in (False, True):
        note(f"fp32 rows T={T} d={d} rot={rot}")
        got, _ = cie.apply_rotary(x.to(DEV), None, pos.to(DEV), freqs.to(DEV), interleaved=interleaved)
        want, size = ref.rotary(x[0], pos.tolist(), freqs.tolist(), interleaved)
        n = rot // 2
        c, s = (t[:, None] for t in exact(pos, freqs, 1.0))
        a, b = (x[0, ..., :n], x[0, ..., n:rot]) if not interleaved else (x[0, ..., :rot:2], x[0, ..., 1:rot:2])
        a, b = a.double(), b.double()
        first, second = (a * c).abs() + 2 * (b * s).abs(), (b * c).abs() + 2 * (a * s).abs()
        terms = torch.cat((first, second), -1) if not interleaved else torch.stack((first, second), -1).flatten(-2)
        off = (got[0].cpu().double() - want).abs()[..., :rot]
        assert (off <= 2.0 ** -24 * terms + ref.rounding(want[..., :rot], F32) + 2.0 ** -37 * size[..., :rot]).all()
