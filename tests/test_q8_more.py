"""The 8-bit cache without a GPU, further cases: how it is built, and what its paths refuse and accept."""
import types

import pytest
import torch
from transformers import Qwen2Config

import custom_inference_engine_amd as cie
from custom_inference_engine_amd import _build


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
