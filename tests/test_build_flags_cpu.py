"""Which sources are compiled with the promise that no value is NaN: none whose code chooses by values that may be
one (NaN is part of the 4-bit cache's format, and the C entries refuse NaN scales)."""
from __future__ import annotations

from pathlib import Path

import pytest

import build_lib

CSRC = Path(build_lib.__file__).resolve().parent / "csrc"
KEEP_NAN = ["kv4.hip", "fa_bwd.hip", "fa_abi.hip", "fa_abi_ops.hip", "fa_schedule.hip"]


@pytest.mark.parametrize("name", KEEP_NAN)
def test_sources_that_may_meet_nan_honour_it(name):
    assert (CSRC / name).exists()
    flags = build_lib.flags_for(CSRC / name)
    assert not any("honor-nan" in f or f in ("-ffast-math", "-ffinite-math-only", "-mno-amdgpu-ieee") for f in flags)


def test_every_source_is_named():
    others = {p.name for p in CSRC.glob("*.hip")} - set(KEEP_NAN)
    assert others == {f"{stem}.hip" for stem in build_lib.NAN_FREE}


@pytest.mark.parametrize("path", sorted(CSRC.glob("*.hip")), ids=lambda p: p.name)
def test_packed_fp32_stays_off(path):
    flags = build_lib.flags_for(path)
    assert "-packed-fp32-ops" in flags and flags[flags.index("-packed-fp32-ops") - 1] == "-Xclang"
