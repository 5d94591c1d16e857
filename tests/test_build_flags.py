"""Which sources the compiler may take to be free of NaN."""
from __future__ import annotations

import os

import build_lib


def test_kernels_that_meet_nan_honour_it():
    sources = [f for f in os.listdir(build_lib.CSRC) if f.endswith(".hip")]
    assert set(build_lib.NO_NANS) < set(sources)
    for s in sources:
        flags = build_lib.flags(s)
        assert "-packed-fp32-ops" in flags
        assert not [f for f in flags if "fast-math" in f or "finite-math" in f]
        assert ("-fno-honor-nans" in flags) == (s in build_lib.NO_NANS)
    for s in ("h3a_window.hip", "h3a_norm.hip", "h3a_prologue.hip"):
        assert s not in build_lib.NO_NANS
