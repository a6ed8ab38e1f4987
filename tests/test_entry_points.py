"""What the repository's entry points need to be there."""
import json
import os

import pytest

from conftest import ROOT


def test_build_compiles_also_where_a_library_is_there(monkeypatch):
    import __graft_entry__ as entry
    from rankfm_amd import _build
    asked = []
    monkeypatch.setattr(_build, "build", lambda force=False, verbose=False: asked.append(force) or _build.LIB)
    monkeypatch.setenv("RANKFM_REFERENCE", os.path.join(ROOT, "no such folder"))
    if not os.path.exists(_build.LIB):
        pytest.skip("nothing is built")
    entry.build()
    assert asked == [True]


@pytest.mark.gpu
def test_the_counters_of_the_bench_line_are_there():
    """bench.py prints `traffic` and the atomic rates from them where it runs"""
    with open(os.path.join(ROOT, "profiles", "traffic.json")) as f:
        counters = json.load(f)
    for config in ("C2", "C3", "C4", "C5"):
        assert counters[config + "_hbm_bytes_per_launch"] > 0 and counters[config + "_atomic_requests_per_launch"] > 0
