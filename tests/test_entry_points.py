"""What the repository's entry points need to be there."""
import json
import os

import pytest

from conftest import ROOT


@pytest.mark.gpu
def test_the_counters_of_the_bench_line_are_there():
    """bench.py prints `traffic` and the atomic rates from them where it runs"""
    with open(os.path.join(ROOT, "profiles", "traffic.json")) as f:
        counters = json.load(f)
    for config in ("C2", "C3", "C4", "C5"):
        assert counters[config + "_hbm_bytes_per_launch"] > 0 and counters[config + "_atomic_requests_per_launch"] > 0
