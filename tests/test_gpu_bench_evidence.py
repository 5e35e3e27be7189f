"""bench.py prices its line with counters and job logs that are committed under profiles/: the tree that it runs in on a GPU holds them."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


def test_the_profiles_are_there():
    sys.path.insert(0, ROOT)
    import bench
    path, peaks, _ = bench.newest_profile("mfma_sustained.json")
    assert path and peaks
    path, blob, key = bench.newest_profile("pmc_panel_summary.json", "gs_tall_kernel<1, false, 0")
    assert path and blob[key]
    assert "no committed log" not in bench.job_gate_evidence()
