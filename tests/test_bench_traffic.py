"""roofline.traffic: the committed counter summaries are of the write's and
gather's sources as they are, whatever stands beside them."""
import json
import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(REPO))

import bench  # noqa: E402

SUMMARIES = sorted((REPO / "profiles").glob("traffic_*.json"))


@pytest.mark.parametrize("path", SUMMARIES, ids=lambda p: p.stem)
def test_committed_summaries_are_of_these_sources(path):
    d = json.loads(path.read_text())
    value, source = bench.load_traffic(d["kind"], d["workload"], d["algorithmic_bytes"])
    assert value == d["bytes_per_launch"] and source == f"profiles/{path.name}"


def test_operators_do_not_touch_the_digest():
    """Every unit of another kind is covered; the operators' are named."""
    from kvx_amd import build as kbuild

    units = [s for s in kbuild.SOURCES if s.endswith(".hip")]
    for prefix in bench.OPERATOR_UNITS:
        assert any(u.startswith(prefix) for u in units)
    covered = [u for u in units if not u.startswith(bench.OPERATOR_UNITS)]
    assert "dispatch.hip" in covered
    assert all(u == "dispatch.hip" or u.startswith(("kernels_write", "kernels_gather",
                                                    "kernels_tiles")) for u in covered)
