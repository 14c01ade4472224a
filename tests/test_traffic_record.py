"""The recorded DRAM traffic of the convolution that bench.py reports in its
roofline (profiles/ncu_traffic.json) belongs to the sources it was captured
from: bench.py leaves the figure out once they differ. A change of those
sources takes a new capture; what other kernels need goes into other files."""
import json
import os
import sys

from conftest import ROOT

sys.path.insert(0, ROOT)


def test_recorded_traffic_is_of_these_sources():
    import bench
    with open(os.path.join(ROOT, "profiles", "ncu_traffic.json")) as f:
        assert json.load(f)["source_sha256"] == bench.conv_source_hash()
