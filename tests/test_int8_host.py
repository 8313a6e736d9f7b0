"""What the sources of the 8-bit products have to hold, where no run can show it."""

import glob
import os
import re

from conftest import ROOT


def test_cluster_barriers_order_the_reads_before_them():
    """A CTA may end, and its shared memory with it, once every CTA of its cluster has arrived: an arrival has to come
    after the arriving CTA's reads of that memory, which a relaxed one does not."""
    arrivals = []
    for path in glob.glob(os.path.join(ROOT, "alphafly_b200", "csrc", "*.cu*")):
        with open(path) as f:
            arrivals += [(os.path.basename(path), kind) for kind in re.findall(r"barrier\.cluster\.arrive(\.\w+)", f.read())]
    assert arrivals and all(kind == ".release" for _, kind in arrivals), arrivals
