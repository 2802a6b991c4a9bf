"""Calls of the 4-bit cache and of eviction that need no GPU to be judged: refusals, and rules that the kernels' sources keep."""
import glob
import os
import re

import rustorch_b200 as rt

CSRC = os.path.join(os.path.dirname(os.path.abspath(rt.__file__)), "csrc")


def test_no_cluster_barrier_needs_a_warp_that_has_met_again():
    """`barrier.cluster` with .aligned is undefined in a warp whose threads left a loop or a branch apart."""
    for path in glob.glob(os.path.join(CSRC, "*.cu*")):
        with open(path) as f:
            code = re.sub(r"//.*", "", f.read())
        assert not re.search(r"barrier\.cluster\.\w+(\.\w+)*\.aligned", code), path
