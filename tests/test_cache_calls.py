"""Calls of the 4-bit cache and of eviction whose outcome needs no GPU: refusals, and rules that the kernels' sources keep."""
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


def test_evict_refuses_destinations_that_overlap():
    """Two planes moved into one place, or weights into a plane: the move has no order."""
    from rustorch_b200 import _lib as L, build
    build.build()
    lib, far = L.lib(), 1 << 40
    src, size = (far, 2 * far), 2 * 8 * 256  # a destination's bytes: 2 heads of 8 rows

    def evict(dst, weights=5 * far, weights_out=6 * far, kept=7 * far, lens_out=8 * far):
        return lib.rt_kv_evict(L.pointers(src), L.pointers(dst), L.int32s((256, 256)), 2, weights, weights_out, kept, lens_out, 1, 2, 64,
                               8, None, 9, 4, 1, None)
    assert evict((3 * far, 3 * far)) == L.RT_ERR_UNSUPPORTED
    assert evict((3 * far, 3 * far + size - 16)) == L.RT_ERR_UNSUPPORTED
    out = (3 * far, 4 * far)
    for name in ("weights_out", "kept", "lens_out"):
        for at in (src[1] + 16, out[0], out[1] + size - 16):  # a plane that is read, one that is written
            assert evict(out, **{name: at}) == L.RT_ERR_UNSUPPORTED, (name, at - far)
    for a, b in (("weights_out", "kept"), ("kept", "lens_out"), ("weights_out", "lens_out"), ("kept", "weights"), ("lens_out", "weights")):
        assert evict(out, **{a: 9 * far, b: 9 * far}) == L.RT_ERR_UNSUPPORTED, (a, b)
