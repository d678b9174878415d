"""Products with MXFP4 weights that no kernel takes are told apart by their launcher, before anything is launched."""
import ctypes

import mx_forms as F

AT = 1 << 20                                                        # never read
NOT_SUPPORTED = 801                                                 # hipErrorNotSupported


def test_more_tiles_than_a_launch_takes(pkg):
    lib, most = pkg.load(), (1 << 31) - 1
    for xt in range(3):
        p, ep = F.prod(xt, most, most, 32, AT, AT, AT, AT), F.F.Ep(out=AT, ldout=most)
        assert lib.ghip_launch_mx(F.LINEAR, ctypes.byref(p), ctypes.byref(ep), None) == NOT_SUPPORTED
