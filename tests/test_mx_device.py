"""The device of the entries of the norm, of microscaled values and of the products
with them, on a stub of the runtime with two of them (tests/c/test_mx_device.c):
launches go to the backend's, and the caller's stays current, the call that
initialises included; the backward passes read the weights that they laid out."""
import os
import subprocess

import pytest

from conftest import ROOT


@pytest.mark.parametrize("first", range(8))
def test_the_callers_device_stays_current(first):
    path = os.path.join(ROOT, "tests", "c", "bin", "test_mx_device")
    if not os.path.exists(path):
        pytest.fail("%s not built (__graft_entry__.build() / make -C tests/c)" % path)
    p = subprocess.run([path, str(first)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)
    assert p.returncode == 0 and p.stdout.rstrip().endswith("PASS"), p.stdout
