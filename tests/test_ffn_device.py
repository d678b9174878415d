"""The device of the dense feed-forward entries, on a stub of the runtime with two
of them (tests/c/test_ffn_device.c): launches go to the backend's, and the
caller's stays current, the call that initialises included."""
import os
import subprocess

import pytest

from conftest import ROOT


@pytest.mark.parametrize("first", range(6))
def test_the_callers_device_stays_current(first):
    path = os.path.join(ROOT, "tests", "c", "bin", "test_ffn_device")
    if not os.path.exists(path):
        pytest.fail("%s not built (__graft_entry__.build() / make -C tests/c)" % path)
    p = subprocess.run([path, str(first)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)
    assert p.returncode == 0 and p.stdout.rstrip().endswith("PASS"), p.stdout
