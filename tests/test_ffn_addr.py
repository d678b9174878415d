"""The loads of the dense feed-forward kernels, address by address on the CPU
(tests/c/test_ffn_addr.cpp over the header that the kernels compute them with)."""
import os
import subprocess

import pytest

from conftest import ROOT


def test_every_load_is_inside_its_matrix_or_marked():
    path = os.path.join(ROOT, "tests", "c", "bin", "test_ffn_addr")
    if not os.path.exists(path):
        pytest.fail("%s not built (__graft_entry__.build() / make -C tests/c)" % path)
    p = subprocess.run([path], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert p.returncode == 0 and p.stdout.rstrip().endswith("PASS"), p.stdout
