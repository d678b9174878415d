"""Every lane of every access of the weight-streaming kernel with MXFP4 weights, on the CPU
(tests/c/test_mx_rows_addr.cpp over k_mx_rows_addr.h)."""
import os
import subprocess

import pytest

from conftest import ROOT


def test_every_access_is_inside_its_matrix():
    path = os.path.join(ROOT, "tests", "c", "bin", "test_mx_rows_addr")
    if not os.path.exists(path):
        pytest.fail("%s not built (__graft_entry__.build() / make -C tests/c)" % path)
    p = subprocess.run([path], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert p.returncode == 0 and p.stdout.rstrip().endswith("PASS"), p.stdout
