"""The compiler keeps a kernel's bounds with the flags that the library is built with.

Rows r0 and r0 + 16 on, each counted by `r < N ? min(N - r, 16) : 0`, the first count taken twice. From the second count's
min(N - r1, 16), whose subtraction wraps where r1 > N, clang's constraint elimination concludes that r1 <= N, and makes the
repeated first count 16 for any N: with such a count in a buffer's descriptor, rows past the matrix are read."""
import os
import re
import subprocess

import pytest

from test_build import _build_mod

SOURCE = """
#include <hip/hip_runtime.h>
#include <stdint.h>
__global__ void counts(uint32_t N, uint32_t *out) {
    const uint32_t r0 = blockIdx.x * 32u, r1 = r0 + 16u;
    out[0] = r0 < N ? min(N - r0, 16u) : 0u;
    out[1] = r1 < N ? min(N - r1, 16u) : 0u;
    out[2] = r0 < N ? min(N - r0, 16u) : 0u;
}
"""


def test_a_count_is_not_folded_by_the_one_beside_it(tmp_path):
    b = _build_mod()
    if not os.path.exists(b.HIPCC):
        pytest.skip("no hipcc here")
    src, out = tmp_path / "counts.hip", tmp_path / "counts.ll"
    src.write_text(SOURCE)
    subprocess.run([b.HIPCC] + b.HIPFLAGS + ["-S", "-emit-llvm", "--cuda-device-only", str(src), "-o", str(out)], check=True,
                   stderr=subprocess.DEVNULL)
    stores = re.findall(r"store i32 ([^,]+), ptr addrspace\(1\)", out.read_text())
    assert len(stores) == 3 and stores[0] == stores[2] != stores[1]
    assert all(v.startswith("%") for v in stores), stores
