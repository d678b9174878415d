"""The built code of every tile of the products with MXFP4 weights, run on the CPU (gfx950_walk.py) over ragged shapes: each
access inside its matrix (a base may lie a step past K, where every lane is put past the buffer), every load waited for, as many
barriers in each wave, each output stored once."""
import os
import re
import struct

import numpy as np
import pytest

import gfx950_walk as W
from test_ffn_asm import BUILD, OBJDUMP

OBJECTS = {0: "k_mx_bf16.hip.o", 1: "k_mx_fp8.hip.o", 2: "k_mx_fp4.hip.o"}
# one value; k cut inside a step, rows inside a vector, more than a tile of some
SHAPES = [(1, 1, 32), (70, 133, 608)]


@pytest.fixture(scope="module")
def tiles(tmp_path_factory):
    """{(mode, type of x, waves along M and N, 16-row and 16-column blocks of a wave, steps in the ring): code}"""
    found = {}
    for name in OBJECTS.values():
        if not (os.path.exists(os.path.join(BUILD, name)) and os.path.exists(OBJDUMP)):
            pytest.skip("no objects of a build here")
        for n, code in W.functions(os.path.join(BUILD, name), "k_mx_gemm", tmp_path_factory.mktemp("tiles")).items():
            found[tuple(map(int, re.search("I" + r"Li(\d+)E" * 7, n).groups()))] = code
    return found


def walk(code, tile, M, N, K, pad=0, ep=True, less=None):
    """ep: with bias and residual; less: a buffer that is declared a row shorter than the kernel is told."""
    mode, xt, wm, wn, rb, cb, ring = tile
    dual, bm, bn = mode == 2, 16 * rb * wm, 16 * cb * wn
    cols = bn // 2 if dual else bn
    units = (0 if xt == 0 else (bm + 63) // 64) + (2 if dual else 1) * ((cols + 63) // 64)
    lds = ring * (bm * (64 if xt == 2 else 128) + bn * (32 if xt == 0 else 64)) + 1024 * units
    ld, wb, xb, out = (K + 127) // 128 * 4, K // 2, (2 * K, K, K // 2)[xt], N + pad
    xld = xb + (16 * pad if xt == 0 else 0)
    rows = {"w": (N, wb), "ws": (N, ld), "w2": (N * dual, wb), "ws2": (N * dual, ld), "x": (M, xld), "xs": (M * (xt > 0), ld), "out": (M, 2 * out),
            "bias": (1, 2 * N * (ep and not dual)), "in": (M * (ep and not dual), 2 * out)}
    last = {"x": xb, "out": 2 * N, "in": 2 * N}
    sizes = {k: (n - 1 - (k == less)) * w + last.get(k, w) if n and w else 0 for k, (n, w) in rows.items()}
    buffers = {k: (0x200000000000 + (i << 40) + 0x300 * i, n, k == "out") for i, (k, n) in enumerate(sizes.items()) if n > 0}
    at = lambda k: buffers[k][0] if k in buffers else 0  # noqa: E731
    mt, nt = -(-M // bm), -(-N // cols)
    args = struct.pack("<6QQ4I", *map(at, ("w", "w2", "ws", "ws2", "x", "xs")), xld, M, N, K, xt)
    args += struct.pack("<4QQQifI4x", at("bias"), at("in"), at("out"), 0, out, out, 3, 1.0, 0) + struct.pack("<2I", mt, nt)
    args += struct.pack("<3I3H", mt * nt, 1, 1, 64 * wm * wn, 1, 1) + bytes(64)
    rng, stores = np.random.default_rng([*tile, M, N, K]), {}
    for block in sorted({0, mt * nt - 1}):
        waves = [W.Wave(code, args, buffers, lds, w, (block, 0), rng, stores, based=False) for w in range(wm * wn)]
        for k, w in enumerate(waves):
            try:
                w.run()
            except W.Fault as f:
                raise W.Fault("%s, workgroup %d, wave %d of %s: %s" % (tile, block, k, (M, N, K), f)) from None
        assert len({w.barriers for w in waves}) == 1
    assert set(stores.values()) == {1}


@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("xt", [0, 1, 2])
def test_every_access_of_the_built_code(tiles, mode, xt):
    found = [t for t in tiles if t[:2] == (mode, xt)]
    assert len(found) >= 5
    for t in found:
        for M, N, K in SHAPES:
            walk(tiles[t], t, M, N, K, pad=M % 3, ep=M % 2 == 1)


@pytest.mark.parametrize("less", ["w", "ws", "x", "xs", "out", "in"])
def test_the_walk_sees_a_row_that_is_not_there(tiles, less):
    tile = min(t for t in tiles if t[:2] == (1, 1))
    with pytest.raises(W.Fault):
        walk(tiles[tile], tile, 15, 17, 160, less=less)
