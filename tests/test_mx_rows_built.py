"""The built code of the weight-streaming kernel with MXFP4 weights, every form, run on the CPU (gfx950_walk.py) over shapes
as those of its test on the device, first and last workgroups: each access inside its matrix, each descriptor's base too, every load waited for, as many barriers in
each wave, each output stored once."""
import os
import re
import struct

import numpy as np
import pytest

import gfx950_walk as W
from test_ffn_asm import BUILD, OBJDUMP

OBJECT = os.path.join(BUILD, "k_mx_rows.hip.o")
XR = (256, 128, 64)                                                 # bytes of x's row in a step of 128
SHAPES = [(1, 1, 32), (3, 300, 544), (16, 33, 1024), (17, 129, 2080), (2, 530, 6400), (3, 9000, 256)]


@pytest.fixture(scope="module")
def forms(tmp_path_factory):
    """{(type of x, waves along k): code}"""
    if not (os.path.exists(OBJECT) and os.path.exists(OBJDUMP)):
        pytest.skip("no objects of a build here")
    found = W.functions(OBJECT, "k_mx_rows", tmp_path_factory.mktemp("rows"))
    return {tuple(map(int, re.search(r"ILi(\d)ELi(\d)E", n).groups())): code for n, code in found.items()}


def cut(xt, ks, M, N, K, ncu=256):
    """k_mx_rows_addr.h's: rows of x a tile, tiles, LDS, blocks, workgroups; None: k is too long."""
    steps, rest = (K + 127) // 128, 8 * 2048 + 8 * 4096
    row = 8 * XR[xt] * 2 * (((steps + 1) // 2 + ks - 1) // ks)
    most = min(16, (163840 - rest) // row)
    if most <= 0:
        return None
    tiles = -(-M // most)
    mr = -(-M // tiles)
    blocks = -(-N // (16 * (8 // ks)))
    room = -(-(ncu * (2 if rest + mr * row <= 81920 else 1)) // tiles)
    return mr, tiles, rest + mr * row, blocks, -(-blocks // -(-blocks // room))


def walk(code, xt, ks, M, N, K, less=None, pad=0):
    """less: a buffer that is declared a row shorter than the kernel is told."""
    mr, tiles, lds, blocks, grid = cut(xt, ks, M, N, K)
    ld, wb, xb = (K + 127) // 128 * 4, K // 2, (2 * K, K, K // 2)[xt]
    xld, out = xb + 16 * pad, N + pad
    sizes = {"w": N * wb, "w2": N * wb, "ws": N * ld, "ws2": N * ld, "x": (M - 1) * xld + xb, "xs": M * ld if xt else 0,
             "out": 2 * ((M - 1) * out + N)}
    if less:
        sizes[less] -= {"w": wb, "w2": wb, "ws": ld, "ws2": ld, "x": xld, "xs": ld, "out": 2 * out}[less]
    buffers = {k: (0x200000000000 + (i << 40) + 0x300 * i, n, k == "out") for i, (k, n) in enumerate(sizes.items()) if n}
    at = lambda k: buffers[k][0] if k in buffers else 0  # noqa: E731
    args = struct.pack("<6QQ4I", *map(at, ("w", "w2", "ws", "ws2", "x", "xs")), xld, M, N, K, xt)
    args += struct.pack("<4QQQifI4x", 0, 0, at("out"), 0, 0, out, 2, 1.0, 0) + struct.pack("<3I4x", blocks, 0, mr)
    args += struct.pack("<3I3H", grid, tiles, 1, 512, 1, 1) + bytes(64)
    rng, stores = np.random.default_rng([xt, ks, M, N, K]), {}
    some = lambda n: sorted({0, n - 1})  # noqa: E731
    for block in [(x, y) for y in some(tiles) for x in some(grid)]:
        waves = [W.Wave(code, args, buffers, lds, w, block, rng, stores) for w in range(8)]
        for k, w in enumerate(waves):
            try:
                w.run()
            except W.Fault as f:
                raise W.Fault("workgroup %s, wave %d of %s: %s" % (block, k, (M, N, K), f)) from None
        assert len({w.barriers for w in waves}) == 1
    assert set(stores.values()) == {1}
    assert len(stores) == M * N or tiles > 2 or grid > 2


@pytest.mark.parametrize("xt", [0, 1, 2])
@pytest.mark.parametrize("ks", [8, 4])
def test_every_access_of_the_built_code(forms, xt, ks):
    for M, N, K in SHAPES:
        if cut(xt, ks, M, N, K):
            walk(forms[xt, ks], xt, ks, M, N, K, pad=M % 3)


@pytest.mark.parametrize("less", ["w", "w2", "ws", "ws2", "x", "xs", "out"])
def test_the_walk_sees_a_row_that_is_not_there(forms, less):
    with pytest.raises(W.Fault):
        walk(forms[1, 4], 1, 4, 3, 300, 544, less)


def test_the_walk_sees_a_missing_wait(forms):
    code, jumps = forms[0, 8]
    without = [(op, ops, more) if op != "s_waitcnt" else ("s_nop", ["0"], "") for op, ops, more in code]
    with pytest.raises(W.Fault, match="in flight"):
        walk((without, jumps), 0, 8, 3, 300, 544)
