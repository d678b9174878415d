"""dbias of more columns than one launch's 2^32 threads take."""
import numpy as np
import pytest

import ffn_ref as R
import gpu_util as G
from test_gpu_ffn import ok

pytestmark = pytest.mark.gpu

SPAN = 1 << 27                                                      # columns of 2^32 threads, 32 a column


@pytest.mark.parametrize("M,N", [(1, SPAN), (2, SPAN + 75)])
def test_bias_gradient_of_very_many_columns(ghip, M, N):
    rng = np.random.default_rng(M)
    row = rng.integers(0x3F00, 0x4080, 1 << 20, dtype=np.uint16)    # 0.5..4, either sign below
    row |= rng.integers(0, 2, row.size, dtype=np.uint16) << 15
    dy = np.tile(row, -(-M * N // row.size))[:M * N].reshape(M, N)
    dd, db = G.dev(dy), G.dev(np.full(N + 64, 0x7E57, np.uint16))
    ok(ghip, ghip.apus_ghip_bf16_linear_ep_backward_dev(None, None, None, G.vp(dd), None, None, G.vp(db), M, N, 8, 0, 0, 0, R.NONE, None,
                                                         0, None))
    got = G.host(db, np.uint16, (N + 64,))
    dd.close()
    db.close()
    f = lambda b: (b.astype(np.uint32) << 16).view(np.float32)      # noqa: E731
    assert np.all(got[N:] == 0x7E57)
    if M == 1:
        assert np.array_equal(got[:N], dy[0])
        return
    want = f(dy[0]) + f(dy[1])                                      # exact in f32: 8 bits each, within 2^3
    assert np.all(np.abs(f(got[:N]) - want) <= 2.0 ** -8 * np.abs(want))
