"""The angles of rows at positions of their own, at the models' rates, against the table of launch_rope_table."""
import ctypes as C

import numpy as np
import pytest

from test_q4_store_gpu import MODELS, _nova

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("model", MODELS)
def test_angles_at_the_models_rates(model):
    """The table's angle is made in fp32.  Its exponent of 2, up to log2(10^6) = 19.94, is a product of a rounded
    logarithm and rounded itself, so its rate is off by up to 19.94 ln 2 2^-23 + 2^-24 of itself and the product with the
    position by another 2^-24; the rates here are off by 2^-24, their angles exact.  Cosines and sines move by no more
    than the angle, and each side rounds them to 2^-25."""
    import nova_amd
    nova, rows, half = _nova(model), 4096, 64
    freq, magnitude = np.zeros(half, np.float32), C.c_double()
    cfg = nova_amd.RopeCfg(2 * half, nova_amd.ROPE_PLAIN, 1e6, 1.0, 0, 1, 32)
    assert nova.nova_rope_freqs(C.byref(cfg), freq.ctypes.data_as(C.POINTER(C.c_float)), C.byref(magnitude)) == half
    pos = np.arange(rows, dtype=np.int32)
    dp, df = nova.upload(pos), nova.upload(freq)
    here, table = ([nova.alloc(rows * half * 4) for _ in range(2)] for _ in range(2))
    nova.launch_rope_angles(dp.ptr, rows, df.ptr, 2 * half, magnitude.value, *(x.ptr for x in here), None)
    nova.launch_rope_table(*(x.ptr for x in table), None)
    nova.dev_sync()
    bound = pos[:, None] * freq.astype(np.float64) * (19.94 * np.log(2) * 2.0 ** -23 + 3 * 2.0 ** -24) * 1.001 + 2.0 ** -24
    for a, b in zip(here, table):
        a, b = (x.numpy((rows, half), np.float32).astype(np.float64) for x in (a, b))
        assert (np.abs(a - b) <= bound).all()
        assert np.abs(a - b).max() > 0                       # (other pairs than the first are compared)
