"""GPU: selective scans of as many sequences as are promised to be accepted, with positions and without."""

import ctypes

import numpy as np
import pytest

from devbuf import DevBuf, hip
from test_gpu_selective_scan import Case, eng, run  # noqa: F401  (eng: the fixture)
from zenjpegai_amd import _lib, nn

pytestmark = pytest.mark.gpu
MOST = 2 ** 20


def test_as_many_sequences_as_are_accepted(eng):  # noqa: F811
    k = Case(41, "f32", MOST, 1, 1, 1)
    run(eng, k, only=[0, 12345, MOST - 1])
    x = DevBuf(np.zeros(1, np.float32))
    with pytest.raises(_lib.HipError) as e:
        nn.selective_scan_noalloc(eng, nn.selective_scan_desc("f32", x, x, x, x, DevBuf(np.zeros(1, np.float32)), channels=1, state_dim=1,
                                                              sequences=MOST + 1, length=1, a=x))
    assert e.value.kind == "LimitExceeded"


@pytest.mark.parametrize("channels,n", [(65, 9), (128, 16)])
def test_no_positions_of_as_many(eng, channels, n):  # noqa: F811
    """Without positions every state is the absent one's zeros."""
    size, a = ctypes.c_size_t(4 * MOST * channels * n), DevBuf(np.zeros((channels, n), np.float32))
    states = ctypes.c_void_p()
    assert hip().hipMalloc(ctypes.byref(states), size) == 0
    try:
        assert hip().hipMemset(states, 0xFF, size) == 0 and hip().hipDeviceSynchronize() == 0
        nn.selective_scan_noalloc(eng, nn.selective_scan_desc("f32", None, None, None, None, None, channels=channels, state_dim=n,
                                                              sequences=MOST, length=0, a=a, state_out=states.value))
        eng.sync()
        for at in (0, MOST // 2, MOST - 1):
            one = np.empty((channels, n), np.float32)
            assert hip().hipMemcpy(one.ctypes.data, ctypes.c_void_p(states.value + at * one.nbytes), one.nbytes, 2) == 0
            assert (one == 0).all()
    finally:
        assert hip().hipFree(states) == 0
