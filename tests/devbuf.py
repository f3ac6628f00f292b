"""Device buffers for tests of entry points that work on the caller's memory, from the HIP runtime the
library itself links (ctypes), and the storage types as numpy arrays."""

import ctypes

import numpy as np

from zenjpegai_amd import _lib

# Half a step of a rounding, relative to the value.
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
RAW = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}
_H2D, _D2H = 1, 2
_hip_lib = None


def hip():
    global _hip_lib
    if _hip_lib is None:
        _lib.lib()  # loads libzjai_hip.so and with it the HIP runtime it links
        h = ctypes.CDLL("libamdhip64.so.7")
        h.hipMalloc.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_size_t]
        h.hipFree.argtypes = [ctypes.c_void_p]
        h.hipMemcpy.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
        for f in (h.hipMalloc, h.hipFree, h.hipMemcpy, h.hipDeviceSynchronize):
            f.restype = ctypes.c_int
        _hip_lib = h
    return _hip_lib


def to_raw(x, prec):
    """float32 values rounded to the storage type, to nearest even."""
    x = np.ascontiguousarray(x, np.float32)
    if prec != "bf16":
        return x.astype(RAW[prec])
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_raw(raw, prec):
    """float64 values of a storage array."""
    if prec != "bf16":
        return raw.astype(np.float64)
    return (raw.astype(np.uint32) << np.uint32(16)).view(np.float32).astype(np.float64)


class DevBuf:
    """A device copy of an array, `offset` bytes into its allocation."""

    def __init__(self, arr, offset=0):
        arr = np.ascontiguousarray(arr)
        self.shape, self.dtype = arr.shape, arr.dtype
        self._base = ctypes.c_void_p()
        assert hip().hipMalloc(ctypes.byref(self._base), arr.nbytes + offset + 256) == 0
        self.address = self._base.value + offset
        self.put(arr)

    def data_ptr(self):
        return self.address

    def put(self, arr):
        arr = np.ascontiguousarray(arr)
        assert arr.shape == self.shape and arr.dtype == self.dtype
        if arr.nbytes:
            assert hip().hipMemcpy(self.address, arr.ctypes.data, arr.nbytes, _H2D) == 0
        assert hip().hipDeviceSynchronize() == 0

    def get(self):
        assert hip().hipDeviceSynchronize() == 0
        a = np.empty(self.shape, self.dtype)
        if a.nbytes:
            assert hip().hipMemcpy(a.ctypes.data, self.address, a.nbytes, _D2H) == 0
        return a

    def __del__(self):
        if _hip_lib is not None and self._base:
            _hip_lib.hipFree(self._base)
