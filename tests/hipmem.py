"""Device memory for tests through the HIP runtime that the library itself uses."""
import ctypes as C

import numpy as np

FENCE = 64  # bytes of 0xA5 on both sides of every allocation's data


class Hip:
    def __init__(self):
        from detllm_amd._lib import lib  # loads libdetllm_amd.so and its HIP runtime

        self.dtl = lib
        rt = self.rt = C.CDLL("libamdhip64.so.7")
        rt.hipMalloc.argtypes = [C.POINTER(C.c_void_p), C.c_size_t]
        rt.hipFree.argtypes = [C.c_void_p]
        rt.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
        rt.hipStreamCreate.argtypes = [C.POINTER(C.c_void_p)]
        rt.hipStreamDestroy.argtypes = [C.c_void_p]
        rt.hipStreamSynchronize.argtypes = [C.c_void_p]
        rt.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
        rt.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
        rt.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
        rt.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
        rt.hipGraphExecDestroy.argtypes = [C.c_void_p]
        rt.hipGraphDestroy.argtypes = [C.c_void_p]
        self.bufs = []
        self.stream = C.c_void_p()
        assert rt.hipStreamCreate(C.byref(self.stream)) == 0

    def sync(self):
        assert self.rt.hipStreamSynchronize(self.stream) == 0

    def put(self, arr, offset=0):
        """Device address of a fenced copy of arr, `offset` bytes off a 16-byte boundary."""
        arr = np.ascontiguousarray(arr)
        raw = np.full(2 * FENCE + offset + arr.nbytes, 0xA5, np.uint8)
        raw[FENCE + offset:FENCE + offset + arr.nbytes] = arr.reshape(-1).view(np.uint8)
        p = C.c_void_p()
        assert self.rt.hipMalloc(C.byref(p), raw.nbytes) == 0
        assert self.rt.hipMemcpy(p, raw.ctypes.data, raw.nbytes, 1) == 0
        self.bufs.append(p)
        return p.value + FENCE + offset

    def fill(self, addr, arr):
        arr = np.ascontiguousarray(arr)
        assert self.rt.hipMemcpy(addr, arr.ctypes.data, arr.nbytes, 1) == 0

    def get(self, addr, dtype, shape):
        """The array at a `put` address; the fences around it must be whole."""
        out = np.empty(shape, dtype)
        raw = np.empty(2 * FENCE + out.nbytes, np.uint8)
        assert self.rt.hipMemcpy(raw.ctypes.data, addr - FENCE, raw.nbytes, 2) == 0
        assert (raw[:FENCE] == 0xA5).all() and (raw[FENCE + out.nbytes:] == 0xA5).all(), "written out of range"
        out.reshape(-1).view(np.uint8)[:] = raw[FENCE:FENCE + out.nbytes]
        return out

    def drop(self):
        """Frees what was put so far."""
        for p in self.bufs:
            self.rt.hipFree(p)
        self.bufs = []

    def close(self):
        self.drop()
        self.rt.hipStreamDestroy(self.stream)
