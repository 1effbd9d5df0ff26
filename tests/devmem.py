"""Device arrays for the tests of the operators on device memory: numpy data in memory of the HIP
runtime that libqxg.so uses (not torch's, which may be another one in the same process)."""
import ctypes

import numpy as np

import qxg  # noqa: F401  (loads libqxg.so and with it the runtime)

_NP = {"float32": np.float32, "float16": np.float16, "bfloat16": np.uint16, "int32": np.int32, "int8": np.int8, "uint8": np.uint8}


class Hip:
    """The runtime's calls that the tests make; every error is raised."""

    def __init__(self):
        self.lib = ctypes.CDLL("libamdhip64.so.7")
        self.held = []

    def __getattr__(self, name):
        f = getattr(self.lib, name)

        def call(*args):
            rc = f(*args)
            assert rc == 0, f"{name}: {rc}"
        return call

    def malloc(self, n):
        p = ctypes.c_void_p()
        self.hipMalloc(ctypes.byref(p), ctypes.c_size_t(max(n, 16)))
        self.held.append(p.value)
        return p.value

    def release(self):
        for p in self.held:
            self.lib.hipFree(ctypes.c_void_p(p))
        self.held = []

    def put(self, a, dtype=None):
        return Array(self, np.ascontiguousarray(a), dtype)

    def workspace(self, n):
        return self.put(np.zeros(max(n, 16), np.uint8))

    def sync(self):
        self.hipDeviceSynchronize()

    def stream(self):
        s = ctypes.c_void_p()
        self.hipStreamCreateWithFlags(ctypes.byref(s), 1)
        return s.value

    def capture(self, stream, work):
        """The graph of what work() queues on the stream, ready to be launched."""
        graph, ready = ctypes.c_void_p(), ctypes.c_void_p()
        self.hipStreamBeginCapture(ctypes.c_void_p(stream), 0)
        work()
        self.hipStreamEndCapture(ctypes.c_void_p(stream), ctypes.byref(graph))
        self.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0))
        return ready


class Array:
    def __init__(self, hip, a, dtype=None, ptr=None):
        self.hip, self.shape, self.np = hip, a.shape, a.dtype
        self.dtype = dtype or str(a.dtype)
        assert np.dtype(_NP[self.dtype]) == a.dtype
        self.strides = tuple(s // a.itemsize for s in a.strides)
        self.base, self.ptr, self.nbytes = None, ptr, a.nbytes
        if ptr is None:
            self.ptr = hip.malloc(a.nbytes)
            self.set(a)

    def set(self, a):
        a = np.ascontiguousarray(a)
        assert a.shape == self.shape and a.dtype == self.np
        if a.nbytes:
            self.hip.hipMemcpy(ctypes.c_void_p(self.ptr), a.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(a.nbytes), 1)

    def get(self):
        a = np.empty(self.shape, self.np)
        if a.nbytes:
            self.hip.hipMemcpy(a.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(self.ptr), ctypes.c_size_t(a.nbytes), 2)
        return a

    def view(self, offset, shape, strides):
        """Elements offset + sum(i * stride); read it through the array that it is a view of."""
        v = Array.__new__(Array)
        v.hip, v.shape, v.np, v.dtype, v.strides = self.hip, tuple(shape), self.np, self.dtype, tuple(strides)
        v.ptr, v.base = self.ptr + offset * self.np.itemsize, self
        return v

    def data_ptr(self):
        return self.ptr

    def stride(self):
        return self.strides


def to_bf16(x):
    """float32 rounded to bfloat16 (to nearest, ties to even), as its 16 bits."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    nan = np.isnan(x)
    r[nan] = ((u[nan] >> 16) | 0x40).astype(np.uint16)
    return r


def encode(x, kind):
    """(array as it is stored, its dtype name) of float values in one of the value types."""
    if kind == "f32":
        return np.asarray(x, np.float32), "float32"
    if kind == "f16":
        with np.errstate(over="ignore"):
            return np.asarray(x, np.float32).astype(np.float16), "float16"
    return to_bf16(np.asarray(x, np.float32)), "bfloat16"


def decode(a, kind):
    if kind == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # a rounding's error relative to the value
