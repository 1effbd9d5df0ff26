"""Errors around the operators on device memory, with the real runtime: a caller's pending error is the caller's."""
import ctypes

import numpy as np
import pytest

import qxg
from test_gpu_kv_evict import chosen, ctx, hip  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu
NO_DEVICE = 101      # hipErrorInvalidDevice


def test_a_pending_error_of_the_caller_stays(ctx, hip):  # noqa: F811
    lib = hip.lib
    account = np.arange(40, dtype=np.float32)[None]
    keep, kept = hip.put(np.zeros((1, 10), np.int32)), hip.put(np.zeros(1, np.int32))
    acc, lens = hip.put(account), hip.put(np.array([40], np.int32))
    lib.hipGetLastError()
    assert lib.hipSetDevice(9999) == NO_DEVICE and lib.hipPeekAtLastError() == NO_DEVICE
    ctx.kv_select(acc, lens, keep, kept, sinks=2)
    assert lib.hipGetLastError() == NO_DEVICE and lib.hipGetLastError() == 0
    assert np.array_equal(keep.get()[0], chosen(account[0], 40, 10, 2, 0))


def test_a_refused_pointer_leaves_no_error(ctx, hip):  # noqa: F811
    lib = hip.lib
    keep, kept, lens = hip.put(np.zeros((1, 10), np.int32)), hip.put(np.zeros(1, np.int32)), hip.put(np.array([40], np.int32))
    mine = np.zeros((1, 40), np.float32)
    host = keep.view(0, (1, 40), (40, 1))
    host.ptr, host.dtype = mine.ctypes.data_as(ctypes.c_void_p).value, "float32"
    lib.hipGetLastError()
    with pytest.raises(qxg.QxgError, match="account is not"):
        ctx.kv_select(host, lens, keep, kept)
    assert lib.hipGetLastError() == 0
