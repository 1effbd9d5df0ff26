"""The host side of the operators on device memory on the CPU: ops_host.cpp compiled with a runtime of its own that writes
down what is asked of it."""
import ctypes
import os
import subprocess
import threading

import pytest

import qxg
from test_gpu_tree_attention_long import PLANS
from test_ops_refusals import Fake, big, logits, tree

INVALID_VALUE, CONFIGURATION, UNKNOWN = 1, 9, 999      # hipErrorInvalidValue, ...InvalidConfiguration, ...Unknown


class Seen(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("last", "fail", "unknown", "device", "launches", "waits", "waits_that_fail")] + [
        (n, ctypes.c_uint32) for n in ("wide", "splits", "tiles", "wgs", "kept", "packed")]


@pytest.fixture(scope="module")
def lib(root, tmp_path_factory):
    out = tmp_path_factory.mktemp("ops_host") / "ops_host.so"
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I/opt/rocm/include",
                    "-I" + os.path.join(root, "include"), "-I" + os.path.join(root, "qx-mini-c_amd", "csrc"),
                    os.path.join(root, "tests", "ops_host.cpp"), "-o", str(out)], check=True, capture_output=True)
    lib = ctypes.CDLL(str(out))
    for name in ("qxg_tree_attention", "qxg_kv_select", "qxg_kv_compact", "qxg_adjust_logits"):
        getattr(lib, name).argtypes = getattr(qxg._g, name).argtypes
    return lib


@pytest.fixture()
def host(lib, monkeypatch):
    """(a context whose calls go to the library, what its runtime has seen)"""
    monkeypatch.setattr(qxg, "_g", lib)
    seen = Seen.in_dll(lib, "seen")
    ctypes.memset(ctypes.addressof(seen), 0, ctypes.sizeof(seen))
    c = qxg.Context.__new__(qxg.Context)
    c._c, c._err = ctypes.c_void_p(1), ctypes.create_string_buffer(1024)
    yield c, seen
    c._c = None      # (nothing to close)


def calls(c):
    yield c.tree_attention, tree()
    yield c.kv_select, dict(account=Fake((3, 40)), lens=Fake((3,), "int32"), keep=Fake((3, 10), "int32"), kept=Fake((3,), "int32"))
    yield c.kv_compact, dict(k=Fake((3, 40, 64), "int8"), v=Fake((3, 40, 64), "int8"), kscale=Fake((3, 40)), vscale=Fake((3, 40)),
                             keep=Fake((3, 10), "int32"), kept=Fake((3,), "int32"), workspace=big())
    yield c.adjust_logits, logits()


def test_calls(host):
    c, seen = host
    for n, (call, args) in enumerate(calls(c), 1):
        call(**args, wait=False)
        assert (seen.launches, seen.waits, seen.last) == (n, 0, 0)
    for call, args in calls(c):
        call(**args)
    assert seen.waits == 4


def test_an_error_that_the_caller_has_yet_to_ask_for_stays(host):
    c, seen = host
    seen.last = UNKNOWN
    for call, args in calls(c):
        call(**args)
        assert seen.last == UNKNOWN


def test_a_failed_launch_is_reported_once(host):
    """By the call, not by the caller's next question; but an error from before it leaves one."""
    c, seen = host
    seen.fail = CONFIGURATION
    for call, args in calls(c):
        with pytest.raises(qxg.QxgError, match="configuration"):
            call(**args, wait=False)
        assert seen.last == 0 and seen.waits == 0
    seen.last = UNKNOWN
    for call, args in calls(c):
        with pytest.raises(qxg.QxgError, match="configuration"):
            call(**args, wait=False)
        assert seen.last != 0


def test_a_failed_launch_waits_for_the_kernels_before_it(host):
    c, seen = host
    seen.fail = CONFIGURATION
    for n, (call, args) in enumerate(calls(c), 1):
        with pytest.raises(qxg.QxgError, match="configuration"):
            call(**args)
        assert seen.waits == n


def test_a_wait_that_fails_is_reported(host):
    c, seen = host
    seen.waits_that_fail = UNKNOWN
    for call, args in calls(c):
        with pytest.raises(qxg.QxgError, match="unknown"):
            call(**args)
        assert seen.last == 0


def test_memory_of_another_runtime_is_refused(host):
    c, seen = host
    seen.unknown = 1
    for call, args in calls(c):
        with pytest.raises(qxg.QxgError, match="is not device memory of this library's HIP runtime"):
            call(**args)
        assert seen.last == 0 and seen.launches == 0
    seen.last = UNKNOWN
    for call, args in calls(c):
        with pytest.raises(qxg.QxgError, match="is not device memory"):
            call(**args)
        assert seen.last != 0


def test_the_callers_device_is_current_again(host):
    c, seen = host
    seen.device = 3
    for call, args in calls(c):
        call(**args)
        assert seen.device == 3
    seen.fail = CONFIGURATION
    for call, args in calls(c):
        with pytest.raises(qxg.QxgError):
            call(**args)
        assert seen.device == 3


def test_threads_have_their_own_messages(monkeypatch):
    """A call that fails while another thread's call on the same context fails, too, has its own message."""
    c = qxg.Context.__new__(qxg.Context)
    c._c, c._err = None, ctypes.create_string_buffer(1024)
    args = dict(account=Fake((3, 40)), lens=Fake((3,), "int32"), keep=Fake((3, 10), "int32"), kept=Fake((3,), "int32"))
    seen = []

    def one():
        with pytest.raises(qxg.QxgError) as e:
            c.kv_select(**args)
        seen.append(str(e.value))

    class Calls:
        left = ["the first's", "the second's"]

        def qxg_kv_select(self, ctx, packed, stream, wait, err, n):
            err.value = self.left.pop(0).encode()
            if self.left:
                other = threading.Thread(target=one)
                other.start()
                other.join()
            return 0

    monkeypatch.setattr(qxg, "_g", Calls())
    one()
    assert seen == ["the second's", "the first's"]


def splits_of(seen, case):
    """(chunks, splits) of every sequence, as the kernels share them out."""
    group = case["heads"] // case["kv_heads"]
    counts = case.get("counts") or (case["nodes"],) * len(case["lens"])
    chunks = [max(1, -(-(n + c) // 32)) for n, c in zip(case["lens"], counts)]
    if seen.splits == 1 or len(chunks) > 64:
        return [(n, seen.splits) for n in chunks]
    if len(chunks) == 1:
        return [(chunks[0], min(chunks[0], seen.splits))]
    busy = sum(n * -(-c * group // (128 if seen.wide else 32)) for n, c in zip(chunks, counts))
    return [(n, min(n, max(1, int(n * seen.splits * min(seen.wgs / busy, 2 / sum(chunks)))))) for n in chunks]


@pytest.mark.parametrize("name", sorted(PLANS))
def test_plans(host, name):
    """The cases of test_gpu_tree_attention_long.py reach the kernels and loops that they are meant for."""
    c, seen = host
    case, wide, splits, least = PLANS[name]
    batch, nodes, dim, longest = case.get("batch", 1), case["nodes"], case.get("dim", 128), max(case["lens"])
    positions = longest + nodes + 3
    cache, scales, q = (batch, positions, case["kv_heads"], dim), Fake((batch, positions)), (batch, nodes, case["heads"], dim)
    c.tree_attention(Fake(q), Fake(cache, "int8"), Fake(cache, "int8"), scales, scales, Fake((batch,), "int32"), Fake(q, ptr=1 << 40), max_len=longest,
                     workspace=big())
    assert bool(seen.wide) == wide
    assert (seen.splits == 1) == (splits == 1)
    assert max(n // s for n, s in splits_of(seen, case)) >= least
