"""Arrays of the operators over a cache of 8 or 4 bits that share memory, on the CPU: outputs that reach into other arrays are refused, rows of one
array that lie between another's are not."""
import ctypes
import itertools
import os
import subprocess

import numpy as np
import pytest

import qxg
from test_cache_ops_refusals import append, attend
from test_ops_refusals import Fake


@pytest.fixture()
def ctx():
    c = qxg.Context.__new__(qxg.Context)
    c._c, c._err = None, ctypes.create_string_buffer(1024)
    return c


BASE = 1 << 32
Q, KV = (2, 3, 8, 128), (2, 3, 4, 128)          # 4096 and 2048 bytes a token in f32
WIDE = (3 * 16 * 128, 16 * 128, 128, 1)         # rows of a projection: 8 q, 4 k, 4 v heads
K = lambda ptr, strides=None: Fake(KV, strides=strides, ptr=ptr)                     # noqa: E731
C8 = lambda ptr, strides=None: Fake((2, 50, 4, 128), "int8", strides, ptr)           # noqa: E731
C4 = lambda ptr, strides=None: Fake((2, 50, 4, 64), "uint8", strides, ptr)           # noqa: E731
S4 = lambda ptr, strides=None: Fake((2, 50, 4, 4), "uint8", strides, ptr)            # noqa: E731
FREE = "invalid context"
MEET = "share memory"

APPEND = [
    # parts of one projection's rows, in place or not
    (dict(q=Fake(Q, strides=WIDE, ptr=BASE), k=K(BASE + 4096, WIDE), v=K(BASE + 6144, WIDE), q_out=Fake(Q, strides=WIDE, ptr=BASE)), FREE),
    (dict(q=Fake(Q, strides=WIDE, ptr=BASE), k=K(BASE + 4096, WIDE), v=K(BASE + 6144, WIDE)), FREE),
    (dict(k=K(BASE + 4096, WIDE), v=K(BASE + 6144, WIDE), q_out=Fake(Q, strides=WIDE, ptr=BASE)), FREE),
    # q_out begins inside k, ends in it, holds it, lies in it; the same of v
    (dict(k=K(BASE + 4080, WIDE), v=K(BASE + 6144, WIDE), q_out=Fake(Q, strides=WIDE, ptr=BASE)), "q_out and k share memory"),
    (dict(k=K(BASE + 4096, WIDE), v=K(BASE + 6160, WIDE), q_out=Fake(Q, strides=WIDE, ptr=BASE)), "q_out and v share memory"),
    (dict(k=K(BASE), q_out=Fake(Q, ptr=BASE + 16)), "q_out and k share memory"),
    (dict(v=K(BASE), q_out=Fake(Q, ptr=BASE + 2 * 3 * 2048 - 16)), "q_out and v share memory"),
    (dict(v=K(BASE), q_out=Fake(Q, ptr=BASE + 2 * 3 * 2048)), FREE),
    (dict(k=K(BASE + 2 * 3 * 4096), q_out=Fake(Q, ptr=BASE)), FREE),
    (dict(k=K(BASE + 2 * 3 * 4096 - 16), q_out=Fake(Q, ptr=BASE)), "q_out and k share memory"),
    # q moved by less than its size
    (dict(q=Fake(Q, ptr=BASE), q_out=Fake(Q, ptr=BASE + 4096)), "q_out and q share memory"),
    (dict(q=Fake(Q, ptr=BASE), q_out=Fake(Q, ptr=BASE - 16)), "q_out and q share memory"),
    (dict(q=Fake(Q, ptr=BASE), q_out=Fake(Q, ptr=BASE + 2 * 3 * 4096)), FREE),
    # a cache, its scales
    (dict(q_out=Fake(Q, ptr=BASE), k_cache=C8(BASE + 6 * 4096 - 16)), "q_out and k_cache share memory"),
    (dict(q_out=Fake(Q, ptr=BASE), v_cache=C8(BASE - 2 * 50 * 512 + 16)), "q_out and v_cache share memory"),
    (dict(q_out=Fake(Q, ptr=BASE), v_cache=C8(BASE - 2 * 50 * 512)), FREE),
    (dict(q_out=Fake(Q, ptr=BASE), kscale=Fake((2, 50), ptr=BASE + 4)), "q_out and kscale share memory"),
    (dict(q_out=Fake(Q, ptr=BASE), vscale=Fake((2, 50), ptr=BASE - 396)), "q_out and vscale share memory"),
    (dict(q_out=Fake(Q, ptr=BASE), vscale=Fake((2, 50), ptr=BASE - 400)), FREE),
    (dict(k=K(BASE), k_cache=C8(BASE + 4096)), "k_cache and k share memory"),
    (dict(v=K(BASE), vscale=Fake((2, 50), ptr=BASE)), "vscale and v share memory"),
    (dict(k_cache=C8(BASE), v_cache=C8(BASE + 16)), "k_cache and v_cache share memory"),
    (dict(k_cache=C8(BASE), v_cache=C8(BASE + 2 * 50 * 512)), FREE),
    (dict(kscale=Fake((2, 50), ptr=BASE), vscale=Fake((2, 50), ptr=BASE + 4)), "kscale and vscale share memory"),
    (dict(k_cache=C8(BASE), kscale=Fake((2, 50), ptr=BASE + 512)), "k_cache and kscale share memory"),
    # K and V of a position side by side; of a sequence one after the other; positions before sequences; too near
    (dict(k_cache=C8(BASE, (50 * 1024, 1024, 128, 1)), v_cache=C8(BASE + 512, (50 * 1024, 1024, 128, 1))), FREE),
    (dict(k_cache=C8(BASE, (2 * 50 * 512, 512, 128, 1)), v_cache=C8(BASE + 50 * 512, (2 * 50 * 512, 512, 128, 1))), FREE),
    (dict(k_cache=C8(BASE, (1024, 2048, 128, 1)), v_cache=C8(BASE + 512, (1024, 2048, 128, 1))), FREE),
    (dict(k_cache=C8(BASE, (2 * 50 * 512, 512, 128, 1)), v_cache=C8(BASE + 49 * 512, (2 * 50 * 512, 512, 128, 1))), "k_cache and v_cache share memory"),
    (dict(k_cache=C8(BASE, (1024, 2048, 128, 1)), v_cache=C8(BASE + 528, (1024, 2048, 128, 1))), "k_cache and v_cache share memory"),
    # a row of 4 bits with all that belongs to a position: 256 + 256 + 16 + 16 bytes
    (dict(bits=4, k_cache=C4(BASE, (50 * 544, 544, 64, 1)), v_cache=C4(BASE + 256, (50 * 544, 544, 64, 1)), kscale=S4(BASE + 512, (50 * 544, 544, 4, 1)),
          vscale=S4(BASE + 528, (50 * 544, 544, 4, 1))), FREE),
    (dict(bits=4, k_cache=C4(BASE, (50 * 544, 544, 64, 1)), v_cache=C4(BASE + 256, (50 * 544, 544, 64, 1)), kscale=S4(BASE + 508, (50 * 544, 544, 4, 1)),
          vscale=S4(BASE + 528, (50 * 544, 544, 4, 1))), "v_cache and kscale share memory"),
    # between each other's rows with other strides: not looked into
    (dict(k_cache=C8(BASE, (51 * 1024, 1024, 128, 1)), v_cache=C8(BASE + 512, (51 * 1024, 1024, 128, 1)), q_out=Fake(Q, strides=(3 * 8192, 8192, 128, 1), ptr=BASE + 512)),
     "q_out and k_cache share memory"),
]


@pytest.mark.parametrize("change,message", APPEND)
def test_kv_append(ctx, change, message):
    with pytest.raises(qxg.QxgError, match=message):
        ctx.kv_append(**append(**change))


ATTEND = [
    (dict(out=Fake(Q, ptr=BASE), q=Fake(Q, ptr=BASE + 16)), "out and q share memory"),
    (dict(out=Fake(Q, ptr=BASE), q=Fake(Q, ptr=BASE - 6 * 4096 + 16)), "out and q share memory"),
    (dict(out=Fake(Q, ptr=BASE), q=Fake(Q, ptr=BASE - 6 * 4096)), FREE),
    (dict(out=Fake(Q, strides=(3 * 2048, 2048, 128, 1), ptr=BASE), q=Fake(Q, strides=(3 * 2048, 2048, 128, 1), ptr=BASE + 4096)), FREE),
    (dict(out=Fake(Q, ptr=BASE), k=C8(BASE + 16)), "out and k share memory"),
    (dict(out=Fake(Q, ptr=BASE), v=C8(BASE - 16)), "out and v share memory"),
    (dict(out=Fake(Q, ptr=BASE), kscale=Fake((2, 50), ptr=BASE)), "out and kscale share memory"),
    (dict(out=Fake(Q, ptr=BASE), vscale=Fake((2, 50), ptr=BASE + 6 * 4096)), FREE),
    (dict(out=Fake(Q, ptr=BASE), lse=Fake((2, 3, 8), ptr=BASE + 6 * 4096 - 4)), "out and lse share memory"),
    (dict(lse=Fake((2, 3, 8), ptr=1 << 23)), "lse and kscale share memory"),
]


@pytest.mark.parametrize("change,message", ATTEND)
def test_cache_attention(ctx, change, message):
    with pytest.raises(qxg.QxgError, match=message):
        ctx.cache_attention(**attend(**change))


@pytest.fixture(scope="module")
def meet(root, tmp_path_factory):
    at = tmp_path_factory.mktemp("rows_meet")
    (at / "rows.cpp").write_text('#include "qxg_ops_host.h"\nextern "C" int meet(uint64_t p, uint64_t a, uint64_t na, uint64_t b, uint64_t nb, uint64_t row, uint64_t q, '
                                 'uint64_t c, uint64_t nc, uint64_t d, uint64_t nd, uint64_t width) {\n'
                                 'return rows_meet({(void *)p, "", a, na, b, nb, row}, {(void *)q, "", c, nc, d, nd, width}); }\n')
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-shared", "-fPIC", "-I/opt/rocm/include", "-I" + os.path.join(root, "include"),
                    "-I" + os.path.join(root, "qx-mini-c_amd", "csrc"), str(at / "rows.cpp"), "-o", str(at / "rows.so")], check=True, capture_output=True)
    f = ctypes.CDLL(str(at / "rows.so")).meet
    f.argtypes = [ctypes.c_uint64] * 12
    return f


def test_rows_that_share_memory_are_found(meet):
    """Small layouts against their bytes: exactly, of like strides; of unlike ones none that does is missed."""
    rng = np.random.default_rng(0)
    found = 0
    for a, b, na, nb in itertools.product((0, 3, 4, 7, 12, 20, 31), (0, 2, 5, 6, 11, 40), (1, 2, 4), (1, 3)):
        for n in range(8):
            wx, wy, d = int(rng.integers(1, 6)), int(rng.integers(1, 6)), int(rng.integers(-90, 90))
            c, e, nc, nd = (a, b, na, nb) if n < 4 else (a, b, *(int(rng.integers(1, 5)) for _ in range(2))) if n < 6 else (*(int(rng.integers(0, 30)) for _ in range(2)), na, nb)
            x = {1000 + i * a + j * b + t for i in range(na) for j in range(nb) for t in range(wx)}
            y = {1000 + d + i * c + j * e + t for i in range(nc) for j in range(nd) for t in range(wy)}
            got, want = bool(meet(1000, a, na, b, nb, wx, 1000 + d, c, nc, e, nd, wy)), bool(x & y)
            assert got == want if n < 6 else got >= want, (a, b, na, nb, c, e, nc, nd, wx, wy, d)
            found += want
    assert found > 300


def test_rows_far_apart(meet):
    """Strides and counts as large as a call's: 2^20 tokens, rows 2^26 bytes apart, sequences 2^46."""
    n, row = 1 << 20, 1 << 26
    args = (65535, row, n, 512)
    assert not meet(1 << 20, 1 << 46, *args, (1 << 20) + 512, 1 << 46, *args)
    assert meet(1 << 20, 1 << 46, *args, (1 << 20) + 511, 1 << 46, *args)
    assert meet(1 << 20, 1 << 46, *args, (1 << 20) + (9 << 46) + 77 * row - 511, 1 << 46, *args)
    assert not meet(1 << 20, 1 << 46, *args, (1 << 20) + (9 << 46) + 77 * row - 512, 1 << 46, *args)
