"""What the operators on device memory refuse, before any device work: on the CPU, without a context.  A
call whose arguments are all right gets as far as "invalid context" there."""
import ctypes

import numpy as np
import pytest

import qxg


class Fake:
    """A device array by its description alone; nothing reads its address."""

    def __init__(self, shape, dtype="float32", strides=None, ptr=1 << 20):
        self.shape, self.dtype, self.ptr = tuple(shape), dtype, ptr
        self.strides = strides or qxg._dense(self.shape)

    def data_ptr(self):
        return self.ptr

    def stride(self):
        return self.strides


@pytest.fixture()
def ctx():
    c = qxg.Context.__new__(qxg.Context)
    c._c, c._err = None, ctypes.create_string_buffer(1024)
    return c


def big(n=1 << 30):
    return Fake((n,), "uint8")


def tree(**kw):
    a = dict(q=Fake((2, 3, 8, 128)), k=Fake((2, 50, 4, 128), "int8"), v=Fake((2, 50, 4, 128), "int8"), kscale=Fake((2, 50)), vscale=Fake((2, 50)),
             lens=Fake((2,), "int32"), out=Fake((2, 3, 8, 128), ptr=1 << 21), mask=Fake((2, 3, 1), "int32"), counts=Fake((2,), "int32"), lse=Fake((2, 3, 8)),
             account=Fake((2, 50)), workspace=big())
    a.update(kw)
    return a


TREE_BYTES = qxg._tree_workspace((2, 3, 8, 128), (2, 50, 4, 128), None, True)


@pytest.mark.parametrize("change,message", [
    ({}, "invalid context"),
    (dict(q=Fake((2, 3, 8, 128), "int32")), "dtype int32"),
    (dict(q=Fake((2, 3, 8, 96)), k=Fake((2, 50, 4, 96), "int8"), v=Fake((2, 50, 4, 96), "int8"), out=Fake((2, 3, 8, 96))), "dim must be 64 or 128"),
    (dict(q=Fake((2, 3, 8, 64))), "q has the dimensions"),
    (dict(q=Fake((3, 3, 8, 128))), "q has the dimensions"),
    (dict(q=Fake((2, 3, 6, 128)), out=Fake((2, 3, 6, 128)), lse=None), "heads must be a multiple of kv_heads"),
    (dict(q=Fake((2, 1025, 8, 128)), out=Fake((2, 1025, 8, 128)), lse=None, mask=None), "nodes must be between 1 and 1024"),
    (dict(q=Fake((2, 0, 8, 128)), out=Fake((2, 0, 8, 128)), lse=None, mask=None), "nodes must be between 1 and 1024"),
    (dict(q=Fake((2, 3, 8, 128), ptr=(1 << 20) + 8)), "q is not aligned to 16 bytes"),
    (dict(q=Fake((2, 3, 8, 128), strides=(3 * 1026, 1026, 128, 1))), "multiples of 16 bytes"),
    (dict(q=Fake((2, 3, 8, 128), strides=(8 * 3 * 128, 128, 3 * 128, 1))), "not contiguous"),
    (dict(k=Fake((2, 50, 4, 128), "int8", strides=(50 * 520, 520, 128, 1)), v=Fake((2, 50, 4, 128), "int8", strides=(50 * 520, 520, 128, 1))),
     "multiples of 16 bytes"),
    (dict(k=Fake((2, 50, 4, 128), "int8", strides=(50 * 528, 528, 128, 1))), "different strides"),
    (dict(v=Fake((2, 51, 4, 128), "int8", strides=(50 * 512, 512, 128, 1))), "v has shape"),
    (dict(out=Fake((2, 3, 8, 128), "float16")), "out has dtype"),
    (dict(kscale=Fake((2, 49), strides=(50, 1))), "kscale has shape"),
    (dict(vscale=Fake((2, 50), strides=(60, 1))), "different strides"),
    (dict(mask=Fake((2, 3, 2), "int32")), "mask has shape"),
    (dict(lens=Fake((2,), "int8")), "lens has dtype"),
    (dict(lens=None), "lens is NULL"),
    (dict(out=Fake((2, 3, 8, 128), ptr=0)), "out is NULL"),
    (dict(workspace=None, lse=None), f"the workspace holds 0 bytes; this call needs {TREE_BYTES}"),
    (dict(workspace=big(TREE_BYTES - 1), lse=None), f"the workspace holds {TREE_BYTES - 1} bytes; this call needs {TREE_BYTES}"),
    (dict(workspace=big(TREE_BYTES), lse=None), "invalid context"),
    (dict(k=Fake((2, 50, 4, 128), "int8", strides=(1 << 34, 1 << 26, 128, 1)), v=Fake((2, 50, 4, 128), "int8", strides=(1 << 34, 1 << 26, 128, 1))),
     "row stride of k and v must be below 2\\^26"),
    (dict(workspace=Fake((300,), "uint8", ptr=(1 << 20) + 8)), "workspace is not aligned to 16 bytes"),
    (dict(out=Fake((2, 3, 8, 128), strides=(0, 1024, 128, 1))), "rows of out overlap"),
    (dict(out=Fake((2, 3, 8, 128), strides=(3 * 1024, 512, 128, 1))), "rows of out overlap"),
    (dict(out=Fake((2, 3, 8, 128), strides=(1024, 2048, 128, 1), ptr=1 << 21)), "invalid context"),
    (dict(out=Fake((2, 3, 8, 128))), "out must be another array than q"),
    (dict(account=Fake((2, 50), strides=(0, 1))), "accounts overlap"),
    (dict(scale=float("nan")), "scale must be positive and finite"),
    (dict(scale=0.0), "scale must be positive and finite"),
    (dict(decay=float("inf")), "decay must be finite"),
])
def test_tree_attention(ctx, change, message):
    with pytest.raises((qxg.QxgError, ValueError), match=message):
        ctx.tree_attention(**tree(**change))


def test_tree_attention_small_calls_need_no_workspace(ctx):
    with pytest.raises(qxg.QxgError, match="invalid context"):
        ctx.tree_attention(**tree(workspace=None, account=None))


@pytest.mark.parametrize("change,message", [
    ({}, "invalid context"),
    (dict(sinks=6, recent=5), "sinks \\+ recent exceed the budget"),
    (dict(sinks=2 ** 32 - 1, recent=2), "sinks \\+ recent exceed the budget"),
    (dict(keep=Fake((3, 0), "int32")), "budget must be positive"),
    (dict(keep=Fake((4, 10), "int32")), "keep has shape|keep has"),
    (dict(account=Fake((3, 40), "float16")), "account has dtype"),
    (dict(account=Fake((3, 0))), "positions and max_len must be below"),
    (dict(account=Fake((3, 40), ptr=(1 << 20) + 2)), "account is not aligned"),
    (dict(kept=Fake((3,), "int32", ptr=0)), "kept is NULL"),
    (dict(keep=Fake((3, 10), "int32", strides=(0, 1))), "lists of keep overlap"),
    (dict(account=Fake((3, 40), strides=(0, 1))), "invalid context"),      # (one account for all groups)
])
def test_kv_select(ctx, change, message):
    a = dict(account=Fake((3, 40)), lens=Fake((3,), "int32"), keep=Fake((3, 10), "int32"), kept=Fake((3,), "int32"))
    a.update(change)
    with pytest.raises((qxg.QxgError, ValueError), match=message):
        ctx.kv_select(**a)


@pytest.mark.parametrize("change,message", [
    ({}, "invalid context"),
    (dict(first=40), "first is outside the cache"),
    (dict(k=Fake((3, 40, 24), "int8"), v=Fake((3, 40, 24), "int8")), "row_bytes must be a multiple of 16"),
    (dict(k=Fake((3, 40, 8192), "int8"), v=Fake((3, 40, 8192), "int8")), "row_bytes must be a multiple of 16 up to 4096"),
    (dict(k=Fake((3, 40, 64), "int8", strides=(40 * 32, 32, 1)), v=Fake((3, 40, 64), "int8", strides=(40 * 32, 32, 1))), "overlap"),
    (dict(k=Fake((3, 40, 64), "int8", strides=(40 * 72, 72, 1)), v=Fake((3, 40, 64), "int8", strides=(40 * 72, 72, 1))), "multiples of 16 bytes"),
    (dict(account=None), "account and account_out go together"),
    (dict(account_out=None), "account and account_out go together"),
    (dict(account_out=Fake((3, 40), ptr=1 << 20)), "another array"),
    (dict(keep=Fake((3, 0), "int32")), "slots must be positive"),
    (dict(kscale=Fake((3, 41), strides=(40, 1))), "kscale has shape"),
    (dict(k=Fake((3, 40, 64), "int8", strides=(0, 64, 1)), v=Fake((3, 40, 64), "int8", strides=(0, 64, 1))), "rows of k and v overlap"),
    (dict(k=Fake((3, 40, 64), "int8", strides=(64, 192, 1)), v=Fake((3, 40, 64), "int8", strides=(64, 192, 1))), "invalid context"),
    (dict(kscale=Fake((3, 40), strides=(0, 1)), vscale=Fake((3, 40), strides=(0, 1))), "scales of groups overlap"),
    (dict(account_out=Fake((3, 40), strides=(0, 1), ptr=1 << 21)), "accounts of groups overlap"),
    (dict(keep=Fake((3, 10), "int32", strides=(0, 1)), kept=Fake((3,), "int32", strides=(0,))), "invalid context"),      # (one list for all)
])
def test_kv_compact(ctx, change, message):
    a = dict(k=Fake((3, 40, 64), "int8"), v=Fake((3, 40, 64), "int8"), kscale=Fake((3, 40)), vscale=Fake((3, 40)), keep=Fake((3, 10), "int32"),
             kept=Fake((3,), "int32"), account=Fake((3, 40)), account_out=Fake((3, 40), ptr=1 << 21), workspace=big())
    a.update(change)
    with pytest.raises((qxg.QxgError, ValueError), match=message):
        ctx.kv_compact(**a)


def logits(**kw):
    a = dict(logits=Fake((3, 500)), out=Fake((3, 500), ptr=1 << 21), history=Fake((3, 20), "int32"), history_lens=Fake((3,), "int32"),
             prompt_lens=Fake((3,), "int32"), penalties=Fake((3, 3)), temperature=Fake((3,)), bias_ids=Fake((3, 4), "int32"),
             bias_values=Fake((3, 4)), mask=Fake((2, 16), "int32"), mask_rows=Fake((3,), "int32"), top_ids=Fake((3, 8), "int32"),
             top_logits=Fake((3, 8)), lse=Fake((3,)), workspace=big())
    a.update(kw)
    return a


@pytest.mark.parametrize("change,message", [
    ({}, "invalid context"),
    (dict(logits=Fake((3, 500), "int8")), "dtype int8"),
    (dict(out=Fake((3, 500), "float16")), "out has dtype"),
    (dict(logits=Fake((3, 0)), out=Fake((3, 0)), mask=None, mask_rows=None), "vocab must be between"),
    (dict(logits=Fake((3, 500), strides=(400, 1))), "overlap"),
    (dict(logits=Fake((3, 500), strides=(500, 2))), "not contiguous"),
    (dict(out=Fake((3, 500), strides=(600, 1))), "the row strides must be equal"),
    (dict(top_ids=Fake((3, 33), "int32"), top_logits=Fake((3, 33))), "top_n must be at most 32"),
    (dict(top_ids=None), "top_logits has shape|go together"),
    (dict(history=None), "without history"),
    (dict(bias_values=None), "go together"),
    (dict(bias_ids=Fake((3, 1025), "int32"), bias_values=Fake((3, 1025))), "biases must be at most 1024"),
    (dict(mask=Fake((2, 15), "int32")), "mask has shape"),
    (dict(mask=None), "go together"),
    (dict(mask_rows=None), "fewer masks than rows"),
    (dict(penalties=Fake((3, 2))), "penalties has shape"),
    (dict(temperature=Fake((2,))), "temperature has shape"),
    (dict(workspace=None), "the workspace holds 0 bytes; this call needs"),
    (dict(logits=Fake((3, 500), ptr=(1 << 20) + 2)), "logits is not aligned"),
])
def test_adjust_logits(ctx, change, message):
    a = logits(**change)
    if "out" in change and message.startswith("the row strides"):
        a["out"].ptr = a["logits"].ptr
    with pytest.raises((qxg.QxgError, ValueError), match=message):
        ctx.adjust_logits(**a)


def test_null_arguments():
    err = ctypes.create_string_buffer(256)
    for name in ("qxg_tree_attention", "qxg_kv_select", "qxg_kv_compact", "qxg_adjust_logits"):
        assert getattr(qxg._g, name)(None, None, None, 1, err, 256) == 0 and err.value == b"invalid argument"
        assert getattr(qxg._g, name)(None, None, None, 1, None, 0) == 0      # (no place for the message)
    assert qxg._g.qxg_tree_attention_workspace(None) == 0


def test_argument_structs_match_the_header(tmp_path, root):
    """The packed structs of the binding have the sizes and offsets that a C compiler gives the header's."""
    import os
    import subprocess
    src = tmp_path / "s.c"
    src.write_text('#include "qxg.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void) { printf("%zu %zu %zu %zu %zu %zu %zu %zu\\n", '
                   "sizeof(qxg_tree_attention_args), offsetof(qxg_tree_attention_args, type), sizeof(qxg_kv_select_args), "
                   "offsetof(qxg_kv_select_args, groups), sizeof(qxg_kv_compact_args), offsetof(qxg_kv_compact_args, groups), "
                   "sizeof(qxg_adjust_logits_args), offsetof(qxg_adjust_logits_args, type)); return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [qxg._TREE.size, 21 * 8, qxg._SELECT.size, 6 * 8, qxg._COMPACT.size, 17 * 8, qxg._ADJUST.size, 19 * 8]


def test_dense_strides():
    assert qxg._dense((2, 3, 4)) == (12, 4, 1) and qxg._dense(()) == ()
    qxg._fits(qxg._layout(Fake((1, 5), strides=(99, 1))), "a", "f32", (1, 5))      # (a dimension of 1 has any stride)
    assert np.prod(qxg._dense((7,))) == 1
