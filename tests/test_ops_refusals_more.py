"""More of what the operators on device memory refuse, on the CPU (as test_ops_refusals.py)."""
import ctypes

import pytest

import qxg
from test_ops_refusals import Fake, big, ctx, tree  # noqa: F401


@pytest.mark.parametrize("change,message", [
    (dict(scale=3.0e38), "scale \\* log2\\(e\\) must be finite"),
    (dict(scale=2.3e38), "invalid context"),
])
def test_tree_attention(ctx, change, message):  # noqa: F811
    with pytest.raises((qxg.QxgError, ValueError), match=message):
        ctx.tree_attention(**tree(**change))


def overlaps(strides, shape, row):
    """By listing where every row starts."""
    starts = sorted(i * strides[0] + j * strides[1] for i in range(shape[0]) for j in range(shape[1]))
    return any(b - a < row for a, b in zip(starts, starts[1:]))


@pytest.mark.parametrize("batch,nodes", [(2, 3), (3, 2), (5, 4), (1, 4), (4, 1)])
@pytest.mark.parametrize("outer", [0, 512, 1024, 1536, 2048, 2560, 3136, 4096, 5120])
@pytest.mark.parametrize("inner", [0, 1024, 1536, 2048, 3584])
def test_rows_of_out_that_overlap(ctx, batch, nodes, outer, inner):  # noqa: F811
    a = tree(q=Fake((batch, nodes, 8, 128)), out=Fake((batch, nodes, 8, 128), strides=(outer, inner, 128, 1), ptr=1 << 21),
             lse=None, account=None, mask=None, counts=None, lens=Fake((batch,), "int32"))
    for name, dtype in (("k", "int8"), ("v", "int8")):
        a[name] = Fake((batch, 50, 4, 128), dtype)
    a["kscale"], a["vscale"] = Fake((batch, 50)), Fake((batch, 50))
    with pytest.raises(qxg.QxgError, match="rows of out overlap" if overlaps((outer, inner), (batch, nodes), 1024) else "invalid context"):
        ctx.tree_attention(**a)


@pytest.mark.parametrize("group,row", [(64, 64), (64, 192), (64, 128), (128, 64), (160, 320), (96, 160), (64, 0), (0, 64), (40 * 64, 64),
                                       (39 * 64, 64), (39 * 64 + 16, 64), (80, 256), (80, 240), (1 << 62, 1 << 63), ((1 << 63) + 64, 1 << 63)])
def test_rows_of_a_cache_that_overlap(ctx, group, row):  # noqa: F811
    k = Fake((3, 40, 64), "int8", strides=(group, row, 1))
    a = dict(k=k, v=k, kscale=Fake((3, 40)), vscale=Fake((3, 40)), keep=Fake((3, 10), "int32"), kept=Fake((3,), "int32"), workspace=big())
    with pytest.raises(qxg.QxgError, match="rows of k and v overlap" if overlaps((group, row), (3, 40), 64) else "invalid context"):
        ctx.kv_compact(**a)


@pytest.mark.parametrize("offset,message", [(0, "invalid context"), (4, "kept overlaps lens"), (-8, "kept overlaps lens"), (12, "invalid context"),
                                            (-12, "invalid context")])
def test_kept_that_overlaps_lens(ctx, offset, message):  # noqa: F811
    a = dict(account=Fake((3, 40)), lens=Fake((3,), "int32"), keep=Fake((3, 10), "int32", ptr=1 << 21), kept=Fake((3,), "int32", ptr=(1 << 20) + offset))
    with pytest.raises(qxg.QxgError, match=message):
        ctx.kv_select(**a)


@pytest.mark.parametrize("groups,message", [((1 << 22) - 1, "invalid context"), (1 << 22, "groups must be between"), (0xffffffff, "groups must be between")])
def test_groups_beyond_a_launch(ctx, groups, message):  # noqa: F811
    a = dict(account=Fake((groups, 40), strides=(0, 1)), lens=Fake((groups,), "int32"), keep=Fake((groups, 10), "int32", ptr=1 << 40),
             kept=Fake((groups,), "int32", ptr=1 << 39))
    with pytest.raises(qxg.QxgError, match=message):
        ctx.kv_select(**a)


@pytest.mark.parametrize("positions,message", [(8 * 256, "invalid context"), (8 * 257, "too many rows for one call"), (8 * 1024, "too many rows")])
def test_rows_beyond_a_launch(ctx, positions, message):  # noqa: F811
    """Tiles of 8 rows of 4096 bytes, 65535 groups."""
    groups, row = 65535, 4096
    k = Fake((groups, positions, row), "int8")
    a = dict(k=k, v=k, kscale=Fake((groups, positions)), vscale=Fake((groups, positions)), keep=Fake((groups, positions), "int32", strides=(0, 1)),
             kept=Fake((groups,), "int32", strides=(0,)), workspace=big())
    with pytest.raises(qxg.QxgError, match=message):
        ctx.kv_compact(**a)


@pytest.mark.parametrize("change", [
    dict(q=Fake((1, 3, 8, 128), strides=(1, 1024, 128, 1))),                     # (of a permuted [nodes, heads, dim, 1])
    dict(out=Fake((1, 3, 8, 128), strides=(0, 1024, 128, 1), ptr=1 << 21)),
    dict(k=Fake((1, 50, 4, 128), "int8", strides=(5, 512, 128, 1))),
    dict(kscale=Fake((1, 50), strides=(1, 1))),
    dict(account=Fake((1, 50), strides=(0, 1))),
])
def test_any_stride_of_a_dimension_of_one(ctx, change):  # noqa: F811
    a = tree(q=Fake((1, 3, 8, 128)), k=Fake((1, 50, 4, 128), "int8"), v=Fake((1, 50, 4, 128), "int8"), kscale=Fake((1, 50)), vscale=Fake((1, 50)),
             lens=Fake((1,), "int32"), out=Fake((1, 3, 8, 128), ptr=1 << 21), mask=None, counts=None, lse=None, account=None)
    a.update(change)
    with pytest.raises(qxg.QxgError, match="invalid context"):
        ctx.tree_attention(**a)


def test_any_stride_of_one_node_or_position(ctx):  # noqa: F811
    one = dict(q=Fake((2, 1, 8, 128), strides=(1024, 3, 128, 1)), k=Fake((2, 1, 4, 128), "int8", strides=(512, 7, 128, 1)),
               v=Fake((2, 1, 4, 128), "int8", strides=(512, 1 << 40, 128, 1)), kscale=Fake((2, 1)), vscale=Fake((2, 1), strides=(1, 9)),
               out=Fake((2, 1, 8, 128), strides=(1024, 0, 128, 1), ptr=1 << 21), lse=None, mask=None, account=None)
    with pytest.raises(qxg.QxgError, match="invalid context"):
        ctx.tree_attention(**tree(**one))


@pytest.mark.parametrize("change", [
    dict(k=Fake((1, 40, 64), "int8", strides=(1, 64, 1))), dict(kscale=Fake((1, 40), strides=(3, 1))), dict(keep=Fake((1, 10), "int32", strides=(0, 1))),
    dict(k=Fake((1, 40, 64), "int8", strides=(7, 64, 1)), v=Fake((1, 40, 64), "int8", strides=(9, 64, 1))),
    dict(account_out=Fake((1, 40), strides=(1, 1), ptr=1 << 22)),
])
def test_any_stride_of_one_group(ctx, change):  # noqa: F811
    k = Fake((1, 40, 64), "int8")
    a = dict(k=k, v=k, kscale=Fake((1, 40)), vscale=Fake((1, 40)), keep=Fake((1, 10), "int32"), kept=Fake((1,), "int32", strides=(5,)),
             account=Fake((1, 40)), account_out=Fake((1, 40), ptr=1 << 22), workspace=big())
    a.update(change)
    with pytest.raises(qxg.QxgError, match="invalid context"):
        ctx.kv_compact(**a)


def test_strides_that_the_c_interface_does_not_use(ctx):  # noqa: F811
    """The same at the C interface: strides over one sequence, node, position or group are not looked at."""
    err = ctypes.create_string_buffer(256)
    p = 1 << 20
    packed = qxg._TREE.pack(p, p, p, p, p, p, 0, 0, 1 << 21, 0, 0, p, 1 << 30, 3, 5, 7, 9, 11, 13, 1, 1, 0, 1, 1, 8, 4, 128, 1, 1, 0.1, 1.0)
    assert qxg._g.qxg_tree_attention(None, packed, None, 1, err, 256) == 0 and err.value == b"invalid context"
    packed = qxg._COMPACT.pack(p, p, p, p, p, p, 0, 0, p, 1 << 30, 3, 5, 1, 1, 1, 1, 1, 1, 1, 1, 0, 64)
    assert qxg._g.qxg_kv_compact(None, packed, None, 1, err, 256) == 0 and err.value == b"invalid context"
