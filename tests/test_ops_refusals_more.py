"""More of what the operators on device memory refuse, on the CPU (as test_ops_refusals.py)."""
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
