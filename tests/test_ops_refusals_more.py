"""More of what the operators on device memory refuse, on the CPU (as test_ops_refusals.py)."""
import pytest

import qxg
from test_ops_refusals import ctx, tree  # noqa: F401


@pytest.mark.parametrize("change,message", [
    (dict(scale=3.0e38), "scale \\* log2\\(e\\) must be finite"),
    (dict(scale=2.3e38), "invalid context"),
])
def test_tree_attention(ctx, change, message):  # noqa: F811
    with pytest.raises((qxg.QxgError, ValueError), match=message):
        ctx.tree_attention(**tree(**change))
