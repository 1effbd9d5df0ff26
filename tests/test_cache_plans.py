"""The cases of test_gpu_cache_attention_scores.py reach the kernels that they are meant for: the host side's plans, on the CPU."""
import pytest

from test_cache_host import host, lib, plan  # noqa: F401
from test_gpu_cache_attention_scores import KERNELS


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_plans(host, name):  # noqa: F811
    c, seen = host
    case, columns = KERNELS[name]
    plan(c, seen, **case)
    assert seen.columns == columns and (seen.splits > 1) == ("splits" in name or name.startswith("32"))
