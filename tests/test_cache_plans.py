"""The cases of test_gpu_cache_attention_scores.py and test_gpu_cache_attention_kernels.py reach the kernels that they are meant for: the host
side's plans, on the CPU."""
import pytest

from test_cache_host import host, lib, plan  # noqa: F401
from test_gpu_cache_attention_kernels import FAR, HEADS, SPLITS, behind
from test_gpu_cache_attention_scores import KERNELS


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_plans(host, name):  # noqa: F811
    c, seen = host
    case, columns = KERNELS[name]
    plan(c, seen, **case)
    assert seen.columns == columns and (seen.splits > 1) == ("splits" in name or name.startswith("32"))


@pytest.mark.parametrize("name", sorted(HEADS))
@pytest.mark.parametrize("n", [640, 2000, 4000])
def test_plans_of_many_heads(host, name, n):  # noqa: F811
    c, seen = host
    plan(c, seen, **behind(name, n))
    assert seen.columns == HEADS[name][1]


@pytest.mark.parametrize("name", sorted(FAR))
def test_plans_of_caches_past_4_gib(host, name):  # noqa: F811
    c, seen = host
    plan(c, seen, **FAR[name][0])
    assert seen.columns == FAR[name][1]


@pytest.mark.parametrize("name", sorted(SPLITS))
def test_plans_of_more_splits_than_lanes(host, name):  # noqa: F811
    c, seen = host
    plan(c, seen, **{k: v for k, v in SPLITS[name].items() if k != "max_len"})
    assert seen.splits > 64
    # the lengths between end behind the 64th split, and before
    chunks = [-(-(n + 1) // 32) for n in (SPLITS[name]["lens"][0] * m // 12 for m in (12, 9, 8))]
    assert chunks[0] > 64 * seen.split_chunks
