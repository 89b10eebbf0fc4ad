"""Refusals of the serving attention calls that need a workspace, without a GPU."""
import pytest

from frame_public_b200 import capi
from test_attention_serving_cpu import PTR, good_cache, good_params, paged, refused


@pytest.mark.parametrize("change", [dict(max_q=1), dict(max_q=5, max_kv=9000)], ids=["decode", "keys in parts"])
def test_paged_refuses_every_workspace_that_is_too_small(change):
    p, c = good_params(**change), good_cache()
    size = capi.attention_paged_workspace(p, c)
    assert size > 4096
    refused(1, "workspace", paged, p, c, size=size - 1)
    refused(1, "workspace", paged, p, c, size=0)
    refused(1, "workspace", paged, p, c, work=None, size=size)
    refused(1, "workspace", paged, p, c, work=PTR + 16, size=size)


@pytest.mark.parametrize("scale", [2.5e38, 3.4e38])
def test_a_score_scale_whose_exponent_overflows_is_refused(scale):
    refused(1, "scale", paged, good_params(scale=scale), good_cache())
    refused(1, "scale", capi.attention_paged_workspace, good_params(scale=scale), good_cache())
