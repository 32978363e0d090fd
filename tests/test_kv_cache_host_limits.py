"""Limits of the packed and paged operators' arguments that are found before any device call (CPU)."""
import pytest
from test_kv_cache_host import A16, ARG, append, packed, paged


@pytest.mark.parametrize("more", [dict(), dict(dt=2), dict(pos=A16), dict(rot=256)])
def test_append_refuses_empty_tables(more):
    """Rotation with tables of no position: every row would be outside them, and no entry may be read."""
    assert append(**{**dict(rot=64, cos=A16, sin=A16, n_pos=0), **more}) == ARG


@pytest.mark.parametrize("call", [packed, paged])
@pytest.mark.parametrize("scale", [2.5e38, 3.4e38])
def test_a_scale_that_is_infinite_in_log2_units_is_refused(call, scale):
    """The softmax runs on scale x log2(e), fp32: where that is infinite a score of 0 would be NaN."""
    assert call(scale=scale) == ARG
