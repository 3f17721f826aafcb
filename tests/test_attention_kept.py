"""The bound of kept query tokens, on the host."""

import ctypes

import pytest

import ekv_hip
from test_attention_refusals import P, attention


def test_a_negative_bound_is_refused():
    a = attention(kept=-1)
    with pytest.raises(ValueError, match="kept"):
        ekv_hip.call("ekv_prefix_attention", ctypes.addressof(a), P, 1 << 40, 0)


def test_the_workspace_is_the_same():
    sizes = {ekv_hip.load().ekv_prefix_attention_workspace(ctypes.addressof(attention(kept=k))) for k in (0, 1, 5)}
    assert len(sizes) == 1 and min(sizes) > 0
