"""Calls of the attention over a paged cache that its C entries refuse, without a GPU."""
import pytest

from test_paged_boundary import _attention


@pytest.mark.parametrize("scale", [1e39, -1e39, 3e38, -3e38, 2.4e38, 1.7e308])
def test_scales_beyond_fp32(capi, scale):
    """The kernels take scale_value * log2(e) in fp32: what is infinite there is refused like an infinite scale."""
    for rc, message in _attention(capi, scale=scale):
        assert rc == 1 and "finite" in message, message


@pytest.mark.parametrize("scale", [2.3e38, -2.3e38, 1e-45, 0.0])
def test_scales_within_fp32(capi, scale):
    for rc, message in _attention(capi, scale=scale, heads=0):
        assert rc == 0, message
