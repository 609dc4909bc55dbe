"""Calls of the attention over a paged cache that its C entries refuse, without a GPU."""
import ctypes

import pytest

from test_paged_boundary import _attention, _cache


@pytest.mark.parametrize("scale", [1e39, -1e39, 3e38, -3e38, 2.4e38, 1.7e308])
def test_scales_beyond_fp32(capi, scale):
    """The kernels take scale_value * log2(e) in fp32: what is infinite there is refused like an infinite scale."""
    for rc, message in _attention(capi, scale=scale):
        assert rc == 1 and "finite" in message, message


@pytest.mark.parametrize("scale", [2.3e38, -2.3e38, 1e-45, 0.0])
def test_scales_within_fp32(capi, scale):
    for rc, message in _attention(capi, scale=scale, heads=0):
        assert rc == 0, message


def test_operands_off_their_alignment(capi):
    """Outputs are written in 16-byte vectors (log-sums: 4), tables and lengths are read as 32-bit words."""
    lib, n = capi.lib(), 1 << 20
    place = dict(out=n, lse=n, table=n, lens=n, start=n)
    for name, off in (("out", 2), ("out", 8), ("lse", 2), ("table", 2), ("lens", 1), ("start", 2)):
        a = {**place, name: n + off}
        calls = {"qmm_paged_prompt_attention": lambda: lib.qmm_paged_prompt_attention(
            n, 0, 2, 4, 256, 64, _cache(capi), a["table"], 4, 4, a["lens"], a["start"], 2, 1.0, 0, 0, a["out"], a["lse"], None, 0, None)}
        if name != "start":
            calls["qmm_paged_attention"] = lambda: lib.qmm_paged_attention(
                n, 0, 2, 4, 256, 64, _cache(capi), a["table"], 4, 4, a["lens"], 1.0, 0, 0, a["out"], a["lse"], None, 0, None)
        for op, call in calls.items():
            assert call() == 1 and "boundaries" in lib.qmm_last_error().decode(), (op, name, lib.qmm_last_error())


def test_keys_and_values_at_one_address(capi):
    """A cache that is written: which of the two would remain is left to chance."""
    lib, one = capi.lib(), (ctypes.c_int64 * 1)(4)

    def call(cache):
        return lib.qmm_rotary_axes_cache(None, 0, 0, None, 0, 0, None, 0, 0, 0, 0, 4, None, 3, 0, 1, None, 4, one, 1, 0, 0, cache, None, 3, 1, None, None)

    assert call(_cache(capi, dim=8)) == 0
    assert call(_cache(capi, dim=8, value=1 << 20)) == 1 and "same address" in lib.qmm_last_error().decode()
    assert call(_cache(capi, dim=8, key=None, value=None, pages=0)) == 0
