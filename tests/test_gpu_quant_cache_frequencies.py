"""Rotary positions with the write into an int8 paged cache, for frequencies that are not finite: rows that turn to NaN say so."""
import math

import pytest
import torch

from oracle import paged_oracle
from oracle import quant_cache_oracle as oracle
from test_gpu_quant_cache_write import make, npu  # noqa: F401  (npu: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["aligned", "offset"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("mode", ["half", "interleave"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,pairs,which", [(64, 32, 0), (64, 32, 31), (128, 64, 17), (80, 32, 5), (128, 32, 31), (256, 128, 100)])
def test_one_frequency(npu, dev, dim, pairs, which, dtype, mode, bad, layout):  # noqa: F811
    """The pair is NaN in every key (position 0 too: 0 * inf), so each key's scale is NaN and its codes 0; values are as ever."""
    for T in (3, 701):
        q, k, v, positions, inv_freq, kc, vc, ks, vs, slots = make(dev, T, dim=dim, pairs=pairs, dtype=dtype, seed=dim + which)
        positions[0, 1] = 0
        inv_freq[which] = bad
        if layout == "offset":
            k = torch.cat([k.new_zeros(1), k.reshape(-1)])[1:].view(k.shape)
        codes, scales = oracle.quantize(paged_oracle.rotary(k, positions, inv_freq, None, mode == "interleave"))
        assert bool(scales.isnan().all())
        wrote = (slots >= 0) & (slots < kc.shape[0] * 16)
        at = slots[wrote]
        npu.npu_rotary_axes_quant_cache(q, k, v, positions, inv_freq, kc, vc, ks, vs, slots, sections=[pairs], rotary_mode=mode)
        assert bool(ks[at // 16, :, at % 16].isnan().all()) and not bool(kc[at // 16, at % 16].any())
        codes, scales = oracle.quantize(v.double())
        assert torch.equal(vc[at // 16, at % 16], codes[wrote]) and torch.equal(vs[at // 16, :, at % 16], scales[wrote])
