"""Attention over an int8 cache in f16: weights keep more bits than the output has."""
import math

import pytest
import torch

from oracle import quant_cache_oracle as oracle
from test_gpu_quant_cache_attention import make, npu  # noqa: F401  (npu: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (32, 8, 128), (32, 2, 128), (4, 1, 256), (12, 1, 256)])
def test_weights_do_not_show(npu, dev, heads, kv, dim):  # noqa: F811
    """Values of both signs, whose sums are far smaller than they: all outputs together are off by what rounding the exact ones to f16 is, not by weights that are
    rounded to f16, too, which would be as much again.  A tenth is left for the rest."""
    q, k, v, ks, vs, table, lens = make(dev, [3000, 4000, 9000], heads=heads, kv=kv, dim=dim, dtype=torch.float16, seed=dim)
    out, _ = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens)
    ref = oracle.attention(q, k, v, ks, vs, table, lens)[0]
    rounded = ((ref.half().double() - ref).norm() / ref.norm()).item()
    assert ((out.double() - ref).norm() / ref.norm()).item() <= 1.1 * rounded


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinite_values(npu, dev, dtype):  # noqa: F811
    """A value whose scale is infinite: infinite with the sign of its code, NaN where that is 0."""
    q, k, v, ks, vs, table, lens = make(dev, [40], heads=4, kv=1, dim=64, dtype=dtype, seed=50)
    v[table[0, 1], 3, 0] = torch.arange(64, device=dev).int().sub(5).sign().to(torch.int8)  # place 19
    vs[table[0, 1], 0, 3] = math.inf
    out, lse = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens)
    assert bool((out[0, :, :5] == -math.inf).all()) and bool(out[0, :, 5].isnan().all()) and bool((out[0, :, 6:] == math.inf).all())
    assert bool(lse.isfinite().all())
