"""Attention over an int8 cache where values of zero come first: what lies behind them keeps its bits, however small it is."""
import math

import pytest
import torch

from oracle import quant_cache_oracle as oracle
from test_gpu_quant_cache_attention import npu  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
PLACES, COPIES = 900, 400
DOWN = 14 * math.log(2.0)


def check(npu, dev, scores, value_scales, kv, dim, dtype=torch.bfloat16, **kw):  # noqa: F811
    """One sequence of a single page, so many times that a CTA has whole ones: place j has the score scores[j], its values the scale value_scales[j]."""
    g = torch.Generator(device=dev).manual_seed(dim + kv)
    v = torch.randint(-127, 128, (1, 1024, kv, dim), generator=g, device=dev, dtype=torch.int8)
    k = torch.zeros_like(v)  # a key's other elements would widen the bound
    k[..., 0] = 1
    q = torch.zeros((1, 2 * kv, dim), dtype=dtype, device=dev)
    q[..., 0] = 1.0
    ks, vs = (torch.full((1, kv, 1024), math.nan, device=dev) for _ in range(2))
    ks[:, :, :PLACES], vs[:, :, :PLACES] = scores.to(dev), value_scales.to(dev)
    table, lens = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.tensor([PLACES], dtype=torch.int32, device=dev)
    ref, ref_lse, bound, lse_bound = oracle.attention(q, k, v, ks, vs, table, lens, scale=1.0, **kw)
    out, lse = npu.npu_paged_quant_attention(q.repeat(COPIES, 1, 1), k, v, ks, vs, table.repeat(COPIES, 1), lens.repeat(COPIES), scale_value=1.0, **kw)
    err = (out.double() - ref).abs()
    assert bool((err <= bound).all()), f"out is off by {(err / bound).max().item():.2f} times its bound"
    err = (lse.double() - ref_lse).abs()
    assert bool((err <= lse_bound).all()), f"lse is off by {(err / lse_bound).max().item():.2f} times its bound"


def tail(n, first, falling):
    """Scores of `first` for n places, or from there down to weights of 2^-14 of the first's."""
    return first - (torch.linspace(0.0, DOWN, n) if falling else torch.zeros(n))


@pytest.mark.parametrize("falling", [False, True])
@pytest.mark.parametrize("small", [1e-2, 1e-6, 2e-8])
@pytest.mark.parametrize("zeros", [1, 32, 64, 300])
@pytest.mark.parametrize("dim,kv", [(64, 1), (64, 4), (128, 1), (128, 4), (256, 1), (256, 4)])
def test_zeros_first(npu, dev, dim, kv, zeros, small, falling):  # noqa: F811
    scores, values = tail(PLACES, 0.0, falling), torch.full((PLACES,), small)
    scores[:zeros], values[:zeros] = 0.0, 0.0
    check(npu, dev, scores, values, kv, dim)
    if falling:  # the zeros outweigh everything
        scores[zeros:] -= DOWN
        check(npu, dev, scores, values, kv, dim, dtype=torch.float16)


@pytest.mark.parametrize("small", [1e-2, 1e-6, 2e-8])
@pytest.mark.parametrize("dim,kv", [(64, 1), (64, 4), (128, 1), (128, 4), (256, 1), (256, 4)])
def test_zero_sinks(npu, dev, dim, kv, small):  # noqa: F811
    """Sinks of value zero, alone in their tile, with the weight of the others and far above them."""
    for above in (0.0, DOWN, 2 * DOWN):
        scores, values = torch.zeros(PLACES), torch.full((PLACES,), small)
        scores[:3], values[:3] = above, 0.0
        check(npu, dev, scores, values, kv, dim, window=64, sinks=3)
        check(npu, dev, scores, values, kv, dim, window=500, sinks=1, dtype=torch.float16)


@pytest.mark.parametrize("falling", [False, True])
@pytest.mark.parametrize("large", [1e6, 2.0 ** 110, 2.0 ** -110])
@pytest.mark.parametrize("small", [1e-2, 1e-6, 2e-8])
@pytest.mark.parametrize("dim,kv", [(64, 1), (64, 4), (128, 1), (128, 4), (256, 1), (256, 4)])
def test_jump_onto_zeros(npu, dev, dim, kv, small, large, falling):  # noqa: F811
    """Scores that rise by 250 (2^360) where values of zero begin: nothing before them counts, and the power of two that suited it is none of those behind."""
    scores, values = torch.zeros(PLACES), torch.full((PLACES,), large)
    scores[320:], values[320:] = tail(PLACES - 320, 250.0, falling), small
    values[320:576] = 0.0
    check(npu, dev, scores, values, kv, dim)
