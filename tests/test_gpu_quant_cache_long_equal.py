"""Attention over an int8 cache along long stretches of equal scores, where an fp32 sum of weights would round every time the same way."""
import math

import pytest
import torch

from test_gpu_quant_cache_attention import npu  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
PAGE = 4096


@pytest.mark.parametrize("weight", [0.7, 0.3, 0.001])
@pytest.mark.parametrize("heads,kv,dim,log_places", [(2, 1, 64, 21), (2, 1, 128, 21), (12, 1, 128, 21), (2, 1, 256, 21),  # more than 131072 places a warp
                                                     (4, 4, 64, 17), (4, 4, 128, 17), (2, 1, 128, 19), (2, 1, 256, 19)])  # as many
def test_equal_weights(npu, dev, heads, kv, dim, log_places, weight):  # noqa: F811
    """A few keys of score 0 in each warp's first tile, all others of score log(weight), and values of 1: as many sequences as CTAs, or a
    multiple, so that a warp has all of its part of one.

    A score is exact here but for the rounding of log2(e) and of the exponent, 2^-24 * |score| each, and its exponential is off by 2^-22; both are the same
    for all keys.  A lane's weights of a tile are up to 8 (2^-24 each at most), what it adds them to keeps what it rounds, and three steps add the lanes, three more the
    parts (three roundings each): 22 * 2^-24.  The logarithm of 2^21 * weight and the largest score add to 15 at most: 2^-20 for each of two roundings.  All
    that is less than 2^-18 + 2^-23 * |log(weight)|.  A plain fp32 chain of 16384 additions is off by up to 2^-12, one of 65536 by up to 2^-10.  In the output the equal weights are rounded to f16 (2^-11), and the
    tensor cores cut sums of 2^16 to 2^17 places (2^-11), as in other long sums.
    """
    places = 1 << log_places
    batch = 2 * torch.cuda.get_device_properties(dev).multi_processor_count
    k = torch.zeros((2, PAGE, kv, dim), dtype=torch.int8, device=dev)
    k[..., 0] = 1
    v = torch.full_like(k, 100)
    low = torch.tensor(math.log(weight), dtype=torch.float32)
    ks = torch.full((2, kv, PAGE), low.item(), device=dev)
    ks[1, :, :256:16] = 0.0
    vs = torch.full((2, kv, PAGE), 2.0 ** -7, device=dev)
    q = torch.zeros((batch, heads, dim), dtype=torch.float16, device=dev)
    q[..., 0] = 1.0
    table = torch.zeros((batch, places // PAGE), dtype=torch.int32, device=dev)
    table[:, 0] = 1
    lens = torch.full((batch,), places, dtype=torch.int32, device=dev)
    out, lse = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens, scale_value=1.0)
    want = math.log(16 + (places - 16) * math.exp(low.double().item()))
    err = (lse.double() - want).abs().max().item()
    assert err <= 2.0 ** -18 + 2.0 ** -23 * abs(low.item()), f"2^{math.log2(err):.2f}"
    assert (out.double() / (100 * 2.0 ** -7) - 1).abs().max().item() <= 2.0 ** -11 + 2.0 ** -10 + 2.0 ** -12
