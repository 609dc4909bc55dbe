"""Attention of single tokens over long stretches of equal scores, where an fp32 sum of weights would round every time the same way."""
import math
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
PKG_DIR = Path(__file__).resolve().parent.parent / "ascend-python_b200"
PAGE = 4096


@pytest.fixture(scope="module")
def npu():
    sys.path.insert(0, str(PKG_DIR))
    try:
        import torch_npu
    finally:
        sys.path.pop(0)
    return torch_npu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("weight", [0.7, 0.3])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("log_places", [15, 17, 19])
def test_equal_weights(npu, dev, log_places, dim, weight, dtype):
    """A few keys of score 0, all others of one score, and values of 1: as many sequences as warps, so that a warp has whole ones, up to 2^19 places.

    The score is exact; log2(e) and the exponent are rounded (2^-24 of |score| each), the exponential is off by 2^-22, the same for all keys.  A lane's weights of a tile
    are 16 at most (2^-24 each), what adding them to those before rounds away is kept, two steps add the lanes and a few more the parts of cut ones: less than
    2^-19.  The log-sum is 14 at most, each of its two roundings 2^-21.  All that is less than 2^-18.  (A plain fp32 chain is off by 2^-15, 2^-12.5 and 2^-10.6.)  The output's equal weights
    are rounded to the type of the query (half a step, as the output is), and the tensor cores cut sums of 2^16 to 2^17 places by up to 2^-11.
    """
    places, batch = 1 << log_places, 8 * torch.cuda.get_device_properties(dev).multi_processor_count
    low = torch.tensor(math.log(weight)).to(dtype)
    k = torch.zeros((2, PAGE, 1, dim), dtype=dtype, device=dev)
    k[..., 0] = low
    k[1, :256:16, :, 0] = 0.0
    q = torch.zeros((batch, 2, dim), dtype=dtype, device=dev)
    q[..., 0] = 1.0
    table = torch.zeros((batch, places // PAGE), dtype=torch.int32, device=dev)
    table[:, 0] = 1
    lens = torch.full((batch,), places, dtype=torch.int32, device=dev)
    out, lse = npu.npu_paged_attention(q, k, torch.ones_like(k), table, lens, scale_value=1.0)
    want = math.log(16 + (places - 16) * math.exp(low.double().item()))
    err = (lse.double() - want).abs().max().item()
    assert err <= 2.0 ** -18, f"2^{math.log2(err):.2f}"
    assert (out.double() - 1).abs().max().item() <= torch.finfo(dtype).eps + 2.0 ** -11
